// 8-bit rows: quantisation with a scale per row, and the matrix product of two such matrices.
#include "i8_device.hpp"
#include "score_i8.hpp"

#include <atomic>

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

static inline int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }
static inline bool dtype_ok(int t) { return t == TFREC_DT_F32 || t == TFREC_DT_BF16 || t == TFREC_DT_F16; }

// ------------------------------------------------------------------------------------------
// quantisation: scale = max|x| / 127, q = nearest-even(x / scale)
// ------------------------------------------------------------------------------------------
// The nearest integer to x / s, ties to even, exactly: r = rint(x * RN(1/s)) is off by at most one, and the remainder
// x - r s is exact in float32 (both are multiples of ulp(s) where |x| >= s, and |x - r s| < s otherwise), so comparing it
// with s / 2 decides.  Scales near the subnormal range are lifted by 2^64 first (exact; |x| <= 127.5 s, or up to 190 s where s was
// rounded to one of the smallest subnormal numbers: such a value ends at 127).
__device__ __forceinline__ int quantize_one(float x, float s, float inv)
{
    float r = rintf(x * inv);
    const float e = fmaf(-r, s, x), half = 0.5f * s;
    const bool odd = ((int)r & 1) != 0;
    if (e > half || (e == half && odd)) r += 1.f;
    else if (e < -half || (e == -half && odd)) r -= 1.f;
    return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// 16 values at the alignment of their type (global memory takes 16-byte accesses at any)
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Values16 { T v[16]; };

// LPR threads hold one row (a power of two up to 64: lanes of a wave; 256: the workgroup), CH runs of 16 columns each in
// registers: one read of the row, one write of a quarter (half) as much.  CH = 0: rows too long for that are read twice,
// the second time from the caches.
// Bound by its vector instructions, 30 a value (the vector pipes are busy at least 70 % of the cycles), with nothing of the next row on its
// way meanwhile: 4096 x 8192 in bfloat16 (100 MB in all) 28 us, 3.6 TB/s; in float32 (168 MB) 29 us.
template <class T, int LPR, int CH>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T *__restrict__ X, int64_t n_rows, int64_t ldx, int64_t d,
                                                            const int32_t *__restrict__ rows, int64_t n, int8_t *__restrict__ q, int64_t ldq,
                                                            float *__restrict__ scale, uint32_t *__restrict__ flags)
{
    constexpr int GPB = 256 / LPR;
    const int gl = threadIdx.x % LPR;
    int64_t r = (int64_t)blockIdx.x * GPB + threadIdx.x / LPR;
    const bool live = r < n;                   // (threads past the last row stay for the workgroup's barrier)
    r = live ? r : n - 1;
    int64_t src = r;
    if (rows) {
        const int32_t id = rows[r];
        src = id < 0 ? 0 : (id >= n_rows ? n_rows - 1 : id);
        if (src != id && gl == 0) atomicOr(flags, TFREC_FLAG_BAD_INDEX);
    }
    const T *x = X + src * ldx;
    const int64_t chunks = (d + 15) / 16;
    auto load = [&](int64_t c) {
        Values16<T> v;
        if (c * 16 + 16 <= d) v = *reinterpret_cast<const Values16<T> *>(x + c * 16);
        else
#pragma unroll
            for (int j = 0; j < 16; ++j) v.v[j] = c * 16 + j < d ? x[c * 16 + j] : (T)0.f;
        return v;
    };
    float mx = 0.f;
    bool bad = false;
    auto look = [&](const Values16<T> &v) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float f = fabsf((float)v.v[j]);
            bad |= !(f < INFINITY);
            mx = fmaxf(mx, f);
        }
    };
    Values16<T> held[CH > 0 ? CH : 1];
    if constexpr (CH > 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i) held[i] = load(gl + i * LPR);          // (past the row: zeros)
#pragma unroll
        for (int i = 0; i < CH; ++i) look(held[i]);
    } else {
        for (int64_t c = gl; c < chunks; c += LPR) look(load(c));
    }
    mx = bad ? INFINITY : mx;
#pragma unroll
    for (int off = (LPR < 64 ? LPR : 64) / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if constexpr (LPR > 64) {
        __shared__ float part[4];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    }
    if (!live) return;
    float s = mx / 127.0f;
    const bool none = !(mx < INFINITY) || !(s > 0.f);
    if (gl == 0) scale[r] = mx < INFINITY ? s : NAN;
    const float up = s < 0x1p-60f ? 0x1p64f : 1.f;
    s *= up;
    const float inv = 1.f / s;
    auto put = [&](int64_t c, const Values16<T> &v) {
        union { int8_t b[16]; uint4 v; } o;
#pragma unroll
        for (int j = 0; j < 16; ++j) o.b[j] = none ? 0 : (int8_t)quantize_one((float)v.v[j] * up, s, inv);
        *reinterpret_cast<uint4 *>(q + r * ldq + c * 16) = o.v;
    };
    if constexpr (CH > 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (gl + i * LPR < chunks) put(gl + i * LPR, held[i]);
    } else {
        for (int64_t c = gl; c < chunks; c += LPR) put(c, load(c));
    }
}

template <class T>
static int launch_quantize(tfrec_ctx *ctx, const void *X, int64_t n_rows, int64_t ldx, int64_t d, const int32_t *rows, int64_t n, int8_t *q,
                           int64_t ldq, float *scale)
{
    auto go = [&]<int LPR, int CH>() -> int {
        constexpr int GPB = 256 / LPR;
        for (int64_t r = 0; r < n; r += TF_LAUNCH_ROWS * GPB) {
            const int64_t m = n - r < TF_LAUNCH_ROWS * GPB ? n - r : TF_LAUNCH_ROWS * GPB;
            quantize_rows_kernel<T, LPR, CH><<<(unsigned)((m + GPB - 1) / GPB), 256, 0, ctx->stream>>>(
                (const T *)X + (rows ? 0 : r * ldx), n_rows, ldx, d, rows ? rows + r : nullptr, m, q + r * ldq, ldq, scale + r, ctx->d_flags);
            TF_HIP(hipGetLastError());
        }
        return TFREC_OK;
    };
    const int64_t chunks = (d + 15) / 16;
    if (chunks <= 4) return go.template operator()<4, 1>();
    if (chunks <= 16) return go.template operator()<16, 1>();
    if (chunks <= 64) return go.template operator()<64, 1>();
    if (chunks <= 256) return go.template operator()<256, 1>();
    if (chunks <= 512) return go.template operator()<256, 2>();
    return go.template operator()<256, 0>();
}

int tfrec_quantize_rows(tfrec_ctx *ctx, const void *d_X, int x_dtype, int64_t n_rows, int64_t ldx, int64_t d, const int32_t *d_rows, int64_t n,
                        int8_t *d_q, int64_t ldq, float *d_scale)
{
    if (x_dtype == TFREC_DT_BF16) return launch_quantize<__bf16>(ctx, d_X, n_rows, ldx, d, d_rows, n, d_q, ldq, d_scale);
    if (x_dtype == TFREC_DT_F16) return launch_quantize<_Float16>(ctx, d_X, n_rows, ldx, d, d_rows, n, d_q, ldq, d_scale);
    return launch_quantize<float>(ctx, d_X, n_rows, ldx, d, d_rows, n, d_q, ldq, d_scale);
}

// the layout every 8-bit matrix has to have
int tfrec_check_i8(const char *name, const int8_t *q, int64_t rows, int64_t ld, int64_t cols)
{
    TF_REQUIRE(rows == 0 || q != nullptr, TFREC_EINVAL, "%s is null", name);
    TF_REQUIRE(((uintptr_t)q & 15u) == 0, TFREC_EINVAL, "%s is not 16-byte aligned", name);
    TF_REQUIRE(ld % 16 == 0 && ld >= up16(cols), TFREC_EINVAL, "%s: a row pitch of %lld bytes, need a multiple of 16 and at least %lld", name,
               (long long)ld, (long long)up16(cols));
    TF_REQUIRE(rows < (1ll << 40) / (ld > 0 ? ld : 1), TFREC_EUNSUP, "%s is too large", name);
    return TFREC_OK;
}

// n rows of len bytes, pitch bytes apart
struct RowBytes { uintptr_t at; int64_t pitch, len, n; };

// [lo, hi) and any of the rows
static bool meets(uintptr_t lo, uintptr_t hi, const RowBytes &b)
{
    const uintptr_t end = b.at + (b.n - 1) * b.pitch + b.len;
    if (hi <= b.at || lo >= end) return false;
    if (lo <= b.at) return true;
    const int64_t r = (int64_t)(lo - b.at) / b.pitch, off = (int64_t)(lo - b.at) % b.pitch;
    return off < b.len || b.at + (r + 1) * b.pitch < hi;         // within row r, or the next row (there is one: lo < end) begins before hi
}

// Any byte in common?  Rows that merely lie between each other's have none.  The spans of two buffers that have nothing to do with
// each other are apart, which is all that is looked at then.
static bool rows_overlap(RowBytes a, RowBytes b)
{
    if (a.n <= 0 || b.n <= 0 || a.len <= 0 || b.len <= 0) return false;
    if (a.n > b.n) { const RowBytes t = a; a = b; b = t; }
    const uintptr_t end_a = a.at + (a.n - 1) * a.pitch + a.len, end_b = b.at + (b.n - 1) * b.pitch + b.len;
    if (end_a <= b.at || end_b <= a.at) return false;
    for (int64_t i = 0; i < a.n; ++i)
        if (meets(a.at + i * a.pitch, a.at + i * a.pitch + a.len, b)) return true;
    return false;
}

// the same for callers without the struct (tests)
extern "C" int tfrec_rows_overlap(uintptr_t at, int64_t pitch, int64_t len, int64_t n, uintptr_t at2, int64_t pitch2, int64_t len2, int64_t n2)
{
    return rows_overlap({at, pitch, len, n}, {at2, pitch2, len2, n2});
}

// a contiguous array as one row (null: none)
static RowBytes array_bytes(const void *p, int64_t n, int64_t size) { return {(uintptr_t)p, n * size, n * size, p ? 1 : 0}; }

extern "C" int tfrec_quantize_rows_i8(tfrec_ctx *ctx, const void *d_X, int x_dtype, int64_t n_rows, int64_t ldx, int64_t d,
                                      const int32_t *d_rows, int64_t n, int8_t *d_q, int64_t ldq, float *d_scale)
{
    TF_REQUIRE(dtype_ok(x_dtype), TFREC_EINVAL, "unknown type %d", x_dtype);
    TF_REQUIRE(d >= 1 && n >= 0 && n_rows >= 0 && ldx >= d, TFREC_EINVAL, "bad shape n=%lld d=%lld ldx=%lld", (long long)n, (long long)d, (long long)ldx);
    TF_REQUIRE(d_rows || n <= n_rows, TFREC_EINVAL, "%lld rows wanted of %lld", (long long)n, (long long)n_rows);
    TF_REQUIRE(!d_rows || n == 0 || (n_rows >= 1 && n_rows < (1ll << 31)), TFREC_EINVAL, "row ids into a table of %lld rows", (long long)n_rows);
    TF_REQUIRE(n == 0 || (d_X && d_scale), TFREC_EINVAL, "null pointer");
    TF_REQUIRE(((uintptr_t)d_X & (x_dtype == TFREC_DT_F32 ? 3u : 1u)) == 0, TFREC_EINVAL, "rows are not aligned to their type");
    TF_TRY(tfrec_check_i8("the 8-bit matrix", d_q, n, ldq, d));
    TF_TRY(tfrec_ctx_enter(ctx));
    if (n == 0) return TFREC_OK;
    const int64_t es = x_dtype == TFREC_DT_F32 ? 4 : 2;
    const RowBytes q{(uintptr_t)d_q, ldq, up16(d), n}, s = array_bytes(d_scale, n, 4), x{(uintptr_t)d_X, ldx * es, d * es, d_rows ? n_rows : n}, ids = array_bytes(d_rows, n, 4);
    for (const RowBytes &o : {q, s})
        TF_REQUIRE(!rows_overlap(o, x) && !rows_overlap(o, ids), TFREC_EINVAL, "an output overlaps the source rows or their list");
    TF_REQUIRE(!rows_overlap(q, s), TFREC_EINVAL, "the 8-bit rows and the scales overlap");
    return tfrec_quantize_rows(ctx, d_X, x_dtype, n_rows, ldx, d, d_rows, n, d_q, ldq, d_scale);
}

// The words W (8 or 16 bytes) as values of type T: one store, at T's alignment, or the first `room` values one by one.  (As a
// vector type on purpose: the compiler takes the store of a struct apart and joins it with the other branch's.)
template <class T, int W>
__device__ __forceinline__ void store_values(T *to, const uint32_t (&w)[W], int64_t room)
{
    typedef uint32_t Words __attribute__((ext_vector_type(W), aligned(sizeof(T)), may_alias));
    struct All { T v[4 * W / sizeof(T)]; };
    if (room >= (int64_t)(4 * W / sizeof(T))) {
        Words o;
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = w[i];
        *reinterpret_cast<Words *>(to) = o;
    } else {
        struct In { uint32_t w[W]; } in;
#pragma unroll
        for (int i = 0; i < W; ++i) in.w[i] = w[i];
        const All all = __builtin_bit_cast(All, in);
#pragma unroll
        for (int x = 0; x < (int)(4 * W / sizeof(T)); ++x)
            if (x < room) to[x] = all.v[x];
    }
}

// ------------------------------------------------------------------------------------------
// product
// ------------------------------------------------------------------------------------------
struct MatmulArgs {
    const int8_t *A, *B;
    const float *sa, *sb, *bias;
    void *C;
    int64_t lda, ldb, ldc, M, N, K;
};

// one value of C before it is rounded to C's type
__device__ __forceinline__ float output(const MatmulArgs &a, int acc, float sa, float sb, float bias)
{
    const float v = scaled_sum(acc, sa, sb);
    return a.bias ? add_rounded(v, bias) : v;
}

// ---- few rows of A, or few tiles: 16 rows of B by 16 MT rows of A per workgroup, its KW waves sharing K ----------------
// Bound by reading B (one row of A) or by latency (small products): B's rows come straight from memory as the matrix
// instruction's A operand (16 x 16 x 64: lane l holds 16 bytes of row l & 15, columns 16 (l >> 4) .. + 16; result register
// j is row 4 (l >> 4) + j, column l & 15), all of a wave's loads of several steps in flight, and the waves' whole-number sums
// are added in LDS.
template <class T, int MT, int KW>
__global__ __launch_bounds__(64 * KW) void matmul_i8_rows_kernel(MatmulArgs a)
{
    __shared__ int32_t part[KW > 1 ? KW - 1 : 1][MT][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, c16 = (lane >> 4) * 16;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
    const int8_t *bp = a.B + (n0 + r < a.N ? n0 + r : a.N - 1) * a.ldb;
    const int8_t *ap[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = m0 + 16 * t + r;
        ap[t] = a.A + (m < a.M ? m : a.M - 1) * a.lda;
    }
    i32x4 acc[MT] = {};
    // steps of 64 columns; wave w takes steps w, w + KW, ...
    const int steps = (int)(a.K / 64);
    constexpr int DEPTH = MT <= 2 ? 4 : (MT == 4 ? 2 : 1);
    int s = wave;
    for (; s + (DEPTH - 1) * KW < steps; s += DEPTH * KW) {
        i32x4 fb[DEPTH], fa[DEPTH][MT];
#pragma unroll
        for (int q = 0; q < DEPTH; ++q) {
            const int64_t k = (int64_t)(s + q * KW) * 64 + c16;
            fb[q] = *reinterpret_cast<const i32x4 *>(bp + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) fa[q][t] = *reinterpret_cast<const i32x4 *>(ap[t] + k);
        }
#pragma unroll
        for (int q = 0; q < DEPTH; ++q)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[q], fa[q][t], acc[t], 0, 0, 0);
    }
    for (; s * 64 < a.K; s += KW) {
        // what is left, up to a last step that ends inside 64 columns: A is zero there, B any bytes of its row
        const int64_t k = (int64_t)s * 64 + c16;
        const i32x4 fb = *reinterpret_cast<const i32x4 *>(bp + (k < a.K ? k : 0));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (k < a.K) v = keep_below(*reinterpret_cast<const uint4 *>(ap[t] + k), k, a.K);
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb, __builtin_bit_cast(i32x4, v), acc[t], 0, 0, 0);
        }
    }
    if constexpr (KW > 1) {
        if (wave > 0)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[wave - 1][t][j][lane] = acc[t][j];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 0; w < KW - 1; ++w)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][j] += part[w][t][j][lane];
    }
    const int64_t n = n0 + (lane >> 4) * 4;
    float sb[4], bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t nj = n + j < a.N ? n + j : a.N - 1;
        sb[j] = a.sb[nj];
        bias[j] = a.bias ? a.bias[nj] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = m0 + 16 * t + r;
        if (m >= a.M) continue;
        const float sa = a.sa[m];
        T *to = reinterpret_cast<T *>(a.C) + m * a.ldc + n;
        struct Four { T v[4]; } o;
        struct Words { uint32_t w[sizeof(T)]; };
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[j] = (T)output(a, acc[t][j], sa, sb[j], bias[j]);
        store_values(to, __builtin_bit_cast(Words, o).w, a.N - n);
    }
}

// ---- short rows: bound by the stores of C ------------------------------------------------------------------------------
// 128 x 128 of C per workgroup, 64 x 64 per wave in four 32 x 32 blocks of v_mfma_i32_32x32x32_i8.  Tiles of 64 columns go
// through LDS (two buffers; rows of 64 bytes, the chunk position XORed with the row so that fragment reads spread over
// the banks).  Operand layout of the instruction: lane l holds 16 bytes of row l & 31, columns 16 (l >> 5) .. + 16;
// result register j of lane l is row (j & 3) + 8 (j >> 2) + 4 (l >> 5), column l & 31.
template <class T>
__global__ __launch_bounds__(256) void matmul_i8_kernel(MatmulArgs a)
{
    constexpr int BM = 128, BN = 128, KB = 64;
    __shared__ __align__(16) char lds[2][(BM + BN) * KB];
    __shared__ float scale_a[BM];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, h = lane >> 5;
    const int64_t n_tiles = (a.N + BN - 1) / BN;
    const int64_t m0 = (int64_t)(blockIdx.x / n_tiles) * BM, n0 = (int64_t)(blockIdx.x % n_tiles) * BN;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    // the scales and biases are requested first: they are here when the products are done
    if (tid < BM) scale_a[tid] = a.sa[m0 + tid < a.M ? m0 + tid : a.M - 1];
    float sb[2], bias[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + wn + 32 * j + r, nc = n < a.N ? n : a.N - 1;
        sb[j] = a.sb[nc];
        bias[j] = a.bias ? a.bias[nc] : 0.f;
    }
    i32x16 acc[2][2] = {};
    uint4 st[4];
    auto load = [&](int64_t kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = (tid + 256 * i) & 511, row = c >> 2;
            const int64_t k = kt * KB + (c & 3) * 16;
            const bool is_a = i < 2;
            int64_t g = (is_a ? m0 : n0) + row;
            const int64_t last = (is_a ? a.M : a.N) - 1;
            g = g < last ? g : last;
            st[i] = make_uint4(0, 0, 0, 0);
            if (k < a.K) st[i] = *reinterpret_cast<const uint4 *>((is_a ? a.A + g * a.lda : a.B + g * a.ldb) + k);
            if (is_a) st[i] = keep_below(st[i], k, a.K);
        }
    };
    auto swz = [](int row, int c) { return row * KB + ((c ^ ((row >> 1) & 3)) * 16); };
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = (tid + 256 * i) & 511, row = c >> 2;
            *reinterpret_cast<uint4 *>(lds[buf] + (i < 2 ? 0 : BM * KB) + swz(row, c & 3)) = st[i];
        }
    };
    const int64_t steps = (a.K + KB - 1) / KB;
    load(0);
    put(0);
    __syncthreads();
    for (int64_t kt = 0; kt < steps; ++kt) {
        const int buf = (int)(kt & 1);
        if (kt + 1 < steps) load(kt + 1);
#pragma unroll
        for (int ks = 0; ks < KB / 32; ++ks) {
            i32x4 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const i32x4 *>(lds[buf] + swz(wm + 32 * i + r, 2 * ks + h));
                fb[i] = *reinterpret_cast<const i32x4 *>(lds[buf] + BM * KB + swz(wn + 32 * i + r, 2 * ks + h));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
        if (kt + 1 < steps) put(buf ^ 1);
        __syncthreads();
    }
    // C through LDS, 16 rows of a wave's 64 columns at a time (rows padded by 16 bytes): stores of 16 bytes a lane that
    // cover whole 128- or 256-byte pieces of C's rows
    constexpr int PITCH = 64 * sizeof(T) + 16, LANES = 64 * sizeof(T) / 16, PER = 16 / sizeof(T);
    char *mine = lds[0] + wave * 16 * PITCH;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int e = 8 * half; e < 8 * half + 8; ++e) {
                const int row = (e & 3) + 8 * (e >> 2) + 4 * h;
                const float sa = scale_a[wm + 32 * i + row];
#pragma unroll
                for (int j = 0; j < 2; ++j) *reinterpret_cast<T *>(mine + (row & 15) * PITCH + (32 * j + r) * sizeof(T)) = (T)output(a, acc[i][j][e], sa, sb[j], bias[j]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 16 * LANES / 64; ++q) {
                const int row = (64 * q + lane) / LANES, col = (64 * q + lane) % LANES * PER;
                const int64_t m = m0 + wm + 32 * i + 16 * half + row, n = n0 + wn + col;
                const uint4 v = *reinterpret_cast<const uint4 *>(mine + row * PITCH + col * sizeof(T));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                if (m < a.M) store_values(reinterpret_cast<T *>(a.C) + m * a.ldc + n, w, a.N - n);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
}

// ---- large products: WM x WN waves, FM x FN blocks of 32 x 32 of C per wave ----------------------------------------------
// 256 x 256 of C per workgroup (2 x 4 waves of 4 x 2 blocks, two waves a SIMD; 8192 x 8192 x 8192 482 us, 2.28 * 10^15
// operations/s), or 128 x 128 (2 x 2 waves of 2 x 2 blocks) where the larger tiles are too few for the chip.  At 4096 x 8192 x 8192
// the matrix pipes are busy 55 % of the cycles, at 1.9 GHz, the clock the chip holds under this load; LDS bank conflicts take 21 %
// of the cycles, the rest are waits between fragments and products.
// A step takes 128 columns: 4 FM FN matrix instructions a wave.  Rows go from memory straight into LDS
// (global_load_lds_dwordx4: one kilobyte, eight rows, per instruction and wave), NB buffers: the loads of step s + NB - 1 are
// issued among the products of step s.  The LDS image has no row padding; position c of row r holds the row's chunk c ^ (r & 7),
// so that fragment reads spread over the banks (the swizzle is on the source address).  Rows past the ends of A and B read
// the last row, columns past K are masked out of A's fragments in the last step.  C goes out through LDS, so that stores cover
// whole 128-byte pieces of its rows.
// With one workgroup a CU (NB = 4) a SIMD has one wave, and nothing hides its waits but itself: fragments are read two
// products ahead, requests cost one vector instruction each (scalar base, 32-bit offsets).  A step is then 0.45 us, 0.7 without
// (the products alone 0.21): 512 x 4096 x 8192 37 us.
template <int WM, int WN, int FM, int FN, int NB>
struct BigGeom {
    static constexpr int NW = WM * WN, SIDE = 32 * FM * WM, KB = 128, HALF = SIDE * KB, BUF = 2 * HALF;
    static_assert(SIDE == 32 * FN * WN && SIDE / 8 == 4 * NW && FN == 2 && 2 * BUF / NW == 16384 && NB >= 2 && NB <= 4, "tiles are square, four loads a wave and side, 64 columns a wave");
    static constexpr int LDS = NB * BUF + SIDE * 4;    // the buffers, and A's scales
    static_assert(LDS <= 160 << 10, "more than a CU's LDS");
};

template <class T, int WM, int WN, int FM, int FN, int NB>
__global__ __launch_bounds__((64 * WM * WN)) void matmul_i8_big_kernel(MatmulArgs a, int tiles_m, int tiles_n)
{
    using G = BigGeom<WM, WN, FM, FN, NB>;
    constexpr int KB = G::KB, HALF = G::HALF, BUF = G::BUF, NW = G::NW, SIDE = G::SIDE;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, h = lane >> 5;
    // consecutive workgroups go to the 8 XCDs in turn: each XCD takes one run of tiles, four tiles of A rows at a time, so
    // that the tiles it works on together share rows of A and B in its L2
    const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
    const int t = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if (t >= tiles || (int)(blockIdx.x / 8) >= per) return;
    const int band = t / (4 * tiles_n), in_band = t - band * 4 * tiles_n;
    const int band_m = tiles_m - 4 * band < 4 ? tiles_m - 4 * band : 4;
    const int64_t m0 = (int64_t)(4 * band + in_band % band_m) * SIDE, n0 = (int64_t)(in_band / band_m) * SIDE;

    // this wave's rows of a step: 8 * (NW i + wave) + lane / 8 of A and of B, i = 0..3, as offsets from the tile's first rows
    // (the launch code sees to it that they fit 32 bits); the step's columns are in the scalar base
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    uint32_t from[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 8 * (NW * i + wave) + (lane >> 3);
        const int64_t last_a = a.M - 1 - m0, last_b = a.N - 1 - n0;
        from[i] = (uint32_t)((row < last_a ? row : last_a) * a.lda) + chunk;
        from[4 + i] = (uint32_t)((row < last_b ? row : last_b) * a.ldb) + chunk;
    }
    const char *base_a = (const char *)a.A + m0 * a.lda, *base_b = (const char *)a.B + n0 * a.ldb;
    float *scale_a = reinterpret_cast<float *>(lds + NB * BUF);
    if (tid < SIDE) scale_a[tid] = a.sa[m0 + tid < a.M ? m0 + tid : a.M - 1];
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + wave * 1024);
    const int steps = (int)((a.K + KB - 1) / KB);        // (K <= 131071)
    // load i of step s into buffer buf; lanes whose chunk of the last step begins past K read its first
    auto request = [&](int s, int buf, int i) {
        const uint32_t back = s + 1 == steps && s * KB + chunk >= (int)a.K ? chunk : 0;
        const char *base = (i < 4 ? base_a : base_b) + s * KB;
        const uint32_t to = lds0 + buf * BUF + (i >> 2) * HALF + NW * (i & 3) * 1024;
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(from[i] - back), "s"(base), "s"(to) : "memory", "m0");
    };
    const int wm = wave / WN * (32 * FM), wn = wave % WN * (32 * FN);
    int off[KB / 32];
#pragma unroll
    for (int ks = 0; ks < KB / 32; ++ks) off[ks] = r * KB + (((2 * ks + h) ^ (r & 7)) * 16);
    i32x16 acc[FM][FN] = {};
#pragma unroll
    for (int q = 0; q < NB - 1; ++q)
        if (q < steps)
#pragma unroll
            for (int i = 0; i < 8; ++i) request(q, q, i);
    // Step s's rows are here: this wave's loads of it have landed (of up to NB - 2 later steps 8 each may be under way; loads
    // return in order, and there are no others), after the barrier everyone's; and everyone's earlier fragment reads are done.
    auto landed = [&](int s) {
        if (NB > 3 && s + 2 < steps) asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)" ::: "memory");
        else if (NB > 2 && s + 1 < steps) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr int KS = KB / 32, SLOTS = NB == 2 ? 2 : KS;
    i32x4 fa[SLOTS][FM], fb[SLOTS][FN];
    auto fragments = [&](int buf, int ks) {
        const char *A = lds + buf * BUF + wm * KB, *B = lds + buf * BUF + HALF + wn * KB;
        const int to = ks % SLOTS;
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[to][i] = *reinterpret_cast<const i32x4 *>(A + off[ks] + 32 * i * KB);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[to][j] = *reinterpret_cast<const i32x4 *>(B + off[ks] + 32 * j * KB);
    };
    // columns from K on (in the last step) count as zeros
    auto cut = [&](int ks) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
            fa[ks % SLOTS][i] = __builtin_bit_cast(i32x4, keep_below(__builtin_bit_cast(uint4, fa[ks % SLOTS][i]), (steps - 1) * KB + 32 * ks + 16 * h, a.K));
    };
    auto products = [&](int ks) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[ks % SLOTS][i], fb[ks % SLOTS][j], acc[i][j], 0, 0, 0);
    };
    if constexpr (NB == 2) {
        for (int s = 0; s < steps; ++s) {
            const int buf = s & 1;
            const bool last = s + 1 == steps;
            landed(s);
            fragments(buf, 0);
            if (last) cut(0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 1 < KS) {
                    fragments(buf, ks + 1);
                    if (last) cut(ks + 1);
                }
                if (!last) {
                    request(s + 1, buf ^ 1, 2 * ks);
                    request(s + 1, buf ^ 1, 2 * ks + 1);
                }
                products(ks);
            }
        }
    } else {
        // one wave a SIMD: fragments are read two products ahead, past the barrier between two steps
        landed(0);
        fragments(0, 0);
        fragments(0, 1);
        int buf = 0;
        for (int s = 0; s + 1 < steps; ++s) {
            const int before = buf == 0 ? NB - 1 : buf - 1, next = buf + 1 == NB ? 0 : buf + 1;      // the buffers of steps s - 1 and s + 1
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 2 == KS) landed(s + 1);
                fragments(ks + 2 < KS ? buf : next, (ks + 2) % KS);
                if (ks < 2 && s + NB - 1 < steps)
#pragma unroll
                    for (int i = 4 * ks; i < 4 * ks + 4; ++i) request(s + NB - 1, before, i);
                __builtin_amdgcn_sched_barrier(0);
                products(ks);
                __builtin_amdgcn_sched_barrier(0);
            }
            buf = next;
        }
        fragments(buf, 2);
        fragments(buf, 3);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            cut(ks);
            products(ks);
        }
    }
    __syncthreads();

    // C: a wave's 32 FM x 64 in pieces of 32 rows through its 16 KB of LDS (rows padded by 16 bytes)
    constexpr int PITCH = 64 * sizeof(T) + 16, LANES = 64 * sizeof(T) / 16, PER = 16 / sizeof(T);
    static_assert(32 * PITCH <= 16384, "a wave's piece exceeds its LDS");
    char *mine = lds + wave * 16384;
    float sb[FN], bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int64_t n = n0 + wn + 32 * j + r, nc = n < a.N ? n : a.N - 1;
        sb[j] = a.sb[nc];
        bias[j] = a.bias ? a.bias[nc] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int row = (e & 3) + 8 * (e >> 2) + 4 * h;
            const float sa = scale_a[wm + 32 * i + row];
#pragma unroll
            for (int j = 0; j < FN; ++j) *reinterpret_cast<T *>(mine + row * PITCH + (32 * j + r) * sizeof(T)) = (T)output(a, acc[i][j][e], sa, sb[j], bias[j]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 32 * LANES / 64; ++q) {
            const int row = (64 * q + lane) / LANES, col = (64 * q + lane) % LANES * PER;
            const int64_t m = m0 + wm + 32 * i + row, n = n0 + wn + col;
            const uint4 v = *reinterpret_cast<const uint4 *>(mine + row * PITCH + col * sizeof(T));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            if (m < a.M) store_values(reinterpret_cast<T *>(a.C) + m * a.ldc + n, w, a.N - n);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <class T, int WM, int WN, int FM, int FN, int NB>
static int launch_big(tfrec_ctx *ctx, const MatmulArgs &a)
{
    using G = BigGeom<WM, WN, FM, FN, NB>;
    const int64_t tm = (a.M + G::SIDE - 1) / G::SIDE, tn = (a.N + G::SIDE - 1) / G::SIDE, tiles = tm * tn;
    TF_TRY(check_launch((tiles + 7) / 8 * 8, 64 * G::NW));
    static std::atomic<uint64_t> done{0};
    TF_TRY(tfrec_raise_lds_limit(ctx, reinterpret_cast<const void *>(&matmul_i8_big_kernel<T, WM, WN, FM, FN, NB>), G::LDS, done));
    matmul_i8_big_kernel<T, WM, WN, FM, FN, NB><<<(unsigned)((tiles + 7) / 8 * 8), 64 * G::NW, G::LDS, ctx->stream>>>(a, (int)tm, (int)tn);
    TF_HIP(hipGetLastError());
    return TFREC_OK;
}

// Which kernel (us, measured on both sides of each rule):
//   256 x 256 tiles where they fill the chip and a row is long enough to repay 128 KB of LDS, one workgroup a CU
//     (4096 x 8192 x 8192: 254; 128 x 128 tiles 284 to 370);
//   128 x 128 tiles where the time that reading B for 16 of its rows at a time takes (what a sweep over M, N and K measured:
//     more with every row of A) exceeds that of the tiles, a chain of K / 128 steps: 16 x 65536 x 4096 47 / 70,
//     512 x 4096 x 4096 22 / 69, 77 x 5003 x 1210 11 / 8.9, 128 x 4096 x 4096 20 / 21, 1 x 8192 x 8192 34 / 15.  Up to one tile a CU with
//     four buffers (512 x 8192 x 4096: 26, with two 32), beyond with two and two workgroups a CU (1024 x 8192 x 4096: 40, 51);
//   short rows (512 columns and a float32 output, 256 and 16 bits) are bound by the stores of C, which the kernel with 33 KB of
//     LDS and several workgroups a CU serves best: 2048 x 200000 x 64 in float32 300 (5.5 TB/s; a fill of C alone 240) against
//     454, 2048 x 50000 x 256 in float32 113 / 151, in bfloat16 even, x 512 even / in bfloat16 128 / 100;
//   16 rows of B at a time for everything else: small products get workgroups enough, few rows of A are bound by reading B.
static int choose_matmul(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int c_bytes)
{
    const int64_t big = ((M + 255) / 256) * ((N + 255) / 256), mid = ((M + 127) / 128) * ((N + 127) / 128);
    const bool near = lda < (1 << 24) && ldb < (1 << 24);        // a tile's rows are within 4 GB of its first
    const double rows_us = (double)N * (double)K * (1.6e-7 + 6.2e-9 * (double)M);
    const double tiles_us = (2.2 + 3.65e-3 * (double)K) * (mid > 256 ? (double)mid / 230. : 1.);
    const bool stores = M > 64 && mid >= 192 && K <= 128 * (int64_t)c_bytes;
    if (near && !stores && M > 128 && K >= 512 && big >= 160) return TFREC_I8_TILES_256;
    if (near && !stores && K >= 256 && rows_us > tiles_us) return mid <= 256 ? TFREC_I8_TILES_128_DEEP : TFREC_I8_TILES_128;
    return stores || (M > 64 && mid >= 192) ? TFREC_I8_SHORT : TFREC_I8_ROWS;
}

template <class T>
static int launch_matmul(tfrec_ctx *ctx, const MatmulArgs &a)
{
    switch (choose_matmul(a.M, a.N, a.K, a.lda, a.ldb, sizeof(T))) {
    case TFREC_I8_TILES_256: return launch_big<T, 2, 4, 4, 2, 2>(ctx, a);
    case TFREC_I8_TILES_128_DEEP: return launch_big<T, 2, 2, 2, 2, 4>(ctx, a);
    case TFREC_I8_TILES_128: return launch_big<T, 2, 2, 2, 2, 2>(ctx, a);
    case TFREC_I8_SHORT: {
        const int64_t tiles = ((a.M + 127) / 128) * ((a.N + 127) / 128);
        TF_TRY(check_launch(tiles, 256));
        matmul_i8_kernel<T><<<(unsigned)tiles, 256, 0, ctx->stream>>>(a);
        break;
    }
    default: {
        const int64_t nb = (a.N + 15) / 16;
        TF_TRY(check_launch(nb, 64 * 8));
        auto go = [&]<int MT, int KW>() { matmul_i8_rows_kernel<T, MT, KW><<<dim3((unsigned)nb, (unsigned)((a.M + 16 * MT - 1) / (16 * MT))), 64 * KW, 0, ctx->stream>>>(a); };
        auto waves = [&]<int MT>() {
            if (a.K <= 256) go.template operator()<MT, 1>();
            else if (a.K <= 2048 || MT == 8) go.template operator()<MT, 4>();
            else if constexpr (MT < 8) go.template operator()<MT, 8>();
        };
        if (a.M <= 16) waves.template operator()<1>();
        else if (a.M <= 32) waves.template operator()<2>();
        else if (a.M <= 64) waves.template operator()<4>();
        else waves.template operator()<8>();
    }
    }
    TF_HIP(hipGetLastError());
    return TFREC_OK;
}

extern "C" int tfrec_matmul_i8_kernel(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int c_dtype)
{
    return choose_matmul(M, N, K, lda, ldb, c_dtype == TFREC_DT_F32 ? 4 : 2);
}

extern "C" int tfrec_matmul_i8(tfrec_ctx *ctx, const int8_t *d_A, int64_t lda, const float *d_sa, int64_t M, const int8_t *d_B, int64_t ldb,
                               const float *d_sb, int64_t N, int64_t K, const float *d_bias, void *d_C, int c_dtype, int64_t ldc)
{
    TF_REQUIRE(dtype_ok(c_dtype), TFREC_EINVAL, "unknown output type %d", c_dtype);
    TF_REQUIRE(M >= 0 && N >= 0 && K >= 1 && ldc >= N, TFREC_EINVAL, "bad shape M=%lld N=%lld K=%lld ldc=%lld", (long long)M, (long long)N, (long long)K,
               (long long)ldc);
    TF_REQUIRE(K <= 131071, TFREC_EUNSUP, "K=%lld: sums beyond 131071 products may leave 32 bits", (long long)K);
    TF_TRY(tfrec_check_i8("A", d_A, M, lda, K));
    TF_TRY(tfrec_check_i8("B", d_B, N, ldb, K));
    TF_REQUIRE(M == 0 || N == 0 || (d_sa && d_sb && d_C), TFREC_EINVAL, "null pointer");
    TF_REQUIRE(((uintptr_t)d_C & (c_dtype == TFREC_DT_F32 ? 3u : 1u)) == 0, TFREC_EINVAL, "C is not aligned to its type");
    TF_TRY(tfrec_ctx_enter(ctx));
    if (M == 0 || N == 0) return TFREC_OK;
    const int64_t es = c_dtype == TFREC_DT_F32 ? 4 : 2;
    const RowBytes c{(uintptr_t)d_C, ldc * es, N * es, M};
    for (const RowBytes &r : {RowBytes{(uintptr_t)d_A, lda, K, M}, RowBytes{(uintptr_t)d_B, ldb, K, N}, array_bytes(d_sa, M, 4), array_bytes(d_sb, N, 4), array_bytes(d_bias, N, 4)})
        TF_REQUIRE(!rows_overlap(c, r), TFREC_EINVAL, "C overlaps an operand, a scale or the bias");
    // (pieces of 2^26 rows of A and of B; the sums are integers: no result depends on it)
    constexpr int64_t PIECE = 16 * TF_LAUNCH_ROWS;
    for (int64_t m = 0; m < M; m += PIECE)
        for (int64_t n = 0; n < N; n += PIECE) {
            const MatmulArgs a{d_A + m * lda, d_B + n * ldb, d_sa + m, d_sb + n, d_bias ? d_bias + n : nullptr, (char *)d_C + (m * ldc + n) * es, lda, ldb, ldc,
                               M - m < PIECE ? M - m : PIECE, N - n < PIECE ? N - n : PIECE, K};
            if (c_dtype == TFREC_DT_BF16) TF_TRY(launch_matmul<__bf16>(ctx, a));
            else if (c_dtype == TFREC_DT_F16) TF_TRY(launch_matmul<_Float16>(ctx, a));
            else TF_TRY(launch_matmul<float>(ctx, a));
        }
    return TFREC_OK;
}
