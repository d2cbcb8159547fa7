// 8-bit rows: quantisation with a scale per row, and the matrix product of two such matrices.
#include "i8_device.hpp"
#include "score_i8.hpp"

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

static inline int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }
static inline bool dtype_ok(int t) { return t == TFREC_DT_F32 || t == TFREC_DT_BF16 || t == TFREC_DT_F16; }

// ------------------------------------------------------------------------------------------
// quantisation: scale = max|x| / 127, q = nearest-even(x / scale)
// ------------------------------------------------------------------------------------------
// The nearest integer to x / s, ties to even, exactly: r = rint(x * RN(1/s)) is off by at most one, and the remainder
// x - r s is exact in float32 (both are multiples of ulp(s) where |x| >= s, and |x - r s| < s otherwise), so comparing it
// with s / 2 decides.  Scales near the subnormal range are lifted by 2^64 first (exact; |x| <= 127.5 s).
__device__ __forceinline__ int quantize_one(float x, float s, float inv)
{
    float r = rintf(x * inv);
    const float e = fmaf(-r, s, x), half = 0.5f * s;
    const bool odd = ((int)r & 1) != 0;
    if (e > half || (e == half && odd)) r += 1.f;
    else if (e < -half || (e == -half && odd)) r -= 1.f;
    return (int)fminf(fmaxf(r, -127.f), 127.f);
}

template <class T>
struct Elem;
template <> struct Elem<float> { static __device__ __forceinline__ float get(const float *p) { return *p; } };
template <> struct Elem<__bf16> { static __device__ __forceinline__ float get(const __bf16 *p) { return (float)*p; } };
template <> struct Elem<_Float16> { static __device__ __forceinline__ float get(const _Float16 *p) { return (float)*p; } };

// LPR lanes (a power of two up to 64) hold one row, 16 columns per lane and round; two rounds over the row (the second
// finds it in the caches).
template <class T, int LPR>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T *__restrict__ X, int64_t n_rows, int64_t ldx, int64_t d,
                                                            const int32_t *__restrict__ rows, int64_t n, int8_t *__restrict__ q, int64_t ldq,
                                                            float *__restrict__ scale, uint32_t *__restrict__ flags)
{
    constexpr int GPB = 256 / LPR;
    const int gl = threadIdx.x % LPR;
    const int64_t r = (int64_t)blockIdx.x * GPB + threadIdx.x / LPR;
    if (r >= n) return;
    int64_t src = r;
    if (rows) {
        const int32_t id = rows[r];
        src = id < 0 ? 0 : (id >= n_rows ? n_rows - 1 : id);
        if (src != id && gl == 0) atomicOr(flags, TFREC_FLAG_BAD_INDEX);
    }
    const T *x = X + src * ldx;
    const int64_t chunks = (d + 15) / 16;
    float mx = 0.f;
    bool bad = false;
    for (int64_t c = gl; c < chunks; c += LPR)
        for (int j = 0; j < 16; ++j)
            if (c * 16 + j < d) {
                const float v = fabsf(Elem<T>::get(x + c * 16 + j));
                bad |= !(v < INFINITY);
                mx = fmaxf(mx, v);
            }
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) {
        mx = fmaxf(mx, __shfl_xor(mx, off, 64));
        bad |= __shfl_xor((int)bad, off, 64) != 0;
    }
    float s = mx / 127.0f;
    if (gl == 0) scale[r] = bad ? NAN : s;
    const bool none = bad || !(s > 0.f);
    const float up = s < 0x1p-60f ? 0x1p64f : 1.f;
    s *= up;
    const float inv = 1.f / s;
    for (int64_t c = gl; c < chunks; c += LPR) {
        union { int8_t b[16]; uint4 v; } o;
        for (int j = 0; j < 16; ++j)
            o.b[j] = !none && c * 16 + j < d ? (int8_t)quantize_one(Elem<T>::get(x + c * 16 + j) * up, s, inv) : 0;
        *reinterpret_cast<uint4 *>(q + r * ldq + c * 16) = o.v;
    }
}

template <class T>
static int launch_quantize(tfrec_ctx *ctx, const void *X, int64_t n_rows, int64_t ldx, int64_t d, const int32_t *rows, int64_t n, int8_t *q,
                           int64_t ldq, float *scale)
{
    auto go = [&]<int LPR>() -> int {
        constexpr int GPB = 256 / LPR;
        const int64_t blocks = (n + GPB - 1) / GPB;
        TF_REQUIRE(blocks < (1ll << 31), TFREC_EUNSUP, "too many rows");
        quantize_rows_kernel<T, LPR><<<(unsigned)blocks, 256, 0, ctx->stream>>>((const T *)X, n_rows, ldx, d, rows, n, q, ldq, scale, ctx->d_flags);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    };
    const int64_t chunks = (d + 15) / 16;
    if (chunks <= 4) return go.template operator()<4>();
    if (chunks <= 16) return go.template operator()<16>();
    return go.template operator()<64>();
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
    return tfrec_quantize_rows(ctx, d_X, x_dtype, n_rows, ldx, d, d_rows, n, d_q, ldq, d_scale);
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

template <class T>
__device__ __forceinline__ void store_out(void *C, int64_t at, float v) { reinterpret_cast<T *>(C)[at] = (T)v; }

// 128 x 128 of C per workgroup, 64 x 64 per wave in four 32 x 32 blocks of v_mfma_i32_32x32x32_i8.  Tiles of 64 columns go
// through LDS (two buffers; rows of 64 bytes, the chunk position XORed with the row so that fragment reads spread over
// the banks).  Operand layout of the instruction: lane l holds 16 bytes of row l & 31, columns 16 (l >> 5) .. + 16;
// result register j of lane l is row (j & 3) + 8 (j >> 2) + 4 (l >> 5), column l & 31.
template <class T>
__global__ __launch_bounds__(256) void matmul_i8_kernel(MatmulArgs a)
{
    constexpr int BM = 128, BN = 128, KB = 64;
    __shared__ __align__(16) char lds[2][(BM + BN) * KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, h = lane >> 5;
    const int64_t n_tiles = (a.N + BN - 1) / BN;
    const int64_t m0 = (int64_t)(blockIdx.x / n_tiles) * BM, n0 = (int64_t)(blockIdx.x % n_tiles) * BN;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
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
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + wn + 32 * j + r;
        if (n >= a.N) continue;
        const float sb = a.sb[n], bias = a.bias ? a.bias[n] : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int64_t m = m0 + wm + 32 * i + (e & 3) + 8 * (e >> 2) + 4 * h;
                if (m < a.M) {
                    float v = scaled_sum(acc[i][j][e], a.sa[m], sb);
                    if (a.bias) v = add_rounded(v, bias);
                    store_out<T>(a.C, m * a.ldc + n, v);
                }
            }
    }
}

template <class T>
static int launch_matmul(tfrec_ctx *ctx, const MatmulArgs &a)
{
    const int64_t tiles = ((a.M + 127) / 128) * ((a.N + 127) / 128);
    TF_REQUIRE(tiles < (1ll << 31), TFREC_EUNSUP, "the product is too large for one launch");
    matmul_i8_kernel<T><<<(unsigned)tiles, 256, 0, ctx->stream>>>(a);
    TF_HIP(hipGetLastError());
    return TFREC_OK;
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
    const MatmulArgs a{d_A, d_B, d_sa, d_sb, d_bias, d_C, lda, ldb, ldc, M, N, K};
    if (c_dtype == TFREC_DT_BF16) return launch_matmul<__bf16>(ctx, a);
    if (c_dtype == TFREC_DT_F16) return launch_matmul<_Float16>(ctx, a);
    return launch_matmul<float>(ctx, a);
}
