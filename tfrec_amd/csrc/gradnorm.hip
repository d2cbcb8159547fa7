// Global l2 norm over many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over all values of g^2),   out = g * max_norm / max(norm, max_norm)
//
// Bound by memory: every value is read once for the norm and, where it is scaled, once more and written.  The tensors are
// cut into chunks of CHUNK values; workgroups take chunks in a fixed pattern and leave one float64 partial sum each, which
// are added in a fixed order, so results do not depend on scheduling.  Squares are formed and summed in float64: no
// float32 value's square leaves its range, and the sum of 10^9 values keeps more bits than the result has.
#include "common.hpp"

static constexpr int GRAD_TENSORS = 96;        // tensors per launch of a call without a list: their table rides in the kernel's arguments (below 4 KB)
static constexpr int GRAD_CHUNK = 8192;        // values per chunk
static constexpr int GRAD_BLOCKS = 2048;       // partial sums (and workgroups at most)
static constexpr int GRAD_SMALL = 8;           // chunks one workgroup holds in its registers
static_assert(GRAD_BLOCKS * sizeof(double) <= TFREC_SMALL_BYTES, "partial sums exceed the context's scratch");

// a chunk: `len` values of one tensor
struct GradChunk {
    const void *src;
    void *dst;
    int32_t len, dtype;
    int64_t unused;                            // (32 bytes: one scalar load)
};

// where a kernel finds chunk c: in a list on the device ...
struct GradListed {
    const GradChunk *at;
    int64_t chunks;
    __device__ __forceinline__ GradChunk get(int64_t c) const { return at[c]; }
};

// ... or by a search among the tensors of a table in its arguments
struct GradTable {
    const void *src[GRAD_TENSORS];
    void *dst[GRAD_TENSORS];
    int64_t count[GRAD_TENSORS];
    int64_t first[GRAD_TENSORS];               // first chunk of the tensor; ascending
    uint8_t dtype[GRAD_TENSORS];
    int n;
    int64_t chunks;
    __device__ __forceinline__ GradChunk get(int64_t c) const
    {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= c) lo = mid; else hi = mid;
        }
        const int64_t at = (c - first[lo]) * GRAD_CHUNK, left = count[lo] - at, es = dtype[lo] == TFREC_DT_F32 ? 4 : 2;
        return GradChunk{(const char *)src[lo] + at * es, dst[lo] ? (char *)dst[lo] + at * es : nullptr, (int32_t)(left < GRAD_CHUNK ? left : GRAD_CHUNK),
                         dtype[lo], 0};
    }
};

// 16 bytes at the alignment of the element type (global memory takes them at any)
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[16 / sizeof(T)]; };

// f.operator()<T>(src, dst) with the chunk's type
template <class F>
__device__ __forceinline__ void by_type(const GradChunk &c, F &&f)
{
    if (c.dtype == TFREC_DT_F32) f.template operator()<float>((const float *)c.src, (float *)c.dst);
    else if (c.dtype == TFREC_DT_BF16) f.template operator()<__bf16>((const __bf16 *)c.src, (__bf16 *)c.dst);
    else f.template operator()<_Float16>((const _Float16 *)c.src, (_Float16 *)c.dst);
}

template <class T>
__device__ __forceinline__ double chunk_squares(const T *__restrict__ x, int m, double s)
{
    constexpr int V = 16 / sizeof(T), R = GRAD_CHUNK / (256 * V);
    if (m == GRAD_CHUNK) {
        Pack<T> p[R];
#pragma unroll
        for (int r = 0; r < R; ++r) p[r] = reinterpret_cast<const Pack<T> *>(x)[r * 256 + threadIdx.x];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) { const double v = (double)(float)p[r].v[j]; s = fma(v, v, s); }
    } else {
        for (int i = threadIdx.x; i < m; i += 256) { const double v = (double)(float)x[i]; s = fma(v, v, s); }
    }
    return s;
}

// The factor s of every value: max_norm / norm in float64, as hi + lo in float32.  hi alone would cost a second half step;
// fma(x, hi, x * lo) is x s rounded once (lo is within 2^-48 of what hi leaves; next to the subnormal numbers x * lo may be half a
// step off), in two instructions.  Factors below 2^-76, whose lo could leave float32's range (bounds of 1e-38 beside gradients of
// 1e30), take the product in float64; all values that way cost 40 MB of bfloat16 in 600 tensors 23.4 us against 22.2.
// A sum of squares of finite float32 values stays finite in float64: a norm that is not finite means an infinity or NaN among the
// values.
struct GradFactor {
    double s;
    float hi, lo;
    __device__ __forceinline__ GradFactor(double norm, double max_norm)
    {
        s = !(norm < (double)INFINITY) ? (double)NAN : (norm <= max_norm ? 1. : max_norm / norm);
        hi = (float)s;
        lo = (float)(s - (double)hi);
    }
    // in place and within the bound: every value is what it was
    __device__ __forceinline__ bool nothing(const GradChunk &c) const { return s == 1. && c.src == c.dst; }
    // calls f(scale) with the form of the product, the same for all values
    template <class F>
    __device__ __forceinline__ void with(F &&f) const
    {
        const float h = hi, l = lo;
        const double d = s;
        if (d < 0x1p-76) f([=](float x) { return (float)((double)x * d); });
        else f([=](float x) { return fmaf(x, h, x * l); });
    }
};

template <class T, class Scale>
__device__ __forceinline__ void chunk_scale(const T *x, T *y, int m, Scale &&f)
{
    constexpr int V = 16 / sizeof(T), R = GRAD_CHUNK / (256 * V);
    if (m == GRAD_CHUNK) {
        Pack<T> p[R];
#pragma unroll
        for (int r = 0; r < R; ++r) p[r] = reinterpret_cast<const Pack<T> *>(x)[r * 256 + threadIdx.x];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < V; ++j) p[r].v[j] = (T)f((float)p[r].v[j]);
            reinterpret_cast<Pack<T> *>(y)[r * 256 + threadIdx.x] = p[r];
        }
    } else {
        for (int i = threadIdx.x; i < m; i += 256) y[i] = (T)f((float)x[i]);
    }
}

// sum over the workgroup's NW waves, the same on every thread, in a fixed order
template <int NW>
__device__ __forceinline__ double block_sum(double v)
{
    __shared__ double red[NW];
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w];
    __syncthreads();
    return v;
}

// 308 MB of float32 in 3 tensors: 77 us, 4.0 TB/s, as much as a plain sum of them reads and two thirds of what grad_scale_kernel
// moves: a workgroup has one chunk on its way at a time.  40 MB of bfloat16 in 600 tensors 16 us.  2048 workgroups: 4096 take 14 us
// and their norm 1 us more, 1024 take 21 us.
// partial sum of workgroup b over its chunks b, b + grid, ...; `first`: the first launch of a call, which sets the partials
template <class Table>
__global__ __launch_bounds__(256) void grad_squares_kernel(Table t, double *__restrict__ part, int first)
{
    double s = 0.;
    for (int64_t k = blockIdx.x; k < t.chunks; k += gridDim.x) {
        const GradChunk c = t.get(k);
        by_type(c, [&]<class T>(const T *x, T *) { s = chunk_squares(x, c.len, s); });
    }
    s = block_sum<4>(s);
    if (threadIdx.x == 0) part[blockIdx.x] = first ? s : part[blockIdx.x] + s;
}

// the norm from the partial sums, on every thread; every workgroup that wants it forms it the same way
__device__ __forceinline__ double norm_of(const double *__restrict__ part, int n_part)
{
    double s = 0.;
    for (int i = threadIdx.x; i < n_part; i += 256) s += part[i];
    return sqrt(block_sum<4>(s));
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double *__restrict__ part, int n_part, float *__restrict__ norm)
{
    const double nm = norm_of(part, n_part);
    if (threadIdx.x == 0) *norm = (float)nm;
}

// 308 MB of float32: 102 us, 6.0 TB/s of reads and writes; 40 MB of bfloat16 in 600 tensors 22 us, of which every workgroup spends
// some adding the partial sums before it requests its first chunk.
template <class Table>
__global__ __launch_bounds__(256) void grad_scale_kernel(Table t, const double *__restrict__ part, int n_part, double max_norm, float *__restrict__ norm)
{
    const double nm = norm_of(part, n_part);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nm;
    const GradFactor f(nm, max_norm);
    // the last chunks first: what the norm read last is still cached
    f.with([&](auto &&scale) {
        for (int64_t k = blockIdx.x; k < t.chunks; k += gridDim.x) {
            const GradChunk c = t.get(t.chunks - 1 - k);
            if (!f.nothing(c)) by_type(c, [&]<class T>(const T *x, T *y) { chunk_scale(x, y, c.len, scale); });
        }
    });
}

// Few values: one workgroup holds all of them in registers between the norm and the product (one launch, one read).
// Up to 8 chunks: 54182 values in 3 tensors 10 us.
template <class Table>
__global__ __launch_bounds__(1024) void grad_clip_small_kernel(Table t, double max_norm, float *__restrict__ norm)
{
    uint4 held[GRAD_SMALL][2];                 // 8 values of each chunk: two packs of 4, or one of 8
    double s = 0.;
    const int n = (int)t.chunks;
    GradChunk cs[GRAD_SMALL];                  // all looked up before the first is used: one wait, not one per chunk
#pragma unroll
    for (int k = 0; k < GRAD_SMALL; ++k) cs[k] = n ? t.get(k < n ? k : n - 1) : GradChunk{};
#pragma unroll
    for (int k = 0; k < GRAD_SMALL; ++k) {
        if (k >= n) break;
        const GradChunk &c = cs[k];
        by_type(c, [&]<class T>(const T *x, T *) {
            constexpr int V = 16 / sizeof(T), R = 8 / V;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int i = (r * 1024 + threadIdx.x) * V;
                Pack<T> p;
                if (i + V <= c.len) p = *reinterpret_cast<const Pack<T> *>(x + i);
                else
#pragma unroll
                    for (int j = 0; j < V; ++j) p.v[j] = i + j < c.len ? x[i + j] : (T)0.f;
                held[k][r] = __builtin_bit_cast(uint4, p);
            }
        });
    }
#pragma unroll
    for (int k = 0; k < GRAD_SMALL; ++k) {
        if (k >= n) break;
        const GradChunk &c = cs[k];
        by_type(c, [&]<class T>(const T *, T *) {
            constexpr int V = 16 / sizeof(T), R = 8 / V;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const Pack<T> p = __builtin_bit_cast(Pack<T>, held[k][r]);
#pragma unroll
                for (int j = 0; j < V; ++j) { const double v = (double)(float)p.v[j]; s = fma(v, v, s); }
            }
        });
    }
    const double nm = sqrt(block_sum<16>(s));
    if (norm && threadIdx.x == 0) *norm = (float)nm;
    const GradFactor f(nm, max_norm);
    f.with([&](auto &&scale) {
#pragma unroll
        for (int k = 0; k < GRAD_SMALL; ++k) {
            if (k >= n) break;
            const GradChunk &c = cs[k];
            if (f.nothing(c)) continue;
            by_type(c, [&]<class T>(const T *, T *y) {
                constexpr int V = 16 / sizeof(T), R = 8 / V;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int i = (r * 1024 + threadIdx.x) * V;
                    Pack<T> p = __builtin_bit_cast(Pack<T>, held[k][r]);
#pragma unroll
                    for (int j = 0; j < V; ++j) p.v[j] = (T)scale((float)p.v[j]);
                    if (i + V <= c.len) *reinterpret_cast<Pack<T> *>(y + i) = p;
                    else
                        for (int j = 0; j < V; ++j)
                            if (i + j < c.len) y[i + j] = p.v[j];
                }
            });
        }
    });
}

static inline size_t dt_size(int t) { return t == TFREC_DT_F32 ? 4 : 2; }

static int check_grads(int n, const void *const *g, const int64_t *counts, const int *dtypes)
{
    TF_REQUIRE(n >= 0, TFREC_EINVAL, "%d tensors", n);
    TF_REQUIRE(n == 0 || (g && counts && dtypes), TFREC_EINVAL, "null host array");
    for (int i = 0; i < n; ++i) {
        TF_REQUIRE(counts[i] >= 0 && counts[i] < (1ll << 40), TFREC_EINVAL, "tensor %d: a length of %lld", i, (long long)counts[i]);
        TF_REQUIRE(dtypes[i] == TFREC_DT_F32 || dtypes[i] == TFREC_DT_BF16 || dtypes[i] == TFREC_DT_F16, TFREC_EINVAL, "tensor %d: unknown type %d", i, dtypes[i]);
        TF_REQUIRE(counts[i] == 0 || g[i], TFREC_EINVAL, "tensor %d is null", i);
        TF_REQUIRE(((uintptr_t)g[i] & (dt_size(dtypes[i]) - 1)) == 0, TFREC_EINVAL, "tensor %d is not aligned to its type", i);
    }
    return TFREC_OK;
}

struct Range { uintptr_t lo, hi; int out; };       // out: index of the output

// by address (no library sort: nothing here may throw)
template <class R>
static void sort_ranges(R *r, size_t m)
{
    for (size_t gap = m / 2; gap > 0; gap /= 2)
        for (size_t i = gap; i < m; ++i) {
            const R x = r[i];
            size_t j = i;
            for (; j >= gap && r[j - gap].lo > x.lo; j -= gap) r[j] = r[j - gap];
            r[j] = x;
        }
}

// No output overlaps another output, or a gradient other than the one it replaces.
static int check_outputs(int n, const void *const *g, void *const *out, const int64_t *counts, const int *dtypes)
{
    TF_REQUIRE(n == 0 || out, TFREC_EINVAL, "null host array");
    Range *r = new (std::nothrow) Range[(size_t)n + 1];
    TF_REQUIRE(r != nullptr, TFREC_ENOMEM, "host allocation failed");
    size_t m = 0;
    int bad = -1, why = 0;
    bool sorted = true;
    for (int i = 0; i < n && bad < 0; ++i) {
        if (!counts[i]) continue;
        const size_t es = dt_size(dtypes[i]);
        if (!out[i]) { bad = i; why = 1; break; }
        if ((uintptr_t)out[i] & (es - 1)) { bad = i; why = 2; break; }
        r[m] = {(uintptr_t)out[i], (uintptr_t)out[i] + (size_t)counts[i] * es, i};
        sorted = sorted && (m == 0 || r[m - 1].hi <= r[m].lo);
        ++m;
    }
    if (bad < 0) {
        // outputs by address, then every gradient against the outputs around it
        if (!sorted) {
            sort_ranges(r, m);
            for (size_t i = 1; i < m; ++i)
                if (r[i - 1].hi > r[i].lo) { bad = r[i].out; why = 3; break; }
        }
        for (int i = 0; i < n && bad < 0; ++i) {
            if (!counts[i]) continue;
            const uintptr_t lo = (uintptr_t)g[i], hi = lo + (size_t)counts[i] * dt_size(dtypes[i]);
            size_t a = 0, b = m;                                   // first output that ends behind lo
            while (a < b) {
                const size_t mid = (a + b) / 2;
                if (r[mid].hi <= lo) a = mid + 1; else b = mid;
            }
            for (; a < m && r[a].lo < hi; ++a)
                if (!(r[a].out == i && r[a].lo == lo)) { bad = r[a].out; why = 4; break; }
        }
    }
    delete[] r;
    TF_REQUIRE(bad < 0, TFREC_EINVAL, why == 1 ? "output %d is null" : why == 2 ? "output %d is not aligned to its type"
               : why == 3 ? "output %d overlaps another output" : "output %d overlaps a gradient that it does not replace", bad);
    return TFREC_OK;
}

// The norm is written while gradients are still read and outputs written: it may be no part of either.
static int check_norm_apart(int n, const void *const *g, void *const *out, const int64_t *counts, const int *dtypes, const float *d_norm)
{
    if (!d_norm) return TFREC_OK;
    const uintptr_t lo = (uintptr_t)d_norm, hi = lo + sizeof(float);
    for (int i = 0; i < n; ++i) {
        const size_t bytes = (size_t)counts[i] * dt_size(dtypes[i]);
        for (const void *p : {g[i], (const void *)out[i]})
            TF_REQUIRE(bytes == 0 || hi <= (uintptr_t)p || (uintptr_t)p + bytes <= lo, TFREC_EINVAL, "the norm lies within tensor %d", i);
    }
    return TFREC_OK;
}

// calls f(table) for the tensors in groups of GRAD_TENSORS, empty ones left out
template <class F>
static int for_tables(int n, const void *const *g, void *const *out, const int64_t *counts, const int *dtypes, F &&f)
{
    GradTable t;
    t.n = 0;
    t.chunks = 0;
    auto flush = [&]() -> int {
        if (t.n) TF_TRY(f(t));
        t.n = 0;
        t.chunks = 0;
        return TFREC_OK;
    };
    for (int i = 0; i < n; ++i) {
        if (!counts[i]) continue;
        t.src[t.n] = g[i];
        t.dst[t.n] = out ? out[i] : nullptr;
        t.count[t.n] = counts[i];
        t.first[t.n] = t.chunks;
        t.dtype[t.n] = (uint8_t)dtypes[i];
        t.chunks += (counts[i] + GRAD_CHUNK - 1) / GRAD_CHUNK;
        if (++t.n == GRAD_TENSORS) TF_TRY(flush());
    }
    return flush();
}

// One launch sequence over `tables` tables (each(f) calls f(table) for every one of them): the partial sums, then what the
// call wants of them.  `most`: the largest number of chunks of a table; `total`: of all.
template <class Each>
static int run_norm(tfrec_ctx *ctx, int64_t most, Each &&each, int *n_part)
{
    const int blocks = most < 1 ? 1 : (most < GRAD_BLOCKS ? (int)most : GRAD_BLOCKS);
    double *part = (double *)ctx->d_small;
    int first = 1;
    TF_TRY(each([&](const auto &t) -> int {
        grad_squares_kernel<<<blocks, 256, 0, ctx->stream>>>(t, part, first);
        TF_HIP(hipGetLastError());
        first = 0;
        return TFREC_OK;
    }));
    if (first) {                                   // nothing but empty tensors
        grad_squares_kernel<<<blocks, 256, 0, ctx->stream>>>(GradListed{nullptr, 0}, part, 1);
        TF_HIP(hipGetLastError());
    }
    *n_part = blocks;
    return TFREC_OK;
}

template <class Each>
static int run_clip(tfrec_ctx *ctx, int64_t most, int tables, Each &&each, double max_norm, float *d_norm)
{
    if (tables == 1 && most <= GRAD_SMALL)
        return each([&](const auto &t) -> int {
            grad_clip_small_kernel<<<1, 1024, 0, ctx->stream>>>(t, max_norm, d_norm);
            TF_HIP(hipGetLastError());
            return TFREC_OK;
        });
    int n_part = 0;
    TF_TRY(run_norm(ctx, most, each, &n_part));
    const double *part = (const double *)ctx->d_small;
    bool any = false;
    TF_TRY(each([&](const auto &t) -> int {
        const int blocks = t.chunks < 2048 ? (int)t.chunks : 2048;
        grad_scale_kernel<<<blocks, 256, 0, ctx->stream>>>(t, part, n_part, max_norm, any ? nullptr : d_norm);
        TF_HIP(hipGetLastError());
        any = true;
        return TFREC_OK;
    }));
    if (!any && d_norm) {
        grad_norm_kernel<<<1, 256, 0, ctx->stream>>>(part, n_part, d_norm);
        TF_HIP(hipGetLastError());
    }
    return TFREC_OK;
}

static int finish_norm(tfrec_ctx *ctx, int n_part, float *d_norm)
{
    grad_norm_kernel<<<1, 256, 0, ctx->stream>>>((const double *)ctx->d_small, n_part, d_norm);
    TF_HIP(hipGetLastError());
    return TFREC_OK;
}

static int check_bound(double max_norm, const float *d_norm)
{
    TF_REQUIRE(max_norm > 0. && max_norm < (double)INFINITY, TFREC_EINVAL, "max_norm must be positive and finite, got %g", max_norm);
    TF_REQUIRE(((uintptr_t)d_norm & 3u) == 0, TFREC_EINVAL, "misaligned output");
    return TFREC_OK;
}

extern "C" int tfrec_grad_norm(tfrec_ctx *ctx, int n, const void *const *h_grads, const int64_t *h_counts, const int *h_dtypes, float *d_norm)
{
    TF_TRY(check_grads(n, h_grads, h_counts, h_dtypes));
    TF_REQUIRE(d_norm && ((uintptr_t)d_norm & 3u) == 0, TFREC_EINVAL, "null or misaligned output");
    TF_TRY(tfrec_ctx_enter(ctx));
    auto each = [&](auto &&f) -> int { return for_tables(n, h_grads, nullptr, h_counts, h_dtypes, f); };
    int64_t most = 0;
    TF_TRY(each([&](const GradTable &t) -> int { most = t.chunks > most ? t.chunks : most; return TFREC_OK; }));
    int n_part = 0;
    TF_TRY(run_norm(ctx, most, each, &n_part));
    return finish_norm(ctx, n_part, d_norm);
}

extern "C" int tfrec_grad_clip(tfrec_ctx *ctx, int n, const void *const *h_grads, void *const *h_out, const int64_t *h_counts,
                               const int *h_dtypes, double max_norm, float *d_norm)
{
    TF_TRY(check_grads(n, h_grads, h_counts, h_dtypes));
    TF_TRY(check_bound(max_norm, d_norm));
    TF_TRY(check_outputs(n, h_grads, h_out, h_counts, h_dtypes));
    TF_TRY(check_norm_apart(n, h_grads, h_out, h_counts, h_dtypes, d_norm));
    TF_TRY(tfrec_ctx_enter(ctx));
    auto each = [&](auto &&f) -> int { return for_tables(n, h_grads, h_out, h_counts, h_dtypes, f); };
    int64_t most = 0;
    int tables = 0;
    TF_TRY(each([&](const GradTable &t) -> int { most = t.chunks > most ? t.chunks : most; ++tables; return TFREC_OK; }));
    return run_clip(ctx, most, tables, each, max_norm, d_norm);
}

// ------------------------------------------------------------------------------------------
// kept lists
// ------------------------------------------------------------------------------------------
struct Span { uintptr_t lo, hi; };

struct tfrec_grads {
    GradChunk *d_chunks = nullptr;
    int64_t chunks = 0;
    int device = 0;
    Span *spans = nullptr;                     // the memory of all gradients and outputs: disjoint, by address
    size_t n_spans = 0;
};

static void free_grads(tfrec_grads *g)
{
    if (g->d_chunks) (void)hipFree(g->d_chunks);
    delete[] g->spans;
    delete g;
}

extern "C" int tfrec_grads_create(tfrec_ctx *ctx, int n, const void *const *h_grads, void *const *h_out, const int64_t *h_counts,
                                  const int *h_dtypes, tfrec_grads **out)
{
    TF_REQUIRE(out != nullptr, TFREC_EINVAL, "out is null");
    *out = nullptr;
    TF_TRY(check_grads(n, h_grads, h_counts, h_dtypes));
    TF_TRY(check_outputs(n, h_grads, h_out, h_counts, h_dtypes));
    TF_TRY(tfrec_ctx_enter(ctx));
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    TF_HIP(hipStreamIsCapturing(ctx->stream, &cap));
    TF_REQUIRE(cap == hipStreamCaptureStatusNone, TFREC_EINVAL, "a list cannot be made while the stream is captured");
    int64_t chunks = 0;
    for (int i = 0; i < n; ++i) chunks += (h_counts[i] + GRAD_CHUNK - 1) / GRAD_CHUNK;
    tfrec_grads *g = new (std::nothrow) tfrec_grads();
    GradChunk *h = new (std::nothrow) GradChunk[(size_t)chunks + 1];
    if (g) g->spans = new (std::nothrow) Span[2 * (size_t)n + 1];
    if (!g || !h || !g->spans) {
        if (g) free_grads(g);
        delete[] h;
        tfrec_set_error("host allocation failed");
        return TFREC_ENOMEM;
    }
    int64_t c = 0;
    size_t m = 0;
    for (int i = 0; i < n; ++i) {
        const size_t es = dt_size(h_dtypes[i]);
        for (int64_t at = 0; at < h_counts[i]; at += GRAD_CHUNK) {
            const int64_t left = h_counts[i] - at;
            h[c++] = GradChunk{(const char *)h_grads[i] + at * es, (char *)h_out[i] + at * es, (int32_t)(left < GRAD_CHUNK ? left : GRAD_CHUNK), h_dtypes[i], 0};
        }
        if (!h_counts[i]) continue;
        g->spans[m++] = {(uintptr_t)h_grads[i], (uintptr_t)h_grads[i] + (size_t)h_counts[i] * es};
        if (h_out[i] != h_grads[i]) g->spans[m++] = {(uintptr_t)h_out[i], (uintptr_t)h_out[i] + (size_t)h_counts[i] * es};
    }
    sort_ranges(g->spans, m);
    for (size_t i = 0; i < m; ++i) {           // (gradients may overlap each other)
        if (g->n_spans && g->spans[i].lo <= g->spans[g->n_spans - 1].hi) {
            Span &last = g->spans[g->n_spans - 1];
            last.hi = g->spans[i].hi > last.hi ? g->spans[i].hi : last.hi;
        } else g->spans[g->n_spans++] = g->spans[i];
    }
    g->chunks = chunks;
    g->device = ctx->device;
    hipError_t e = hipMalloc((void **)&g->d_chunks, sizeof(GradChunk) * (size_t)(chunks > 0 ? chunks : 1));
    if (e != hipSuccess) g->d_chunks = nullptr;
    if (e == hipSuccess && chunks) e = hipMemcpyAsync(g->d_chunks, h, sizeof(GradChunk) * (size_t)chunks, hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    delete[] h;
    if (e != hipSuccess) {
        const int code = g->d_chunks ? TFREC_EHIP : TFREC_ENOMEM;
        free_grads(g);
        tfrec_set_error("the list of %lld chunks could not be stored: %s", (long long)chunks, hipGetErrorString(e));
        return code;
    }
    *out = g;
    return TFREC_OK;
}

extern "C" int tfrec_grads_destroy(tfrec_ctx *ctx, tfrec_grads *g)
{
    if (!g) return TFREC_OK;
    (void)hipSetDevice(g->device);
    if (ctx) (void)hipStreamSynchronize(ctx->stream);
    else (void)hipDeviceSynchronize();
    free_grads(g);
    return TFREC_OK;
}

// check_norm_apart for a kept list
static int check_norm_outside(const tfrec_grads *g, const float *d_norm)
{
    const uintptr_t lo = (uintptr_t)d_norm;
    size_t a = 0, b = g->n_spans;              // first span that ends behind the norm's first byte
    while (a < b) {
        const size_t mid = (a + b) / 2;
        if (g->spans[mid].hi <= lo) a = mid + 1; else b = mid;
    }
    TF_REQUIRE(!d_norm || a == g->n_spans || g->spans[a].lo >= lo + sizeof(float), TFREC_EINVAL, "the norm lies within a tensor of the list");
    return TFREC_OK;
}

static int check_list(tfrec_ctx *ctx, const tfrec_grads *g)
{
    TF_REQUIRE(g->device == ctx->device, TFREC_EINVAL, "the list was made on device %d, the context is on device %d", g->device, ctx->device);
    return TFREC_OK;
}

extern "C" int tfrec_grads_norm(tfrec_ctx *ctx, const tfrec_grads *g, float *d_norm)
{
    TF_REQUIRE(g != nullptr, TFREC_EINVAL, "null list");
    TF_REQUIRE(d_norm && ((uintptr_t)d_norm & 3u) == 0, TFREC_EINVAL, "null or misaligned output");
    TF_TRY(tfrec_ctx_enter(ctx));
    TF_TRY(check_list(ctx, g));
    int n_part = 0;
    TF_TRY(run_norm(ctx, g->chunks, [&](auto &&f) -> int { return f(GradListed{g->d_chunks, g->chunks}); }, &n_part));
    return finish_norm(ctx, n_part, d_norm);
}

extern "C" int tfrec_grads_clip(tfrec_ctx *ctx, const tfrec_grads *g, double max_norm, float *d_norm)
{
    TF_REQUIRE(g != nullptr, TFREC_EINVAL, "null list");
    TF_TRY(check_bound(max_norm, d_norm));
    TF_TRY(tfrec_ctx_enter(ctx));
    TF_TRY(check_list(ctx, g));
    TF_TRY(check_norm_outside(g, d_norm));
    if (g->chunks == 0 && !d_norm) return TFREC_OK;
    return run_clip(ctx, g->chunks, 1, [&](auto &&f) -> int { return f(GradListed{g->d_chunks, g->chunks}); }, max_norm, d_norm);
}
