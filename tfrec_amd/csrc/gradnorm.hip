// Global l2 norm over many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over all values of g^2),   out = g * max_norm / max(norm, max_norm)
//
// Bound by memory: every value is read once for the norm and, where it is scaled, once more and written.  The tensors are
// cut into chunks of CHUNK values; workgroups take chunks in a fixed pattern and leave one float64 partial sum each, which
// are added in a fixed order, so results do not depend on scheduling.  Squares are formed and summed in float64: no
// float32 value's square leaves its range, and the sum of 10^9 values keeps more bits than the result has.
#include "common.hpp"

static constexpr int GRAD_TENSORS = 96;        // tensors per launch: their table rides in the kernel's arguments (below 4 KB)
static constexpr int GRAD_CHUNK = 8192;        // values per chunk
static constexpr int GRAD_BLOCKS = 1024;       // partial sums (and workgroups at most)
static_assert(GRAD_BLOCKS * sizeof(double) <= TFREC_SMALL_BYTES, "partial sums exceed the context's scratch");

struct GradTable {
    const void *src[GRAD_TENSORS];
    void *dst[GRAD_TENSORS];
    int64_t count[GRAD_TENSORS];
    int64_t first[GRAD_TENSORS];               // first chunk of the tensor; ascending
    uint8_t dtype[GRAD_TENSORS];
    int n;
    int64_t chunks;
};

// 16 bytes at the alignment of the element type (global memory takes them at any)
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[16 / sizeof(T)]; };

// tensor of chunk c (wave-uniform)
__device__ __forceinline__ int tensor_of(const GradTable &t, int64_t c)
{
    int lo = 0, hi = t.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
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

template <class T>
__device__ __forceinline__ void chunk_scale(const T *x, T *y, int m, float s, float p2)
{
    constexpr int V = 16 / sizeof(T), R = GRAD_CHUNK / (256 * V);
    if (m == GRAD_CHUNK) {
        Pack<T> p[R];
#pragma unroll
        for (int r = 0; r < R; ++r) p[r] = reinterpret_cast<const Pack<T> *>(x)[r * 256 + threadIdx.x];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < V; ++j) p[r].v[j] = (T)((float)p[r].v[j] * s * p2);
            reinterpret_cast<Pack<T> *>(y)[r * 256 + threadIdx.x] = p[r];
        }
    } else {
        for (int i = threadIdx.x; i < m; i += 256) y[i] = (T)((float)x[i] * s * p2);
    }
}

// sum over the 256 threads, the same on every thread, in a fixed order
__device__ __forceinline__ double block_sum(double v)
{
    __shared__ double red[4];
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return v;
}

// partial sum of workgroup b over its chunks b, b + grid, ...; `first`: the first launch of a call, which sets the partials
__global__ __launch_bounds__(256) void grad_squares_kernel(GradTable t, double *__restrict__ part, int first)
{
    double s = 0.;
    for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const int64_t at = (c - t.first[i]) * GRAD_CHUNK, left = t.count[i] - at;
        const int m = left < GRAD_CHUNK ? (int)left : GRAD_CHUNK;
        if (t.dtype[i] == TFREC_DT_F32) s = chunk_squares((const float *)t.src[i] + at, m, s);
        else if (t.dtype[i] == TFREC_DT_BF16) s = chunk_squares((const __bf16 *)t.src[i] + at, m, s);
        else s = chunk_squares((const _Float16 *)t.src[i] + at, m, s);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = first ? s : part[blockIdx.x] + s;
}

// the norm from the partial sums, on every thread; every workgroup that wants it forms it the same way
__device__ __forceinline__ double norm_of(const double *__restrict__ part, int n_part)
{
    double s = 0.;
    for (int i = threadIdx.x; i < n_part; i += 256) s += part[i];
    return sqrt(block_sum(s));
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double *__restrict__ part, int n_part, float *__restrict__ norm)
{
    const double nm = norm_of(part, n_part);
    if (threadIdx.x == 0) *norm = (float)nm;
}

__global__ __launch_bounds__(256) void grad_scale_kernel(GradTable t, const double *__restrict__ part, int n_part, double max_norm, float *__restrict__ norm)
{
    const double nm = norm_of(part, n_part);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nm;
    // (a sum of squares of finite float32 values stays finite in float64: not finite = an infinity or NaN among the values)
    // A scale near or below the subnormal range of float32 (gradients of 1e35 and more) is applied as s 2^64 and then 2^-64.
    const double sd = nm <= max_norm ? 1. : max_norm / nm;
    const bool tiny = sd < 0x1p-100;
    const float s = !(nm < (double)INFINITY) ? NAN : (float)(tiny ? sd * 0x1p64 : sd), p2 = tiny ? 0x1p-64f : 1.f;
    // the last chunks first: what the norm read last is still cached
    for (int64_t k = blockIdx.x; k < t.chunks; k += gridDim.x) {
        const int64_t c = t.chunks - 1 - k;
        const int i = tensor_of(t, c);
        if (s == 1.f && t.src[i] == t.dst[i]) continue;        // in place and within the bound: every value is what it was
        const int64_t at = (c - t.first[i]) * GRAD_CHUNK, left = t.count[i] - at;
        const int m = left < GRAD_CHUNK ? (int)left : GRAD_CHUNK;
        if (t.dtype[i] == TFREC_DT_F32) chunk_scale((const float *)t.src[i] + at, (float *)t.dst[i] + at, m, s, p2);
        else if (t.dtype[i] == TFREC_DT_BF16) chunk_scale((const __bf16 *)t.src[i] + at, (__bf16 *)t.dst[i] + at, m, s, p2);
        else chunk_scale((const _Float16 *)t.src[i] + at, (_Float16 *)t.dst[i] + at, m, s, p2);
    }
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

struct Range { uintptr_t lo, hi; int out; };       // out: index of the output, or -1 for a gradient

// No output overlaps another output, or a gradient other than the one it replaces.
static int check_outputs(int n, const void *const *g, void *const *out, const int64_t *counts, const int *dtypes)
{
    TF_REQUIRE(n == 0 || out, TFREC_EINVAL, "null host array");
    Range *r = new (std::nothrow) Range[2 * (size_t)n + 1];
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
            for (size_t gap = m / 2; gap > 0; gap /= 2)            // (no library sort: nothing here may throw)
                for (size_t i = gap; i < m; ++i) {
                    const Range x = r[i];
                    size_t j = i;
                    for (; j >= gap && r[j - gap].lo > x.lo; j -= gap) r[j] = r[j - gap];
                    r[j] = x;
                }
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

// leaves the partial sums in the context's scratch; *n_part = how many
static int grad_squares(tfrec_ctx *ctx, int n, const void *const *g, const int64_t *counts, const int *dtypes, int *n_part)
{
    int64_t most = 1;
    TF_TRY(for_tables(n, g, nullptr, counts, dtypes, [&](const GradTable &t) -> int { most = t.chunks > most ? t.chunks : most; return TFREC_OK; }));
    const int blocks = most < GRAD_BLOCKS ? (int)most : GRAD_BLOCKS;
    double *part = (double *)ctx->d_small;
    int first = 1;
    TF_TRY(for_tables(n, g, nullptr, counts, dtypes, [&](const GradTable &t) -> int {
        grad_squares_kernel<<<blocks, 256, 0, ctx->stream>>>(t, part, first);
        TF_HIP(hipGetLastError());
        first = 0;
        return TFREC_OK;
    }));
    if (first) {                                   // nothing but empty tensors
        GradTable t;
        t.n = 0;
        t.chunks = 0;
        grad_squares_kernel<<<blocks, 256, 0, ctx->stream>>>(t, part, 1);
        TF_HIP(hipGetLastError());
    }
    *n_part = blocks;
    return TFREC_OK;
}

extern "C" int tfrec_grad_norm(tfrec_ctx *ctx, int n, const void *const *h_grads, const int64_t *h_counts, const int *h_dtypes, float *d_norm)
{
    TF_TRY(check_grads(n, h_grads, h_counts, h_dtypes));
    TF_REQUIRE(d_norm && ((uintptr_t)d_norm & 3u) == 0, TFREC_EINVAL, "null or misaligned output");
    TF_TRY(tfrec_ctx_enter(ctx));
    int n_part = 0;
    TF_TRY(grad_squares(ctx, n, h_grads, h_counts, h_dtypes, &n_part));
    grad_norm_kernel<<<1, 256, 0, ctx->stream>>>((const double *)ctx->d_small, n_part, d_norm);
    TF_HIP(hipGetLastError());
    return TFREC_OK;
}

extern "C" int tfrec_grad_clip(tfrec_ctx *ctx, int n, const void *const *h_grads, void *const *h_out, const int64_t *h_counts,
                               const int *h_dtypes, float max_norm, float *d_norm)
{
    TF_TRY(check_grads(n, h_grads, h_counts, h_dtypes));
    TF_REQUIRE(max_norm > 0.f && max_norm < INFINITY, TFREC_EINVAL, "max_norm must be positive and finite, got %g", (double)max_norm);
    TF_REQUIRE(((uintptr_t)d_norm & 3u) == 0, TFREC_EINVAL, "misaligned output");
    TF_TRY(check_outputs(n, h_grads, h_out, h_counts, h_dtypes));
    TF_TRY(tfrec_ctx_enter(ctx));
    int n_part = 0;
    TF_TRY(grad_squares(ctx, n, h_grads, h_counts, h_dtypes, &n_part));
    const double *part = (const double *)ctx->d_small;
    bool any = false;
    TF_TRY(for_tables(n, h_grads, h_out, h_counts, h_dtypes, [&](const GradTable &t) -> int {
        const int blocks = t.chunks < 2 * GRAD_BLOCKS ? (int)t.chunks : 2 * GRAD_BLOCKS;
        grad_scale_kernel<<<blocks, 256, 0, ctx->stream>>>(t, part, n_part, (double)max_norm, any ? nullptr : d_norm);
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
