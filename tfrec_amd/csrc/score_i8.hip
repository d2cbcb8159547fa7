// Top-k of the scores of 8-bit factor rows against an 8-bit item table (tfrec_quantize_rows_i8).
//
//   score[u][i] = ((float)(sum_f Pq[u][f] Qq[i][f]) * sp[u]) * sq[i] + b[i]       (each step rounded to float32)
//
// The order is (score descending, item id ascending), train items are left out, and the [users, items] matrix is never
// formed.  A NaN score (a NaN scale) passes no comparison and so enters no list.
#include "i8_device.hpp"
#include "score_i8.hpp"

#include "topk_list.hpp"

// row of the user table that listed user r reads, and the user's id (the row of the train CSR)
__device__ __forceinline__ int64_t user_row(const ScoreI8Args &a, int64_t r, int32_t *id)
{
    const int32_t u = a.users[r];
    *id = u;
    if (a.p_compact) return r;
    const int64_t c = u < 0 ? 0 : (u >= a.U ? a.U - 1 : u);
    if (c != u) atomicOr(a.flags, TFREC_FLAG_BAD_INDEX);
    *id = (int32_t)c;
    return c;
}

// One wave per user and range of items, a lane per item: 64 rows of the item table at a time, four products per
// instruction (v_dot4_i32_i8).  Scores above the running threshold go to a list in LDS that is cut back to the k best
// when it is full.
template <int CAP>
__global__ __launch_bounds__(256) void score_rows_i8_kernel(ScoreI8Args a)
{
    __shared__ uint64_t lists[4][CAP], sortbuf[4][CAP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * 4 + wave;
    if (r >= a.n) return;
    int32_t user;
    const int64_t prow = user_row(a, r, &user);
    const int8_t *p = a.Pq + prow * a.ldp;
    const float sp = a.sp[prow];
    const int64_t mlo = a.train_indptr ? a.train_indptr[user] : 0, mhi = a.train_indptr ? a.train_indptr[user + 1] : 0;
    const int64_t it0 = (int64_t)blockIdx.y * a.split_items, it1 = it0 + a.split_items < a.n_items ? it0 + a.split_items : a.n_items;
    const int chunks = (a.d + 15) / 16;
    const int32_t id0 = (int32_t)(a.id_offset + a.item_lo);
    uint64_t *list = lists[wave];
    int cnt = 0, ver = 0;
    float tau = -INFINITY;
    for (int64_t base = it0; base < it1; base += 64) {
        if (cnt > CAP - 64) {
            cnt = wave_compact<CAP>(list, cnt, ver, a.k, a.train_indices, mlo, mhi, sortbuf[wave], lane, &tau);
            ver = cnt;
        }
        const int64_t it = base + lane;
        float v = -INFINITY;
        if (it < it1) {
            const uint4 *q = reinterpret_cast<const uint4 *>(a.Qq + (a.item_lo + it) * a.ldq);
            int acc = 0;
            for (int c = 0; c < chunks; ++c) {
                const uint4 qv = q[c];
                const uint4 pv = keep_below(reinterpret_cast<const uint4 *>(p)[c], 16 * c, a.d);
                acc = __builtin_amdgcn_sdot4((int)qv.x, (int)pv.x, acc, false);
                acc = __builtin_amdgcn_sdot4((int)qv.y, (int)pv.y, acc, false);
                acc = __builtin_amdgcn_sdot4((int)qv.z, (int)pv.z, acc, false);
                acc = __builtin_amdgcn_sdot4((int)qv.w, (int)pv.w, acc, false);
            }
            v = add_rounded(scaled_sum(acc, sp, a.sq[a.item_lo + it]), a.b ? a.b[a.item_lo + it] : 0.f);
        }
        const bool pass = v > tau;
        const uint64_t m = __ballot(pass);
        if (pass) list[cnt + __popcll(m & ((1ull << lane) - 1))] = make_key(v, id0 + (int32_t)it);
        cnt += __popcll(m);
    }
    cnt = wave_compact<CAP>(list, cnt, ver, a.k, a.train_indices, mlo, mhi, sortbuf[wave], lane, &tau);
    int32_t *oi = a.out_ids + ((size_t)blockIdx.y * a.n + r) * a.k;
    float *os = a.out_scores + ((size_t)blockIdx.y * a.n + r) * a.k;
    for (int e = lane; e < a.k; e += 64) {
        const uint64_t key = e < cnt ? sortbuf[wave][e] : 0;
        oi[e] = e < cnt ? key_id(key) : -1;
        os[e] = e < cnt ? key_score(key) : -INFINITY;
    }
}

__global__ __launch_bounds__(256) void no_entries_kernel(int32_t *__restrict__ ids, float *__restrict__ scores, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) { ids[i] = -1; scores[i] = -INFINITY; }
}

struct ScoreI8Plan { int cap, splits; int64_t split_items; size_t part_bytes, total; };

static ScoreI8Plan plan_i8(int64_t n, int64_t n_items, int k)
{
    ScoreI8Plan p;
    p.cap = k <= 112 ? 256 : 512;
    // fewer than 2048 waves: the items are split too, as far as one merge of the partial lists goes
    int64_t s = n < 2048 ? 2048 / n : 1;
    const int64_t most = (n_items + 1023) / 1024;
    s = s < most ? s : most;
    s = s < 2048 / k ? s : 2048 / k;
    s = s < 1 ? 1 : s;
    p.split_items = ((n_items + s - 1) / s + 63) / 64 * 64;
    p.splits = (int)((n_items + p.split_items - 1) / p.split_items);
    p.part_bytes = p.splits > 1 ? tf_align((size_t)p.splits * n * k * 4) : 0;
    p.total = 2 * p.part_bytes + 1024;
    return p;
}

size_t tfrec_score_i8_bytes(int64_t n, int64_t n_items, int k) { return n > 0 && n_items > 0 ? plan_i8(n, n_items, k).total : 0; }

size_t tfrec_score_i8_bytes_most(int64_t n, int k)
{
    if (n <= 0 || k < 1 || k > 240) return 0;
    return plan_i8(n, (int64_t)1 << 30, k).total;
}

int tfrec_score_i8(tfrec_ctx *ctx, ScoreI8Args a)
{
    if (a.n == 0) return TFREC_OK;
    if (a.n_items == 0) {
        no_entries_kernel<<<(unsigned)((a.n * a.k + 255) / 256), 256, 0, ctx->stream>>>(a.out_ids, a.out_scores, a.n * a.k);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    }
    const ScoreI8Plan p = plan_i8(a.n, a.n_items, a.k);
    TF_TRY(tfrec_ws_require(ctx, ctx->ws_used + p.total));
    TF_TRY(tfrec_note_capture(ctx));
    a.flags = ctx->d_flags;
    a.split_items = p.split_items;
    int32_t *const ids = a.out_ids;
    float *const scores = a.out_scores;
    if (p.splits > 1) {
        a.out_ids = (int32_t *)tfrec_ws_take(ctx, p.part_bytes);
        a.out_scores = (float *)tfrec_ws_take(ctx, p.part_bytes);
        TF_REQUIRE(a.out_ids && a.out_scores, TFREC_ENOMEM, "internal: workspace carve failed");
    }
    const dim3 grid((unsigned)((a.n + 3) / 4), p.splits);
    if (p.cap == 256) score_rows_i8_kernel<256><<<grid, 256, 0, ctx->stream>>>(a);
    else score_rows_i8_kernel<512><<<grid, 256, 0, ctx->stream>>>(a);
    TF_HIP(hipGetLastError());
    if (p.splits > 1) TF_TRY(tfrec_merge_lists(ctx, a.out_ids, a.out_scores, p.splits, a.n, a.k, ids, scores));
    return TFREC_OK;
}

extern "C" int tfrec_score_topk_i8(tfrec_ctx *ctx, const int8_t *d_Pq, int64_t ldp, const float *d_sp, int64_t U, int p_compact, const int8_t *d_Qq,
                                   int64_t ldq, const float *d_sq, const float *d_b, int64_t I, int d, int64_t item_lo, int64_t item_hi,
                                   const int32_t *d_eval_users, int64_t n, const int64_t *d_train_indptr, const int32_t *d_train_indices, int k,
                                   int32_t *d_out_ids, float *d_out_scores)
{
    TF_REQUIRE(n >= 0 && k >= 1 && d >= 1, TFREC_EINVAL, "bad shape n=%lld k=%d d=%d", (long long)n, k, d);
    TF_REQUIRE(k <= 240, TFREC_EUNSUP, "top-k above 240 is not supported (k=%d)", k);
    TF_REQUIRE(d <= 256, TFREC_EUNSUP, "factor size d=%d is not supported (max 256)", d);
    TF_REQUIRE(0 <= item_lo && item_lo <= item_hi && item_hi <= I, TFREC_EINVAL, "bad item range [%lld,%lld) of %lld", (long long)item_lo,
               (long long)item_hi, (long long)I);
    TF_REQUIRE(I < (1ll << 31) && U < (1ll << 31) && n < (1ll << 31), TFREC_EUNSUP, "user and item ids must fit in int32");
    TF_REQUIRE(p_compact == 0 || p_compact == 1, TFREC_EINVAL, "p_compact must be 0 or 1");
    TF_REQUIRE(n == 0 || (p_compact ? U >= n : U >= 1), TFREC_EINVAL, "%lld user rows for %lld users", (long long)U, (long long)n);
    TF_REQUIRE((d_train_indptr == nullptr) == (d_train_indices == nullptr), TFREC_EINVAL, "train CSR needs both arrays");
    TF_TRY(tfrec_check_i8("P", d_Pq, U, ldp, d));
    TF_TRY(tfrec_check_i8("Q", d_Qq, I, ldq, d));
    TF_REQUIRE(n == 0 || (d_sp && d_eval_users && d_out_ids && d_out_scores), TFREC_EINVAL, "null pointer");
    TF_REQUIRE(item_lo == item_hi || d_sq, TFREC_EINVAL, "null pointer");
    TF_TRY(tfrec_ctx_enter(ctx));
    ScoreI8Args a{};
    a.Pq = d_Pq; a.ldp = ldp; a.sp = d_sp; a.U = U; a.p_compact = p_compact;
    a.Qq = d_Qq; a.ldq = ldq; a.sq = d_sq; a.b = d_b;
    a.d = d; a.item_lo = item_lo; a.n_items = item_hi - item_lo;
    a.users = d_eval_users; a.n = n; a.train_indptr = d_train_indptr; a.train_indices = d_train_indices; a.k = k;
    a.out_ids = d_out_ids; a.out_scores = d_out_scores;
    return tfrec_score_i8(ctx, a);
}
