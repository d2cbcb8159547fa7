// What the 8-bit kernels share: the layout of 8-bit rows, and the host side of the 8-bit top-k.
#pragma once
#include "common.hpp"

#include <atomic>

struct ScoreI8Args {
    const int8_t *Pq;          // user rows: the table [U, ldp], or the listed users' rows in order (p_compact)
    int64_t ldp;
    const float *sp;
    int64_t U;
    int p_compact;
    const int8_t *Qq;          // item rows [.., ldq]; rows item_lo .. item_lo + n_items are scored
    int64_t ldq;
    const float *sq, *b;       // scales and biases by row of Qq; b may be null
    int d;
    int64_t item_lo, n_items;
    int64_t id_offset;         // added to the row of Qq to form the reported id
    const int32_t *users;      // [n]
    int64_t n;
    const int64_t *train_indptr;
    const int32_t *train_indices;
    int k;
    int32_t *out_ids;          // [n, k]
    float *out_scores;
    uint32_t *flags;
};

// A launch has to stay below 2^32 threads.  What has a workgroup per row, user or 16 columns is launched in pieces of this many.
static constexpr int64_t TF_LAUNCH_ROWS = 1ll << 22;
static inline int check_launch(int64_t blocks, int threads)
{
    TF_REQUIRE(blocks * threads < (1ll << 32), TFREC_EUNSUP, "%lld workgroups of %d threads are too many for one launch", (long long)blocks, threads);
    return TFREC_OK;
}

// raises a kernel's dynamic-LDS limit once per device (eval.hip)
int tfrec_raise_lds_limit(tfrec_ctx *ctx, const void *kernel, int bytes, std::atomic<uint64_t> &done);
// the layout every 8-bit matrix has to have (quant.hip)
int tfrec_check_i8(const char *name, const int8_t *q, int64_t rows, int64_t ld, int64_t cols);
// tfrec_quantize_rows_i8 without the checks (quant.hip)
int tfrec_quantize_rows(tfrec_ctx *ctx, const void *d_X, int x_dtype, int64_t n_rows, int64_t ldx, int64_t d, const int32_t *d_rows, int64_t n,
                        int8_t *d_q, int64_t ldq, float *d_scale);
// Scores and ranks; scratch from the workspace above what is in use (score_i8.hip).
int tfrec_score_i8(tfrec_ctx *ctx, ScoreI8Args a);
size_t tfrec_score_i8_bytes(int64_t n, int64_t n_items);        // its scratch
