// Top-k of the scores of 8-bit factor rows against an 8-bit item table (tfrec_quantize_rows_i8).
//
//   score[u][i] = ((float)(sum_f Pq[u][f] Qq[i][f]) * sp[u]) * sq[i] + b[i]       (each step rounded to float32)
//
// The order is (score descending, item id ascending), train items are left out, and the [users, items] matrix is never
// formed.  A NaN score (a NaN scale or bias) passes no comparison and so is never listed; neither is a score of -inf.
//
// Up to SMALL_ITEMS items, one workgroup scores them all for its user and keeps the scores in registers
// (score_small_i8_kernel).  Beyond that:
//   1. score_max_i8_kernel: all scores on the matrix cores; of every 32 items (a block) only the best score of every user
//      is kept: the table is read once however few the users are, and 1/32 of the scores is written.
//   2. pick_i8_kernel, a workgroup per user: the k-th largest of the best scores of disjoint groups of blocks that hold no
//      train item is a lower bound T of the user's k-th best score (k different rankable items reach it).  Only blocks whose
//      best score reaches T can hold a listed item: k blocks and few more, which are scored again, item by item.
// Neither depends on the order of the items, and nothing is kept between calls.
#include "i8_device.hpp"
#include "score_i8.hpp"
#include "topk_list.hpp"

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
struct __attribute__((packed, aligned(4))) Float4 { float v[4]; };       // 16 bytes at the alignment of a float

static constexpr int BLOCK = 32;               // items per block
static constexpr int SMALL_ITEMS = 4096;       // (16 scores per thread of score_small_i8_kernel)
static constexpr uint32_t KEY_NONE = 0x007fffffu;      // orderable form of -inf: nothing below or at it is listed

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

// score of item `it` (row item_lo + it of the table) for the user row p; the row's bytes from column d on are left out
__device__ __forceinline__ float score_item(const ScoreI8Args &a, const int8_t *__restrict__ p, float sp, int64_t it)
{
    const uint4 *__restrict__ q = reinterpret_cast<const uint4 *>(a.Qq + (a.item_lo + it) * a.ldq);
    const int chunks = (a.d + 15) / 16;
    int acc = 0;
    for (int c = 0; c < chunks; ++c) {
        const uint4 qv = q[c], pv = keep_below(reinterpret_cast<const uint4 *>(p)[c], 16 * c, a.d);
        acc = __builtin_amdgcn_sdot4((int)qv.x, (int)pv.x, acc, false);
        acc = __builtin_amdgcn_sdot4((int)qv.y, (int)pv.y, acc, false);
        acc = __builtin_amdgcn_sdot4((int)qv.z, (int)pv.z, acc, false);
        acc = __builtin_amdgcn_sdot4((int)qv.w, (int)pv.w, acc, false);
    }
    return add_rounded(scaled_sum(acc, sp, a.sq[a.item_lo + it]), a.b ? a.b[a.item_lo + it] : 0.f);
}

// ------------------------------------------------------------------------------------------
// step 1: the best score of every block of 32 items, for every user
// ------------------------------------------------------------------------------------------
struct MaxArgs {
    ScoreI8Args s;
    float *best;               // [n, pitch]; blocks beyond the last hold -inf
    int64_t pitch;             // blocks per user row, a multiple of 8
    int64_t groups;            // groups of 8 blocks
    int64_t groups_per_split;
    int user_groups, splits;
};

// KS = steps of 32 columns, UW = sets of 32 users a wave holds (as the matrix instruction's B operand, resident; the items
// are its A operand and come straight from memory, a block ahead).  A lane gets 16 scores of one user per block.
template <int KS, int UW>
__global__ __launch_bounds__(256) void score_max_i8_kernel(MaxArgs m)
{
    __shared__ __align__(16) float out[4][UW][32][8];
    const ScoreI8Args &a = m.s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    // consecutive workgroups go to the 8 XCDs in turn: an XCD takes every 8th slice of the items, for all users one after
    // the other, so that its L2 holds the slice
    const int wgs = (m.user_groups + 3) / 4;
    const int64_t idx = blockIdx.x >> 3;
    const int split = (int)(idx / wgs) * 8 + (blockIdx.x & 7);
    const int ug = (int)(idx % wgs) * 4 + wave;
    if (split >= m.splits || ug >= m.user_groups) return;
    const int64_t g0 = split * m.groups_per_split, g1 = g0 + m.groups_per_split < m.groups ? g0 + m.groups_per_split : m.groups;

    i32x4 pb[UW][KS];
    float sp[UW];
#pragma unroll
    for (int s = 0; s < UW; ++s) {
        const int64_t ur = (int64_t)ug * 32 * UW + 32 * s + r;
        int32_t id;
        const int64_t row = user_row(a, ur < a.n ? ur : a.n - 1, &id);
        sp[s] = a.sp[row];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = 32 * ks + 16 * h;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (c < a.d) v = keep_below(*reinterpret_cast<const uint4 *>(a.Pq + row * a.ldp + c), c, a.d);
            pb[s][ks] = __builtin_bit_cast(i32x4, v);
        }
    }
    // columns from d on meet zeros of the user rows: any bytes of the row will do there
    int off[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = 32 * ks + 16 * h;
        off[ks] = c < (int)a.ldq ? c : (int)a.ldq - 16;
    }
    const int8_t *__restrict__ Q = a.Qq + a.item_lo * a.ldq;
    const float *__restrict__ sq = a.sq + a.item_lo, *__restrict__ bias = a.b ? a.b + a.item_lo : nullptr;
    struct Block { i32x4 q[KS]; Float4 sq[4], b[4]; };
    auto load = [&](Block &o, int64_t blk) {
        const int64_t it = blk * BLOCK;
        const int64_t row = it + r < a.n_items ? it + r : a.n_items - 1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) o.q[ks] = *reinterpret_cast<const i32x4 *>(Q + row * a.ldq + off[ks]);
        if (it + BLOCK <= a.n_items) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                o.sq[g] = *reinterpret_cast<const Float4 *>(sq + it + 8 * g + 4 * h);
                if (bias) o.b[g] = *reinterpret_cast<const Float4 *>(bias + it + 8 * g + 4 * h);
                else o.b[g] = Float4{{0.f, 0.f, 0.f, 0.f}};
            }
        } else {
            // the last block, or one past it: items that do not exist score -inf
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t i = it + 8 * g + 4 * h + j;
                    o.sq[g].v[j] = i < a.n_items ? sq[i] : 0.f;
                    o.b[g].v[j] = i < a.n_items ? (bias ? bias[i] : 0.f) : -INFINITY;
                }
        }
    };
    Block cur;
    load(cur, g0 * 8);
    for (int64_t g = g0; g < g1; ++g) {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            Block next;
            load(next, g * 8 + i + 1);
#pragma unroll
            for (int s = 0; s < UW; ++s) {
                i32x16 acc = {};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(cur.q[ks], pb[s][ks], acc, 0, 0, 0);
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, add_rounded(scaled_sum(acc[e], sp[s], cur.sq[e >> 2].v[e & 3]), cur.b[e >> 2].v[e & 3]));
                mx = fmaxf(mx, __uint_as_float(swap32(__float_as_uint(mx), lane)));
                if (h == 0) out[wave][s][r][i] = mx;
            }
            cur = next;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < UW; ++s) {
            const int64_t ur = (int64_t)ug * 32 * UW + 32 * s + r;
            if (ur < a.n) *reinterpret_cast<float4 *>(m.best + ur * m.pitch + g * 8 + 4 * h) = *reinterpret_cast<const float4 *>(&out[wave][s][r][4 * h]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------------
// a workgroup's list of keys (256 threads)
// ------------------------------------------------------------------------------------------
static constexpr int LIST = 1024;
struct GroupList {
    uint64_t list[LIST], sorted[LIST];
    uint64_t kth;              // keys at or below it are not wanted
    int count;
    uint32_t hist[2][64];
    uint32_t lo[4], hi[4];
    int valid[4];
};

// A lower bound of the k-th largest of the workgroup's orderable values (V per thread; values at or below KEY_NONE are
// none): the lower edge of a bucket of a two-level histogram below the highest bit in which the values differ.
// KEY_NONE + 1 if fewer than k values are held.
template <int V>
__device__ __forceinline__ uint32_t rank_bound(const uint32_t (&key)[V], int k, GroupList &g)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t lo = 0xffffffffu, hi = 0;
    int valid = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (key[v] > KEY_NONE) {
            lo = key[v] < lo ? key[v] : lo;
            hi = key[v] > hi ? key[v] : hi;
            valid += 1;
        }
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t l2 = __shfl_xor((int)lo, o, 64), h2 = __shfl_xor((int)hi, o, 64);
        lo = l2 < lo ? l2 : lo;
        hi = h2 > hi ? h2 : hi;
        valid += __shfl_xor(valid, o, 64);
    }
    if (lane == 0) { g.lo[wave] = lo; g.hi[wave] = hi; g.valid[wave] = valid; }
    if (threadIdx.x < 128) g.hist[threadIdx.x >> 6][threadIdx.x & 63] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        lo = g.lo[w] < lo ? g.lo[w] : lo;
        hi = g.hi[w] > hi ? g.hi[w] : hi;
    }
    valid = g.valid[0] + g.valid[1] + g.valid[2] + g.valid[3];
    if (valid < k) return KEY_NONE + 1;
    if (lo == hi) return hi;
    const int top = 31 - __builtin_clz(lo ^ hi);
    const int s1 = top >= 5 ? top - 5 : 0;
    // level 1: six bits from the highest differing one down (all values share the bits above)
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (key[v] > KEY_NONE) atomicAdd(&g.hist[0][(key[v] >> s1) & 63u], 1u);
    __syncthreads();
    auto level = [&](const uint32_t *hist, int want, int *above, int *in) {
        const int c = (int)hist[lane], incl = wave_prefix_sum(c), total = __builtin_amdgcn_readlane(incl, 63);
        const int up = total - incl + c;                  // values in this bucket and higher
        const uint64_t b = __ballot(up >= want);
        const int at = b ? 63 - __builtin_clzll(b) : 0;
        *in = __builtin_amdgcn_readlane(c, at);
        *above = __builtin_amdgcn_readlane(up, at) - *in;
        return (uint32_t)at;
    };
    int above, in;
    const uint32_t b1 = level(g.hist[0], k, &above, &in);
    const int width1 = s1 + 6;
    uint32_t cut = (width1 >= 32 ? 0u : (hi >> width1) << width1) | (b1 << s1);
    if (above + in > k && s1 > 0) {
        const int s2 = s1 >= 6 ? s1 - 6 : 0;
        const uint32_t mask = (1u << (s1 - s2)) - 1u;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (key[v] > KEY_NONE && key[v] >> s1 == cut >> s1) atomicAdd(&g.hist[1][(key[v] >> s2) & mask], 1u);
        __syncthreads();
        int above2, in2;
        cut |= level(g.hist[1], k - above, &above2, &in2) << s2;
    }
    return cut;
}

// a wave's keys that pass go to the list; all lanes call it
__device__ __forceinline__ void group_append(GroupList &g, bool pass, uint64_t key)
{
    const int lane = threadIdx.x & 63;
    const uint64_t m = __ballot(pass);
    if (!m) return;
    int base = 0;
    if (lane == 0) base = atomicAdd(&g.count, __popcll(m));
    base = __builtin_amdgcn_readfirstlane(base);
    if (pass) g.list[base + __popcll(m & ((1ull << lane) - 1))] = key;
}

// called by all threads after a step that appended at most 256 keys: cuts the list back to its k best once the next step might
// not fit
__device__ __forceinline__ void group_check(GroupList &g, int k, const int32_t *midx, int64_t mlo, int64_t mhi)
{
    __syncthreads();
    if (g.count > LIST - 256) {
        if (threadIdx.x < 64) {
            float tau;
            const int kept = wave_compact<LIST>(g.list, g.count, 0, k, midx, mlo, mhi, g.sorted, threadIdx.x, &tau);
            if (threadIdx.x == 0) {
                g.count = kept;
                if (kept >= k) g.kth = g.sorted[k - 1];
            }
        }
    }
    __syncthreads();
}

// the list's k best in order, by the first wave
__device__ __forceinline__ void group_finish(GroupList &g, const ScoreI8Args &a, int64_t r, const int32_t *midx, int64_t mlo, int64_t mhi)
{
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x, cnt = g.count;
    float tau;
    int kept;
    if (cnt <= 256) kept = wave_compact<256>(g.list, cnt, 0, a.k, midx, mlo, mhi, g.sorted, lane, &tau);
    else kept = wave_compact<LIST>(g.list, cnt, 0, a.k, midx, mlo, mhi, g.sorted, lane, &tau);
    for (int e = lane; e < a.k; e += 64) {
        const uint64_t key = e < kept ? g.sorted[e] : 0;
        a.out_ids[r * a.k + e] = e < kept ? key_id(key) : -1;
        a.out_scores[r * a.k + e] = e < kept ? key_score(key) : -INFINITY;
    }
}

// ------------------------------------------------------------------------------------------
// step 2: the blocks that can hold a listed item, scored again
// ------------------------------------------------------------------------------------------
static constexpr int SLICES = 1024;            // groups of blocks: block x belongs to slice x % SLICES
static constexpr int CAND = 2048;              // blocks per round

__global__ __launch_bounds__(256) void pick_i8_kernel(MaxArgs m)
{
    __shared__ GroupList g;
    __shared__ uint32_t cand[CAND];
    __shared__ uint16_t slices[SLICES];
    __shared__ uint8_t train[SLICES];
    __shared__ int n_slices, n_cand;
    const ScoreI8Args &a = m.s;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    int32_t user;
    const int64_t prow = user_row(a, r, &user);
    const int8_t *__restrict__ p = a.Pq + prow * a.ldp;
    const float sp = a.sp[prow];
    const int64_t mlo = a.train_indptr ? a.train_indptr[user] : 0, mhi = a.train_indptr ? a.train_indptr[user + 1] : 0;
    const int64_t id0 = a.id_offset + a.item_lo;
    const int64_t blocks = (a.n_items + BLOCK - 1) / BLOCK;
    const float *__restrict__ best = m.best + r * m.pitch;

    for (int i = tid; i < SLICES; i += 256) train[i] = 0;
    if (tid == 0) { g.count = 0; n_slices = 0; n_cand = 0; }
    __syncthreads();
    for (int64_t t = mlo + tid; t < mhi; t += 256) {
        const int64_t i = a.train_indices[t] - id0;
        if (i >= 0 && i < a.n_items) train[(i / BLOCK) % SLICES] = 1;
    }
    __syncthreads();
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    for (int64_t x0 = 0; x0 < blocks; x0 += SLICES) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int64_t x = x0 + 256 * v + tid;
            if (x < blocks) mx[v] = fmaxf(mx[v], best[x]);
        }
    }
    uint32_t key[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) key[v] = train[256 * v + tid] ? 0u : f32_orderable(mx[v]);
    const uint32_t cut = rank_bound(key, a.k, g);
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (f32_orderable(mx[v]) >= cut) slices[atomicAdd(&n_slices, 1)] = (uint16_t)(256 * v + tid);
    if (tid == 0) g.kth = ((uint64_t)cut << 32) - 1;
    __syncthreads();

    const uint32_t per = (uint32_t)((blocks + SLICES - 1) / SLICES), total = (uint32_t)n_slices * per;      // (at most blocks + SLICES: below 2^27)
    for (uint32_t e0 = 0; e0 < total; e0 += CAND) {
        const uint64_t kth = g.kth;
#pragma unroll
        for (int i = 0; i < CAND / 256; ++i) {
            const uint32_t e = e0 + 256 * i + tid;
            if (e < total) {
                const int64_t x = slices[e / per] + (int64_t)(e % per) * SLICES;
                // the block's best score under its lowest id: if that is not wanted, nothing in the block is
                if (x < blocks && make_key(best[x], (int32_t)(id0 + x * BLOCK)) > kth) cand[atomicAdd(&n_cand, 1)] = (uint32_t)x;
            }
        }
        __syncthreads();
        const int c = n_cand;
        for (int c0 = 0; c0 < c; c0 += 256 / BLOCK) {
            const int at = c0 + tid / BLOCK;
            bool pass = false;
            uint64_t k64 = 0;
            if (at < c) {
                const int64_t it = (int64_t)cand[at] * BLOCK + tid % BLOCK;
                if (it < a.n_items) {
                    const float v = score_item(a, p, sp, it);
                    k64 = make_key(v, (int32_t)(id0 + it));
                    pass = v > -INFINITY && k64 > g.kth;
                }
            }
            group_append(g, pass, k64);
            group_check(g, a.k, a.train_indices, mlo, mhi);
        }
        if (tid == 0) n_cand = 0;
        __syncthreads();
    }
    group_finish(g, a, r, a.train_indices, mlo, mhi);
}

// ------------------------------------------------------------------------------------------
// few items: a workgroup scores them all for one user, V per thread
// ------------------------------------------------------------------------------------------
template <int V>
__global__ __launch_bounds__(256) void score_small_i8_kernel(ScoreI8Args a)
{
    __shared__ GroupList g;
    __shared__ uint32_t train[V * 256 / 32];
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    int32_t user;
    const int64_t prow = user_row(a, r, &user);
    const int8_t *__restrict__ p = a.Pq + prow * a.ldp;
    const float sp = a.sp[prow];
    const int64_t id0 = a.id_offset + a.item_lo;
    for (int i = tid; i < V * 8; i += 256) train[i] = 0;
    if (tid == 0) g.count = 0;
    __syncthreads();
    if (a.train_indptr)
        for (int64_t t = a.train_indptr[user] + tid, e = a.train_indptr[user + 1]; t < e; t += 256) {
            const int64_t i = a.train_indices[t] - id0;
            if (i >= 0 && i < a.n_items) atomicOr(&train[i >> 5], 1u << (i & 31));
        }
    __syncthreads();
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = 256 * v + tid;
        key[v] = 0;
        if (i < a.n_items && !(train[i >> 5] >> (i & 31) & 1u)) {
            const float s = score_item(a, p, sp, i);
            key[v] = s > -INFINITY ? f32_orderable(s) : 0u;
        }
    }
    const uint32_t cut = rank_bound(key, a.k, g);
    if (tid == 0) g.kth = ((uint64_t)cut << 32) - 1;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const uint64_t k64 = ((uint64_t)key[v] << 32) | (uint32_t)~(uint32_t)(id0 + 256 * v + tid);
        group_append(g, key[v] > KEY_NONE && k64 > g.kth, k64);
        group_check(g, a.k, nullptr, 0, 0);
    }
    group_finish(g, a, r, nullptr, 0, 0);
}

__global__ __launch_bounds__(256) void no_entries_kernel(int32_t *__restrict__ ids, float *__restrict__ scores, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) { ids[i] = -1; scores[i] = -INFINITY; }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
// users per pass of steps 1 and 2: their table of best scores stays below 512 MB (or holds 32 users)
static int64_t users_per_pass(int64_t n, int64_t n_items)
{
    const int64_t pitch = (n_items + 8 * BLOCK - 1) / (8 * BLOCK) * 8;
    int64_t u = ((int64_t)512 << 20) / (pitch * 4) / 128 * 128;
    u = u < 32 ? 32 : u;
    return n < u ? n : u;
}

size_t tfrec_score_i8_bytes(int64_t n, int64_t n_items, int k)
{
    if (n <= 0 || n_items <= SMALL_ITEMS) return 0;
    const int64_t pitch = (n_items + 8 * BLOCK - 1) / (8 * BLOCK) * 8;
    return tf_align((size_t)users_per_pass(n, n_items) * pitch * 4) + 512;
}

static int launch_max(tfrec_ctx *ctx, MaxArgs m)
{
    const ScoreI8Args &a = m.s;
    auto go = [&]<int KS, int UW>() -> int {
        m.user_groups = (int)((a.n + 32 * UW - 1) / (32 * UW));
        const int wgs = (m.user_groups + 3) / 4;
        // enough waves for the chip (8 a CU), each with at least one group of 8 blocks
        int64_t splits = (2048 + m.user_groups - 1) / m.user_groups;
        splits = splits < m.groups ? splits : m.groups;
        m.groups_per_split = (m.groups + splits - 1) / splits;
        m.splits = (int)((m.groups + m.groups_per_split - 1) / m.groups_per_split);
        const int64_t grid = (int64_t)((m.splits + 7) / 8) * 8 * wgs;
        TF_REQUIRE(grid < (1ll << 31), TFREC_EUNSUP, "too many users and items for one launch");
        score_max_i8_kernel<KS, UW><<<(unsigned)grid, 256, 0, ctx->stream>>>(m);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    };
    auto users = [&]<int KS>() -> int {
        if (a.n <= 32) return go.template operator()<KS, 1>();
        if (a.n <= 64 || KS == 8) return go.template operator()<KS, 2>();
        return go.template operator()<KS, KS == 8 ? 2 : 4>();
    };
    if (a.d <= 32) return users.template operator()<1>();
    if (a.d <= 64) return users.template operator()<2>();
    if (a.d <= 128) return users.template operator()<4>();
    return users.template operator()<8>();
}

int tfrec_score_i8(tfrec_ctx *ctx, ScoreI8Args a)
{
    if (a.n == 0) return TFREC_OK;
    if (a.n_items == 0) {
        no_entries_kernel<<<(unsigned)((a.n * a.k + 255) / 256), 256, 0, ctx->stream>>>(a.out_ids, a.out_scores, a.n * a.k);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    }
    a.flags = ctx->d_flags;
    if (a.n_items <= SMALL_ITEMS) {
        const unsigned n = (unsigned)a.n;
        if (a.n_items <= 256) score_small_i8_kernel<1><<<n, 256, 0, ctx->stream>>>(a);
        else if (a.n_items <= 512) score_small_i8_kernel<2><<<n, 256, 0, ctx->stream>>>(a);
        else if (a.n_items <= 1024) score_small_i8_kernel<4><<<n, 256, 0, ctx->stream>>>(a);
        else if (a.n_items <= 2048) score_small_i8_kernel<8><<<n, 256, 0, ctx->stream>>>(a);
        else score_small_i8_kernel<16><<<n, 256, 0, ctx->stream>>>(a);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    }
    MaxArgs m{};
    m.groups = (a.n_items + 8 * BLOCK - 1) / (8 * BLOCK);
    m.pitch = m.groups * 8;
    const int64_t per_pass = users_per_pass(a.n, a.n_items);
    TF_TRY(tfrec_ws_require(ctx, ctx->ws_used + tfrec_score_i8_bytes(a.n, a.n_items, a.k)));
    TF_TRY(tfrec_note_capture(ctx));
    m.best = (float *)tfrec_ws_take(ctx, (size_t)per_pass * m.pitch * 4);
    TF_REQUIRE(m.best != nullptr, TFREC_ENOMEM, "internal: workspace carve failed");
    for (int64_t u0 = 0; u0 < a.n; u0 += per_pass) {
        m.s = a;
        m.s.n = a.n - u0 < per_pass ? a.n - u0 : per_pass;
        m.s.users = a.users + u0;
        if (a.p_compact) { m.s.Pq = a.Pq + u0 * a.ldp; m.s.sp = a.sp + u0; }
        m.s.out_ids = a.out_ids + u0 * a.k;
        m.s.out_scores = a.out_scores + u0 * a.k;
        TF_TRY(launch_max(ctx, m));
        pick_i8_kernel<<<(unsigned)m.s.n, 256, 0, ctx->stream>>>(m);
        TF_HIP(hipGetLastError());
    }
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
