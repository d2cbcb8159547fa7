// Top-k of the scores of 8-bit factor rows against an 8-bit item table (tfrec_quantize_rows_i8).
//
//   score[u][i] = ((float)(sum_f Pq[u][f] Qq[i][f]) * sp[u]) * sq[i] + b[i]       (each step rounded to float32)
//
// The order is (score descending, item id ascending), train items are left out, and the [users, items] matrix is never
// formed.  A NaN score (a NaN scale or bias) passes no comparison and so is never listed; neither is a score of -inf.
//
// Up to SMALL_ITEMS items, one workgroup scores them all for its user and keeps the scores in registers
// (score_small_i8_kernel).  Beyond that:
//   1. score_max_i8_kernel: all scores on the matrix cores; of every 16 items (a cell: the items whose scores one lane holds)
//      only an upper bound of the best score is kept for every user, and per user how far below its bound a cell's best
//      score can be: the table is read once however few the users are, and 1/16 of the scores is written.
//   2. pick_i8_kernel, a workgroup per user: the k-th largest of the bounds of disjoint groups of cells that hold no train
//      item, less that distance, is a lower bound T of the user's k-th best score (k different rankable items reach it).
//      Only cells whose bound reaches T can hold a listed item: k and few more, which are scored again, item by item.
// Neither depends on the order of the items, and nothing is kept between calls.
#include "i8_device.hpp"
#include "score_i8.hpp"
#include "topk_list.hpp"

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

struct __attribute__((packed, aligned(4))) Float4 { float v[4]; };       // 16 bytes at the alignment of a float

static constexpr int BLOCK = 32, CELL = 16;    // items per block (a matrix instruction's rows) and per cell
// Up to this many items (16 scores per thread) one launch does it, score_small_i8_kernel.  Against the two steps, us: one user x
// 1682 items x 20 columns 8 / 17, 943 users x 1682 x 20 13 / 23, 943 x 4000 x 128 32 / 33, 6000 x 1000 x 64 51 / 84, 20000 x 1682 x 20
// 140 / 211; even where many users meet the most items: 6000 x 3700 x 64 86 / 86, 20000 x 4000 x 64 260 / 256, 4096 x 4096 x 128 97 / 89.
static constexpr int SMALL_ITEMS = 4096;
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

// Scores of items by groups of LPI lanes (a power of two, at least the row's 16-byte chunks): a lane holds chunk lane % LPI of
// the user's row and reads that chunk of an item's row, so that a wave's load covers whole rows.
template <int LPI>
struct RowDot {
    uint4 p;
    float sp;
    int off;                   // byte offset of this lane's chunk in an item row
    __device__ __forceinline__ void init(const ScoreI8Args &a, int64_t prow)
    {
        const int c = 16 * (threadIdx.x % LPI);
        p = make_uint4(0, 0, 0, 0);
        if (c < a.d) p = keep_below(*reinterpret_cast<const uint4 *>(a.Pq + prow * a.ldp + c), c, a.d);
        off = c < a.d ? c : 0;                 // (a lane without a chunk reads the first, against zeros)
        sp = a.sp[prow];
    }
    __device__ __forceinline__ uint4 load(const ScoreI8Args &a, int64_t it) const
    {
        return *reinterpret_cast<const uint4 *>(a.Qq + (a.item_lo + it) * a.ldq + off);
    }
    // the sum over the group's lanes, on all of them
    __device__ __forceinline__ int dot(uint4 q) const
    {
        int s = __builtin_amdgcn_sdot4((int)q.x, (int)p.x, 0, false);
        s = __builtin_amdgcn_sdot4((int)q.y, (int)p.y, s, false);
        s = __builtin_amdgcn_sdot4((int)q.z, (int)p.z, s, false);
        s = __builtin_amdgcn_sdot4((int)q.w, (int)p.w, s, false);
        if constexpr (LPI > 1) s += __builtin_amdgcn_mov_dpp(s, 0xB1, 0xf, 0xf, true);       // quad_perm [1,0,3,2]
        if constexpr (LPI > 2) s += __builtin_amdgcn_mov_dpp(s, 0x4E, 0xf, 0xf, true);       // quad_perm [2,3,0,1]
        if constexpr (LPI > 4) s += __builtin_amdgcn_mov_dpp(s, 0x141, 0xf, 0xf, true);      // mirror of half a row of 16 lanes
        if constexpr (LPI > 8) s += __builtin_amdgcn_mov_dpp(s, 0x140, 0xf, 0xf, true);      // mirror of the row
        return s;
    }
    // an item's scale and bias, requested with its row
    struct Scale { float sq, b; };
    __device__ __forceinline__ Scale scale(const ScoreI8Args &a, int64_t it) const { return {a.sq[a.item_lo + it], a.b ? a.b[a.item_lo + it] : 0.f}; }
    __device__ __forceinline__ float score(int acc, Scale s) const { return add_rounded(scaled_sum(acc, sp, s.sq), s.b); }
    // Of 256 positions scored together, thread t owns this one: after LPI steps of 256 / LPI positions every thread has one.
    static __device__ __forceinline__ int owned() { return (threadIdx.x % LPI) * (256 / LPI) + (threadIdx.x & 255) / LPI; }
};

// ------------------------------------------------------------------------------------------
// step 1: a bound of the best score of every cell of 16 items, for every user
// ------------------------------------------------------------------------------------------
struct MaxArgs {
    ScoreI8Args s;
    float *bound;              // [n, pitch]: cells
    float *group_bound;        // [n, groups]: the largest bound of a group's 16 cells
    float *slack;              // [n, splits]: 1.6 |sp sq|, the largest over a split
    int64_t pitch;             // cells per user row: 16 per group of 8 blocks
    int64_t groups;            // groups of 8 blocks
    int64_t groups_per_split;
    int user_groups, splits;
};

static constexpr float LOWEST = -3.402823466e38f;
// A cell bound at or below this may stand for a cell without a score.
static constexpr float NO_SCORE = LOWEST * (1.f - 0x1p-19f);

// KS = steps of 32 columns, UW = sets of 32 users a wave holds (as the matrix instruction's B operand, resident; the items
// are its A operand and come straight from memory, a block ahead).  A lane gets 16 scores of one user per block: its cell
// is items 8 g + 4 h + 0..3, g = 0..3, of the block.
//
// The vector work per score is what bounds this kernel once there are users enough, so a score is formed in two
// instructions instead of the definition's four (its maximum is a third): the accumulator starts at 1.5 * 2^23 as the BITS of a float, so that its
// bits ARE the float 1.5 * 2^23 + sum (|sum| <= 256 * 2^14 = 2^22), and
//     v = fma(fma(acc, sp, -1.5 * 2^23 * sp), sq, b).
// Against the defined score e: the inner step is off by at most half an ulp of 1.5 * 2^23 sp (0.75 sp) and of the result
// (2^-24 * 2^22 sp), the defined products by 2 * 2^-24 of theirs (0.5 sp sq at most), and both sums by half an ulp of what
// they give: |v - e| <= 1.6 |sp sq| + 2^-22 |v|, plus a few steps of 2^-149.  A cell's bound is its largest v plus that
// (with 2^-21 for its own rounding), its best e at least the bound less twice that; the first term, which does not show in
// the bound, is kept per user and slice of the items.
// 4096 users, 200k items of 64 columns: 125 to 140 us (0.8 * 10^15 operations/s): 3.65 vector instructions a score all in all keep the
// vector pipes busy 61 % of the cycles, the matrix pipes 17 %, and 285 MB are written, a third more than the bounds are; without
// its stores it takes 100 to 105.  33 users, 2M items of 128 columns: 69 us, 3.9 TB/s: vector pipes 21 %, the waves wait for the one
// block each has on its way.
// Scales above 2^50 (of either sign) could leave float32's range in one form and not in the other: users and blocks that have such scales
// take the definition itself.
template <int KS, int UW>
__global__ __launch_bounds__(256, 2) void score_max_i8_kernel(MaxArgs m)
{
    __shared__ float out[4][UW][16][32];
    __shared__ __align__(16) float scales[4][2][64];
    __shared__ float tops[4][UW][4][32];
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
    float sp[UW], off_sp[UW], err_sp[UW], slack[UW];
    bool wide_user = false;
#pragma unroll
    for (int s = 0; s < UW; ++s) {
        const int64_t ur = (int64_t)ug * 32 * UW + 32 * s + r;
        int32_t id;
        const int64_t row = user_row(a, ur < a.n ? ur : a.n - 1, &id);
        sp[s] = a.sp[row];
        off_sp[s] = -12582912.f * sp[s];
        err_sp[s] = sp[s] == sp[s] ? 1.6f * fabsf(sp[s]) : 0.f;        // (a user without a scale has no scores to bound)
        slack[s] = 0.f;
        wide_user |= fabsf(sp[s]) > 0x1p50f;
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
    // a block as this lane holds it before its turn: its chunks of row r, and (h = 0) the scale or (h = 1) the bias of item r
    struct Block { i32x4 q[KS]; float sb; };
    const float *__restrict__ sb_src = h && bias ? bias : sq;
    auto load = [&](Block &o, int64_t blk) {
        const int64_t i = blk * BLOCK + r, row = i < a.n_items ? i : a.n_items - 1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) o.q[ks] = *reinterpret_cast<const i32x4 *>(Q + row * a.ldq + off[ks]);
        o.sb = sb_src[row];
        if (h && !bias) o.sb = 0.f;
        if (i >= a.n_items) o.sb = h ? -INFINITY : 0.f;        // (past the last item: a score of -inf)
    };
    i32x16 start;
#pragma unroll
    for (int e = 0; e < 16; ++e) start[e] = 0x4B400000;
    // kept in registers, not made again for every product, where there are registers for it
    if constexpr (KS < 4) asm volatile("" : "+v"(start));
    // long rows leave no registers to hold the next block's first products
    constexpr bool AHEAD = KS < 6;
    auto products = [&](const Block &o, int s) {
        i32x16 acc = start;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(o.q[ks], pb[s][ks], acc, 0, 0, 0);
        return acc;
    };
    i32x16 acc;                // products of the set whose vector work comes next
    auto step = [&](Block &cur, Block &next, int64_t g, int i) {
        // the scales and biases of the lane's 16 items come through LDS: as loads from memory, eight of 16 bytes a lane for
        // 2 * 16 values, they would keep the memory pipe as busy as the vector pipe
        scales[wave][i & 1][lane] = cur.sb;
        if constexpr (!AHEAD) acc = products(cur, 0);
        load(next, g * 8 + i + 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float sqv[16], bv[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 x = *reinterpret_cast<const float4 *>(&scales[wave][i & 1][8 * q + 4 * h]);
            const float4 y = *reinterpret_cast<const float4 *>(&scales[wave][i & 1][32 + 8 * q + 4 * h]);
            sqv[4 * q] = x.x; sqv[4 * q + 1] = x.y; sqv[4 * q + 2] = x.z; sqv[4 * q + 3] = x.w;
            bv[4 * q] = y.x; bv[4 * q + 1] = y.y; bv[4 * q + 2] = y.z; bv[4 * q + 3] = y.w;
        }
        float sqm = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sqm = fmaxf(sqm, fabsf(sqv[e]));
        auto keep = [&](int s, float mx, float d) {
            slack[s] = fmaxf(slack[s], d);
            out[wave][s][2 * i + h][r] = mx + fmaf(fabsf(mx), 0x1p-21f, d);
        };
        // the products of the next set (after the last, of the next block's first) are issued before the vector work on this
        // set's, and the matrix pipe has them done when their turn comes
        auto sets = [&]<bool PLAIN>() {
#pragma unroll
            for (int s = 0; s < UW; ++s) {
                const i32x16 x = acc;
                __builtin_amdgcn_sched_barrier(0);
                if (s + 1 < UW) acc = products(cur, s + 1);
                else if constexpr (AHEAD) acc = products(next, 0);
                __builtin_amdgcn_sched_barrier(0);
                float mx = LOWEST;
                if constexpr (PLAIN) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, fmaf(fmaf(__int_as_float(x[e]), sp[s], off_sp[s]), sqv[e], bv[e]));
                    keep(s, mx, fmaf(err_sp[s], sqm, 0x1p-140f));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        mx = fmaxf(mx, add_rounded(scaled_sum(x[e] - 0x4B400000, sp[s], sqv[e]), bv[e]));
                    keep(s, mx, 0x1p-140f);
                }
            }
        };
        if (__ballot(wide_user || sqm > 0x1p50f) == 0) [[likely]] sets.template operator()<true>();
        else sets.template operator()<false>();
    };
    Block even, odd;
    load(even, g0 * 8);
    if (AHEAD) acc = products(even, 0);
    for (int64_t g = g0; g < g1; ++g) {
#pragma unroll 1
        for (int i = 0; i < 8; i += 2) {
            step(even, odd, g, i);
            step(odd, even, g, i + 1);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < UW; ++s) {
            const int64_t ur = (int64_t)ug * 32 * UW + 32 * s + r;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = out[wave][s][8 * h + j][r];
            if (ur < a.n) {
                float4 *to = reinterpret_cast<float4 *>(m.bound + ur * m.pitch + g * 16 + 8 * h);
                to[0] = make_float4(v[0], v[1], v[2], v[3]);
                to[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
            float top = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
            top = fmaxf(top, __uint_as_float(swap32(__float_as_uint(top), lane)));
            // four groups' bounds are stored together: one store per row and group would be as many as the cells take
            const int at = (int)(g - g0) & 3;
            tops[wave][s][at][r] = top;
            if (at == 3 || g + 1 == g1) {
                float *to = m.group_bound + ur * m.groups + g - at;
                if (h == 0 && ur < a.n) {
                    if (at == 3) *reinterpret_cast<Float4 *>(to) = Float4{{tops[wave][s][0][r], tops[wave][s][1][r], tops[wave][s][2][r], top}};
                    else
                        for (int j = 0; j <= at; ++j) to[j] = tops[wave][s][j][r];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int s = 0; s < UW; ++s) {
        const int64_t ur = (int64_t)ug * 32 * UW + 32 * s + r;
        slack[s] = fmaxf(slack[s], __uint_as_float(swap32(__float_as_uint(slack[s]), lane)));
        if (h == 0 && ur < a.n) m.slack[ur * m.splits + split] = slack[s];
    }
}

// ------------------------------------------------------------------------------------------
// a workgroup's list of keys
// ------------------------------------------------------------------------------------------
// LIST keys at most: room for k and for the 256 that one step may add.  512 up to k = 112 (a quarter of the registers and
// half the LDS of 1024, which is what bounds the workgroups a CU holds: pick_i8_kernel for 4096 users of 200k items 80 us
// against 110 when it was chosen), else 1024.
static inline int list_for(int k) { return k <= 112 ? 512 : 1024; }
template <int LIST>
struct GroupList {
    uint64_t list[LIST], sorted[LIST];
    uint64_t kth;              // keys at or below it are not wanted
    int count;
    uint32_t hist[2][64];
    uint32_t lo[16], hi[16];
    int valid[16];
};

// A lower bound of the k-th largest of the workgroup's orderable values (V per thread; values at or below `none` are
// none): the lower edge of a bucket of a two-level histogram below the highest bit in which the values differ.
// 0 if fewer than k values are held.
template <int NT, int V, class List>
__device__ __forceinline__ uint32_t rank_bound(const uint32_t (&key)[V], uint32_t none, int k, List &g)
{
    constexpr int NW = NT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t lo = 0xffffffffu, hi = 0;
    int valid = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (key[v] > none) {
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
    valid = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        lo = g.lo[w] < lo ? g.lo[w] : lo;
        hi = g.hi[w] > hi ? g.hi[w] : hi;
        valid += g.valid[w];
    }
    if (valid < k) return 0;
    if (lo == hi) return hi;
    const int top = 31 - __builtin_clz(lo ^ hi);
    const int s1 = top >= 5 ? top - 5 : 0;
    // level 1: six bits from the highest differing one down (all values share the bits above)
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (key[v] > none) atomicAdd(&g.hist[0][(key[v] >> s1) & 63u], 1u);
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
            if (key[v] > none && key[v] >> s1 == cut >> s1) atomicAdd(&g.hist[1][(key[v] >> s2) & mask], 1u);
        __syncthreads();
        int above2, in2;
        cut |= level(g.hist[1], k - above, &above2, &in2) << s2;
    }
    return cut;
}

// a wave's keys that pass go to the list; all lanes call it
template <class List>
__device__ __forceinline__ void group_append(List &g, bool pass, uint64_t key)
{
    const int lane = threadIdx.x & 63;
    const uint64_t m = __ballot(pass);
    if (!m) return;
    int base = 0;
    if (lane == 0) base = atomicAdd(&g.count, __popcll(m));
    base = __builtin_amdgcn_readfirstlane(base);
    if (pass) g.list[base + __popcll(m & ((1ull << lane) - 1))] = key;
}

// The same for N keys a lane (key(i) is 0 for none) with one atomic a wave, and no look at the room: keys behind the list's end
// are dropped, the count tells (the caller then goes over them again, checked).
template <int N, int LIST, class Key>
__device__ __forceinline__ void group_append_many(GroupList<LIST> &g, Key &&key)
{
    const int lane = threadIdx.x & 63;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mine += key(i) != 0;
    const int incl = wave_prefix_sum(mine), total = __builtin_amdgcn_readlane(incl, 63);
    if (!total) return;
    int base = 0;
    if (lane == 0) base = atomicAdd(&g.count, total);
    int at = __builtin_amdgcn_readfirstlane(base) + incl - mine;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t k = key(i);
        if (k != 0 && at < LIST) g.list[at] = k;
        at += k != 0;
    }
}

// called by all threads after a step that appended at most 256 keys: cuts the list back to its k best once the next step might
// not fit
template <int LIST>
__device__ __forceinline__ void group_check(GroupList<LIST> &g, int k, const int32_t *midx, int64_t mlo, int64_t mhi)
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
template <int LIST>
__device__ __forceinline__ void group_finish(GroupList<LIST> &g, const ScoreI8Args &a, int64_t r, const int32_t *midx, int64_t mlo, int64_t mhi)
{
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x, cnt = g.count;
    float tau;
    int kept;
    if (cnt <= 128) kept = wave_compact<128>(g.list, cnt, 0, a.k, midx, mlo, mhi, g.sorted, lane, &tau);
    else if (cnt <= 256) kept = wave_compact<256>(g.list, cnt, 0, a.k, midx, mlo, mhi, g.sorted, lane, &tau);
    else kept = wave_compact<LIST>(g.list, cnt, 0, a.k, midx, mlo, mhi, g.sorted, lane, &tau);
    for (int e = lane; e < a.k; e += 64) {
        const uint64_t key = e < kept ? g.sorted[e] : 0;
        a.out_ids[r * a.k + e] = e < kept ? key_id(key) : -1;
        a.out_scores[r * a.k + e] = e < kept ? key_score(key) : -INFINITY;
    }
}

// ------------------------------------------------------------------------------------------
// step 2: the cells that can hold a listed item, scored again
// ------------------------------------------------------------------------------------------
// The cut is taken over groups of 16 cells where there are groups enough (a sixteenth of the bounds is then read), else over
// the cells themselves: "units" below.
static constexpr int SLICES = 1024;            // unit u belongs to slice u % SLICES
static constexpr int UNITS = 2048;             // units listed at a time
static constexpr int CAND = 2048;              // cells scored between two looks at the lists

// first item of cell y, and item e of it
__device__ __forceinline__ int64_t cell_first(int64_t y) { return (y >> 1) * BLOCK + 4 * (y & 1); }
__device__ __forceinline__ int64_t cell_item(int64_t y, int e) { return cell_first(y) + 8 * (e >> 2) + (e & 3); }

// NT = 256 threads, or 1024 where there are few users and one workgroup's time is the call's; LPI: see RowDot.
// Some twenty dependent steps a user.  4096 users of 200k items 68 to 78 us (vector pipes busy 60 % of the cycles; five workgroups a
// CU, more of them at fewer registers gain nothing; with a look at the list's room every 256 items 80), one user of 200k items 12.5 us,
// 33 of 2M items 20 us (with 256 of the 1024 threads scoring 15 and 25), both bound by latency.
// A train item takes its slice out of the cut.  Of 1024 slices about 1024 exp(-n / 1024) are left for n train items at random: with
// some thousands there are fewer than k, or the cut is loose, and the user's workgroup scores many cells or all: one user of 200k
// items 20 us with 40 train items, 100 with 3000, 187 with 10000.
template <int NT, int LPI, int LIST>
__global__ __launch_bounds__(NT) void pick_i8_kernel(MaxArgs m)
{
    __shared__ GroupList<LIST> g;
    __shared__ uint32_t cand[CAND], units[UNITS];
    __shared__ uint16_t slices[SLICES];
    __shared__ uint8_t train[SLICES];
    __shared__ int n_slices, n_units, n_cand;
    __shared__ uint32_t slack;
    constexpr int V = SLICES / NT;
    const ScoreI8Args &a = m.s;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    int32_t user;
    const int64_t prow = user_row(a, r, &user);
    RowDot<LPI> dot;
    dot.init(a, prow);
    const int64_t mlo = a.train_indptr ? a.train_indptr[user] : 0, mhi = a.train_indptr ? a.train_indptr[user + 1] : 0;
    const int64_t id0 = a.id_offset + a.item_lo;
    const bool by_group = m.groups >= 2 * (a.k + (mhi - mlo)) + 64;
    const uint32_t count = by_group ? (uint32_t)m.groups : 2u * (uint32_t)((a.n_items + BLOCK - 1) / BLOCK);
    const float *__restrict__ bound = m.bound + r * m.pitch;
    const float *__restrict__ top = by_group ? m.group_bound + r * m.groups : bound;
    auto first_id = [&](uint32_t u) { return (int32_t)(id0 + (by_group ? (int64_t)u * (8 * BLOCK) : cell_first(u))); };
    int64_t t = mlo + tid;
    const int32_t train0 = t < mhi ? a.train_indices[t] : -1;

    // the largest bound of every slice
    float mx[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mx[v] = LOWEST;
    constexpr int DEPTH = V >= 4 ? 4 : 8;              // loads in flight: DEPTH * V
    for (uint32_t u0 = 0; u0 < count; u0 += DEPTH * SLICES) {
        float w[DEPTH][V];
#pragma unroll
        for (int q = 0; q < DEPTH; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const uint32_t u = u0 + q * SLICES + NT * v + tid;
                w[q][v] = u < count ? top[u] : LOWEST;
            }
#pragma unroll
        for (int q = 0; q < DEPTH; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v) mx[v] = fmaxf(mx[v], w[q][v]);
    }
    for (int i = tid; i < SLICES; i += NT) train[i] = 0;
    if (tid == 0) { g.count = 0; n_slices = 0; n_units = 0; n_cand = 0; }
    if (tid == 0) slack = 0u;
    __syncthreads();
    {
        // (not negative: the order of the bits is the order of the values, and a maximum has no order of arrival)
        float w = 0.f;
        for (int i = tid; i < m.splits; i += NT) w = fmaxf(w, m.slack[r * m.splits + i]);
        for (int o = 32; o > 0; o >>= 1) w = fmaxf(w, __shfl_xor(w, o, 64));
        if ((tid & 63) == 0) atomicMax(&slack, __float_as_uint(w));
    }
    // (an index of any other sign or size is another shard's item)
    auto mark = [&](int32_t id) {
        const int64_t i = id - id0;
        if (id >= 0 && i >= 0 && i < a.n_items) train[(by_group ? i / (8 * BLOCK) : 2 * (i / BLOCK) + (i >> 2 & 1)) % SLICES] = 1;
    };
    mark(train0);
    for (t += NT; t < mhi; t += NT) mark(a.train_indices[t]);
    __syncthreads();
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = train[NT * v + tid] ? 0u : f32_orderable(mx[v]);
    const uint32_t cut = rank_bound<NT, V>(key, f32_orderable(NO_SCORE), a.k, g);
    // T: the cut less what a bound may be off (twice the slack, and this arithmetic's rounding); without a cut all cells pass
    float T = -INFINITY;
    if (cut) {
        const float c = fminf(orderable_f32(cut), -LOWEST);
        T = c - 2.1f * __uint_as_float(slack) - fabsf(c) * 0x1p-19f;
        T = T > LOWEST ? T : -INFINITY;           // (also where T is not a number)
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (mx[v] >= T) slices[atomicAdd(&n_slices, 1)] = (uint16_t)(NT * v + tid);
    if (tid == 0) g.kth = T > -INFINITY ? ((uint64_t)f32_orderable(T) << 32) - 1 : ((uint64_t)KEY_NONE << 32 | 0xffffffffu);
    __syncthreads();

    // 256 threads (a team) score 256 items in a round; the rows of ROUNDS rounds are requested together
    constexpr int TEAMS = NT / 256, ROUNDS = TEAMS > 1 ? (LPI <= 2 ? 2 : 1) : (LPI <= 2 ? 4 : (LPI <= 8 ? 2 : 1)), STEP = 256 * TEAMS * ROUNDS;
    const int team = tid >> 8, lane_row = (tid & 255) / LPI;
    const int sub = by_group ? 16 : 1;                                  // cells of a unit
    const uint32_t per = (count + SLICES - 1) / SLICES, total = dot.sp == dot.sp ? (uint32_t)n_slices * per : 0u;
    for (uint32_t e0 = 0; e0 < total;) {
        // units of the wanted slices whose bound, under its lowest id, is wanted (else nothing in them is)
        uint64_t kth = g.kth;
        const uint32_t e1 = total - e0 < UNITS ? total : e0 + UNITS;
        for (uint32_t e = e0 + tid; e < e1; e += NT) {
            const uint32_t u = slices[e / per] + (e % per) * SLICES;
            if (u < count && make_key(top[u], first_id(u)) > kth) units[atomicAdd(&n_units, 1)] = u;
        }
        e0 = e1;
        __syncthreads();
        const int nu = n_units;
        for (int v0 = 0; v0 < nu; v0 += CAND / 16) {
            const int nv = nu - v0 < CAND / 16 ? nu - v0 : CAND / 16;
            kth = g.kth;
            for (int i = tid; i < nv * sub; i += NT) {
                const uint32_t u = units[v0 + i / sub], y = u * sub + i % sub;
                if (make_key(bound[y], (int32_t)(id0 + cell_first(y))) > kth) cand[atomicAdd(&n_cand, 1)] = y;
            }
            const int held = g.count;
            __syncthreads();
            const int c = n_cand;
            // once without a look at the list's room (the cut lets little more than k items pass), and once more, checked
            // every 256 items, where it did not do
#pragma unroll 1
            for (int turn = 0;; ++turn) {
                for (int c0 = 0; c0 < c * CELL; c0 += STEP) {
                    int acc[ROUNDS];
                    int64_t own[ROUNDS];
                    typename RowDot<LPI>::Scale sc[ROUNDS];
                    uint4 q[ROUNDS][LPI];
#pragma unroll
                    for (int o = 0; o < ROUNDS; ++o) {
                        const int i = c0 + 256 * (o * TEAMS + team) + RowDot<LPI>::owned();
                        own[o] = i < c * CELL ? cell_item(cand[i / CELL], i % CELL) : a.n_items;
                        sc[o] = dot.scale(a, own[o] < a.n_items ? own[o] : 0);
                    }
#pragma unroll
                    for (int o = 0; o < ROUNDS; ++o)
#pragma unroll
                        for (int j = 0; j < LPI; ++j) {
                            const int i = c0 + 256 * (o * TEAMS + team) + j * (256 / LPI) + lane_row;
                            int64_t it = i < c * CELL ? cell_item(cand[i / CELL], i % CELL) : 0;
                            it = it < a.n_items ? it : 0;
                            q[o][j] = dot.load(a, it);
                        }
                    uint64_t k64[ROUNDS];
#pragma unroll
                    for (int o = 0; o < ROUNDS; ++o) {
#pragma unroll
                        for (int j = 0; j < LPI; ++j) {
                            const int s = dot.dot(q[o][j]);
                            if (tid % LPI == j) acc[o] = s;
                        }
                        const float v = dot.score(acc[o], sc[o]);
                        k64[o] = own[o] < a.n_items && v > -INFINITY ? make_key(v, (int32_t)(id0 + own[o])) : 0;
                    }
                    if (turn == 0) {
                        const uint64_t least = g.kth;
                        group_append_many<ROUNDS>(g, [&](int o) { return k64[o] > least ? k64[o] : 0; });
                    } else {
#pragma unroll 1
                        for (int t = 0; t < ROUNDS * TEAMS && c0 + 256 * t < c * CELL; ++t) {
                            uint64_t mine = k64[0];
#pragma unroll
                            for (int i = 1; i < ROUNDS; ++i) mine = i == t / TEAMS ? k64[i] : mine;
                            if (team == t % TEAMS) group_append(g, mine > g.kth, mine);
                            group_check(g, a.k, a.train_indices, mlo, mhi);
                        }
                    }
                }
                if (turn) break;
                __syncthreads();
                if (g.count <= LIST) break;
                __syncthreads();
                if (tid == 0) g.count = held;
                group_check(g, a.k, a.train_indices, mlo, mhi);
            }
            if (tid == 0) n_cand = 0;
            __syncthreads();
        }
        if (tid == 0) n_units = 0;
        __syncthreads();
    }
    group_finish(g, a, r, a.train_indices, mlo, mhi);
}

// ------------------------------------------------------------------------------------------
// few items: a workgroup scores them all for one user, 16 per thread at most (943 users of 1682 items, 20 columns: 13.4 us,
// nearly all of it the dependent steps of one workgroup)
// ------------------------------------------------------------------------------------------
template <int LPI, int LIST>
__global__ __launch_bounds__(256) void score_small_i8_kernel(ScoreI8Args a)
{
    constexpr int V = SMALL_ITEMS / 256;
    __shared__ GroupList<LIST> g;
    __shared__ uint32_t train[SMALL_ITEMS / 32];
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    int32_t user;
    const int64_t prow = user_row(a, r, &user);
    RowDot<LPI> dot;
    dot.init(a, prow);
    const int64_t id0 = a.id_offset + a.item_lo;
    const int n_items = (int)a.n_items, own = RowDot<LPI>::owned();
    // (the train row is requested ahead of the items and looked at behind them)
    const int64_t mlo = a.train_indptr ? a.train_indptr[user] : 0, mhi = a.train_indptr ? a.train_indptr[user + 1] : 0;
    const int32_t train0 = mlo + tid < mhi ? a.train_indices[mlo + tid] : -1;
    for (int i = tid; i < SMALL_ITEMS / 32; i += 256) train[i] = 0;
    if (tid == 0) g.count = 0;
    __syncthreads();
    uint32_t key[V];
    constexpr int BATCH = LPI <= 4 ? 4 : (LPI == 8 ? 2 : 1);           // rounds of 256 items whose rows are requested together
#pragma unroll
    for (int v0 = 0; v0 < V; v0 += BATCH) {
#pragma unroll
        for (int o = 0; o < BATCH; ++o) key[v0 + o] = 0;
        if (256 * v0 >= n_items) continue;
        uint4 q[BATCH][LPI];
        typename RowDot<LPI>::Scale sc[BATCH];
#pragma unroll
        for (int o = 0; o < BATCH; ++o) {
            const int i = 256 * (v0 + o) + own;
            sc[o] = dot.scale(a, i < n_items ? i : 0);
#pragma unroll
            for (int j = 0; j < LPI; ++j) {
                const int it = 256 * (v0 + o) + j * (256 / LPI) + tid / LPI;
                q[o][j] = dot.load(a, it < n_items ? it : 0);
            }
        }
#pragma unroll
        for (int o = 0; o < BATCH; ++o) {
            int acc = 0;
#pragma unroll
            for (int j = 0; j < LPI; ++j) {
                const int s = dot.dot(q[o][j]);
                if (tid % LPI == j) acc = s;
            }
            const int i = 256 * (v0 + o) + own;
            if (i < n_items) {
                const float s = dot.score(acc, sc[o]);
                key[v0 + o] = s > -INFINITY ? f32_orderable(s) : 0u;
            }
        }
    }
    auto mark = [&](int32_t id) {
        const int64_t i = id - id0;
        if (id >= 0 && i >= 0 && i < n_items) atomicOr(&train[i >> 5], 1u << (i & 31));
    };
    mark(train0);
    for (int64_t t = mlo + tid + 256; t < mhi; t += 256) mark(a.train_indices[t]);
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = 256 * v + own;
        if (train[i >> 5] >> (i & 31) & 1u) key[v] = 0;
    }
    // the k-th largest of the threads' best is a lower bound of the k-th largest of all, for few k nearly as high (k = 50: about
    // 56 keys reach it) and found from one value a thread: 943 users of 1682 items 16.1 -> 13.4 us
    uint32_t cut;
    if constexpr (LIST == 512) {
        uint32_t best[1] = {0};
#pragma unroll
        for (int v = 0; v < V; ++v) best[0] = key[v] > best[0] ? key[v] : best[0];
        cut = rank_bound<256, 1>(best, KEY_NONE, a.k, g);
    } else cut = rank_bound<256, V>(key, KEY_NONE, a.k, g);
    if (tid == 0) g.kth = cut ? ((uint64_t)cut << 32) - 1 : ((uint64_t)KEY_NONE << 32 | 0xffffffffu);
    __syncthreads();
    // (as in pick_i8_kernel: all keys at once where they fit the list, else 256 at a time)
    auto k64 = [&](int v) { return ((uint64_t)key[v] << 32) | (uint32_t)~(uint32_t)(id0 + 256 * v + own); };
    const uint64_t least = g.kth;
    group_append_many<V>(g, [&](int v) { return key[v] > KEY_NONE && k64(v) > least ? k64(v) : 0; });
    __syncthreads();
    if (g.count > LIST) {
        __syncthreads();
        if (tid == 0) g.count = 0;
        __syncthreads();
#pragma unroll 1
        for (int v = 0; 256 * v < n_items; ++v) {
            uint64_t mine = k64(0);
#pragma unroll
            for (int i = 1; i < V; ++i) mine = i == v ? k64(i) : mine;
            group_append(g, (uint32_t)(mine >> 32) > KEY_NONE && mine > g.kth, mine);
            group_check(g, a.k, nullptr, 0, 0);
        }
    }
    group_finish(g, a, r, nullptr, 0, 0);
}

__global__ __launch_bounds__(256) void no_entries_kernel(int32_t *__restrict__ ids, float *__restrict__ scores, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) { ids[i] = -1; scores[i] = -INFINITY; }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
// users per pass of steps 1 and 2: their table of bounds stays below 512 MB (or holds 32 users)
static int64_t users_per_pass(int64_t n, int64_t groups)
{
    int64_t u = ((int64_t)512 << 20) / (groups * 68) / 128 * 128;
    u = u < 32 ? 32 : u;
    return n < u ? n : u;
}

// sets of 32 users a wave of step 1 holds: as many as its 256 registers take beside two blocks of items (4 for rows of up to
// 64 bytes, 3 up to 128, 2 beyond: rows of 256 columns, 4096 users, 200k items 600 us, with one set 870)
static int sets_per_wave(int64_t n, int d) { return n <= 32 ? 1 : (n <= 64 || d > 128 ? 2 : (d > 64 ? 3 : 4)); }

// slices of the items: enough waves for the chip (8 a CU), each with at least one group of 8 blocks
static int split_items(int64_t n, int64_t groups, int d, int64_t *groups_per_split)
{
    const int64_t user_groups = (n + 32 * sets_per_wave(n, d) - 1) / (32 * sets_per_wave(n, d));
    int64_t splits = (2048 + user_groups - 1) / user_groups;
    splits = splits < groups ? splits : groups;
    *groups_per_split = (groups + splits - 1) / splits;
    return (int)((groups + *groups_per_split - 1) / *groups_per_split);
}

static size_t slack_bytes(int64_t n)
{
    // (a later, shorter pass has fewer user groups and so up to 2048 splits for its users)
    return tf_align((size_t)4 * (n + 2048 * 32 * 4));
}

size_t tfrec_score_i8_bytes(int64_t n, int64_t n_items)
{
    if (n <= 0 || n_items <= SMALL_ITEMS) return 0;
    const int64_t groups = (n_items + 8 * BLOCK - 1) / (8 * BLOCK), per_pass = users_per_pass(n, groups);
    return tf_align((size_t)per_pass * groups * 64) + tf_align((size_t)per_pass * groups * 4) + slack_bytes(per_pass) + 1024;
}

// calls f.operator()<LPI>() with the lanes an item's row takes
template <class F>
static int by_row_lanes(int d, F &&f)
{
    if (d <= 16) return f.template operator()<1>();
    if (d <= 32) return f.template operator()<2>();
    if (d <= 64) return f.template operator()<4>();
    if (d <= 128) return f.template operator()<8>();
    return f.template operator()<16>();
}

static int launch_max(tfrec_ctx *ctx, const MaxArgs &m)
{
    const int64_t grid = (int64_t)((m.splits + 7) / 8) * 8 * ((m.user_groups + 3) / 4);
    TF_TRY(check_launch(grid, 256));
    auto go = [&]<int KS, int UW>() -> int {
        score_max_i8_kernel<KS, UW><<<(unsigned)grid, 256, 0, ctx->stream>>>(m);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    };
    const int uw = sets_per_wave(m.s.n, m.s.d);
    auto users = [&]<int KS>() -> int {
        if (uw == 1) return go.template operator()<KS, 1>();
        if (uw == 2) return go.template operator()<KS, 2>();
        return go.template operator()<KS, KS <= 2 ? 4 : (KS == 4 ? 3 : 2)>();
    };
    if (m.s.d <= 32) return users.template operator()<1>();
    if (m.s.d <= 64) return users.template operator()<2>();
    if (m.s.d <= 128) return users.template operator()<4>();
    // (rows of 160 columns, 4096 users, 200k items: 394 us against 458 in eight steps)
    if (m.s.d <= 192) return users.template operator()<6>();
    return users.template operator()<8>();
}

static int launch_pick(tfrec_ctx *ctx, const MaxArgs &m)
{
    return by_row_lanes(m.s.d, [&]<int LPI>() -> int {
        // few users leave most of the chip idle whatever their workgroups do: larger ones end sooner
        const unsigned n = (unsigned)m.s.n;
        if (list_for(m.s.k) == 512) {
            if (n <= 256) pick_i8_kernel<1024, LPI, 512><<<n, 1024, 0, ctx->stream>>>(m);
            else pick_i8_kernel<256, LPI, 512><<<n, 256, 0, ctx->stream>>>(m);
        } else {
            if (n <= 256) pick_i8_kernel<1024, LPI, 1024><<<n, 1024, 0, ctx->stream>>>(m);
            else pick_i8_kernel<256, LPI, 1024><<<n, 256, 0, ctx->stream>>>(m);
        }
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    });
}

int tfrec_score_i8(tfrec_ctx *ctx, ScoreI8Args a)
{
    if (a.n == 0) return TFREC_OK;
    if (a.n_items == 0) {
        const int64_t blocks = (a.n * a.k + 255) / 256;
        no_entries_kernel<<<(unsigned)(blocks < TF_LAUNCH_ROWS ? blocks : TF_LAUNCH_ROWS), 256, 0, ctx->stream>>>(a.out_ids, a.out_scores, a.n * a.k);
        TF_HIP(hipGetLastError());
        return TFREC_OK;
    }
    a.flags = ctx->d_flags;
    // users u0 .. u0 + n of the call
    auto listed = [&](int64_t u0, int64_t n) {
        ScoreI8Args s = a;
        s.n = n;
        s.users = a.users + u0;
        if (a.p_compact) { s.Pq = a.Pq + u0 * a.ldp; s.sp = a.sp + u0; }
        s.out_ids = a.out_ids + u0 * a.k;
        s.out_scores = a.out_scores + u0 * a.k;
        return s;
    };
    if (a.n_items <= SMALL_ITEMS)
        return by_row_lanes(a.d, [&]<int LPI>() -> int {
            for (int64_t u0 = 0; u0 < a.n; u0 += TF_LAUNCH_ROWS) {
                const ScoreI8Args s = listed(u0, a.n - u0 < TF_LAUNCH_ROWS ? a.n - u0 : TF_LAUNCH_ROWS);
                if (list_for(a.k) == 512) score_small_i8_kernel<LPI, 512><<<(unsigned)s.n, 256, 0, ctx->stream>>>(s);
                else score_small_i8_kernel<LPI, 1024><<<(unsigned)s.n, 256, 0, ctx->stream>>>(s);
                TF_HIP(hipGetLastError());
            }
            return TFREC_OK;
        });
    MaxArgs m{};
    m.groups = (a.n_items + 8 * BLOCK - 1) / (8 * BLOCK);
    m.pitch = m.groups * 16;
    const int64_t per_pass = users_per_pass(a.n, m.groups);
    TF_TRY(tfrec_ws_require(ctx, ctx->ws_used + tfrec_score_i8_bytes(a.n, a.n_items)));
    m.bound = (float *)tfrec_ws_take(ctx, (size_t)per_pass * m.pitch * 4);
    m.group_bound = (float *)tfrec_ws_take(ctx, (size_t)per_pass * m.groups * 4);
    const size_t slack = slack_bytes(per_pass);
    m.slack = (float *)tfrec_ws_take(ctx, slack);
    TF_REQUIRE(m.bound != nullptr && m.group_bound != nullptr && m.slack != nullptr, TFREC_ENOMEM, "internal: workspace carve failed");
    for (int64_t u0 = 0; u0 < a.n; u0 += per_pass) {
        m.s = listed(u0, a.n - u0 < per_pass ? a.n - u0 : per_pass);
        m.splits = split_items(m.s.n, m.groups, a.d, &m.groups_per_split);
        const int users = 32 * sets_per_wave(m.s.n, a.d);
        m.user_groups = (int)((m.s.n + users - 1) / users);
        TF_REQUIRE((size_t)m.s.n * m.splits * 4 <= slack, TFREC_ENOMEM, "internal: scratch too small");
        TF_TRY(launch_max(ctx, m));
        TF_TRY(launch_pick(ctx, m));
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
