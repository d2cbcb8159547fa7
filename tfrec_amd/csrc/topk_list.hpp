// Candidate lists of a running top-k, shared by the scoring kernels: keys that order (score descending, item id
// ascending), the wave-wide sorts and selections that compact a list, and the final pass that puts it in order.
#pragma once
#include "common.hpp"

// cycle counts of developer builds (the including file may define them first)
#ifndef TF_PROF_T
#define TF_PROF_T() 0ull
#define TF_PROF_ADD(i, t0) (void)(t0)
#endif

// ------------------------------------------------------------------------------------------
// keys: (score, id) packed so that a larger 64-bit key means "ranks earlier"
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t f32_orderable(float x)
{
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float orderable_f32(uint32_t o)
{
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t make_key(float score, int32_t id)
{
    return ((uint64_t)f32_orderable(score) << 32) | (uint32_t)(~(uint32_t)id);
}
__device__ __forceinline__ float key_score(uint64_t k) { return orderable_f32((uint32_t)(k >> 32)); }
__device__ __forceinline__ int32_t key_id(uint64_t k) { return (int32_t)(~(uint32_t)k); }

__device__ __forceinline__ bool csr_row_contains(const int32_t *__restrict__ idx, int64_t lo, int64_t hi, int32_t id)
{
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        const int32_t v = idx[mid];
        if (v == id) return true;
        if (v < id) lo = mid + 1; else hi = mid;
    }
    return false;
}

// Wave-wide bitonic sort of CAP 64-bit keys in LDS, descending.  All 64 lanes must call it.
template <int CAP>
__device__ __forceinline__ void wave_sort_desc(volatile uint64_t *buf, int lane)
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int k2 = 2; k2 <= CAP; k2 <<= 1) {
        for (int j = k2 >> 1; j > 0; j >>= 1) {
#pragma unroll
            for (int t = lane; t < CAP / 2; t += 64) {
                const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
                const int p = i | j;
                const uint64_t a = buf[i], b = buf[p];
                const bool desc = (i & k2) == 0;
                if ((a < b) == desc) { buf[i] = b; buf[p] = a; }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Wave-wide bitonic sort, descending, of CAP 64-bit keys held EPL = CAP/64 per lane: key[q] of lane
// l is element q*64 + l.  Partners 64 or more elements apart sit in the same lane (register
// compare-exchange); nearer partners are fetched with cross-lane moves, no LDS round trips.
template <int CAP, int K2, int J>
__device__ __forceinline__ void bitonic_step(uint64_t (&key)[CAP / 64], int lane)
{
    constexpr int EPL = CAP / 64;
    if constexpr (J >= 64) {
        constexpr int JQ = J / 64;
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            if ((q & JQ) == 0) {
                const bool desc = (((q * 64 + lane) & K2) == 0);
                const uint64_t x = key[q], y = key[q | JQ];
                const bool swap = desc ? (x < y) : (x > y);
                key[q] = swap ? y : x;
                key[q | JQ] = swap ? x : y;
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const uint64_t x = key[q];
            const uint32_t plo = xor_lane_u32<J>((uint32_t)x, lane), phi = xor_lane_u32<J>((uint32_t)(x >> 32), lane);
            const uint64_t y = ((uint64_t)phi << 32) | plo;
            const bool desc = (((q * 64 + lane) & K2) == 0);
            const bool lower = (lane & J) == 0;
            const bool take_max = (lower == desc);
            key[q] = take_max ? (x > y ? x : y) : (x < y ? x : y);
        }
    }
}
template <int CAP, int K2, int J>
__device__ __forceinline__ void bitonic_merge(uint64_t (&key)[CAP / 64], int lane)
{
    bitonic_step<CAP, K2, J>(key, lane);
    if constexpr (J > 1) bitonic_merge<CAP, K2, J / 2>(key, lane);
}
template <int CAP, int K2>
__device__ __forceinline__ void bitonic_sort(uint64_t (&key)[CAP / 64], int lane)
{
    if constexpr (K2 > 2) bitonic_sort<CAP, K2 / 2>(key, lane);
    bitonic_merge<CAP, K2, K2 / 2>(key, lane);
}

// Compacts one candidate list.  list[0..cnt) holds keys; entries [0,ver) are known not to be
// masked.  Drops masked ids, sorts, keeps the best k.  Returns the new count; *tau_out gets the
// k-th best score (or -inf while fewer than k are held).  Wave-uniform arguments.
// The user's sorted row of masked ids is first copied into the (still unused) sort buffer when it
// fits there, so that the binary searches run in LDS after one coalesced read instead of a chain
// of dependent global loads each.
template <int CAP>
__device__ __forceinline__ int wave_compact(uint64_t *__restrict__ list, int cnt, int ver, int k,
                                            const int32_t *__restrict__ mask_idx, int64_t mlo, int64_t mhi,
                                            volatile uint64_t *sortbuf, int lane, float *tau_out)
{
    constexpr int EPL = CAP / 64;             // entries per lane
    constexpr int ROWCAP = CAP * 2;           // int32 ids that fit the sort buffer
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");   // this wave's own appends are visible
    const int64_t L = mhi - mlo;
    const bool check = mask_idx != nullptr && L > 0 && ver < cnt;
    const bool staged = check && L <= ROWCAP;
    volatile int32_t *rowbuf = reinterpret_cast<volatile int32_t *>(sortbuf);
    // the list entries and the masked row are requested together (one memory round trip, not two)
    uint64_t keys[EPL];
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = lane + 64 * q;
        keys[q] = e < cnt ? list[e] : 0;
    }
    if (staged) {
        for (int j = lane; j < (int)L; j += 64) rowbuf[j] = mask_idx[mlo + j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (check) {
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const int e = lane + 64 * q;
            if (e < cnt && e >= ver) {
                const int32_t id = key_id(keys[q]);
                bool hit;
                if (staged) {
                    int lo = 0, hi = (int)L;
                    hit = false;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        const int32_t v = rowbuf[mid];
                        if (v == id) { hit = true; break; }
                        if (v < id) lo = mid + 1; else hi = mid;
                    }
                } else {
                    hit = csr_row_contains(mask_idx, mlo, mhi, id);
                }
                if (hit) keys[q] = 0;
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();          // every lane is done with the staged row
    int kept = 0;
#pragma unroll
    for (int q = 0; q < EPL; ++q) kept += __popcll(__ballot(keys[q] != 0));
    bitonic_sort<CAP, CAP>(keys, lane);
#pragma unroll
    for (int q = 0; q < EPL; ++q) sortbuf[lane + 64 * q] = keys[q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int newc = kept < k ? kept : k;
    for (int e = lane; e < newc; e += 64) list[e] = sortbuf[e];
    *tau_out = newc >= k ? key_score(sortbuf[k - 1]) : -INFINITY;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return newc;
}

// Inclusive sum over the lanes 0..lane of a wave, by DPP row shifts and row broadcasts (six vector adds, no LDS trip).
__device__ __forceinline__ int wave_prefix_sum(int x)
{
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);   // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);   // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);   // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
    return x;
}

// One level of a histogram selection among the keys a wave holds (EPL per lane).  A key takes part when its score bits from
// `match_shift` up equal `match_value`; its bucket is the `nbits` (<= 6) bits from `shift` up.  Finds the highest bucket L
// such that at least `want` taking-part keys lie in buckets >= L (the caller makes sure that `want` of them take part);
// returns L, *above = keys in buckets > L, *in_bucket = keys in bucket L.  hist: 64 counters in LDS, this wave's own.
// Wave-uniform arguments and results.
template <int EPL>
__device__ __forceinline__ int hist_select_level(const uint64_t (&keys)[EPL], int match_shift, uint32_t match_value, int shift, int nbits, int want,
                                                 volatile uint32_t *hist, int lane, int *above, int *in_bucket)
{
    hist[lane] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t bmask = (1u << nbits) - 1u;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const uint32_t hi = (uint32_t)(keys[q] >> 32);
        if (keys[q] != 0 && (uint32_t)((uint64_t)hi >> match_shift) == match_value) atomicAdd(const_cast<uint32_t *>(hist) + ((hi >> shift) & bmask), 1u);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int c = (int)hist[lane];
    const int incl = wave_prefix_sum(c);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    const int at_or_above = total - incl + c;                     // keys in buckets >= lane
    const uint64_t m = __ballot(at_or_above >= want);
    const int L = m ? 63 - __builtin_clzll(m) : 0;
    *in_bucket = __builtin_amdgcn_readlane(c, L);
    *above = __builtin_amdgcn_readlane(at_or_above, L) - *in_bucket;
    __builtin_amdgcn_wave_barrier();
    return L;
}

// Compaction by selection: like wave_compact, but the k survivors are SELECTED, not sorted -- a list
// only has to be in order when it is written out, and then only its k survivors (wave_finish).  The k-th largest key is found by descending over its
// bits (one wave-uniform count per bit: compares, ballots and scalar population counts; the low
// half -- the id -- only when scores tie at the cut), which costs an order of magnitude fewer
// vector instructions than the sort.  The survivors are written back in lane order.
// A candidate list is two regions of CAP/2 entries, one per lane that holds items of the user (each lane appends to
// its own region without asking the other): region r holds cnt_r entries, the first ver_r of them known not to be
// masked.  INTERLEAVE: survivor j is written to region j & 1, slot j >> 1 (the list itself: both regions get half);
// else to out[j] (the sort buffer of the final pass).
// APPROX (compactions during the scan): the cut is found by two levels of a 64-way histogram over the score bits below the
// highest bit in which the held scores differ, and is the lower edge of a bucket: at least k and in practice k or k + 1 keys
// survive, *tau_out is a lower bound of the k-th best score -- all a filter threshold has to be.  When more than k + 16 keys
// would survive (ties, or scores that differ only in their last bits), the exact descent runs instead.
template <int CAP, bool INTERLEAVE, bool APPROX = false, class Out>
__device__ __forceinline__ int wave_select(const uint64_t *list, int cnt0, int cnt1, int ver0, int ver1, int k,
                                           const int32_t *__restrict__ mask_idx, int64_t mlo, int64_t mhi,
                                           volatile uint64_t *sortbuf, int lane, float *tau_out, Out out,
                                           [[maybe_unused]] unsigned long long *prof_acc = nullptr)
{
    [[maybe_unused]] unsigned long long prof_t = TF_PROF_T();
    constexpr int EPL = CAP / 64;
    constexpr int ROWCAP = CAP * 2;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
#ifdef TF_EVAL_PROFILE
    if (prof_acc) { prof_acc[8] += TF_PROF_T() - prof_t; prof_t = TF_PROF_T(); }
#endif
    const int64_t L = mhi - mlo;
    const bool check = mask_idx != nullptr && L > 0 && (ver0 < cnt0 || ver1 < cnt1);
    const bool staged = check && L <= ROWCAP;
    volatile int32_t *rowbuf = reinterpret_cast<volatile int32_t *>(sortbuf);
    constexpr int HQ = EPL / 2;               // register slots per region
    uint64_t keys[EPL];
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const int e = lane + 64 * (q % HQ);
        keys[q] = e < (q < HQ ? cnt0 : cnt1) ? list[(q / HQ) * (CAP / 2) + e] : 0;
    }
    // short rows are padded to whole groups of four with an id no key carries
    constexpr int LINEAR_MAX = 64;
    const bool linear = staged && L <= LINEAR_MAX;
    if (staged) {
        const int Lp = linear ? (((int)L + 3) & ~3) : (int)L;
        for (int j = lane; j < Lp; j += 64) rowbuf[j] = j < (int)L ? mask_idx[mlo + j] : -2;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
#ifdef TF_EVAL_PROFILE
    if (prof_acc) { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); prof_acc[9] += TF_PROF_T() - prof_t; prof_t = TF_PROF_T(); }
#endif
    if (linear) {
        // every row id against every held id: the row is read four ids at a time (all lanes the same
        // address, one LDS access), independent reads instead of a chain of dependent probes per key
        const int4 *row4 = reinterpret_cast<const int4 *>(const_cast<const int32_t *>(rowbuf));
        bool hit[EPL];
#pragma unroll
        for (int q = 0; q < EPL; ++q) hit[q] = false;
        for (int j = 0; j < (int)L; j += 4) {
            const int4 r = row4[j >> 2];
#pragma unroll
            for (int q = 0; q < EPL; ++q) {
                const int32_t id = key_id(keys[q]);
                hit[q] = hit[q] | (id == r.x) | (id == r.y) | (id == r.z) | (id == r.w);
            }
        }
#pragma unroll
        for (int q = 0; q < EPL; ++q)
            if (hit[q]) keys[q] = 0;
    } else if (check) {
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const int e = lane + 64 * (q % HQ);
            if (e < (q < HQ ? cnt0 : cnt1) && e >= (q < HQ ? ver0 : ver1)) {
                const int32_t id = key_id(keys[q]);
                bool hit;
                if (staged) {
                    int lo = 0, hi = (int)L;
                    hit = false;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        const int32_t v = rowbuf[mid];
                        if (v == id) { hit = true; break; }
                        if (v < id) lo = mid + 1; else hi = mid;
                    }
                } else {
                    hit = csr_row_contains(mask_idx, mlo, mhi, id);
                }
                if (hit) keys[q] = 0;
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();          // every lane is done with the staged row
#ifdef TF_EVAL_PROFILE
    if (prof_acc) { prof_acc[10] += TF_PROF_T() - prof_t; prof_t = TF_PROF_T(); }
#endif
    int kept = 0;
#pragma unroll
    for (int q = 0; q < EPL; ++q) kept += __popcll(__ballot(keys[q] != 0));
    uint64_t cut = 1;                          // keep every real key while fewer than k are held
    if (kept >= k) {
        // the bits all held scores share need no descent: start below the highest bit in which they differ
        uint32_t all_or = 0, all_and = 0xffffffffu;
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
            const uint32_t hi = (uint32_t)(keys[q] >> 32);
            all_or |= hi;
            all_and &= keys[q] != 0 ? hi : 0xffffffffu;
        }
        all_or |= xor_lane_u32<32>(all_or, lane);  all_and &= xor_lane_u32<32>(all_and, lane);
        all_or |= xor_lane_u32<16>(all_or, lane);  all_and &= xor_lane_u32<16>(all_and, lane);
        all_or |= xor_lane_u32<8>(all_or, lane);   all_and &= xor_lane_u32<8>(all_and, lane);
        all_or |= xor_lane_u32<4>(all_or, lane);   all_and &= xor_lane_u32<4>(all_and, lane);
        all_or |= xor_lane_u32<2>(all_or, lane);   all_and &= xor_lane_u32<2>(all_and, lane);
        all_or |= xor_lane_u32<1>(all_or, lane);   all_and &= xor_lane_u32<1>(all_and, lane);
        const uint32_t differ = __builtin_amdgcn_readfirstlane(all_or ^ all_and);
        bool cut_found = false;
        if constexpr (APPROX) {
            if (differ) {
                volatile uint32_t *hist = reinterpret_cast<volatile uint32_t *>(sortbuf);     // the staged row is no longer needed
                const int top = 31 - __builtin_clz(differ);
                const uint32_t common = __builtin_amdgcn_readfirstlane(all_and);
                // level 1: the six bits from the highest differing one down (every held key shares the bits above them)
                const int shift1 = top >= 5 ? top - 5 : 0;
                int above1, in1;
                const int L1 = hist_select_level<EPL>(keys, shift1 + 6, (uint32_t)((uint64_t)common >> (shift1 + 6)), shift1, 6, k, hist, lane, &above1, &in1);
                uint32_t hi_cut = (uint32_t)(((uint64_t)common >> (shift1 + 6)) << (shift1 + 6)) | ((uint32_t)L1 << shift1);
                int survivors = above1 + in1;
                if (survivors > k && shift1 > 0) {
                    // level 2: the next (up to) six bits, among the keys of the level-1 bucket that holds the k-th
                    const int shift2 = shift1 >= 6 ? shift1 - 6 : 0;
                    int above2, in2;
                    const int L2 = hist_select_level<EPL>(keys, shift1, hi_cut >> shift1, shift2, shift1 - shift2, k - above1, hist, lane, &above2, &in2);
                    hi_cut |= (uint32_t)L2 << shift2;
                    survivors = above1 + above2 + in2;
                }
                if (survivors <= k + 16) {
                    cut = (uint64_t)hi_cut << 32;
                    cut_found = true;
                }
            }
        }
        if (!cut_found) {
        // highest differing bit, moved up to an odd position so that whole pairs of bits remain (a shared
        // bit taken into the descent is simply found again)
        int bit = differ ? ((31 - __builtin_clz(differ)) | 1) : -1;
        uint32_t hi_cut = __builtin_amdgcn_readfirstlane(all_and) & (bit >= 0 ? ~(uint32_t)((2ull << bit) - 1ull) : 0xffffffffu);
        int exact = 0;
        const int may_stop = kept > k ? 1 : 0;        // with exactly k held, all bits are resolved: the cut is then the lowest score
        // two bits per round: three counts, then the largest candidate that still has k keys at or above it
#pragma unroll 1
        for (; bit >= 1; bit -= 2) {
#ifdef TF_EVAL_PROFILE
            if (prof_acc) prof_acc[13] += 1;
#endif
            const uint32_t step = 1u << (bit - 1);
            const uint32_t t1 = hi_cut + step, t2 = hi_cut + 2 * step, t3 = hi_cut + 3 * step;
            // all compares first, each into its own mask, then the scalar counts: one shared condition
            // register would chain every compare to the count before it
            uint64_t m1[EPL], m2[EPL], m3[EPL];
#pragma unroll
            for (int q = 0; q < EPL; ++q) {
                const uint32_t hi = (uint32_t)(keys[q] >> 32);
                m1[q] = __ballot(hi >= t1);
                m2[q] = __ballot(hi >= t2);
                m3[q] = __ballot(hi >= t3);
            }
            __builtin_amdgcn_sched_barrier(0);
            int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
            for (int q = 0; q < EPL; ++q) {
                c1 += __popcll(m1[q]);
                c2 += __popcll(m2[q]);
                c3 += __popcll(m3[q]);
            }
            // the counts fall from c1 to c3, so the number of candidates that still have k keys is the choice
            const uint32_t sel = (uint32_t)(c1 >= k) + (uint32_t)(c2 >= k) + (uint32_t)(c3 >= k);
            const int cs = sel == 3u ? c3 : (sel == 2u ? c2 : c1);
            hi_cut += sel * step;
            exact = sel != 0u ? (cs == k ? 1 : 0) : exact;
            if (exact & may_stop) break;
        }
        cut = (uint64_t)hi_cut << 32;
        if (!exact) {                          // equal scores may straddle the cut: the id decides
#ifdef TF_EVAL_PROFILE
            if (prof_acc) prof_acc[14] += 1;
#endif
#pragma unroll 1
            for (int bit = 31; bit >= 0; --bit) {
                const uint64_t t2 = cut | (1ull << bit);
                int c2 = 0;
#pragma unroll
                for (int q = 0; q < EPL; ++q) c2 += __popcll(__ballot(keys[q] >= t2));
                if (c2 >= k) {
                    cut = t2;
                    if (c2 == k) break;
                }
            }
        }
        }   // !cut_found
    }
#ifdef TF_EVAL_PROFILE
    if (prof_acc) { prof_acc[11] += TF_PROF_T() - prof_t; prof_t = TF_PROF_T(); }
#endif
    int base = 0;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
        const bool keep = keys[q] >= cut;
        const uint64_t m = __ballot(keep);
        const int j = base + __popcll(m & ((1ull << lane) - 1ull));
        if (keep) out[INTERLEAVE ? (j & 1) * (CAP / 2) + (j >> 1) : j] = keys[q];
        base += __popcll(m);
    }
    *tau_out = kept >= k ? key_score(cut) : -INFINITY;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#ifdef TF_EVAL_PROFILE
    if (prof_acc) { prof_acc[12] += TF_PROF_T() - prof_t; }
#endif
    return base;
}

// End of the scan: select the k survivors into the wave's LDS buffer (the staged row is no longer
// needed once the selection has its keys in registers), sort just those, leave them in sortbuf[0..n).
template <int CAP>
__device__ __forceinline__ int wave_finish(const uint64_t *__restrict__ list, int cnt0, int cnt1, int ver0, int ver1, int k,
                                           const int32_t *__restrict__ mask_idx, int64_t mlo, int64_t mhi,
                                           volatile uint64_t *sortbuf, int lane)
{
    constexpr int SN = (CAP / 2 & (CAP / 2 - 1)) == 0 ? CAP / 2 : 128;     // a power of two (the sort); k <= SN - 16 for every capacity in use
    float tau;
    // a list that fits the sort as it is needs no selection first (asking for more survivors than it can
    // hold makes the selection keep every unmasked entry); the sort then puts the best k in front
    const bool small = cnt0 + cnt1 <= SN;
    const int held = wave_select<CAP, false>(list, cnt0, cnt1, ver0, ver1, small ? CAP : k, mask_idx, mlo, mhi, sortbuf, lane, &tau, sortbuf);
    const int nc = held < k ? held : k;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    uint64_t keys[SN / 64];
#pragma unroll
    for (int q = 0; q < SN / 64; ++q) {
        const int e = lane + 64 * q;
        keys[q] = e < held ? sortbuf[e] : 0;
    }
    bitonic_sort<SN, SN>(keys, lane);
#pragma unroll
    for (int q = 0; q < SN / 64; ++q) sortbuf[lane + 64 * q] = keys[q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return nc;
}
