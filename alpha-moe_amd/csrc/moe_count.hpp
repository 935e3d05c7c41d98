// A stable counting sort of routing slots by expert, in pieces: what the aligner and the sort of tokens share.
#pragma once
#include "moe_common.hpp"

namespace alpha_moe {
namespace {

typedef unsigned long long lanes_t;
constexpr int kMasks = 256;   // entries of a wavefront's table of lane masks: the experts' low eight bits

// LDS accesses of one wavefront complete in order; this keeps the compiler to the written order
__device__ __forceinline__ void lds_order()
{
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// The lanes of this wavefront whose slot has the same expert as this lane's (e < 0: no slot, no lanes); all 64 lanes
// call it.  masks: the wavefront's table, zero before and after (its LDS accesses complete in order).
// Lanes that add to one table entry take turns.  FEW (few experts, many slots: few_experts()) is for inputs on which that is the
// rule and not the exception: up to eight experts a ballot per bit of the id instead, otherwise the first lane's expert - the hot
// one, if there is one - by a ballot and the others by the table.
template <bool FEW>
__device__ __forceinline__ lanes_t same_expert(int e, int id_bits, lanes_t *masks)
{
    lanes_t first = 0;
    bool other = e >= 0;
    if constexpr (FEW) {
        if (id_bits <= 3) {
            lanes_t same = __ballot(e >= 0);
            for (int b = 0; b < id_bits; b++) {
                const bool set = (e >> b) & 1;
                const lanes_t with = __ballot(set);
                same &= set ? with : ~with;
            }
            return e >= 0 ? same : 0;
        }
        const int e0 = __builtin_amdgcn_readfirstlane(e);
        first = __ballot(e == e0);
        first = e == e0 && e >= 0 ? first : 0;
        other = e >= 0 && e != e0;
    }
    lanes_t same = 0;
    if (other) atomicOr(&masks[e & (kMasks - 1)], 1ull << (threadIdx.x & 63));
    lds_order();
    if (other) same = masks[e & (kMasks - 1)];
    lds_order();
    if (other) masks[e & (kMasks - 1)] = 0;
    lds_order();
    for (int b = 8; b < id_bits; b++) {   // the upper bits, one ballot each
        const bool set = (e >> b) & 1;
        const lanes_t with = __ballot(set);
        same &= set ? with : ~with;
    }
    return same | first;
}

// The bucket of slot i: its expert, -1 behind the end; a slot whose id names no expert has none, or with OTHERS the one behind the
// experts', E.
template <bool OTHERS>
__device__ __forceinline__ int bucket_of_slot(const int32_t *ids, int i, int end, int E)
{
    const int e = i < end ? ids[i] : -1;
    if constexpr (OTHERS) return i >= end ? -1 : (unsigned)e < (unsigned)E ? e : E;
    return e < E ? e : -1;
}

__device__ __forceinline__ lanes_t lanes_below() { return (1ull << (threadIdx.x & 63)) - 1ull; }

// The 64-slot chunks of ids[lo, hi) that a wavefront keeps in registers between counting and placing.
constexpr int kKept = 4;
struct Chunks {
    int e[kKept];
    lanes_t same[kKept];
};

template <bool OTHERS = false>
__device__ __forceinline__ void load_chunks(const int32_t *ids, int lo, int hi, int E, Chunks &c)
{
#pragma unroll
    for (int k = 0; k < kKept; k++) c.e[k] = bucket_of_slot<OTHERS>(ids, lo + k * 64 + (threadIdx.x & 63), hi, E);
}

// counts[at] += n, 16-bit counts, without a round trip.  (Neighbouring wavefronts' counters may share a word.)
__device__ __forceinline__ void add_count(uint16_t *counts, int at, int n)
{
    atomicAdd(reinterpret_cast<unsigned *>(counts) + (at >> 1), (unsigned)n << (16 * (at & 1)));
}

// cursors[e][column] += slots of expert e in ids[lo, hi).  One wavefront, its own column; c holds the first chunks' experts.
template <bool FEW, bool OTHERS = false>
__device__ __forceinline__ void count_run(const int32_t *ids, int lo, int hi, int E, int id_bits, lanes_t *masks,
                                          uint16_t *cursors, int column, int n_waves, Chunks &c)
{
    auto count = [&](int e, lanes_t same) {
        if (e >= 0 && (same & lanes_below()) == 0) add_count(cursors, e * n_waves + column, __builtin_popcountll(same));
    };
#pragma unroll
    for (int k = 0; k < kKept; k++)
        if (lo + k * 64 < hi) c.same[k] = same_expert<FEW>(c.e[k], id_bits, masks);
#pragma unroll
    for (int k = 0; k < kKept; k++)
        if (lo + k * 64 < hi) count(c.e[k], c.same[k]);
    for (int base = lo + kKept * 64; base < hi; base += 64) {
        const int e = bucket_of_slot<OTHERS>(ids, base + (threadIdx.x & 63), hi, E);
        count(e, same_expert<FEW>(e, id_bits, masks));
    }
}

// put(place, slot, e) for the slots of ids[lo, hi): those of expert e go to start(e) + cursor[e] ..., in order.  One wavefront, its
// own cursors (a chunk's are read before they move on: LDS accesses of a wavefront complete in order).
template <bool FEW, bool OTHERS = false, typename Start, typename Put>
__device__ __forceinline__ void place_run(const int32_t *ids, int lo, int hi, int E, int id_bits, lanes_t *masks, Start start,
                                          uint16_t *cursors, int column, int n_waves, const Chunks &c, Put put)
{
    auto place = [&](int e, lanes_t same) {   // the slot's place
        int at = 0;
        if (e >= 0) at = start(e) + cursors[e * n_waves + column];
        lds_order();
        if (e >= 0 && (same & lanes_below()) == 0) add_count(cursors, e * n_waves + column, __builtin_popcountll(same));
        lds_order();
        return at + __builtin_popcountll(same & lanes_below());
    };
    int at[kKept];
#pragma unroll
    for (int k = 0; k < kKept; k++)
        if (lo + k * 64 < hi) at[k] = place(c.e[k], c.same[k]);
#pragma unroll
    for (int k = 0; k < kKept; k++)
        if (lo + k * 64 < hi && c.e[k] >= 0) put(at[k], lo + k * 64 + (int)(threadIdx.x & 63), c.e[k]);
    for (int base = lo + kKept * 64; base < hi; base += 64) {
        const int i = base + (threadIdx.x & 63);
        const int e = bucket_of_slot<OTHERS>(ids, i, hi, E);
        const int to = place(e, same_expert<FEW>(e, id_bits, masks));
        if (e >= 0) put(to, i, e);
    }
}

// cursors[e][w] of the n_waves (2, 4, 8 or 16) wavefronts: counts -> exclusive prefix over the wavefronts; returns the sum
__device__ __forceinline__ int prefix_over_waves(uint16_t *cursors, int e, int n_waves)
{
    int run = 0;
    auto step = [&](unsigned two) {
        const unsigned c0 = two & 0xffffu, c1 = two >> 16, first = run;
        run += (int)(c0 + c1);
        return first | (first + c0) << 16;
    };
    if (n_waves >= 8) {
        v4i *c = reinterpret_cast<v4i *>(cursors + (size_t)e * n_waves);
        v4i a = c[0], b = c[n_waves > 8 ? 1 : 0];
#pragma unroll
        for (int k = 0; k < 4; k++) a[k] = (int)step((unsigned)a[k]);
        c[0] = a;
        if (n_waves > 8) {
#pragma unroll
            for (int k = 0; k < 4; k++) b[k] = (int)step((unsigned)b[k]);
            c[1] = b;
        }
    } else {
        unsigned *c = reinterpret_cast<unsigned *>(cursors + (size_t)e * n_waves);
        const unsigned a = c[0], b = c[n_waves > 2 ? 1 : 0];
        c[0] = step(a);
        if (n_waves > 2) c[1] = step(b);
    }
    return run;
}

// Inclusive prefix sum over the wavefront, in registers (a step is a shift within rows of 16 lanes, or the last lane of the rows
// before; through LDS, as __shfl_up goes, a step is a round trip).
__device__ __forceinline__ int row_inclusive_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // from 1, 2, 4, 8 lanes below in the row
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    return v;
}
__device__ __forceinline__ int wave_inclusive_scan(int v)
{
    v = row_inclusive_scan(v);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // lane 15 of rows 0 and 2 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // lane 31 to rows 2 and 3
    return v;
}

// Exclusive prefix sum over the n values of LDS array `vals`, in place; returns their sum.  All 1024 threads call it.
__device__ __forceinline__ int block_exclusive_scan(int *vals, int n, int *wave_sums /* [16] */)
{
    const int per = (n + 1023) / 1024;
    const int lo = min((int)threadIdx.x * per, n), hi = min(lo + per, n);
    int sum = 0, incl = 0;
    if (__builtin_amdgcn_readfirstlane(lo < n)) {   // (a wavefront without values leaves the others its cycles)
        for (int i = lo; i < hi; i++) sum += vals[i];
        incl = wave_inclusive_scan(sum);
    }
    if ((threadIdx.x & 63) == 63) wave_sums[threadIdx.x >> 6] = incl;
    lds_barrier();
    const int sums = row_inclusive_scan(wave_sums[threadIdx.x & 15]);   // (of all sixteen wavefronts, in every row)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), total = __builtin_amdgcn_readlane(sums, 15);
    int run = incl - sum + (wave > 0 ? __builtin_amdgcn_readlane(sums, wave - 1) : 0);
    for (int i = lo; i < hi; i++) {
        const int v = vals[i];
        vals[i] = run;
        run += v;
    }
    lds_barrier();
    return total;
}

// bytes of the cursors of n_waves wavefronts, whole 16 bytes
__host__ __device__ constexpr size_t cursor_bytes(int n_waves, int E) { return ((size_t)n_waves * E * sizeof(uint16_t) + 15) & ~(size_t)15; }

}  // namespace
}  // namespace alpha_moe
