// Tokens sorted by expert and back, with the gradients of both.
//
//   slot i = t top_k + s of token t goes to row r(i): slots by ascending expert, equal experts by ascending slot; slots whose id names no
//   expert behind all others.  row_of_slot[i] = r(i), or ~r(i) where the slot has no expert, so that the map is a permutation of all
//   rows either way: every row is written by exactly one slot, and nothing is filled beforehand.
//   sort:      rows[r(i)] = x[t], 0 for a slot without an expert          grad_x[t] = sum over s of grad_rows[r(t, s)]   (a combine)
//   combine:   out[t] = c * sum over s of w[t, s] rows[r(t, s)]
//   backward:  grad_rows[r(t, s)] = c w[t, s] g[t],  grad_w[t, s] = c (g[t] . rows[r(t, s)])
//
// Sums are taken in fp32, slots in ascending order, and rounded once; there are no atomics on results.  What is negative in the map
// takes no part: neither its row nor its weight is looked at.  An index of a row is checked against the rows before it is used.
//
// All of it is memory traffic: a row is read once and written once for each slot, in pieces of 16 bytes a thread, a token's row in registers
// while it goes to all its slots.  MI355X: 8192 tokens of 7168 codes to 8 rows each 103 us, 93 of them the copies (545 MB, 5.9 TB/s; a copy
// of 1 GiB runs at 5.1); sums of 4096 x 8 rows of 2048 bf16 24 us (151 MB, 6.2 TB/s, part of it out of the last-level cache), their backward
// pass 55 (285 MB, 5.2).  What is left of small calls is the launch and one chain of dependent loads: 7.3 us for a token's 9 slots, 5.3 for
// the sums of 61 tokens, of 2.2 for an empty kernel.
#include "moe_count.hpp"

namespace alpha_moe {
namespace {

// 16 bytes of a row that starts at any multiple of A bytes (16, or 2: rows whose length is no multiple of 16, or a tensor that does not
// start at one; memory takes such loads and stores as a whole).
template <int A>
struct Piece;
template <>
struct Piece<16> {
    typedef uint32_t type __attribute__((ext_vector_type(4)));
};
template <>
struct Piece<2> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
typedef uint32_t v4w __attribute__((ext_vector_type(4)));

// Piece v of a row of `bytes` bytes, the last one short if A is 2 (what is behind the row's end is 0).
template <int A>
__device__ __forceinline__ v4w load_piece(const uint8_t *row, int v, int64_t bytes)
{
    const int64_t at = (int64_t)v * 16;
    if (A == 16 || at + 16 <= bytes) return *reinterpret_cast<const typename Piece<A>::type *>(row + at);
    v4w r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (at + 2 * i < bytes) r[i / 2] |= (uint32_t) * reinterpret_cast<const uint16_t *>(row + at + 2 * i) << (16 * (i & 1));
    return r;
}
// Non-temporal: rows are written once, and most of them are many (8192 tokens of 7168 codes to 8 rows each 127 us without, 103 with it;
// sums of 4096 x 8 rows of 2048 bf16 33 and 29).
template <int A>
__device__ __forceinline__ void store_piece(uint8_t *row, int v, int64_t bytes, v4w r)
{
    const int64_t at = (int64_t)v * 16;
    if (A == 16 || at + 16 <= bytes) {
        __builtin_nontemporal_store((typename Piece<A>::type)r, reinterpret_cast<typename Piece<A>::type *>(row + at));
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (at + 2 * i < bytes) *reinterpret_cast<uint16_t *>(row + at + 2 * i) = (uint16_t)(r[i / 2] >> (16 * (i & 1)));
}

struct SortParams {
    const uint8_t *x;
    const float *x_scale;
    const int32_t *ids;
    uint8_t *rows;
    float *scale;
    int32_t *offsets, *row_of_slot;
    int *hist;
    int64_t row_bytes;
    int scale_cols, M, top_k, E, numel, pieces;
};

// The U pieces v0, v0 + step, ... of token t's row.
template <int A, int U>
__device__ __forceinline__ void gather(const SortParams &p, int t, int v0, int step, v4w (&piece)[U])
{
    const uint8_t *from = p.x + (int64_t)t * p.row_bytes;
#pragma unroll
    for (int u = 0; u < U; u++)
        if (v0 + u * step < p.pieces) piece[u] = load_piece<A>(from, v0 + u * step, p.row_bytes);
}
// They go to the rows of its slots, and so do (columns c0, c0 + c_step, ...) its scales.  at(s): the slot's entry in the map.
template <int A, int U, typename At>
__device__ __forceinline__ void spread(const SortParams &p, int t, int v0, int step, const v4w (&piece)[U], int c0, int c_step, At at)
{
    for (int s = 0; s < p.top_k; s++) {
        const int m = at(s);
        const int64_t row = m < 0 ? ~m : m;
        uint8_t *to = p.rows + row * p.row_bytes;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (v0 + u * step < p.pieces)
                store_piece<A>(to, v0 + u * step, p.row_bytes, m < 0 ? (v4w){0, 0, 0, 0} : piece[u]);
    }
    if (p.scale_cols > 0)
        for (int c = c0; c < p.scale_cols; c += c_step) {
            const float v = p.x_scale[(int64_t)t * p.scale_cols + c];
            for (int s = 0; s < p.top_k; s++) {
                const int m = at(s);
                p.scale[(int64_t)(m < 0 ? ~m : m) * p.scale_cols + c] = m < 0 ? 0.f : v;
            }
        }
}

__device__ __forceinline__ int bucket(int id, int E) { return (unsigned)id < (unsigned)E ? id : E; }

// Few slots, in one launch: a workgroup to a token (and 16 KiB of its row) finds its slots' rows by itself - a slot's row is the number
// of slots in front of it, by (expert, slot) - and one more workgroup counts the experts.  Its row is on the way meanwhile.
// MI355X: 9 slots 5.0 us, three launches 11.5.
constexpr int kSortMaxExperts = 4096, kMaxTopK = 64;
template <int A>
__global__ __launch_bounds__(256) void sort_few_kernel(const SortParams p)
{
    __shared__ int lds[kSortMaxExperts + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if ((int)blockIdx.x == p.M) {   // offsets
        if (blockIdx.y > 0) return;
        __shared__ int sums[4];
        for (int e = tid; e <= p.E; e += 256) lds[e] = 0;
        __syncthreads();
        for (int i = tid; i < p.numel; i += 256) atomicAdd(&lds[bucket(p.ids[i], p.E)], 1);
        __syncthreads();
        const int per = (p.E + 1 + 255) / 256, lo = min(tid * per, p.E + 1), hi = min(lo + per, p.E + 1);
        int sum = 0;
        for (int e = lo; e < hi; e++) sum += lds[e];
        const int incl = wave_inclusive_scan(sum);
        if (lane == 63) sums[wave] = incl;
        __syncthreads();
        int run = incl - sum;
        for (int w = 0; w < wave; w++) run += sums[w];
        for (int e = lo; e < hi; e++) {
            p.offsets[e] = run;
            run += lds[e];
        }
        return;
    }
    const int t = blockIdx.x, part = blockIdx.y;
    v4w piece[4];
    gather<A, 4>(p, t, part * 1024 + tid, 256, piece);
    constexpr int G = 8;   // slots looked at together
    for (int s0 = 0; s0 < p.top_k; s0 += G) {
        int key[G], count[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int i = t * p.top_k + min(s0 + g, p.top_k - 1);
            key[g] = __builtin_amdgcn_readfirstlane(bucket(p.ids[i], p.E) * p.numel + i);
            count[g] = 0;
        }
#pragma unroll 4
        for (int j0 = wave * 64; j0 < p.numel; j0 += 256) {
            const int j = j0 + lane;
            const int other = j < p.numel ? bucket(p.ids[j], p.E) * p.numel + j : INT32_MAX;
#pragma unroll
            for (int g = 0; g < G; g++) count[g] += __builtin_popcountll(__ballot(other < key[g]));
        }
        if (lane == 0)
#pragma unroll
            for (int g = 0; g < G; g++)
                if (s0 + g < p.top_k) lds[(s0 + g) * 4 + wave] = count[g];
    }
    __syncthreads();
    int *entry = lds + 4 * kMaxTopK;
    if (tid < p.top_k) {
        const int row = lds[tid * 4] + lds[tid * 4 + 1] + lds[tid * 4 + 2] + lds[tid * 4 + 3], i = t * p.top_k + tid;
        entry[tid] = (unsigned)p.ids[i] < (unsigned)p.E ? row : ~row;
        if (part == 0) p.row_of_slot[i] = entry[tid];
    }
    __syncthreads();
    auto at = [&](int s) { return entry[s]; };
    spread<A, 4>(p, t, part * 1024 + tid, 256, piece, part == 0 ? tid : p.scale_cols, 256, at);
}

// Many slots: histograms of segments, places, copies.  65536 slots: 5.0, 5.5 and, of 7168 codes, 93 us.
__global__ __launch_bounds__(256) void sort_hist_kernel(const SortParams p, int words, int seg)
{
    extern __shared__ int counts[];   // [words], 16 bits each
    for (int i = threadIdx.x; i < words; i += 256) counts[i] = 0;
    __syncthreads();
    const int lo = blockIdx.x * seg, hi = min(lo + seg, p.numel);
    for (int i = lo + (int)threadIdx.x; i < hi; i += 256) {
        const int e = bucket(p.ids[i], p.E);
        atomicAdd(&counts[e >> 1], 1 << (16 * (e & 1)));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < words; i += 256) p.hist[(size_t)blockIdx.x * words + i] = counts[i];
}

// One workgroup to a segment: it adds up the segments' histograms, all of them and those in front of its own, and places its slots (as the
// aligner does, so that equal experts stay in order without a sort of keys).  Adding them up in every workgroup instead of in a launch
// of its own saves a launch for n_seg * words * 4 bytes more from the L2.
template <bool FEW>
__global__ __launch_bounds__(1024) void sort_place_kernel(const SortParams p, int words, int seg, int id_bits, int n_waves)
{
    // [n_waves] tables of lane masks | [E + 1][n_waves] cursors (16 bit, whole 16 bytes) | [2 words] starts | [2 words] slots of
    // earlier segments | [16] the scan's sums
    extern __shared__ __attribute__((aligned(16))) uint8_t mem[];
    const int buckets = p.E + 1;
    lanes_t *masks = reinterpret_cast<lanes_t *>(mem);
    uint16_t *cursors = reinterpret_cast<uint16_t *>(masks + n_waves * kMasks);
    int *start = reinterpret_cast<int *>(mem + n_waves * kMasks * sizeof(lanes_t) + cursor_bytes(n_waves, buckets));
    int *before = start + 2 * words, *wave_sums = before + 2 * words;
    const int wave = threadIdx.x >> 6, n_seg = gridDim.x, mine = blockIdx.x;
    const int run = seg / n_waves;
    const int lo = mine * seg + wave * run, hi = wave < n_waves ? min(lo + run, p.numel) : lo;
    Chunks c;
    load_chunks<true>(p.ids, lo, hi, p.E, c);
    const int zero_quads = (int)(reinterpret_cast<uint8_t *>(wave_sums) - mem) / 16;
    for (int i = threadIdx.x; i < zero_quads; i += blockDim.x) reinterpret_cast<v4i *>(mem)[i] = (v4i){0, 0, 0, 0};
    masks += wave * kMasks;
    lds_barrier();
    const int share = words < 1024 ? 1024 / words : 1, part = words < 1024 ? (int)threadIdx.x / words : 0;   // threads of a column
    for (int col = (int)threadIdx.x - part * words; col < words && part < share; col += 1024) {
        int all[2] = {0, 0}, front[2] = {0, 0};
        for (int s0 = part; s0 < n_seg; s0 += 4 * share) {
            unsigned v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = (unsigned)p.hist[(size_t)min(s0 + k * share, n_seg - 1) * words + col];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int s = s0 + k * share;
                const unsigned w = s < n_seg ? v[k] : 0u, f = s < mine ? w : 0u;
                all[0] += (int)(w & 0xffffu), all[1] += (int)(w >> 16);
                front[0] += (int)(f & 0xffffu), front[1] += (int)(f >> 16);
            }
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            atomicAdd(&start[2 * col + k], all[k]);
            atomicAdd(&before[2 * col + k], front[k]);
        }
    }
    count_run<FEW, true>(p.ids, lo, hi, p.E, id_bits, masks, cursors, wave, n_waves, c);
    lds_barrier();
    for (int e = threadIdx.x; e < buckets; e += blockDim.x) prefix_over_waves(cursors, e, n_waves);
    (void)block_exclusive_scan(start, buckets, wave_sums);
    place_run<FEW, true>(p.ids, lo, hi, p.E, id_bits, masks, [&](int e) { return start[e] + before[e]; }, cursors, wave, n_waves, c,
                         [&](int at, int slot, int e) { p.row_of_slot[slot] = e < p.E ? at : ~at; });
    if (mine == 0)
        for (int e = threadIdx.x; e < buckets; e += blockDim.x) p.offsets[e] = start[e];
}

// A token's row to its slots' rows: U pieces a thread, which are read before the map's entries are there.  Rows shorter than a workgroup
// share one; with ONE token to a workgroup its entries come by scalar loads (8192 tokens of 7168 codes 125 us before, 104 with it and
// the stores above).
template <int A, int U, bool ONE>
__global__ __launch_bounds__(256) void spread_kernel(const SortParams p)
{
    const int t = ONE ? (int)blockIdx.x : (int)(blockIdx.x * blockDim.y + threadIdx.y);
    if (t >= p.M) return;
    const int32_t *map = p.row_of_slot + (int64_t)t * p.top_k;
    const int part = blockIdx.y, step = blockDim.x, first = part * U * step + (int)threadIdx.x;
    v4w piece[U];
    gather<A, U>(p, t, first, step, piece);
    spread<A, U>(p, t, first, step, piece, part == 0 ? (int)threadIdx.x : p.scale_cols, step, [&](int s) { return map[s]; });
}

// ---- combine -----------------------------------------------------------------------------------------------
struct CombineParams {
    const uint8_t *rows, *grad;
    const int32_t *map;
    const float *weights;
    uint8_t *out;            // sums, or the rows' gradients
    float *grad_weights;
    int64_t row_bytes, numel;
    float scaling;
    int M, top_k, pieces;
};

template <typename T>
struct Values;   // the values of 16 bytes
template <>
struct Values<uint16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float get(const v4w &v, int i)
    {
        return __builtin_bit_cast(float, i % 2 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
    }
    static __device__ __forceinline__ v4w put(const float (&f)[8])
    {
        return (v4w){pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    }
};
template <>
struct Values<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float get(const v4w &v, int i)
    {
        return __builtin_bit_cast(float, i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
    }
    static __device__ __forceinline__ v4w put(const float (&f)[4])
    {
        return (v4w){__builtin_bit_cast(uint32_t, f[0]), __builtin_bit_cast(uint32_t, f[1]), __builtin_bit_cast(uint32_t, f[2]),
                     __builtin_bit_cast(uint32_t, f[3])};
    }
};

// A thread to 16 bytes of a token's sum, up to eight rows in flight: rows are anywhere, so it is the loads in flight that carry it.
constexpr int kCombineInFlight = 8;
template <typename T, int A, bool ONE>
__global__ __launch_bounds__(256) void combine_kernel(const CombineParams p)
{
    constexpr int N = Values<T>::N;
    const int64_t t = ONE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int v = blockIdx.y * blockDim.x + threadIdx.x;
    if (t >= p.M || v >= p.pieces) return;
    const int32_t *map = p.map + t * p.top_k;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; i++) sum[i] = 0.f;
    for (int s0 = 0; s0 < p.top_k; s0 += kCombineInFlight) {
        v4w row[kCombineInFlight];
        float w[kCombineInFlight];
        bool on[kCombineInFlight];
#pragma unroll
        for (int j = 0; j < kCombineInFlight; j++) {
            const int m = s0 + j < p.top_k ? map[s0 + j] : -1;
            on[j] = m >= 0 && m < p.numel;
            if (on[j]) {
                row[j] = load_piece<A>(p.rows + (int64_t)m * p.row_bytes, v, p.row_bytes);
                w[j] = p.weights ? p.weights[t * p.top_k + s0 + j] : 1.f;
            }
        }
#pragma unroll
        for (int j = 0; j < kCombineInFlight; j++)
            if (on[j])
#pragma unroll
                for (int i = 0; i < N; i++) sum[i] = __builtin_fmaf(w[j], Values<T>::get(row[j], i), sum[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i++) sum[i] *= p.scaling;
    store_piece<A>(p.out + t * p.row_bytes, v, p.row_bytes, Values<T>::put(sum));
}

__device__ __forceinline__ float sum_of_wave(float v)   // in lane 63
{
#define SUM_STEP(ctrl, rows) \
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, false))
    SUM_STEP(0x111, 0xf);   // from 1, 2, 4, 8 lanes below in the row
    SUM_STEP(0x112, 0xf);
    SUM_STEP(0x114, 0xf);
    SUM_STEP(0x118, 0xf);
    SUM_STEP(0x142, 0xa);   // lane 15 of rows 0 and 2 to rows 1 and 3
    SUM_STEP(0x143, 0xc);   // lane 31 to rows 2 and 3
#undef SUM_STEP
    return v;
}

// A workgroup to a token.  Its gradient stays in registers where U pieces a thread hold it (U > 0), otherwise it is read once for each
// slot.  Both gradients in one pass: g times a weight goes out while g times the row is added up.
template <typename T, int A, int U>
__global__ __launch_bounds__(256) void combine_grad_kernel(const CombineParams p)
{
    constexpr int N = Values<T>::N, P = U > 0 ? U : 2;
    extern __shared__ float dots[];   // [top_k][wavefronts]
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, step = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = step >> 6;
    const int32_t *map = p.map + t * p.top_k;
    const uint8_t *grad = p.grad + t * p.row_bytes;
    v4w g[P];
    auto load_grad = [&](int v0) {
#pragma unroll
        for (int u = 0; u < P; u++) {
            const int v = v0 + u * step;
            g[u] = v < p.pieces ? load_piece<A>(grad, v, p.row_bytes) : (v4w){0, 0, 0, 0};
        }
    };
    if constexpr (U > 0) load_grad(tid);
    for (int s = 0; s < p.top_k; s++) {
        const int m = map[s];
        const int64_t row = m < 0 ? ~m : m;
        const bool there = row < p.numel, on = m >= 0 && there;
        float w = on ? (p.weights ? p.weights[t * p.top_k + s] : 1.f) * p.scaling : 0.f;
        float dot = 0.f;
        for (int v0 = tid; v0 < p.pieces; v0 += P * step) {
            if constexpr (U == 0) load_grad(v0);
            v4w y[P];
#pragma unroll
            for (int u = 0; u < P; u++)
                if (p.grad_weights && on && v0 + u * step < p.pieces) y[u] = load_piece<A>(p.rows + row * p.row_bytes, v0 + u * step, p.row_bytes);
#pragma unroll
            for (int u = 0; u < P; u++) {
                const int v = v0 + u * step;
                if (v >= p.pieces) break;
                float f[N];
#pragma unroll
                for (int i = 0; i < N; i++) f[i] = Values<T>::get(g[u], i);
                if (p.grad_weights && on)
#pragma unroll
                    for (int i = 0; i < N; i++) dot = __builtin_fmaf(f[i], Values<T>::get(y[u], i), dot);
                if (p.out && there) {
#pragma unroll
                    for (int i = 0; i < N; i++) f[i] *= w;
                    store_piece<A>(p.out + row * p.row_bytes, v, p.row_bytes, on ? Values<T>::put(f) : (v4w){0, 0, 0, 0});
                }
            }
        }
        if (p.grad_weights) {
            dot = sum_of_wave(dot);
            if (lane == 63) dots[s * waves + wave] = on ? dot : 0.f;
        }
    }
    if (!p.grad_weights) return;
    __syncthreads();
    for (int s = tid; s < p.top_k; s += step) {
        float sum = dots[s * waves];
        for (int w = 1; w < waves; w++) sum += dots[s * waves + w];
        p.grad_weights[t * p.top_k + s] = sum * p.scaling;
    }
}

// ---- launches ----------------------------------------------------------------------------------------------
constexpr int kSortSeg = 1024, kSortMaxSeg = 512;
constexpr size_t kDefaultLds = 64 << 10;   // dynamic LDS a kernel may have without a word

struct Segments {
    int seg, n, words;
    Segments(int numel, int E) : seg(kSortSeg)
    {
        while (seg < (32 << 10) && (numel - 1) / seg >= kSortMaxSeg) seg *= 2;   // (counts and cursors are 16 bits wide)
        n = (numel - 1) / seg + 1;
        words = (E + 2) / 2;
    }
};

int status(hipError_t err) { return err == hipSuccess ? ALPHA_MOE_OK : ALPHA_MOE_ERR_LAUNCH; }

template <typename... Args>
hipError_t launch(void (*kernel)(Args...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, Args... args)
{
    void *list[] = {&args...};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, list, lds, stream);
}

// Threads along a row of `pieces` 16-byte pieces, U pieces each: a power of two up to 256.
int threads_along(int pieces, int U)
{
    int n = 8;
    while (n < 256 && n * U < pieces) n *= 2;
    return n;
}

// Whether the workgroups find their slots' rows by themselves: every wavefront looks at a quarter of the slots for each eight of its token's.
// MI355X, us, so / in three launches: 2048 rows of 2048 bf16 6.5 / 10.7, 5120 10.4 / 11.4, 6144 12.1 / 12.3, 7200 14.4 / 13.3; a token of
// 61 with 9 rows of 7168 codes 7.0 / 11.5; 8000 rows of 4000 tokens 30 / 9.5, 8192 rows of 128 tokens 73 / 23.
bool sort_few(int64_t M, int64_t top_k)
{
    const int64_t looks = (top_k + 7) / 8 * M * top_k;
    return looks <= 6400 && looks * M <= 5000000;
}

template <int A>
int sort_rows(SortParams p, int id_bits, hipStream_t hs)
{
    if (sort_few(p.M, p.top_k))
        return status(launch(sort_few_kernel<A>, dim3(p.M + 1, (p.pieces + 1023) / 1024), dim3(256), 0, hs, p));
    const Segments g(p.numel, p.E);
    hipError_t err = launch(sort_hist_kernel, dim3(g.n), dim3(256), g.words * sizeof(int), hs, p, g.words, g.seg);
    if (err != hipSuccess) return status(err);
    int n_waves = 16;
    auto lds_of = [&](int waves) {
        return waves * kMasks * sizeof(lanes_t) + cursor_bytes(waves, p.E + 1) + (4 * g.words + 16) * sizeof(int);
    };
    while (n_waves > 2 && lds_of(n_waves) > kDefaultLds) n_waves /= 2;
    const bool few = id_bits <= 7;
    err = launch(few ? sort_place_kernel<true> : sort_place_kernel<false>, dim3(g.n), dim3(1024), lds_of(n_waves), hs, p, g.words,
                 g.seg, id_bits, n_waves);
    if (err != hipSuccess) return status(err);
    const int U = p.pieces <= 256 ? 1 : p.pieces <= 512 ? 2 : 4, along = threads_along(p.pieces, U), tokens = 256 / along;
    const dim3 grid((p.M + tokens - 1) / tokens, (p.pieces + along * U - 1) / (along * U)), block(along, tokens);
    const auto kernel = tokens > 1 ? spread_kernel<A, 1, false> : U == 1 ? spread_kernel<A, 1, true>
                      : U == 2   ? spread_kernel<A, 2, true> : spread_kernel<A, 4, true>;
    err = launch(kernel, grid, block, 0, hs, p);
    return status(err);
}

template <typename T, int A>
int combine_rows(const CombineParams &p, hipStream_t hs)
{
    const int along = threads_along(p.pieces, 1), tokens = 256 / along;
    return status(launch(tokens == 1 ? combine_kernel<T, A, true> : combine_kernel<T, A, false>,
                         dim3((p.M + tokens - 1) / tokens, (p.pieces + along - 1) / along), dim3(along, tokens), 0, hs, p));
}

template <typename T, int A>
int combine_rows_grad(const CombineParams &p, hipStream_t hs)
{
    const int along = threads_along(p.pieces, 1), threads = along < 64 ? 64 : along;
    const size_t lds = p.top_k * (threads / 64) * sizeof(float);
    const int each = (p.pieces + threads - 1) / threads;
    const auto kernel = each <= 1 ? combine_grad_kernel<T, A, 1> : each <= 2 ? combine_grad_kernel<T, A, 2>
                      : each <= 4 ? combine_grad_kernel<T, A, 4> : combine_grad_kernel<T, A, 0>;
    return status(launch(kernel, dim3(p.M), dim3(threads), lds, hs, p));
}

// The largest power of two up to 16 that rows of `row_bytes` bytes of all these tensors start at multiples of.
template <typename... Ptr>
int alignment(int64_t row_bytes, Ptr... tensors)
{
    const uintptr_t all = (uintptr_t)row_bytes | (reinterpret_cast<uintptr_t>(tensors) | ...) | 16;
    return (int)(all & (~all + 1));
}

// Sizes that all calls share: M tokens of top_k slots, rows of K values of 1, 2 or 4 bytes.  A launch has less than 2^32 threads and
// a row at most 65535 pieces of 4 KiB.
bool sizes_fit(int M, int top_k, int K, int value_bytes)
{
    return M >= 0 && top_k > 0 && top_k <= kMaxTopK && K > 0 && M < (1 << 24) - 1 && (int64_t)M * top_k <= INT32_MAX &&
           (int64_t)K * value_bytes <= ((int64_t)1 << 27);
}

}  // namespace
}  // namespace alpha_moe

using namespace alpha_moe;

extern "C" size_t alpha_moe_sort_workspace_bytes(int M, int top_k, int num_experts)
{
    if (!sizes_fit(M, top_k, 1, 1) || num_experts <= 0 || sort_few(M, top_k)) return 0;
    const Segments g(M * top_k, num_experts);
    return (size_t)g.n * g.words * sizeof(int);
}

extern "C" int alpha_moe_sort_tokens(const void *x, int value_bytes, const float *x_scale, const int32_t *topk_ids, void *rows,
                                     float *scale, int32_t *offsets, int32_t *row_of_slot, int M, int K, int top_k, int num_experts,
                                     void *workspace, size_t workspace_bytes, void *stream)
{
    if ((value_bytes != 1 && value_bytes != 2 && value_bytes != 4) || !sizes_fit(M, top_k, K, value_bytes) || num_experts <= 0 ||
        num_experts > kSortMaxExperts || (value_bytes == 1 && K % 128 != 0))
        return ALPHA_MOE_ERR_SHAPE;
    if (!offsets || (M > 0 && (!x || !topk_ids || !rows || !row_of_slot)) || (!x_scale) != (!scale)) return ALPHA_MOE_ERR_NULL_POINTER;
    if (x_scale && value_bytes != 1) return ALPHA_MOE_ERR_SHAPE;
    const int starts = alignment((int64_t)K * value_bytes, x, rows);
    if (starts < (value_bytes == 1 ? 16 : value_bytes)) return ALPHA_MOE_ERR_ALIGNMENT;
    SortParams p = {};
    p.x = static_cast<const uint8_t *>(x), p.x_scale = x_scale, p.ids = topk_ids;
    p.rows = static_cast<uint8_t *>(rows), p.scale = scale, p.offsets = offsets, p.row_of_slot = row_of_slot;
    p.hist = static_cast<int *>(workspace);
    p.row_bytes = (int64_t)K * value_bytes;
    p.pieces = (int)((p.row_bytes + 15) / 16);
    p.scale_cols = x_scale ? K / 128 : 0;
    p.M = M, p.top_k = top_k, p.E = num_experts, p.numel = M * top_k;
    const size_t need = alpha_moe_sort_workspace_bytes(M, top_k, num_experts);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0))
        return ALPHA_MOE_ERR_WORKSPACE;
    int id_bits = 0;
    while ((1 << id_bits) < num_experts + 1) id_bits++;
    hipStream_t hs = static_cast<hipStream_t>(stream);
    return starts == 16 ? sort_rows<16>(p, id_bits, hs) : sort_rows<2>(p, id_bits, hs);
}

extern "C" int alpha_moe_combine_tokens(const void *rows, int is_f32, const int32_t *row_of_slot, const float *topk_weights, void *out,
                                        int M, int K, int top_k, float scaling_factor, void *stream)
{
    const int size = is_f32 ? 4 : 2;
    if (!sizes_fit(M, top_k, K, size)) return ALPHA_MOE_ERR_SHAPE;
    if (M == 0) return ALPHA_MOE_OK;
    if (!rows || !row_of_slot || !out) return ALPHA_MOE_ERR_NULL_POINTER;
    const int starts = alignment((int64_t)K * size, rows, out);
    if (starts < size) return ALPHA_MOE_ERR_ALIGNMENT;
    CombineParams p = {};
    p.rows = static_cast<const uint8_t *>(rows), p.map = row_of_slot, p.weights = topk_weights, p.out = static_cast<uint8_t *>(out);
    p.row_bytes = (int64_t)K * size, p.numel = (int64_t)M * top_k, p.pieces = (int)((p.row_bytes + 15) / 16);
    p.scaling = scaling_factor, p.M = M, p.top_k = top_k;
    hipStream_t hs = static_cast<hipStream_t>(stream);
    const bool whole = starts == 16;
    if (is_f32) return whole ? combine_rows<float, 16>(p, hs) : combine_rows<float, 2>(p, hs);
    return whole ? combine_rows<uint16_t, 16>(p, hs) : combine_rows<uint16_t, 2>(p, hs);
}

extern "C" int alpha_moe_combine_tokens_grad(const void *grad, const void *rows, int is_f32, const int32_t *row_of_slot,
                                             const float *topk_weights, void *grad_rows, float *grad_weights, int M, int K, int top_k,
                                             float scaling_factor, void *stream)
{
    const int size = is_f32 ? 4 : 2;
    if (!sizes_fit(M, top_k, K, size)) return ALPHA_MOE_ERR_SHAPE;
    if (M == 0 || (!grad_rows && !grad_weights)) return ALPHA_MOE_OK;
    if (!grad || !row_of_slot || (grad_weights && !rows)) return ALPHA_MOE_ERR_NULL_POINTER;
    const int starts = alignment((int64_t)K * size, rows, grad, grad_rows);
    if (starts < size) return ALPHA_MOE_ERR_ALIGNMENT;
    CombineParams p = {};
    p.rows = static_cast<const uint8_t *>(rows), p.grad = static_cast<const uint8_t *>(grad), p.map = row_of_slot;
    p.weights = topk_weights, p.out = static_cast<uint8_t *>(grad_rows), p.grad_weights = grad_weights;
    p.row_bytes = (int64_t)K * size, p.numel = (int64_t)M * top_k, p.pieces = (int)((p.row_bytes + 15) / 16);
    p.scaling = scaling_factor, p.M = M, p.top_k = top_k;
    hipStream_t hs = static_cast<hipStream_t>(stream);
    const bool whole = starts == 16;
    if (is_f32) return whole ? combine_rows_grad<float, 16>(p, hs) : combine_rows_grad<float, 2>(p, hs);
    return whole ? combine_rows_grad<uint16_t, 16>(p, hs) : combine_rows_grad<uint16_t, 2>(p, hs);
}
