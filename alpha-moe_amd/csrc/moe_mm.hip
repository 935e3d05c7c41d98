// The block-scaled FP8 product of dense layers: out[m, n] = sum over K blocks kb of 128 of
//   x_scale[m, kb] * w_scale[n / 128, kb] * (sum over k in kb of x[m, k] w[n, k]),
// rounded once, to bf16.  A block's sum is the matrix core's, the blocks' sums are added up in fp32.  The two scales are multiplied
// first, in fp32 (one product for four results; the scales one after the other onto the results would be four more instructions for each
// matrix instruction): what overflows there is infinite, or NaN, even where the block's sum is small or 0.
//
// What the matrix core's FP8 sum is good for (MI355X, pairs of products of known sizes): of each eight products along K it keeps
// the bits down to 2^-13 of the largest one's power of two, and adds the eights up in fp32.  On normally distributed operands the
// result is 1.5e-5 off, relatively (2-norm), which a bf16 result's own 1.7e-3 covers and a fp32 result would not: there is none.
//
// Both kernels use the conventions of moe_common.hpp (weight rows are the A operand, tokens the B operand, one instruction
// contracts one block of K) and bring everything to LDS with direct loads of whole 128-byte lines.  A matrix result is scaled into
// its fp32 accumulator by four multiply-adds, which run beside the next matrix instruction (MI355X: 14.8 ns for the
// instruction with them, 14.2 without).
//
//   mm_stream_kernel   few tokens: weights are what is read, and how many bytes are in flight is what counts
//   mm_tile_kernel     many tokens: matrix cores, and the path into a compute unit (a tile's rows of both operands per K block)
//
// plan() chooses between them and their tiles.
#include <type_traits>
#include <utility>

#include "moe_common.hpp"

namespace alpha_moe {
namespace {

struct MmParams {
    const uint8_t *x;
    const float *x_scale;
    const uint8_t *w;
    const float *w_scale;
    uint16_t *out;
    int M, N, K, nkb;
    int row_groups, token_groups;   // tiles of the launch
    int quads;   // 1: there are four K blocks, whose scales of a token are loaded together
};

__device__ __forceinline__ int rfl(int v) { return __builtin_amdgcn_readfirstlane(v); }

// f(0), f(1), ..., f(N - 1) with compile-time numbers
template <typename F, int... I>
__device__ __forceinline__ void for_each_of(F &&f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each(F &&f)
{
    for_each_of(f, std::make_integer_sequence<int, N>{});
}

// A buffer at a wavefront-uniform base, of no end (bytes = -1) or empty (0: its loads give zeros).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *uniform_base, int bytes)
{
    const uint64_t v = reinterpret_cast<uint64_t>(uniform_base);
    const uint64_t u = ((uint64_t)(uint32_t)rfl((int)(uint32_t)(v >> 32)) << 32) | (uint32_t)rfl((int)(uint32_t)v);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), 0, rfl(bytes), 0x00020000);
}

// Direct-to-LDS loads of 16 and 4 bytes per lane from (wavefront-uniform base) + (per-lane offset) + (uniform offset).
template <int AUX>
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t base, unsigned voff, unsigned soff, void *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lptr_t)(uint32_t)(uintptr_t)lds, 16, (int)voff, (int)soff, 0, AUX);
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t base, unsigned voff, unsigned soff, void *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lptr_t)(uint32_t)(uintptr_t)lds, 4, (int)voff, (int)soff, 0, 0);
}
typedef const v4i __attribute__((address_space(3))) * lds_v4i;
typedef const float __attribute__((address_space(3))) * lds_f32;
__device__ __forceinline__ lds_v4i lds_tile(const void *p) { return (lds_v4i)(uint32_t)(uintptr_t)p; }   // [128 * tile]
__device__ __forceinline__ v4i lds_read(const void *p) { return *lds_tile(p); }
__device__ __forceinline__ float lds_float(const void *p) { return *(lds_f32)(uint32_t)(uintptr_t)p; }

// The scales of a tile's tokens in LDS, loaded four K blocks at a time if there are four (one by one, every scale is a line of its own
// on the path into the compute unit, half as many again as the data is; 8192 x 4096 x 7168 221 us, by fours 207, x 7296 229 and 220, 2048 x
// 4096 x 7168 57.0 and 56.0): two places of [token][four K blocks], or eight of [token].
struct TokenScales {
    int quads, tokens, last;   // last: the K block at which the last four of a row begin (which a row's last load takes, so that it ends with
                               // the row; a load of 16 bytes may start at any multiple of four)
    __device__ __forceinline__ bool loads(int kb, bool first) const { return !quads || first || (kb & 3) == 0; }
    __device__ __forceinline__ int begin(int kb) const { return (kb & ~3) < last ? kb & ~3 : last; }   // of the four with kb
    __device__ __forceinline__ int place(int kb) const
    {
        return quads ? ((kb >> 2) & 1) * tokens * 16 + (kb - begin(kb)) * 4 : (kb & 7) * tokens * 4;
    }
    __device__ __forceinline__ int stride() const { return quads ? 16 : 4; }   // from token to token
    // lanes [0, count) load the scales of as many tokens, from `token` on, that K block kb is the first to ask for
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t base, unsigned offset, int kb, int token, bool mine, uint8_t *area) const
    {
        if (quads) {
            if (mine) dma16<0>(base, offset, 4u * (unsigned)begin(kb), area + ((kb >> 2) & 1) * tokens * 16 + token * 16);
        } else {
            if (mine) dma4(base, offset, 4u * (unsigned)kb, area + place(kb) + token * 4);
        }
    }
};

// Results at any multiple of their two bytes: a row of an odd N starts at one.  (Memory takes stores of 8 and 16 bytes there as a whole;
// value by value 8192 x 4095 x 1024 takes 124 us, so 62; 4094 columns 128 and 48, 4096 43.)
typedef uint32_t any2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));

// Columns n .. n + 3 of row m; what is behind the last row or column is not there.
__device__ __forceinline__ void store4(const MmParams &p, int m, int n, v4f v)
{
    if (m >= p.M || n >= p.N) return;
    uint16_t *at = p.out + (size_t)m * p.N + n;
    const any2 two = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    if (n + 3 < p.N) {
        *reinterpret_cast<any2 *>(at) = two;
    } else {
        at[0] = (uint16_t)two[0];
        if (n + 1 < p.N) at[1] = (uint16_t)(two[0] >> 16);
        if (n + 2 < p.N) at[2] = (uint16_t)two[1];
    }
}

// Few tokens: a workgroup multiplies R * 16 rows of w with T * 16 tokens, its wavefronts taking K blocks in turn, each through a
// ring of its own in LDS (D K blocks of weights, tokens and scales), so that nobody waits for anybody until the sums over the
// wavefronts at the end.  HALF: at most eight tokens, whose second eight places in a tile are left as they are - a matrix
// column's result depends on its own token alone, and theirs are not stored.
//
// What bounds it: the weights' way from memory at few tokens, the path into a compute unit (128 bytes times rows plus tokens per K
// block, 70 - 100 GB/s) from some thirty on.  MI355X, back to back: 1 x 4096 x 7168 (29 MB) 6.0 us, of which 2.5 are an
// empty call's, 61 x 2112 x 7168 8.3, 64 x 7168 x 2048 6.0, 256 x 4096 x 7168 15.  The contraction split over workgroups with a
// second launch for the partial sums costs 3 - 4 us, more than the idle compute units it fills (61 x 2112 x 7168 in seven parts 11.6 us);
// split within one launch, the last workgroup adding up, has not been tried.
// Why through LDS, though no wavefront reads what another has loaded: a load into a matrix operand's registers takes 64 bytes of sixteen
// lines, and lines are what the path counts (61 x 2112 x 7168 so 15.4 us, 1 x 4096 x 7168 7.8).
// Weights are loaded non-temporally only with at most eight tokens, where they are read once and there is little else to read
// (1 x 4096 x 7168 from HBM 7.1 us against 7.6, 3 x 1280 x 5120 4.7 and 5.0; but 61 x 2112 x 7168 11.9 and 8.3.  A loop over one small
// matrix would rather keep it in L2, 3 x 1280 x 5120 4.7 and 3.4 us; a model's layers come back after all the others).
// Deeper rings change nothing (16 x 4096 x 7168 with two, four K blocks 7.0, 7.05 us).  Eight wavefronts where a tile is 16 x 16 or
// the tokens are few, four for larger ones, of which two fit a compute unit (17 x 4096 x 7168, 32 x 16 tile, eight 7.7, four 6.9 us; 32 x
// 4096 x 7168 7.4, 7.1; 32 x 32 tile 61 x 2112 x 7168 8.7, 8.4; 16 x 16 tile, 16 x 4096 x 7168, 6.8 with eight).
template <int R, int T, int WAVES, int D, bool HALF>
struct StreamRing {
    static constexpr bool kRun = T >= 4;   // the tokens' scales four K blocks at a time
    static constexpr int kSlot = (R + T) * 2048 + (kRun ? 0 : 256);
    static constexpr int kScales = 4 * (kMaxKBlocks / WAVES);   // bytes: the weights' scales of a wavefront's K blocks
    static constexpr int kData = 2 * R + (HALF ? 1 : 2 * T), kLoads = kData + 1;   // loads of a slot without, with tokens' scales
    static constexpr int kWave = D * kSlot + kScales + (kRun ? T * 512 : 0);
    static constexpr bool kSpread = R * T <= 8;   // the refill's loads between the matrix instructions, or in front of them
    static constexpr int kSums = WAVES * R * T * 1024;              // the sums at the end take the rings' place
    static constexpr int kBytes = WAVES * kWave > kSums ? WAVES * kWave : kSums;
    static_assert(kBytes <= 160 * 1024, "");
};

template <int R, int T, int WAVES, int D, bool HALF>
__global__ __launch_bounds__(WAVES * 64) void mm_stream_kernel(const MmParams p)
{
    typedef StreamRing<R, T, WAVES, D, HALF> Ring;
    constexpr int L = Ring::kLoads, DATA = Ring::kData;
    __shared__ __attribute__((aligned(128))) uint8_t lds[Ring::kBytes];
    const int tid = threadIdx.x, lane = tid & 63, w = rfl(tid >> 6);
    const int n = lane & 15, q = lane >> 4;

    // workgroups are dealt to the eight XCDs in turn: each gets a run of tiles, token groups of one row group next to each other
    const int tiles = p.row_groups * p.token_groups, run = (tiles + 7) >> 3;
    const int tile = (int)(blockIdx.x & 7) * run + (int)(blockIdx.x >> 3);
    if (tile >= tiles) return;
    const int rg = tile / p.token_groups, tg = tile - rg * p.token_groups;
    const int c0 = rg * (R * 16), m0 = tg * (T * 16);
    const int K = p.K, nkb = p.nkb;
    // This wavefront's K blocks: every WAVES-th one, so that a workgroup reads on along its rows; with four tiles of tokens a run of
    // them, for the sake of the tokens' scales.  61 tokens, 2112 columns, K = 7168: with four tiles 14.4 us as a run against 16.5 in turn,
    // with two of 32 columns 8.7 against 8.3; one token, 4096 columns: 6.2 against 6.0.
    constexpr bool RUN = Ring::kRun;
    constexpr int STEP = RUN ? 1 : WAVES;
    const int first = RUN ? w * nkb / WAVES : w;
    const int count = RUN ? (w + 1) * nkb / WAVES - first : w < nkb ? (nkb - w + WAVES - 1) / WAVES : 0;

    const __amdgpu_buffer_rsrc_t wbuf = agent_buffer(p.w + (size_t)c0 * K);
    const __amdgpu_buffer_rsrc_t xbuf = agent_buffer(p.x + (size_t)m0 * K);
    const __amdgpu_buffer_rsrc_t xsbuf = agent_buffer(p.x_scale + (size_t)m0 * nkb);
    const __amdgpu_buffer_rsrc_t wsbuf = agent_buffer(p.w_scale + (size_t)(c0 >> 7) * nkb);
    // load h of a tile: lane l fills position l & 7 of row 8 h + l / 8.  Matrix row r of weight tile k is column
    // 4 R (r / 4) + 4 k + r % 4: a lane's results of all tiles are 4 R adjacent columns.  Rows behind the last: the last.
    const int ld_row = lane >> 3;
    unsigned w_off[R][2], x_off[T][2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = 8 * h + ld_row;
        const unsigned chunk = 16u * ((lane & 7) ^ ((r >> 1) & 7));
#pragma unroll
        for (int k = 0; k < R; k++) {
            int c = 4 * R * (r >> 2) + 4 * k + (r & 3);
            c = c0 + c < p.N ? c : p.N - 1 - c0;
            w_off[k][h] = (unsigned)c * (unsigned)K + chunk;
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
            int m = 16 * t + r;
            m = m0 + m < p.M ? m : p.M - 1 - m0;
            x_off[t][h] = (unsigned)m * (unsigned)K + chunk;
        }
    }
    const unsigned xs_off = 4u * (unsigned)((m0 + lane < p.M ? lane : p.M - 1 - m0) * nkb);

    uint8_t *ring = lds + w * Ring::kWave;
    uint8_t *ws = ring + D * Ring::kSlot, *xs = ws + Ring::kScales;
    const TokenScales scales = {p.quads, T * 16, nkb - 4};   // (RUN)
    for (int c = 0; c < count; c += 64)
        if (c + lane < count) dma4(wsbuf, 4u * (unsigned)(first + (c + lane) * STEP), 0u, ws + 4 * c);
    // Load j of a slot for the i-th of this wavefront's K blocks: weights and tokens, the tokens' scales between them, or in front of
    // both where there are not always any.
    auto issue = [&](int slot, int i, auto jc) {
        constexpr int at_scales = RUN ? 0 : 2 * R, at_j = decltype(jc)::value;
        constexpr int j = at_j == at_scales ? -1 : at_j > at_scales ? at_j - 1 : at_j, tj = j - 2 * R;
        const int kb = first + i * STEP;
        uint8_t *at = ring + slot * Ring::kSlot;
        if constexpr (j < 0) {
            if (!RUN && lane < T * 16) dma4(xsbuf, xs_off, 4u * (unsigned)kb, at + (R + T) * 2048);
            if (RUN && scales.loads(kb, i == 0)) scales.load(xsbuf, xs_off, kb, 0, lane < T * 16, xs);
        } else if constexpr (j < 2 * R) {
            dma16<HALF ? 2 : 0>(wbuf, w_off[j / 2][j % 2], 128u * kb, at + j * 1024);
        } else {
            constexpr int t = HALF ? tj : tj / 2, h = HALF ? 0 : tj % 2;
            dma16<0>(xbuf, x_off[t][h], 128u * kb, at + (R + t) * 2048 + h * 1024);
        }
    };
#pragma unroll
    for (int i = 0; i < D; i++)
        if (i < count) for_each<L>([&](auto j) { issue(i, i, j); });

    const int f_n = (n >> 1) & 7;
    const int frag_lo = n * 128 + 16 * (q ^ f_n), frag_hi = n * 128 + 16 * ((q ^ f_n) ^ 4);
    v4f acc[R][T] = {};
    int slot = 0;
    for (int i = 0; i < count; i++) {
        // of what was issued behind this K block, all may still be on its way (with a run, at least the data)
        static_assert(D <= 2, "the last K blocks are waited for as if there were nothing behind them");
        if (i + D <= count) wait_vmcnt<(RUN ? DATA : L) * (D - 1)>();
        else wait_vmcnt<0>();
        const uint8_t *at = ring + slot * Ring::kSlot;
        const uint8_t *my_xs = RUN ? xs + scales.place(first + i) : at + (R + T) * 2048;
        const int xs_token = RUN ? scales.stride() : 4;
        v8i a[R], b[T];
        float f[T];
#pragma unroll
        for (int k = 0; k < R; k++) a[k] = cat(lds_read(at + k * 2048 + frag_lo), lds_read(at + k * 2048 + frag_hi));
#pragma unroll
        for (int t = 0; t < T; t++) {
            b[t] = cat(lds_read(at + (R + t) * 2048 + frag_lo), lds_read(at + (R + t) * 2048 + frag_hi));
            f[t] = lds_float(my_xs + xs_token * (16 * t + n));
        }
        const float sc = lds_float(ws + 4 * i);
#pragma unroll
        for (int k = 0; k < R; k++) asm volatile("" : "+v"(a[k]));
#pragma unroll
        for (int t = 0; t < T; t++) asm volatile("" : "+v"(b[t]), "+v"(f[t]));
        wait_lds_reads();
        // the slot is refilled between the matrix instructions: handed out in a burst, the loads of four wavefronts keep the path
        // into the compute unit busy for longer than the matrix instructions behind them take
        auto multiply = [&](auto refill) {
            for_each<T>([&](auto tc) {
                constexpr int t = decltype(tc)::value;
                const float by = f[t] * sc;
                for_each<R>([&](auto kc) {
                    constexpr int k = decltype(kc)::value, o = t * R + k;
                    const v4f prod = mfma_fp8(a[k], b[t]);
                    if constexpr (decltype(refill)::value) {
                        __builtin_amdgcn_sched_barrier(0);
                        for_each<L>([&](auto j) {
                            if constexpr (decltype(j)::value * (R * T) / L == o) issue(slot, i + D, j);
                        });
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    acc[k][t] += prod * by;
                });
            });
        };
        if (i + D < count && !Ring::kSpread) for_each<L>([&](auto j) { issue(slot, i + D, j); });
        if (i + D < count && Ring::kSpread) multiply(std::true_type{});
        else multiply(std::false_type{});
        slot = slot + 1 < D ? slot + 1 : 0;
    }

    // sums over the wavefronts, in their order
    __syncthreads();
    v4f *sums = reinterpret_cast<v4f *>(lds);
#pragma unroll
    for (int k = 0; k < R; k++)
#pragma unroll
        for (int t = 0; t < T; t++) sums[((w * T + t) * R + k) * 64 + lane] = acc[k][t];
    __syncthreads();
    for (int e = tid; e < R * T * 64; e += WAVES * 64) {
        v4f sum = sums[e];
#pragma unroll
        for (int o = 1; o < WAVES; o++) sum += sums[o * R * T * 64 + e];
        const int l = e & 63, k = (e >> 6) % R, t = (e >> 6) / R;
        store4(p, m0 + 16 * t + (l & 15), c0 + 4 * R * (l >> 4) + 4 * k, sum);
    }
}

int64_t tiles_of(int M, int N, int cols, int tokens)
{
    return (int64_t)((N + cols - 1) / cols) * ((M + tokens - 1) / tokens);
}

// A launch has less than 2^32 threads.
bool grid_fits(int64_t tiles, int threads) { return (tiles + 7) * threads < (int64_t(1) << 32); }

template <int R, int T, int WAVES, int D, bool HALF>
hipError_t launch_stream_mm(MmParams p, hipStream_t stream)
{
    if (!grid_fits(tiles_of(p.M, p.N, R * 16, T * 16), WAVES * 64)) return hipErrorInvalidConfiguration;
    p.row_groups = (p.N + R * 16 - 1) / (R * 16);
    p.token_groups = (p.M + T * 16 - 1) / (T * 16);
    const int run = (p.row_groups * p.token_groups + 7) / 8;
    void *args[] = {&p};
    return hipLaunchKernel(reinterpret_cast<const void *>(mm_stream_kernel<R, T, WAVES, D, HALF>), dim3((unsigned)run * 8),
                           dim3(WAVES * 64), args, 0, stream);
}

// Many tokens: WN x WM wavefronts, each with TN * 16 columns x TM * 16 tokens of a workgroup's tile, through S stages of one K
// block in LDS.
//
// One barrier to a K block, in front of the last token tile's pass: by then all fragments of the stage are in registers, so the stage
// behind the barrier can be refilled at once and has nearly S - 1 K blocks of time for it, and the pass replaces each weight
// fragment by the next K block's as it is used for the last time, so the next K block starts without a wait.
//
// The loads: a wavefront that hands loads to the path into the compute unit (four cycles for a line of 128 bytes) waits for it, and its
// matrix instructions with it.  Where registers allow, LOADERS more wavefronts do nothing but load (128 x 128 tile, 1024 x 4096 x 7168 43.5 ->
// 35.8 us, 128 x 64, 256 x 7168 x 2048 9.9 -> 9.3).  The 256 x 256 tile has no registers left for them: there the loads of a stage go
// out one by one between matrix instructions, over the first three eighths of a K block (8192 x 4096 x 7168 in a burst 226, over three
// eighths 221, over all of it 231; with the tokens' scales four K blocks at a time then 207).
//
// What bounds it: up to 256 x 128 the path into a compute unit, which takes four cycles for a line of 128 bytes (128 x 64 tile 0.38 us a
// K block of 192 lines, 128 x 128 0.50, 256 x 128 0.70).  In the largest tile matrix instructions and their scaling multiply-adds
// (19.3 ns a pair on random operands, where the clock gives way: 138 us for 8192 x 4096 x 7168; on equal operands 14.8), and LDS,
// which takes loads in at 64 bytes a cycle while fragments are read from it (without any loads the same kernel takes 137 us).
// MI355X: 8192 x 4096 x 7168 207 - 217 us by card (2.2 - 2.3 PFLOP/s; a library product of the same size without block scales 188),
// 4096 x 4096 x 7168 99, 1024 x 7168 x 2048 18.7, 256 x 7168 x 2048 9.4.  Also tried, against 221: 128 columns x 64 tokens a wavefront
// 237; token fragments read two passes ahead 228; all fragments read behind the barrier 239; against 213: weights loaded a K block
// further ahead, behind a barrier of their own, so that loads go out over all of a K block, 214.
template <int TN, int TM, int WN, int WM, int S, int LOADERS>
struct Tile {
    static constexpr int kWaves = WN * WM, kLoaders = LOADERS > 0 ? LOADERS : kWaves, kCols = TN * 16 * WN, kTokens = TM * 16 * WM;
    static constexpr int kStage = (kCols + kTokens) * 128;
    static constexpr int kScaleRows = (kCols + 127) / 128;   // a tile starts at a multiple of its columns
    static constexpr int kBytes = S * kStage + kTokens * 32 + kScaleRows * kMaxKBlocks * 4;
    static constexpr int kW = kCols / 8 / kLoaders, kX = kTokens / 8 / kLoaders;   // 1 KiB pieces a loading wavefront has per stage
    static constexpr int kData = kW + kX, kLoads = kData + 1;   // of a wavefront and stage, the first: its share of the tokens' scales, if any
    static constexpr int kScaleLanes = kTokens / kLoaders;
    // Piece j of a stage is issued behind matrix instruction at(j) of the TN * TM that follow the barrier which frees its place.
    static constexpr int at(int j) { return j * (S == 2 ? TN * TM * 3 / 8 : TN * TM) / kLoads; }
    static constexpr int early() { int c = 0; while (c < kLoads && at(c) < TN) c++; return c; }   // those in the first TN
    static_assert(kCols % (8 * kLoaders) == 0 && kTokens % (8 * kLoaders) == 0 && kScaleLanes <= 64 && S <= 4 && kBytes <= 160 * 1024, "");
    static_assert(kCols >= 128 ? (TN * 16) <= 128 : 128 % kCols == 0, "a wavefront's columns share their scales");
};

template <int TN, int TM, int WN, int WM, int S, int LOADERS>
__global__ __launch_bounds__((WN * WM + LOADERS) * 64, 2) void mm_tile_kernel(const MmParams p)
{
    typedef Tile<TN, TM, WN, WM, S, LOADERS> T;
    __shared__ __attribute__((aligned(128))) uint8_t lds[T::kBytes];
    const int tid = threadIdx.x, lane = tid & 63, w = rfl(tid >> 6);
    const int wn = w % WN, wm = w / WN;
    const int lw = LOADERS > 0 ? w - T::kWaves : w;   // which of the loading wavefronts it is
    const bool loads = LOADERS == 0 || lw >= 0;
    const int n = lane & 15, q = lane >> 4;

    // each XCD gets a run of tiles, in groups of eight tiles of tokens, so that those at work at a time share rows and columns
    const int tiles = p.row_groups * p.token_groups, run = (tiles + 7) >> 3;
    const int tile = (int)(blockIdx.x & 7) * run + (int)(blockIdx.x >> 3);
    if (tile >= tiles) return;
    constexpr int kGroup = 8;
    const int per_group = kGroup * p.row_groups, group = tile / per_group, in_group = tile - group * per_group;
    const int high = p.token_groups - group * kGroup < kGroup ? p.token_groups - group * kGroup : kGroup;
    const int rg = in_group / high, tg = group * kGroup + in_group - rg * high;
    const int c0 = rg * T::kCols, m0 = tg * T::kTokens;
    const int K = p.K, nkb = p.nkb;

    // Matrix row r of a wavefront's weight tile k is its column 4 TN (r / 4) + 4 k + r % 4, so a lane's results of all tiles are 4 TN
    // adjacent columns.  Piece i of a stage: rows 8 (i % 2) .. + 7 of tile i / 2, tiles counted through the wavefronts.
    unsigned w_off[T::kW], x_off[T::kX];
    const int ld_row = lane >> 3;
#pragma unroll
    for (int j = 0; j < T::kW; j++) {
        const int i = lw * T::kW + j, r = 8 * (i & 1) + ld_row, k = (i >> 1) % TN;
        int c = (i >> 1) / TN * (TN * 16) + 4 * TN * (r >> 2) + 4 * k + (r & 3);
        c = c0 + c < p.N ? c : p.N - 1 - c0;
        w_off[j] = (unsigned)c * (unsigned)K + 16u * ((lane & 7) ^ ((r >> 1) & 7));
    }
#pragma unroll
    for (int j = 0; j < T::kX; j++) {
        const int i = lw * T::kX + j, r = 8 * (i & 1) + ld_row;
        int m = (i >> 1) * 16 + r;
        m = m0 + m < p.M ? m : p.M - 1 - m0;
        x_off[j] = (unsigned)m * (unsigned)K + 16u * ((lane & 7) ^ ((r >> 1) & 7));
    }
    const int my_token = lw * T::kScaleLanes + (lane < T::kScaleLanes ? lane : 0);
    const unsigned xs_off = 4u * (unsigned)((m0 + my_token < p.M ? my_token : p.M - 1 - m0) * nkb);
    uint8_t *xs = lds + S * T::kStage, *ws = xs + T::kTokens * 32;
    const TokenScales scales = {p.quads, T::kTokens, nkb - 4};

    // (a tile's offsets are below 2^25: rows of up to 64 KiB)
    const uint8_t *w_base = p.w + (size_t)c0 * K, *x_base = p.x + (size_t)m0 * K;
    const float *xs_base = p.x_scale + (size_t)m0 * nkb;
    // Load j of a stage.  Behind the last K block nothing is loaded, but the loads are still counted.
    auto issue = [&](int stage, int kb, auto jc) {
        constexpr int j = decltype(jc)::value - 1;
        uint8_t *at = lds + stage * T::kStage;
        const int limit = kb < nkb ? -1 : 0;
        if constexpr (j < 0) {
            if (scales.loads(kb, false)) scales.load(buffer(xs_base, limit), xs_off, kb, lw * T::kScaleLanes, lane < T::kScaleLanes, xs);
        } else if constexpr (j < T::kW) dma16<0>(buffer(w_base, limit), w_off[j], 128u * kb, at + (lw * T::kW + j) * 1024);
        else dma16<0>(buffer(x_base, limit), x_off[j - T::kW], 128u * kb, at + T::kCols * 128 + (lw * T::kX + j - T::kW) * 1024);
    };
    for (int i = lw; loads && i < T::kScaleRows * ((nkb + 63) >> 6); i += T::kLoaders) {   // the columns' scales of all K blocks
        const int row = i % T::kScaleRows, c = i / T::kScaleRows * 64;
        const int last = (p.N - 1) >> 7;
        const int block = (c0 >> 7) + row < last ? (c0 >> 7) + row : last;
        if (c + lane < nkb)
            dma4(agent_buffer(p.w_scale + (size_t)block * nkb + c), 4u * lane, 0u, ws + 4 * (row * kMaxKBlocks + c));
    }
    if constexpr (LOADERS > 0) {
        if (loads) {
#pragma unroll
            for (int i = 0; i < S; i++) for_each<T::kLoads>([&](auto j) { issue(i, i, j); });
            wait_vmcnt<T::kData *(S - 1)>();
            lds_barrier();
            int stage = 0;
            for (int kb = 0; kb < nkb; kb++) {
                wait_vmcnt<T::kData *(S - 2)>();   // the next K block's loads have landed
                lds_barrier();                     // and this one's stage has been read
                for_each<T::kLoads>([&](auto j) { issue(stage, kb + S, j); });
                stage = stage + 1 < S ? stage + 1 : 0;
            }
            wait_vmcnt<0>();   // (the workgroup's memory is given back)
            return;
        }
    } else {
#pragma unroll
        for (int i = 0; i < S - 1; i++) for_each<T::kLoads>([&](auto j) { issue(i, i, j); });
        for_each<T::early()>([&](auto j) { issue(S - 1, S - 1, j); });
    }

    const int f_n = (n >> 1) & 7;
    const int frag_lo = n * 128 + 16 * (q ^ f_n), frag_hi = n * 128 + 16 * ((q ^ f_n) ^ 4);
    const uint8_t *my_ws = ws + 4 * kMaxKBlocks * ((wn * TN * 16) >> 7);
    lds_v4i w_lo, w_hi, x_lo, x_hi;   // this wavefront's part of a stage
    const uint8_t *my_xs;
    const int xs_row = (wm * TM * 16 + n) * scales.stride(), xs_tile = 16 * scales.stride();
    auto aim = [&](int stage, int kb) {
        const uint8_t *at = lds + stage * T::kStage;
        w_lo = lds_tile(at + wn * TN * 2048 + frag_lo);
        w_hi = lds_tile(at + wn * TN * 2048 + frag_hi);
        x_lo = lds_tile(at + T::kCols * 128 + wm * TM * 2048 + frag_lo);
        x_hi = lds_tile(at + T::kCols * 128 + wm * TM * 2048 + frag_hi);
        my_xs = xs + scales.place(kb) + xs_row;
    };
    v4f acc[TN][TM] = {};
    // A product is scaled into its accumulator two matrix instructions after its own, so no wait states stand between the two.
    v4f prod[2] = {};
    float fac[2] = {0.f, 0.f};
    v8i a[TN];
    if constexpr (LOADERS == 0) wait_vmcnt<T::kData *(S - 2) + T::early() - 1>();
    lds_barrier();
    aim(0, 0);
    v4i b_lo = x_lo[0], b_hi = x_hi[0];
    float f = lds_float(my_xs), sc = lds_float(my_ws);
#pragma unroll
    for (int k = 0; k < TN; k++) a[k] = cat(w_lo[k * 128], w_hi[k * 128]);
    int stage = 0, freed = S - 1;   // freed: the stage whose loads are being issued, for K block kb + S - 1, then kb + S
    for (int kb = 0; kb < nkb; kb++) {
        auto pass = [&](auto tc) {
            constexpr int t = decltype(tc)::value;
            const v8i b = cat(b_lo, b_hi);
            const float by = f * sc;
            if constexpr (t + 1 < TM) {
                b_lo = x_lo[(t + 1) * 128];
                b_hi = x_hi[(t + 1) * 128];
                f = lds_float(my_xs + (t + 1) * xs_tile);
            } else {
                // The last token tile is in registers: behind the barrier everybody is done with this stage, and its place is
                // refilled.  The weight tiles are replaced by the next K block's as they are used for the last time.
                // (Behind the last K block, what is read is not used.)
                if constexpr (LOADERS == 0) wait_vmcnt<T::kData *(S - 2)>();   // the next K block's loads have landed
                lds_barrier();
                freed = stage;
                stage = stage + 1 < S ? stage + 1 : 0;
                aim(stage, kb + 1);
                b_lo = x_lo[0];
                b_hi = x_hi[0];
                f = lds_float(my_xs);
                sc = lds_float(my_ws + 4 * (kb + 1 < nkb ? kb + 1 : kb));
            }
            __builtin_amdgcn_sched_barrier(0);
            auto one = [&](auto kc) {
                constexpr int k = decltype(kc)::value;
                const v4f cur = mfma_fp8(a[k], b);
                __builtin_amdgcn_sched_barrier(0);
                constexpr int kAll = TN * TM, j = t * TN + k, done = (j + kAll - 2) % kAll;
                v4f &dst = acc[done % TN][done / TN];
                dst += prod[j & 1] * fac[j & 1];
                asm volatile("" : "+v"(dst));
                prod[j & 1] = cur;
                fac[j & 1] = by;
                if constexpr (t + 1 == TM) a[k] = cat(w_lo[k * 128], w_hi[k * 128]);
                constexpr int slot = t + 1 == TM ? k : TN + j;   // matrix instructions since the barrier
                for_each<T::kLoads>([&](auto piece) {
                    if constexpr (LOADERS == 0 && T::at(decltype(piece)::value) == slot) issue(freed, t + 1 == TM ? kb + S : kb + S - 1, piece);
                });
                __builtin_amdgcn_sched_barrier(0);
            };
            for_each<TN>(one);
        };
        for_each<TM>(pass);
    }
    if constexpr (LOADERS == 0) wait_vmcnt<0>();   // (the workgroup's memory is given back)
    static_assert(TN * TM % 2 == 0, "");
    acc[TN - 2][TM - 1] += prod[0] * fac[0];
    acc[TN - 1][TM - 1] += prod[1] * fac[1];
    const int col = c0 + wn * TN * 16 + 4 * TN * q;
#pragma unroll
    for (int t = 0; t < TM; t++) {
        const int m = m0 + (wm * TM + t) * 16 + n;
        if (col + 4 * TN <= p.N) {
            if (m < p.M) {
                any4 *to = reinterpret_cast<any4 *>(p.out + (size_t)m * p.N + col);
#pragma unroll
                for (int k = 0; k < TN; k += 2)
                    to[k / 2] = (any4){pack_bf16x2(acc[k][t][0], acc[k][t][1]), pack_bf16x2(acc[k][t][2], acc[k][t][3]),
                                       pack_bf16x2(acc[k + 1][t][0], acc[k + 1][t][1]),
                                       pack_bf16x2(acc[k + 1][t][2], acc[k + 1][t][3])};
            }
        } else {
#pragma unroll
            for (int k = 0; k < TN; k++) store4(p, m, col + 4 * k, acc[k][t]);
        }
    }
}

template <int TN, int TM, int WN, int WM, int S, int LOADERS>
hipError_t launch_tile_mm(MmParams p, hipStream_t stream)
{
    typedef Tile<TN, TM, WN, WM, S, LOADERS> T;
    if (!grid_fits(tiles_of(p.M, p.N, T::kCols, T::kTokens), (T::kWaves + LOADERS) * 64)) return hipErrorInvalidConfiguration;
    p.row_groups = (p.N + T::kCols - 1) / T::kCols;
    p.token_groups = (p.M + T::kTokens - 1) / T::kTokens;
    const int run = (p.row_groups * p.token_groups + 7) / 8;
    void *args[] = {&p};
    return hipLaunchKernel(reinterpret_cast<const void *>(mm_tile_kernel<TN, TM, WN, WM, S, LOADERS>), dim3((unsigned)run * 8),
                           dim3((T::kWaves + LOADERS) * 64), args, 0, stream);
}

// What a call takes.  Few tiles: the largest tile of the streaming kernel of which there are more than half as many as compute
// units - a smaller one reads more, a larger one leaves the memory idle (MI355X, us, K = 7168; M x N, 32x32 / 64x32 / 64x64 tile:
// 61 x 2112 8.4 / 11.3 / 14.5, 128 x 4096 14.3 / 11.6 / 14.6, 192 x 4096 19.2 / 20.9 / 14.6).  More: the tile whose rounds over the compute
// units take the least time.  What a round takes for each K block was measured, us: with tiles for half the units, and with as many
// as run at a time; between the two it is taken in proportion where a unit holds one tile, and as a whole where it holds two.
// (K = 7168, us, 128x64 / 128x128 / 256x128 / 256x256 tile: 384 x 4096 22.7 / 30.2 / 41.1 / 77, 700 x 4096 34.6 / 30.8 / 41.6 / 78,
// 1500 x 4096 57 / 61 / 46 / 79, 3000 x 4096 109 / 98 / 92 / 83, 8192 x 2112 168 / 166 / 145 / 172.)
enum Plan { kStreamHalf1, kStreamHalf2, kStream1x1, kStream2x1, kStream2x2, kStream4x2, kStream4x4, kTile128x64, kTile128x128,
            kTile256x128, kTile256x256 };
constexpr int kUnits = 256;

Plan plan(int M, int N)
{
    auto few = [&](int cols, int tokens) { return tiles_of(M, N, cols, tokens) <= kUnits / 2; };
    if (M <= 8) return few(32, 16) ? kStreamHalf1 : kStreamHalf2;
    if (few(64, 64)) return !few(64, 32) ? kStream4x2 : !few(32, 32) ? kStream2x2 : !few(32, 16) ? kStream2x1 : kStream1x1;
    static const struct {
        Plan plan;
        int cols, tokens, resident;
        float half, full;
    } kinds[] = {
        {kStream4x4, 64, 64, 2, 0.23f, 0.43f},      {kTile128x64, 128, 64, 2, 0.38f, 0.67f},   {kTile128x128, 128, 128, 1, 0.50f, 0.59f},
        {kTile256x128, 256, 128, 1, 0.70f, 0.97f}, {kTile256x256, 256, 256, 1, 1.36f, 1.80f},
    };
    Plan best = kStream4x4;
    float least = 0.f;
    for (const auto &k : kinds) {
        const int64_t tiles = tiles_of(M, N, k.cols, k.tokens), slots = kUnits * k.resident, rest = tiles % slots;
        float time = (float)(tiles / slots) * k.full;
        if (rest > 0 && rest <= slots / 2) time += k.half;
        else if (rest > 0) time += k.resident > 1 ? k.full : k.half + (k.full - k.half) * (float)(2 * rest - slots) / (float)slots;
        if (k.plan == kStream4x4 || time < least) best = k.plan, least = time;
    }
    return best;
}

}  // namespace
}  // namespace alpha_moe

extern "C" int alpha_moe_block_scaled_mm(const uint8_t *x, const float *x_scale, const uint8_t *w, const float *w_scale,
                                         uint16_t *out, int M, int N, int K, void *stream)
{
    using namespace alpha_moe;
    if (M < 0 || N <= 0 || K <= 0 || K % 128 != 0 || K > 128 * kMaxKBlocks || M > INT32_MAX - 255 || N > INT32_MAX - 255)
        return ALPHA_MOE_ERR_SHAPE;
    if (M == 0) return ALPHA_MOE_OK;
    if (!x || !x_scale || !w || !w_scale || !out) return ALPHA_MOE_ERR_NULL_POINTER;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
        return ALPHA_MOE_ERR_ALIGNMENT;
    MmParams p = {};
    p.x = x, p.x_scale = x_scale, p.w = w, p.w_scale = w_scale, p.out = out;
    p.M = M, p.N = N, p.K = K, p.nkb = K / 128;
    p.quads = p.nkb >= 4;
    hipStream_t hs = static_cast<hipStream_t>(stream);
    hipError_t err = hipErrorInvalidValue;
    switch (plan(M, N)) {
    case kStreamHalf1: err = launch_stream_mm<1, 1, 8, 2, true>(p, hs); break;
    case kStreamHalf2: err = launch_stream_mm<2, 1, 8, 2, true>(p, hs); break;
    case kStream1x1: err = launch_stream_mm<1, 1, 8, 2, false>(p, hs); break;
    case kStream2x1: err = launch_stream_mm<2, 1, 4, 2, false>(p, hs); break;
    case kStream2x2: err = launch_stream_mm<2, 2, 4, 2, false>(p, hs); break;
    case kStream4x2: err = launch_stream_mm<4, 2, 4, 2, false>(p, hs); break;
    case kStream4x4: err = launch_stream_mm<4, 4, 4, 1, false>(p, hs); break;
    case kTile128x64: err = launch_tile_mm<4, 2, 2, 2, 3, 4>(p, hs); break;
    case kTile128x128: err = launch_tile_mm<4, 4, 2, 2, 4, 4>(p, hs); break;
    case kTile256x128: err = launch_tile_mm<4, 4, 4, 2, 3, 4>(p, hs); break;
    case kTile256x256: err = launch_tile_mm<4, 8, 4, 2, 2, 0>(p, hs); break;
    }
    return err == hipSuccess ? ALPHA_MOE_OK : err == hipErrorInvalidConfiguration ? ALPHA_MOE_ERR_SHAPE : ALPHA_MOE_ERR_LAUNCH;
}
