// Low-rank adapters of many requests beside a shared projection:
//   out[m, :] = base[m, :] + scale[l] (x[m, :] a[l]^T) b[l]^T,  l = adapter_ids[m];  out[m] = base[m] where l names no adapter.
//
// Two kernels.  The first contracts tokens with the adapters' a, K split over wavefronts and workgroups, into partial sums in fp32
// (workspace, [split][token][rank]); the second adds them up, in their order, times scale, and contracts with b.  Between the two, a token's
// `rank` values are taken as sums of two bf16 numbers, high and low part, so that the second product on the bf16 matrix cores is as
// good as one of fp32 values: the high part is the value's upper 16 bits, the low part the rest rounded to 8 bits, together 2^-16 off.
// Both parts lie next to each other along the contraction, in front of b's values twice.
//
// A token's adapter is its own, whatever its neighbours have: a workgroup takes a tile of neighbouring tokens, and the distinct adapters
// among them one after the other (or P workgroups share them).  Tokens are columns of the matrix instructions, whose results depend on
// their own column alone, so a tile is multiplied as a whole and what belongs to other adapters is not stored: nothing of
// them, NaN or infinity, reaches a token.
//
// Operands as in moe_common.hpp: adapters' rows are A, tokens B, results (row 4q + j, token n) in register j of lane (n, q).
#include "moe_common.hpp"

namespace alpha_moe {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));   // rows of an odd N start at any multiple of two bytes

constexpr int kMaxRank = 128;

struct AdaptParams {
    const uint16_t *base, *a, *b;
    const uint8_t *x;          // bf16, or FP8 codes with x_scale
    const float *x_scale, *scale;
    const int32_t *ids;
    uint16_t *out;
    float *part;               // [splits][M][rank]
    int M, N, K, rank, adapters, nkb, splits, sharers;
};

// The distinct adapters of a tile of tokens, in the order of their first tokens: f(adapter, tokens that have it), every `sharers`-th one.
template <typename F>
__device__ __forceinline__ void for_each_adapter(int id, int adapters, int mine, int sharers, F f)
{
    unsigned long long left = __ballot((unsigned)id < (unsigned)adapters);
    int turn = 0;
    while (left != 0) {
        const int which = __builtin_amdgcn_readlane(id, (int)__builtin_ctzll(left));
        const unsigned long long same = __ballot(id == which);
        left &= ~same;
        if (turn == mine) f(which, same);
        turn = turn + 1 < sharers ? turn + 1 : 0;
    }
}

// The bf16 values of 16 codes (a code's value has 4 bits: exact).
__device__ __forceinline__ void widen(v4i codes, v8bf (&to)[2])
{
    typedef float v2f __attribute__((ext_vector_type(2)));
    v4i half[2];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes[i], true);
        half[i / 2][2 * (i % 2)] = (int)pack_bf16x2(lo.x, lo.y);
        half[i / 2][2 * (i % 2) + 1] = (int)pack_bf16x2(hi.x, hi.y);
    }
    to[0] = __builtin_bit_cast(v8bf, half[0]);
    to[1] = __builtin_bit_cast(v8bf, half[1]);
}

// part[split][token][rank]: RT tiles of 16 ranks, T tiles of 16 tokens; the four wavefronts take the split's K blocks in turn.
template <int RT, int T, bool FP8>
__global__ __launch_bounds__(256) void adapt_in_kernel(const AdaptParams p)
{
    __shared__ v4f sums[4][RT * T][64];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.x * (16 * T), split = blockIdx.y;
    const int first = (int)((int64_t)split * p.nkb / p.splits), last = (int)((int64_t)(split + 1) * p.nkb / p.splits);
    const int id = lane < 16 * T && m0 + lane < p.M ? p.ids[m0 + lane] : -1;
    const int K = p.K;
    int token[T];
#pragma unroll
    for (int t = 0; t < T; t++) token[t] = min(m0 + 16 * t + n, p.M - 1);
    for_each_adapter(id, p.adapters, blockIdx.z, p.sharers, [&](int adapter, unsigned long long same) {
        const uint16_t *a = p.a + (size_t)adapter * p.rank * K;
        v4f acc[RT][T] = {};
        for (int kb = first + w; kb < last; kb += 4) {
            // lane (n, q) has the 32 columns [32 q, 32 q + 32) of the block, of rank n's row and of token n's
            v8bf av[RT][4], xv[T][4];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const v8bf *at = reinterpret_cast<const v8bf *>(a + (size_t)min(16 * r + n, p.rank - 1) * K + kb * 128 + q * 32);
#pragma unroll
                for (int i = 0; i < 4; i++) av[r][i] = at[i];
            }
            float f[T];
#pragma unroll
            for (int t = 0; t < T; t++) {
                if constexpr (FP8) {
                    const v4i *at = reinterpret_cast<const v4i *>(p.x + (size_t)token[t] * K + kb * 128 + q * 32);
                    v8bf two[2];
                    widen(at[0], two);
                    xv[t][0] = two[0], xv[t][1] = two[1];
                    widen(at[1], two);
                    xv[t][2] = two[0], xv[t][3] = two[1];
                    f[t] = p.x_scale[(size_t)token[t] * p.nkb + kb];
                } else {
                    const v8bf *at = reinterpret_cast<const v8bf *>(p.x + 2 * ((size_t)token[t] * K + kb * 128 + q * 32));
#pragma unroll
                    for (int i = 0; i < 4; i++) xv[t][i] = at[i];
                }
            }
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int t = 0; t < T; t++) {
                    v4f s = FP8 ? (v4f){0.f, 0.f, 0.f, 0.f} : acc[r][t];
#pragma unroll
                    for (int i = 0; i < 4; i++) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[r][i], xv[t][i], s, 0, 0, 0);
                    if constexpr (FP8) acc[r][t] += s * f[t];
                    else acc[r][t] = s;
                }
        }
        __syncthreads();   // (what the adapter before has left has been read)
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int t = 0; t < T; t++) sums[w][r * T + t][lane] = acc[r][t];
        __syncthreads();
        for (int e = tid; e < RT * T * 64; e += 256) {
            const int l = e & 63, t = (e >> 6) % T, r = (e >> 6) / T, rank = 16 * r + 4 * (l >> 4), at = 16 * t + (l & 15);
            const v4f s = sums[0][e >> 6][l] + sums[1][e >> 6][l] + sums[2][e >> 6][l] + sums[3][e >> 6][l];
            if (rank < p.rank && ((same >> at) & 1))
                *reinterpret_cast<v4f *>(p.part + ((size_t)split * p.M + m0 + at) * p.rank + rank) = s;
        }
    });
}

// out: each wavefront 64 columns of T tiles of 16 tokens; STEPS matrix instructions of 32 along the two parts of the ranks.
template <int STEPS, int T>
__global__ __launch_bounds__(256) void adapt_out_kernel(const AdaptParams p)
{
    constexpr int kRow = STEPS * 64 + 16;   // bytes of a token's parts in LDS, and 16 so that tokens' rows begin at other banks
    __shared__ __attribute__((aligned(16))) uint8_t parts[16 * T * kRow];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * (16 * T), c0 = (blockIdx.x * 4 + w) * 64, rank = p.rank;
    const int id = lane < 16 * T && m0 + lane < p.M ? p.ids[m0 + lane] : -1;
    const unsigned long long there = __ballot(lane < 16 * T && m0 + lane < p.M);
    // matrix row r of column tile k is column 16 (r / 4) + 4 k + r % 4: a lane's results are the 16 columns from 16 q on
    const int col = c0 + 16 * q;
    auto finish = [&](int t, const v4f (&acc)[4]) {
        const size_t at = (size_t)(m0 + 16 * t + n) * p.N + col;
        if (col + 16 <= p.N) {
            const any4 *from = reinterpret_cast<const any4 *>(p.base + at);
            any4 *to = reinterpret_cast<any4 *>(p.out + at);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                any4 v = from[h];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const v4f s = acc[2 * h + i / 2];
                    const float lo = __builtin_bit_cast(float, v[i] << 16), hi = __builtin_bit_cast(float, v[i] & 0xffff0000u);
                    v[i] = i % 2 == 0 ? pack_bf16x2(lo + s[0], hi + s[1]) : pack_bf16x2(lo + s[2], hi + s[3]);
                }
                to[h] = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (col + i < p.N)
                    p.out[at + i] = (uint16_t)pack_bf16x2(__builtin_bit_cast(float, (uint32_t)p.base[at + i] << 16) + acc[i / 4][i % 4], 0.f);
        }
    };
    if (blockIdx.z == 0) {   // tokens without an adapter
        const unsigned long long none = there & ~__ballot((unsigned)id < (unsigned)p.adapters);
#pragma unroll
        for (int t = 0; t < T; t++)
            if ((none >> (16 * t + n)) & 1) {
                const v4f zero[4] = {};
                finish(t, zero);
            }
    }
    for_each_adapter(id, p.adapters, blockIdx.z, p.sharers, [&](int adapter, unsigned long long same) {
        const float scale = p.scale ? p.scale[adapter] : 1.f;
        __syncthreads();   // (the parts of the adapter before have been read)
        for (int i = tid; i < 16 * T * rank; i += 256) {
            const int t = i / rank, r = i - t * rank;
            if (!((same >> t) & 1)) continue;
            const float *from = p.part + (size_t)(m0 + t) * rank + r;
            float v = 0.f;
            for (int s = 0; s < p.splits; s++) v += from[(size_t)s * p.M * rank];
            v *= scale;
            const uint32_t high = __builtin_bit_cast(uint32_t, v) & 0xffff0000u;
            const float low = fabsf(v) == __builtin_inff() ? 0.f : v - __builtin_bit_cast(float, high);
            uint16_t *to = reinterpret_cast<uint16_t *>(parts + t * kRow) + r;
            to[0] = (uint16_t)(high >> 16);
            to[rank] = (uint16_t)pack_bf16x2(low, 0.f);
        }
        __syncthreads();
        const uint16_t *b = p.b + (size_t)adapter * p.N * rank;
        v4f acc[T][4] = {};
        if (c0 < p.N) {
            const int chunks = rank / 8;
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int chunk = 4 * s + q;   // eight values of the high parts, then of the low ones; nothing behind them
                const bool some = chunk < 2 * chunks;
                v8bf bv[4], vv[T];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int c = min(c0 + 16 * (n >> 2) + 4 * k + (n & 3), p.N - 1);
                    bv[k] = some ? *reinterpret_cast<const v8bf *>(b + (size_t)c * rank + (chunk < chunks ? chunk : chunk - chunks) * 8) : (v8bf){};
                }
#pragma unroll
                for (int t = 0; t < T; t++)
                    vv[t] = some ? *reinterpret_cast<const v8bf *>(parts + (16 * t + n) * kRow + chunk * 16) : (v8bf){};
#pragma unroll
                for (int t = 0; t < T; t++)
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[t][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[k], vv[t], acc[t][k], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < T; t++)
            if ((same >> (16 * t + n)) & 1) finish(t, acc[t]);
    });
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tokens of a tile, workgroups that share a tile's adapters, and parts of K.
struct AdaptPlan {
    int T, sharers, splits;
    AdaptPlan(int M, int K, int rank, int adapters)
    {
        const int nkb = K / 128;
        T = M <= 1024 || rank > 64 ? 1 : rank > 32 ? 2 : 4;
        const int64_t tiles = ceil_div(M, 16 * T);
        const int most = adapters < 16 * T ? adapters : 16 * T;
        sharers = (int)ceil_div(256, tiles);
        sharers = sharers > most ? most : sharers;
        sharers = sharers > M ? M : sharers;
        const int64_t want = ceil_div(512, tiles * sharers), can = ceil_div(nkb, 4);
        splits = (int)(want > can ? can : want);
    }
};

template <typename... Args>
hipError_t launch(void (*kernel)(Args...), dim3 grid, dim3 block, hipStream_t stream, Args... args)
{
    void *list[] = {&args...};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, list, 0, stream);
}

template <int RT, int T>
hipError_t adapt(const AdaptParams &p, hipStream_t hs)
{
    const unsigned tiles = (unsigned)ceil_div(p.M, 16 * T);
    const auto in = p.x_scale ? adapt_in_kernel<RT, T, true> : adapt_in_kernel<RT, T, false>;
    const hipError_t err = launch(in, dim3(tiles, p.splits, p.sharers), dim3(256), hs, p);
    if (err != hipSuccess) return err;
    return launch(adapt_out_kernel<RT, T>, dim3((unsigned)ceil_div(p.N, 256), tiles, p.sharers), dim3(256), hs, p);
}

bool sizes_fit(int M, int N, int K, int rank, int adapters)
{
    return M >= 0 && N > 0 && K > 0 && K % 128 == 0 && K <= 128 * kMaxKBlocks && rank > 0 && rank % 8 == 0 && rank <= kMaxRank &&
           adapters > 0 && M <= 16 * 65535 && N <= INT32_MAX - 255;
}

}  // namespace
}  // namespace alpha_moe

using namespace alpha_moe;

extern "C" size_t alpha_moe_adapters_workspace_bytes(int M, int K, int rank, int num_adapters)
{
    if (M <= 0 || !sizes_fit(M, 1, K, rank, num_adapters)) return 0;
    return (size_t)AdaptPlan(M, K, rank, num_adapters).splits * M * rank * sizeof(float);
}

extern "C" int alpha_moe_add_adapters(const uint16_t *base, const void *x, const float *x_scale, const uint16_t *a, const uint16_t *b,
                                      const int32_t *adapter_ids, const float *scale, uint16_t *out, int M, int N, int K, int rank,
                                      int num_adapters, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!sizes_fit(M, N, K, rank, num_adapters)) return ALPHA_MOE_ERR_SHAPE;
    if (M == 0) return ALPHA_MOE_OK;
    if (!base || !x || !a || !b || !adapter_ids || !out) return ALPHA_MOE_ERR_NULL_POINTER;
    uintptr_t all = 0;
    for (const void *ptr : {static_cast<const void *>(base), x, static_cast<const void *>(a), static_cast<const void *>(b),
                            static_cast<const void *>(out)})
        all |= reinterpret_cast<uintptr_t>(ptr);
    if ((all & 15) != 0) return ALPHA_MOE_ERR_ALIGNMENT;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
        workspace_bytes < alpha_moe_adapters_workspace_bytes(M, K, rank, num_adapters))
        return ALPHA_MOE_ERR_WORKSPACE;
    const AdaptPlan plan(M, K, rank, num_adapters);
    AdaptParams p = {};
    p.base = base, p.a = a, p.b = b, p.x = static_cast<const uint8_t *>(x), p.x_scale = x_scale, p.scale = scale;
    p.ids = adapter_ids, p.out = out, p.part = static_cast<float *>(workspace);
    p.M = M, p.N = N, p.K = K, p.rank = rank, p.adapters = num_adapters, p.nkb = K / 128;
    p.splits = plan.splits, p.sharers = plan.sharers;
    hipStream_t hs = static_cast<hipStream_t>(stream);
    const int T = plan.T;
    const hipError_t err = rank <= 16   ? (T == 1 ? adapt<1, 1>(p, hs) : adapt<1, 4>(p, hs))
                           : rank <= 32 ? (T == 1 ? adapt<2, 1>(p, hs) : adapt<2, 4>(p, hs))
                           : rank <= 64 ? (T == 1 ? adapt<4, 1>(p, hs) : adapt<4, 2>(p, hs))
                                        : adapt<8, 1>(p, hs);
    return err == hipSuccess ? ALPHA_MOE_OK : ALPHA_MOE_ERR_LAUNCH;
}
