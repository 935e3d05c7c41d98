// Low-rank adapters of many requests beside a shared projection:
//   out[m, :] = base[m, :] + scale[l] (x[m, :] a[l]^T) b[l]^T,  l = adapter_ids[m];  out[m] = base[m] where l names no adapter.
//
// Two kernels.  The first contracts tokens with the adapters' a, K split over wavefronts and workgroups, into partial sums in fp32
// (workspace, [split][token][rank]); the second adds them up, in their order, times scale, and contracts with b.  Between the two, a token's
// `rank` values are taken as sums of three bf16 numbers, eight of their 24 bits each, so that the second product on the bf16 matrix
// cores is one of the fp32 values themselves: what base and adapter leave of each other where they cancel is as good as theirs.
// The parts lie behind each other along the contraction, in front of b's values again.
//
// A token's adapter is its own, whatever its neighbours have: a workgroup takes a tile of neighbouring tokens, and the distinct adapters
// among them one after the other (or P workgroups share them).  Tokens are columns of the matrix instructions, whose results depend on
// their own column alone, so a tile is multiplied as a whole and what belongs to other adapters is not stored: nothing of
// them, NaN or infinity, reaches a token.
//
// What bounds it: of many tokens memory, x once, base and result once each (8192 tokens, K = 2048, N = 7168, rank 64: 271 MB, 53 us at a
// copy's rate; MI355X 20 us the first kernel and 70 the second, whose b is read again by every tile out of the L2; it was 65 with two parts,
// 2^-16 off, whose tiles fit a compute unit once more); of few tokens two launches, each one chain of loads and a sum over wavefronts (1 token 4.2
// and 3.8 us, 61 tokens of 48 adapters 8.4 and 5.0).  One kernel for both would have every column's workgroup contract all of K again, or
// wait for the others.
//
// Operands as in moe_common.hpp: adapters' rows are A, tokens B, results (row 4q + j, token n) in register j of lane (n, q).
#include "moe_common.hpp"

namespace alpha_moe {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));

constexpr int kMaxRank = 128;

struct AdaptParams {
    const uint16_t *base, *a, *b;
    const uint8_t *x;          // bf16, or FP8 codes with x_scale
    const float *x_scale, *scale;
    const int32_t *ids;
    uint16_t *out;
    float *part;               // [splits][M][rank]
    int M, N, K, rank, adapters, nkb, splits, sharers, run, tiles, pieces, rank_groups;
};

// LDS accesses of one wavefront complete in order; this keeps the compiler to the written order
__device__ __forceinline__ void lds_order()
{
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// Workgroups are dealt to the eight XCDs in turn: each gets a run of tiles, so that an adapter's a and b are read into few of their
// L2s.  A tile's workgroups: `pieces` times `sharers`.
struct Place {
    int tile, piece, turn;
};
__device__ __forceinline__ bool find_place(int tiles, int pieces, Place &at)
{
    // (the sharers behind each other: most of a tile's have nothing to do, and every so-many-th workgroup is the same few compute units')
    const int all = tiles * pieces, run = (all + 7) >> 3, in_run = (int)(blockIdx.x >> 3);
    at.turn = in_run / run;
    const int i = (int)(blockIdx.x & 7) * run + in_run - at.turn * run;
    if (i >= all) return false;
    at.tile = i / pieces;
    at.piece = i - at.tile * pieces;
    return true;
}

// A buffer at a wavefront-uniform base: loads behind its end give 0.  (Rows of an odd N start at any multiple of two bytes, and memory
// takes 16 bytes there as a whole.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *uniform_base, uint32_t bytes)
{
    const uint64_t v = reinterpret_cast<uint64_t>(uniform_base);
    const uint64_t u = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32) |
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

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

// part[split][token][rank]: RT tiles of 16 ranks of p.rank_groups times as many, T tiles of 16 tokens; the four wavefronts take the
// split's K blocks in turn, operands straight from memory: each value of x is used by one wavefront only, and an adapter's a comes out of
// the L2 (staged through LDS for all four it was no faster).
template <int RT, int T, bool FP8>
__global__ __launch_bounds__(256, 2) void adapt_in_kernel(const AdaptParams p)
{
    __shared__ v4f sums[4][RT * T][64];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    Place place;
    if (!find_place(p.tiles, p.splits * p.rank_groups, place)) return;
    const int m0 = place.tile * (16 * T), split = place.piece / p.rank_groups, r0 = (place.piece - split * p.rank_groups) * (16 * RT);
    const int first = (int)((int64_t)split * p.nkb / p.splits), last = (int)((int64_t)(split + 1) * p.nkb / p.splits);
    const int id = lane < 16 * T && m0 + lane < p.M ? p.ids[m0 + lane] : -1;
    const int K = p.K;
    int token[T];
#pragma unroll
    for (int t = 0; t < T; t++) token[t] = min(m0 + 16 * t + n, p.M - 1);
    for_each_adapter(id, p.adapters, place.turn, p.sharers, [&](int adapter, unsigned long long same) {
        const uint16_t *a = p.a + (size_t)adapter * p.rank * K;
        v4f acc[RT][T] = {};
        for (int kb = first + w; kb < last; kb += 4) {
            // lane (n, q) has columns [16 q, 16 q + 16) of either half of the block, of rank n's row and of token n's: a load of all lanes
            // is sixteen lines (any other share of the columns made it thirty-two, and lines are what the path into a compute unit counts)
            v8bf av[RT][4], xv[T][4];
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const v8bf *at = reinterpret_cast<const v8bf *>(a + (size_t)min(r0 + 16 * r + n, p.rank - 1) * K + kb * 128 + q * 16);
#pragma unroll
                for (int i = 0; i < 4; i++) av[r][i] = at[8 * (i / 2) + i % 2];
            }
            float f[T];
#pragma unroll
            for (int t = 0; t < T; t++) {
                if constexpr (FP8) {
                    const v4i *at = reinterpret_cast<const v4i *>(p.x + (size_t)token[t] * K + kb * 128 + q * 16);
                    v8bf two[2];
                    widen(at[0], two);
                    xv[t][0] = two[0], xv[t][1] = two[1];
                    widen(at[4], two);
                    xv[t][2] = two[0], xv[t][3] = two[1];
                    f[t] = p.x_scale[(size_t)token[t] * p.nkb + kb];
                } else {
                    const v8bf *at = reinterpret_cast<const v8bf *>(p.x + 2 * ((size_t)token[t] * K + kb * 128 + q * 16));
#pragma unroll
                    for (int i = 0; i < 4; i++) xv[t][i] = at[8 * (i / 2) + i % 2];
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
            const int l = e & 63, t = (e >> 6) % T, r = (e >> 6) / T, rank = r0 + 16 * r + 4 * (l >> 4), at = 16 * t + (l & 15);
            const v4f s = sums[0][e >> 6][l] + sums[1][e >> 6][l] + sums[2][e >> 6][l] + sums[3][e >> 6][l];
            if (rank < p.rank && ((same >> at) & 1))
                *reinterpret_cast<v4f *>(p.part + ((size_t)split * p.M + m0 + at) * p.rank + rank) = s;
        }
    });
}

// out: each wavefront 64 columns of T tiles of 16 tokens, whose b values stay in registers over the tiles.  Up to 16 ranks (RT = 1) two parts
// lie behind each other in one matrix instruction, and b's values twice; beyond, b's values of 32 ranks are multiplied with each.
template <int RT, int T>
__global__ __launch_bounds__(256, RT == 8 ? 3 : 4) void adapt_out_kernel(const AdaptParams p)
{
    constexpr int S = RT == 1 ? 1 : RT / 2, PARTS = RT == 1 ? 2 : 3;   // matrix instructions along the ranks, and for each of them
    constexpr int kRow = 64 * S * PARTS + 16;   // bytes of a token's parts in LDS, and 16 so that tokens' rows begin at other banks
    __shared__ __attribute__((aligned(16))) uint8_t parts[16 * T * kRow];
    __shared__ __attribute__((aligned(16))) float turned[4][16][68];   // of each wavefront: 64 columns of 16 tokens, from columns to rows
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    Place place;
    if (!find_place(p.tiles, p.pieces, place)) return;
    const int m0 = place.tile * (16 * T), rank = p.rank, chunks = rank / 8;
    // this wavefront's columns: 64 of every 256, `run` times
    const int c_begin = place.piece * p.run * 256 + 64 * w, c_end = min((place.piece + 1) * p.run * 256, p.N);
    const int id = lane < 16 * T && m0 + lane < p.M ? p.ids[m0 + lane] : -1;
    const unsigned long long there = __ballot(lane < 16 * T && m0 + lane < p.M);
    // base and out go by rows, eight tokens' 128 bytes at a time (as the matrix instructions' results lie, sixteen tokens' 64, a load
    // or store takes twice the lines): lane l has eight columns of tokens l / 8 and 8 + l / 8 of a tile
    const int row = lane >> 3, col = 8 * (lane & 7);
    // (a tile has at most 64 rows of 2^24 columns; what is behind the last row is not there: a row's part of an offset is in the register
    // that is compared with the buffer's size, whether or not the uniform part, a column of the first row, is added before)
    const uint32_t tile_bytes = (uint32_t)min(16 * T, p.M - m0) * (uint32_t)p.N * 2u;
    const __amdgpu_buffer_rsrc_t base_tile = buffer(p.base + (size_t)m0 * p.N, tile_bytes), out_tile = buffer(p.out + (size_t)m0 * p.N, tile_bytes);
    const uint32_t at = ((uint32_t)row * (uint32_t)p.N + (uint32_t)col) * 2u, eight_rows = 16u * (uint32_t)p.N;
    auto load_base = [&](int c0, int t, int h) {   // of a whole 64 columns
        return __builtin_bit_cast(v4w, __builtin_amdgcn_raw_buffer_load_b128(base_tile, (int)(at + (2 * t + h) * eight_rows), 2 * c0, 0));
    };
    auto store = [&](int c0, int t, int h, v4w v) {
        __builtin_amdgcn_raw_buffer_store_b128(v, out_tile, (int)(at + (2 * t + h) * eight_rows), 2 * c0, 0);
    };
    auto add = [](v4w base, v4f lo, v4f hi) {
        auto two = [](uint32_t b, float x, float y) {
            return pack_bf16x2(__builtin_bit_cast(float, b << 16) + x, __builtin_bit_cast(float, b & 0xffff0000u) + y);
        };
        return (v4w){two(base[0], lo[0], lo[1]), two(base[1], lo[2], lo[3]), two(base[2], hi[0], hi[1]), two(base[3], hi[2], hi[3])};
    };
    // The tokens of `tokens` in tile t: base plus lo, hi (of either half).
    auto finish = [&](int c0, int t, unsigned long long tokens, const v4w (&base)[2], const v4f (&lo)[2], const v4f (&hi)[2]) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const v4w sum = add(base[h], lo[h], hi[h]);
            if ((tokens >> (16 * t + 8 * h + row)) & 1) store(c0, t, h, sum);
        }
    };
    // The same behind the last whole 64 columns, as far as there are any.
    auto finish_ragged = [&](int c0, int t, unsigned long long tokens, const v4f (&lo)[2], const v4f (&hi)[2]) {
        for (int h = 0; h < 2; h++) {
            const int token = 16 * t + 8 * h + row;
            if (!((tokens >> token) & 1)) continue;
            const size_t from = (size_t)(m0 + token) * p.N + c0 + col;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c0 + col + i < p.N)
                    p.out[from + i] = (uint16_t)pack_bf16x2(
                        __builtin_bit_cast(float, (uint32_t)p.base[from + i] << 16) + (i < 4 ? lo[h][i % 4] : hi[h][i % 4]), 0.f);
        }
    };
    const unsigned long long with = __ballot((unsigned)id < (unsigned)p.adapters);
    if (place.turn == 0 && with != there) {   // tokens without an adapter: base's bits
        const unsigned long long tokens = there & ~with;
#pragma unroll 1
        for (int c0 = c_begin; c0 < c_end; c0 += 256)
#pragma unroll 1
            for (int t = 0; t < T; t++)
                if (c0 + 64 <= p.N) {
                    const v4w base[2] = {load_base(c0, t, 0), load_base(c0, t, 1)};
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if ((tokens >> (16 * t + 8 * h + row)) & 1) store(c0, t, h, base[h]);
                } else {
                    for (int h = 0; h < 2; h++) {
                        const int token = 16 * t + 8 * h + row;
                        const size_t from = (size_t)(m0 + token) * p.N + c0 + col;
                        for (int i = 0; i < 8; i++)
                            if (((tokens >> token) & 1) && c0 + col + i < p.N) p.out[from + i] = p.base[from + i];
                    }
                }
    }
    // eight values of a chunk of b: the ranks' chunks one behind the other (RT == 1: twice), 0 behind the last one
    struct Weights {
        v8bf v[S][4];
    };
    uint32_t b_at[S];
#pragma unroll
    for (int s = 0; s < S; s++) {
        const bool some = RT == 1 ? q < 2 * chunks : 4 * s + q < chunks;
        const int chunk = RT == 1 && q >= chunks ? q - chunks : 4 * s + q;
        b_at[s] = some ? 2u * (uint32_t)(n * rank + 8 * chunk) : 0x40000000u;
    }
    // (the parts' places behind the last rank; what is multiplied there is 0 on both sides)
    for (int i = tid; i < 16 * T * kRow / 16; i += 256) reinterpret_cast<v4i *>(parts)[i] = (v4i){0, 0, 0, 0};
    for_each_adapter(id, p.adapters, place.turn, p.sharers, [&](int adapter, unsigned long long same) {
        const uint16_t *b = p.b + (size_t)adapter * p.N * rank;
        auto load_weights = [&](int c0, Weights &bv) {
            const int cols = min(64, p.N - c0);
            const __amdgpu_buffer_rsrc_t from = buffer(b + (size_t)c0 * rank, cols > 0 ? 2u * (uint32_t)(cols * rank) : 0u);
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    bv.v[s][k] = __builtin_bit_cast(
                        v8bf, __builtin_amdgcn_raw_buffer_load_b128(from, (int)(b_at[s] + 32u * (uint32_t)(k * rank)), 0, 0));
        };
        Weights bv;
        load_weights(c_begin, bv);   // (in front of the parts' loads)
        const float scale = p.scale ? p.scale[adapter] : 1.f;
        __syncthreads();   // (the parts of the adapter before have been read)
        for (int i = tid; i < 16 * T * rank / 4; i += 256) {   // four ranks of a token
            const int t = i / (rank / 4), r = 4 * (i - t * (rank / 4));
            if (!((same >> t) & 1)) continue;
            const float *from = p.part + (size_t)(m0 + t) * rank + r;
            const size_t step = (size_t)p.M * rank;
            v4f v = {0.f, 0.f, 0.f, 0.f};
            constexpr int F = T == 1 ? 8 : 4;   // loads in flight
            for (int s0 = 0; s0 < p.splits; s0 += F) {
                v4f in[F];
#pragma unroll
                for (int s = 0; s < F; s++) in[s] = *reinterpret_cast<const v4f *>(from + (size_t)min(s0 + s, p.splits - 1) * step);
#pragma unroll
                for (int s = 0; s < F; s++)
                    if (s0 + s < p.splits) v += in[s];
            }
            float rest[4];
#pragma unroll
            for (int j = 0; j < 4; j++) rest[j] = v[j] * scale;
            // the upper 16 bits of what is left, three times: 24 bits, exact down to 2^-103 (the last part of less may be subnormal)
            uint8_t *to = parts + t * kRow + 2 * r;
#pragma unroll
            for (int h = 0; h < 3; h++) {
                uint32_t part[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    part[j] = __builtin_bit_cast(uint32_t, rest[j]) & 0xffff0000u;
                    rest[j] = fabsf(rest[j]) == __builtin_inff() ? 0.f : rest[j] - __builtin_bit_cast(float, part[j]);
                }
                *reinterpret_cast<uint2 *>(to + (RT > 1 ? 64 * S * h : h == 1 ? 2 * rank : 32 * h)) =
                    make_uint2(part[0] >> 16 | part[1], part[2] >> 16 | part[3]);
            }
        }
        __syncthreads();
        // Tile t: matrix row r of column tile k is column 16 k + r; the results go through LDS into rows.
        auto multiply = [&](int t, const Weights &bv, v4f (&lo)[2], v4f (&hi)[2]) {
            v4f acc[4] = {};
#pragma unroll
            for (int s = 0; s < S; s++) {
#pragma unroll
                for (int h = 0; h < PARTS; h++) {
                    const v8bf v = *reinterpret_cast<const v8bf *>(parts + (16 * t + n) * kRow + 64 * S * h + 64 * s + 16 * q);
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv.v[s][k], v, acc[k], 0, 0, 0);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) *reinterpret_cast<v4f *>(&turned[w][n][16 * k + 4 * q]) = acc[k];
            lds_order();   // (of one wavefront: its LDS accesses complete in order)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                lo[h] = *reinterpret_cast<const v4f *>(&turned[w][8 * h + row][col]);
                hi[h] = *reinterpret_cast<const v4f *>(&turned[w][8 * h + row][col + 4]);
            }
            lds_order();
        };
#pragma unroll 1
        for (int c0 = c_begin; c0 < c_end; c0 += 256) {
            if (c0 > c_begin) load_weights(c0, bv);
            v4f lo[2], hi[2];
            if (c0 + 64 <= p.N) {
                v4w base[T][2];
#pragma unroll
                for (int t = 0; t < T; t++)
#pragma unroll
                    for (int h = 0; h < 2; h++) base[t][h] = load_base(c0, t, h);
#pragma unroll
                for (int t = 0; t < T; t++) {
                    multiply(t, bv, lo, hi);
                    finish(c0, t, same, base[t], lo, hi);
                    __builtin_amdgcn_sched_barrier(0);   // (one tile's registers at a time)
                }
            } else {
#pragma unroll 1
                for (int t = 0; t < T; t++) {
                    multiply(t, bv, lo, hi);
                    finish_ragged(c0, t, same, lo, hi);
                }
            }
        }
    });
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Each kernel's tokens of a tile and workgroups that share a tile's adapters, and the parts of K.  A tile of 64 tokens reads its adapters a
// quarter as often; one of 16 is seldom of two requests, and has less to do one behind the other.  MI355X, us, 16 / 64 tokens in the first
// kernel: 2048 tokens of 64 requests, K = 7168, N = 2112, rank 32 28.8 / 33.5, 3890 of 40, K = 5120, N = 173, rank 64 48 / 40, 7759 of one, K =
// 3200, N = 177, rank 16 22 / 19; in the second: 8192 of 37, K = 2048, N = 7168, rank 64 113 / 85, 3890 of 40 as before 40 / 50.  One workgroup
// to a tile's adapters instead of two to sixteen: 61 tokens of 48 adapters 28 for 13, 8192 of 37 requests 109 for 87 (those a tile has no
// adapters for end at once, but take their turn).
struct AdaptPlan {
    struct Tiles {
        int tokens, sharers;
    } in, out;
    int splits, run;   // parts of K, and 256 columns that a workgroup of the second kernel takes one behind the other
    AdaptPlan(int M, int N, int K, int rank, int adapters)
    {
        auto shared = [&](int tokens) {
            const int64_t tiles = ceil_div(M, tokens);
            int64_t n = tiles < 32 ? ceil_div(128, tiles) : tokens == 16 && tiles >= 96 ? 2 : 4;
            for (const int most : {adapters, tokens, M}) n = n < most ? n : most;
            return Tiles{tokens, (int)n};
        };
        in = shared((int64_t)M * rank > 65536 ? 64 : 16);
        out = shared(M <= 2048 || N <= 1024 ? 16 : rank > 64 ? 32 : 64);
        const int64_t groups = ceil_div(M, in.tokens) * in.sharers, can = ceil_div(K / 128, 4);
        int64_t want = in.tokens == 16 ? (groups <= 512 ? 8 : 4) : ceil_div(1024, groups);
        if (in.tokens == 64 && M > 2048 && want > 4) want = 4;
        splits = (int)(want > can ? can : want);
        const int64_t pieces = ceil_div(N, 256) * ceil_div(M, out.tokens) / 1536;   // 256 columns of a tile
        run = pieces < 1 ? 1 : pieces > 4 ? 4 : (int)pieces;
    }
};

template <typename... Args>
hipError_t launch(void (*kernel)(Args...), dim3 grid, dim3 block, hipStream_t stream, Args... args)
{
    void *list[] = {&args...};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, list, 0, stream);
}

// The workgroups of a kernel with `each` times `sharers` to a tile.
int64_t workgroups(const AdaptParams &p, const AdaptPlan::Tiles &tiles, int64_t each)
{
    return 8 * ceil_div(ceil_div(p.M, tiles.tokens) * each, 8) * tiles.sharers;
}

hipError_t launch_tiles(void (*kernel)(AdaptParams), AdaptParams p, const AdaptPlan::Tiles &tiles, int64_t each, hipStream_t hs)
{
    p.tiles = (int)ceil_div(p.M, tiles.tokens), p.sharers = tiles.sharers;
    return launch(kernel, dim3((unsigned)workgroups(p, tiles, each)), dim3(256), hs, p);
}

// Of many ranks, each workgroup of the first kernel takes a group: 32 of few tokens, whose parts are little work for many units (44 tokens,
// K = 4736, N = 1357, rank 128 15 us in one, 11.5 in four), 64 of many, so that 64 tokens' sums fit the registers.
template <int RT>
hipError_t adapt(AdaptParams p, const AdaptPlan &plan, hipStream_t hs)
{
    constexpr int kFew = RT < 2 ? RT : 2, kMany = RT < 4 ? RT : 4, kOut = RT == 8 ? 2 : 4;
    const bool many = plan.in.tokens == 64, fp8 = p.x_scale != nullptr;
    p.rank_groups = (int)ceil_div(p.rank, 16 * (many ? kMany : kFew));
    p.pieces = (int)ceil_div(p.N, 256 * (int64_t)p.run);
    const auto in = many ? (fp8 ? adapt_in_kernel<kMany, 4, true> : adapt_in_kernel<kMany, 4, false>)
                         : (fp8 ? adapt_in_kernel<kFew, 1, true> : adapt_in_kernel<kFew, 1, false>);
    const auto out = plan.out.tokens == 16 ? adapt_out_kernel<RT, 1> : adapt_out_kernel<RT, kOut>;
    const int64_t of_in = (int64_t)p.splits * p.rank_groups, most = (int64_t(1) << 32) / 256;
    if (workgroups(p, plan.in, of_in) >= most || workgroups(p, plan.out, p.pieces) >= most)
        return hipErrorInvalidConfiguration;   // (a launch has less than 2^32 threads)
    const hipError_t err = launch_tiles(in, p, plan.in, of_in, hs);
    return err != hipSuccess ? err : launch_tiles(out, p, plan.out, p.pieces, hs);
}

bool sizes_fit(int M, int N, int K, int rank, int adapters)
{
    return M >= 0 && N > 0 && K > 0 && K % 128 == 0 && K <= 128 * kMaxKBlocks && rank > 0 && rank % 8 == 0 && rank <= kMaxRank &&
           adapters > 0 && M <= 16 * 65535 && N <= (1 << 24);
}

}  // namespace
}  // namespace alpha_moe

using namespace alpha_moe;

extern "C" size_t alpha_moe_adapters_workspace_bytes(int M, int N, int K, int rank, int num_adapters)
{
    if (M <= 0 || !sizes_fit(M, N, K, rank, num_adapters)) return 0;
    return (size_t)AdaptPlan(M, N, K, rank, num_adapters).splits * M * rank * sizeof(float);
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
        workspace_bytes < alpha_moe_adapters_workspace_bytes(M, N, K, rank, num_adapters))
        return ALPHA_MOE_ERR_WORKSPACE;
    const AdaptPlan plan(M, N, K, rank, num_adapters);
    AdaptParams p = {};
    p.base = base, p.a = a, p.b = b, p.x = static_cast<const uint8_t *>(x), p.x_scale = x_scale, p.scale = scale;
    p.ids = adapter_ids, p.out = out, p.part = static_cast<float *>(workspace);
    p.M = M, p.N = N, p.K = K, p.rank = rank, p.adapters = num_adapters, p.nkb = K / 128;
    p.splits = plan.splits, p.run = plan.run;
    hipStream_t hs = static_cast<hipStream_t>(stream);
    const hipError_t err = rank <= 16   ? adapt<1>(p, plan, hs)
                           : rank <= 32 ? adapt<2>(p, plan, hs)
                           : rank <= 64 ? adapt<4>(p, plan, hs)
                                        : adapt<8>(p, plan, hs);
    return err == hipSuccess ? ALPHA_MOE_OK : err == hipErrorInvalidConfiguration ? ALPHA_MOE_ERR_SHAPE : ALPHA_MOE_ERR_LAUNCH;
}

extern "C" int alpha_moe_adapters_plan(int M, int N, int K, int rank, int num_adapters, int plan[6])
{
    if (M <= 0 || !sizes_fit(M, N, K, rank, num_adapters)) return ALPHA_MOE_ERR_SHAPE;
    const AdaptPlan a(M, N, K, rank, num_adapters);
    const int values[6] = {a.in.tokens, a.in.sharers, a.out.tokens, a.out.sharers, a.splits, a.run};
    for (int i = 0; i < 6; i++) plan[i] = values[i];
    return ALPHA_MOE_OK;
}
