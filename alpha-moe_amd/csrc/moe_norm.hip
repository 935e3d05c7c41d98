// The two operators that write FP8 activations for a product that follows: the RMS norm (with the residual's addition in front of
// it) and the SwiGLU between the two products of a dense layer.
//
//   norm:    h = x (+ residual), r = 1 / sqrt(mean(h^2) + eps), y = h r weight
//   swiglu:  y = g / (1 + exp(-g)) u of a row [g | u]
//   both:    per group of 128 columns scale = max(max|y|, 1e-10) / 448, q = e4m3(clamp(y / scale, +-448))
//
// Everything between the loads and the stores is fp32: h and y are rounded once each, where they are stored (the residual stream
// and, if asked for, the normalised row in x's type; the codes from y itself, not from its rounded copy).
//
// A NaN makes its group's scale and codes NaN (the maxima are taken over the bits of |y|, where a NaN is larger than anything), so
// what was lost upstream stays visible behind the product.
//
// Both are bound by memory, or by the launch: MI355X, bf16, 8192 x 7168 with a residual 72.5 us (411 MB, 5.7 TB/s; a copy of a GiB 5.1),
// 1 x 7168 3.0 us, SwiGLU of 8192 x 2 x 2048 14.0 us (84 MB, some of it from the last-level cache), 7 x 2 x 768 1.9; an empty call 2.2.
// The norm's rows stay in registers, so that a row is read once; a group's maximum takes a few data-parallel steps in registers
// (through shuffles, with a second pass over the row for the codes, the two took 76 and 19 us).  Above 32768 columns this holds for bf16
// rows and weights only: a lane of 1024 threads has 128 registers, and what fp32 rows (or fp32 weights of bf16 rows) need beyond
// goes to scratch memory, 348 to 476 (136) bytes a lane.  1024 rows with a residual: bf16 of 32768, 65536 columns 42, 107 us, with a fp32
// weight 144; fp32 98, 337 (5.6, 4.4, 3.3, 4.5, 2.6 TB/s).
#include "moe_common.hpp"

namespace alpha_moe {
namespace {

// What a lane loads at a time: N values in 16 bytes (of a row of another type than the activations', the same N values).
template <typename T>
struct Lane;
template <>
struct Lane<uint16_t> {
    static constexpr int N = 8;
};
template <>
struct Lane<float> {
    static constexpr int N = 4;
};

template <typename T, int N>
struct Raw {
    static constexpr int kBytes = N * (int)sizeof(T);   // 8, 16 or 32
    static constexpr int kWords = kBytes < 16 ? kBytes / 4 : 4;
    typedef uint32_t Piece __attribute__((ext_vector_type(kWords)));
    Piece piece[kBytes / (4 * kWords)];
    __device__ __forceinline__ void load(const void *p, size_t at)
    {
#pragma unroll
        for (int i = 0; i < kBytes / (4 * kWords); i++) piece[i] = reinterpret_cast<const Piece *>(static_cast<const T *>(p) + at)[i];
    }
    __device__ __forceinline__ void store(void *p, size_t at) const
    {
#pragma unroll
        for (int i = 0; i < kBytes / (4 * kWords); i++) reinterpret_cast<Piece *>(static_cast<T *>(p) + at)[i] = piece[i];
    }
    __device__ __forceinline__ float value(int i) const
    {
        // (a copy first: the builtin takes element 0 of a vector for any element of it)
        const uint32_t word = sizeof(T) == 4 ? piece[i / 4][i % 4] : piece[0][i / 2];
        return __builtin_bit_cast(float, sizeof(T) == 4 ? word : i % 2 ? word & 0xffff0000u : word << 16);
    }
    __device__ __forceinline__ explicit Raw(const float (&v)[N])
    {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (sizeof(T) == 4) piece[i / 4][i % 4] = __builtin_bit_cast(uint32_t, v[i]);
            else if (i % 2 == 0) piece[0][i / 2] = pack_bf16x2(v[i], v[i + 1]);
        }
    }
    Raw() = default;
};

__device__ __forceinline__ float wave_sum(float v)   // in lane 63
{
#define NORM_STEP(ctrl, rows) \
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, false))
    NORM_STEP(0x111, 0xf);   // from 1, 2, 4, 8 lanes below in the row
    NORM_STEP(0x112, 0xf);
    NORM_STEP(0x114, 0xf);
    NORM_STEP(0x118, 0xf);
    NORM_STEP(0x142, 0xa);   // lane 15 of rows 0 and 2 to rows 1 and 3
    NORM_STEP(0x143, 0xc);   // lane 31 to rows 2 and 3
#undef NORM_STEP
    return v;
}

// The largest of the 16 or 32 lanes of a group, in all of them.
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t m)
{
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, false));    // lanes 1, 0, 3, 2
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, false));    // lanes 2, 3, 0, 1
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, false));   // mirrored in eight
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xf, 0xf, false));   // mirrored in sixteen
    if constexpr (LANES == 32) m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    return m;
}

// The codes of N values of a lane whose group of 128 is held by 128 / N neighbouring lanes; every lane of the group calls it.
template <int N>
struct GroupQuant {
    float scale;
    uint32_t code[N / 4];
    __device__ __forceinline__ explicit GroupQuant(const float (&y)[N])
    {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; i++) m = max(m, __builtin_bit_cast(uint32_t, y[i]) & 0x7fffffffu);
        m = group_max<128 / N>(m);
        scale = m < 0x7f800000u ? fmaxf(__builtin_bit_cast(float, m), kAmaxFloor) / kFp8Max : __builtin_bit_cast(float, m);
        if (m < 0x7f800000u) {
            float r = __builtin_amdgcn_rcpf(scale);
            r = __builtin_fmaf(__builtin_fmaf(-scale, r, 1.0f), r, r);
            auto one = [&](float v) { return clamp_fp8(divide(v, scale, r)); };
#pragma unroll
            for (int i = 0; i < N / 4; i++) code[i] = pack_fp8x4(one(y[4 * i]), one(y[4 * i + 1]), one(y[4 * i + 2]), one(y[4 * i + 3]));
        } else {   // an infinity over an infinite scale is NaN, a finite value 0; everything over NaN is NaN
            const bool nan = m > 0x7f800000u;
#pragma unroll
            for (int i = 0; i < N / 4; i++) {
                code[i] = 0;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (nan || !(fabsf(y[4 * i + j]) < __builtin_inff())) code[i] |= 0x7fu << (8 * j);
            }
        }
    }
    __device__ __forceinline__ void store(uint8_t *q, size_t at) const
    {
        if constexpr (N == 8) *reinterpret_cast<uint2 *>(q + at) = make_uint2(code[0], code[1]);
        else *reinterpret_cast<uint32_t *>(q + at) = code[0];
    }
};

struct NormParams {
    const void *x, *residual, *weight;
    void *residual_out, *norm_out;
    uint8_t *q;
    float *scale;
    float eps;
    int M, K;
};

// One workgroup to a row, which stays in registers between its sum of squares and its codes (for the longest rows see above): P
// pieces of 16 bytes a thread, all loads of them in flight at once (pieces behind the row's end: its last one again, and not used).
template <typename T, typename W, int P>
__global__ __launch_bounds__(1024) void rms_norm_kernel(const NormParams s)
{
    constexpr int N = Lane<T>::N;
    __shared__ float sums[16];
    const int K = s.K, tid = threadIdx.x, step = (int)blockDim.x * N;
    const size_t row = (size_t)blockIdx.x * K;
    Raw<T, N> x[P], add[P];
    Raw<W, N> weight[P];
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = min(p * step + tid * N, K - N);
        x[p].load(s.x, row + c);
        if (s.residual) add[p].load(s.residual, row + c);
    }
#pragma unroll
    for (int p = 0; p < P; p++) weight[p].load(s.weight, min(p * step + tid * N, K - N));
    float h[P][N];
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = p * step + tid * N;
#pragma unroll
        for (int i = 0; i < N; i++) h[p][i] = x[p].value(i);
        if (s.residual) {
#pragma unroll
            for (int i = 0; i < N; i++) h[p][i] += add[p].value(i);
            if (c < K) Raw<T, N>(h[p]).store(s.residual_out, row + c);
        }
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) part += h[p][i] * h[p][i];
        sum += c < K ? part : 0.f;
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 63) sums[tid >> 6] = sum;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < (int)blockDim.x >> 6; w++) sum += sums[w];
    const float r = 1.0f / sqrtf(sum / (float)K + s.eps);
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = p * step + tid * N;
        if (c < K) {   // (a group's lanes agree)
            float y[N];
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = h[p][i] * r * weight[p].value(i);
            if (s.norm_out) Raw<T, N>(y).store(s.norm_out, row + c);
            const GroupQuant<N> g(y);
            g.store(s.q, row + c);
            if ((c & 127) == 0) s.scale[(row + c) >> 7] = g.scale;
        }
    }
}

// g / (1 + exp(-g)) within (1.25 |g| + 9) roundings: the exponent's counts 1.25 |g|, the others one or two each.  The reciprocal is of
// a quarter of 1 + exp(-g): where that is infinite the result is g * 0, and elsewhere it is a normal number.
__device__ __forceinline__ float silu(float g)
{
    const float den = __builtin_fmaf(__builtin_amdgcn_exp2f(g * -1.44269504f), 0.25f, 0.25f);
    return 0.25f * g * __builtin_amdgcn_rcpf(den);
}

template <typename T>
__global__ __launch_bounds__(256) void swiglu_kernel(const void *gate_up, uint8_t *q, float *scale, int I, long long n_groups)
{
    constexpr int N = Lane<T>::N, LANES = 128 / N;
    const int sub = threadIdx.x % LANES;
    const int per_row = I >> 7;
    const long long stride = (long long)gridDim.x * (256 / LANES);
    for (long long g = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; g < n_groups; g += stride) {
        const long long row = g / per_row;
        const size_t at = (size_t)row * 2 * I + (size_t)(g - row * per_row) * 128 + sub * N;
        Raw<T, N> gate, up;
        gate.load(gate_up, at);
        up.load(gate_up, at + I);
        float a[N];
#pragma unroll
        for (int i = 0; i < N; i++) a[i] = silu(gate.value(i)) * up.value(i);
        const GroupQuant<N> c(a);
        c.store(q, (size_t)g * 128 + sub * N);
        if (sub == 0) scale[g] = c.scale;
    }
}

template <typename T, typename W>
hipError_t launch_norm(const NormParams &s, hipStream_t stream)
{
    const int pieces = s.K / Lane<T>::N;
    typedef void (*Fn)(const NormParams);
    Fn fn;
    int per;
    // (one piece a thread: 8192 x 7168 bf16 79 us, two 73, four 75; up to 512 threads the first is as good or better: 64 x 4096 3.3, 3.4)
    if (pieces <= 512) fn = rms_norm_kernel<T, W, 1>, per = 1;
    else if (pieces <= 2048) fn = rms_norm_kernel<T, W, 2>, per = 2;
    else if (pieces <= 4096) fn = rms_norm_kernel<T, W, 4>, per = 4;
    else if (sizeof(T) == 2 || pieces <= 8192) fn = rms_norm_kernel<T, W, 8>, per = 8;   // (K is 65536 at most)
    else if constexpr (sizeof(T) == 4) fn = rms_norm_kernel<T, W, 16>, per = 16;
    const int threads = ((pieces + per - 1) / per + 63) & ~63;
    void *args[] = {const_cast<NormParams *>(&s)};
    return hipLaunchKernel(reinterpret_cast<const void *>(fn), dim3((unsigned)s.M), dim3((unsigned)threads), args, 0, stream);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace alpha_moe

extern "C" int alpha_moe_rms_norm_quant_fp8(const void *x, const void *residual, const void *weight, int x_is_f32,
                                            int weight_is_f32, float eps, uint8_t *q, float *scale, void *residual_out,
                                            void *norm_out, int M, int K, void *stream)
{
    using namespace alpha_moe;
    if (M < 0 || M >= 1 << 22 || K <= 0 || K % 128 != 0 || K > 128 * kMaxKBlocks) return ALPHA_MOE_ERR_SHAPE;   // (2^32 threads a launch)
    if (M == 0) return ALPHA_MOE_OK;
    if (!x || !weight || !q || !scale || !residual != !residual_out) return ALPHA_MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(q) || !aligned16(residual_out) ||
        !aligned16(norm_out))
        return ALPHA_MOE_ERR_ALIGNMENT;
    const NormParams s = {x, residual, weight, residual_out, norm_out, q, scale, eps, M, K};
    hipStream_t hs = static_cast<hipStream_t>(stream);
    hipError_t err;
    if (x_is_f32) err = weight_is_f32 ? launch_norm<float, float>(s, hs) : launch_norm<float, uint16_t>(s, hs);
    else err = weight_is_f32 ? launch_norm<uint16_t, float>(s, hs) : launch_norm<uint16_t, uint16_t>(s, hs);
    return err == hipSuccess ? ALPHA_MOE_OK : ALPHA_MOE_ERR_LAUNCH;
}

extern "C" int alpha_moe_swiglu_quant_fp8(const void *gate_up, int is_f32, uint8_t *q, float *scale, int M, int I, void *stream)
{
    using namespace alpha_moe;
    if (M < 0 || I <= 0 || I % 128 != 0 || I > INT32_MAX / 2) return ALPHA_MOE_ERR_SHAPE;
    if (M == 0) return ALPHA_MOE_OK;
    if (!gate_up || !q || !scale) return ALPHA_MOE_ERR_NULL_POINTER;
    if (!aligned16(gate_up) || !aligned16(q)) return ALPHA_MOE_ERR_ALIGNMENT;
    const long long n_groups = (long long)M * (I >> 7);
    const long long blocks = (n_groups + (is_f32 ? 7 : 15)) / (is_f32 ? 8 : 16);
    const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
    void *args[] = {&gate_up, &q, &scale, &I, const_cast<long long *>(&n_groups)};
    const void *fn = is_f32 ? reinterpret_cast<const void *>(swiglu_kernel<float>)
                            : reinterpret_cast<const void *>(swiglu_kernel<uint16_t>);
    return hipLaunchKernel(fn, dim3(grid), dim3(256), args, 0, static_cast<hipStream_t>(stream)) == hipSuccess
               ? ALPHA_MOE_OK : ALPHA_MOE_ERR_LAUNCH;
}
