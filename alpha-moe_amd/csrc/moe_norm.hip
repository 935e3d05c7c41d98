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
#include "moe_common.hpp"

namespace alpha_moe {
namespace {

template <typename T>
struct Lane;   // what a lane loads at a time: 16 bytes
template <>
struct Lane<uint16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const void *p, size_t at, float (&v)[N])
    {
        const v4i raw = *reinterpret_cast<const v4i *>(static_cast<const uint16_t *>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __builtin_bit_cast(float, (uint32_t)raw[i] << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, (uint32_t)raw[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(void *p, size_t at, const float (&v)[N])
    {
        v4i raw;
#pragma unroll
        for (int i = 0; i < 4; i++) raw[i] = (int)pack_bf16x2(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<v4i *>(static_cast<uint16_t *>(p) + at) = raw;
    }
};
template <>
struct Lane<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const void *p, size_t at, float (&v)[N])
    {
        const v4f raw = *reinterpret_cast<const v4f *>(static_cast<const float *>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = raw[i];
    }
    static __device__ __forceinline__ void store(void *p, size_t at, const float (&v)[N])
    {
        *reinterpret_cast<v4f *>(static_cast<float *>(p) + at) = (v4f){v[0], v[1], v[2], v[3]};
    }
};

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
#pragma unroll
        for (int d = 1; d < 128 / N; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
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

// N values of a row of another type than the activations'
template <typename W, int N>
__device__ __forceinline__ void load_weight(const void *p, int at, float (&v)[N])
{
    if constexpr (Lane<W>::N == N) {
        Lane<W>::load(p, at, v);
    } else if constexpr (sizeof(W) == 4) {
        float lo[4], hi[4];
        Lane<W>::load(p, at, lo);
        Lane<W>::load(p, at + 4, hi);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = lo[i], v[4 + i] = hi[i];
    } else {
        const uint2 raw = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
        v[0] = __builtin_bit_cast(float, raw.x << 16);
        v[1] = __builtin_bit_cast(float, raw.x & 0xffff0000u);
        v[2] = __builtin_bit_cast(float, raw.y << 16);
        v[3] = __builtin_bit_cast(float, raw.y & 0xffff0000u);
    }
}

struct NormParams {
    const void *x, *residual, *weight;
    void *residual_out, *norm_out;
    uint8_t *q;
    float *scale;
    float eps;
    int M, K;
};

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// One workgroup to a row, which stays in registers between its sum of squares and its codes: P pieces of 16 bytes a thread.
template <typename T, typename W, int P>
__global__ __launch_bounds__(1024) void rms_norm_kernel(const NormParams s)
{
    constexpr int N = Lane<T>::N;
    __shared__ float sums[16];
    const int K = s.K, tid = threadIdx.x;
    const size_t row = (size_t)blockIdx.x * K;
    float h[P][N];
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (p * (int)blockDim.x + tid) * N;
        if (c < K) {
            Lane<T>::load(s.x, row + c, h[p]);
            if (s.residual) {
                float add[N];
                Lane<T>::load(s.residual, row + c, add);
#pragma unroll
                for (int i = 0; i < N; i++) h[p][i] += add[i];
                Lane<T>::store(s.residual_out, row + c, h[p]);
            }
#pragma unroll
            for (int i = 0; i < N; i++) sum += h[p][i] * h[p][i];
        }
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) sums[tid >> 6] = sum;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < (int)blockDim.x >> 6; w++) sum += sums[w];
    const float r = 1.0f / sqrtf(sum / (float)K + s.eps);
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (p * (int)blockDim.x + tid) * N;
        if (c < K) {   // (a group's lanes agree)
            float y[N];
            load_weight<W>(s.weight, c, y);
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = h[p][i] * r * y[i];
            if (s.norm_out) Lane<T>::store(s.norm_out, row + c, y);
            const GroupQuant<N> g(y);
            g.store(s.q, row + c);
            if ((c & 127) == 0) s.scale[(row + c) >> 7] = g.scale;
        }
    }
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
        float a[N], u[N];
        Lane<T>::load(gate_up, at, a);
        Lane<T>::load(gate_up, at + I, u);
#pragma unroll
        for (int i = 0; i < N; i++) a[i] = a[i] / (1.0f + expf(-a[i])) * u[i];
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
    if (pieces <= 1024) fn = rms_norm_kernel<T, W, 1>, per = 1;
    else if (pieces <= 2048) fn = rms_norm_kernel<T, W, 2>, per = 2;
    else if (pieces <= 4096) fn = rms_norm_kernel<T, W, 4>, per = 4;
    else if (pieces <= 8192) fn = rms_norm_kernel<T, W, 8>, per = 8;
    else fn = rms_norm_kernel<T, W, 16>, per = 16;
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
    if (M < 0 || K <= 0 || K % 128 != 0 || K > 128 * kMaxKBlocks) return ALPHA_MOE_ERR_SHAPE;
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
