// The router's selection: from a token's logits of E experts the top_k experts and their weights, in the form the aligner and the
// fused operator take.
//
//   score  s = softmax(l) or sigmoid(l)
//   choice c = s + bias in 64 bits, or l itself without a bias (s is monotonic in l, but rounds different logits to one score)
//   groups   num_groups runs of E / num_groups experts, valued by the sum of their two best choices (with a bias) or by their best
//            one; the experts of the top_groups best groups stay, the others are out
//   result   the top_k best of the experts that stay, in descending order; weights s, divided by their sum if renormalised;
//            behind them the fused shared experts E, E + 1, ... with a weight of their own
//
// Of equal choices, and of equal groups, the lower index comes first.  The order is decided in 64 bits: of 256 experts' scores two
// neighbours are closer than fp32 tells in one token of a few thousand, and which expert a token visits is not a rounding.
//
// A NaN choice ranks as -infinity.  Every id is a valid one whatever the logits hold; a row with a NaN logit has NaN weights, a row
// without scores (every chosen logit -infinity) weights of 0.
//
// One wavefront to a token.  Lane l holds the V experts l V .. l V + V - 1, so that the lowest lane of several with the same value
// has the lowest expert.
#include "moe_common.hpp"

namespace alpha_moe {
namespace {

struct RouteParams {
    const void *logits;
    const float *bias;
    float *weights;
    int32_t *ids;
    int M, E, top_k, num_groups, top_groups, shared;
    float shared_weight;
    int sigmoid, renormalize;
};

constexpr int kRouteMaxExperts = 4096;
constexpr int kRouteMaxTopK = 64;     // a lane each
constexpr int kRouteMaxGroups = 64;

template <typename C>
__device__ __forceinline__ C wave_max(C v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const C o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

template <typename T>
__device__ __forceinline__ float logit_at(const void *p, size_t at)
{
    if constexpr (sizeof(T) == 4) return static_cast<const float *>(p)[at];
    else return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t *>(p)[at] << 16);
}

// C: the type of a choice, float without a bias and double with one.
template <typename T, typename C, int V>
__global__ __launch_bounds__(64) void route_kernel(const RouteParams s)
{
    constexpr bool BIAS = sizeof(C) == 8;
    const C lowest = -(C)__builtin_inff();
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x;
    const int E = s.E, e0 = lane * V;
    const size_t row = (size_t)blockIdx.x * E;

    float l[V];
    C c[V];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; v++) {
        l[v] = e0 + v < E ? logit_at<T>(s.logits, row + e0 + v) : -__builtin_inff();
        nan |= l[v] != l[v];
    }
    const bool any_nan = __ballot(nan) != 0;

    float top = -__builtin_inff();   // the softmax's largest logit and sum, over all experts
    double total = 1.0;
    if (!s.sigmoid) {
#pragma unroll
        for (int v = 0; v < V; v++) top = l[v] > top ? l[v] : top;
        top = wave_max(top);
        if (BIAS || !s.renormalize) {
            double sum = 0.0;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (l[v] > -__builtin_inff()) sum += exp((double)l[v] - (double)top);
            total = wave_sum(sum);
        }
    }
    auto score = [&](float x) {   // in 64 bits; before the renormalisation
        if (s.sigmoid) return 1.0 / (1.0 + exp(-(double)x));
        if (x == -__builtin_inff()) return 0.0;
        return exp((double)x - (double)top) / total;
    };
    unsigned long long out_of = 0;   // experts that are out: not there, in a group that is, or chosen already
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (e0 + v >= E) out_of |= 1ull << v;
        if constexpr (BIAS) c[v] = e0 + v < E ? score(l[v]) + (double)s.bias[e0 + v] : lowest;
        else c[v] = l[v];
        if (!(c[v] == c[v])) c[v] = lowest;
    }

    if (s.num_groups > 1) {
        C *all = reinterpret_cast<C *>(lds);
#pragma unroll
        for (int v = 0; v < V; v++)
            if (e0 + v < E) all[e0 + v] = c[v];
        __syncthreads();
        const int size = E / s.num_groups;
        C first = lowest, second = lowest;
        if (lane < s.num_groups)
            for (int i = 0; i < size; i++) {
                const C x = all[lane * size + i];
                if (x > first) second = first, first = x;
                else if (x > second) second = x;
            }
        C value = BIAS && size > 1 ? first + second : first;
        if (!(value == value)) value = lowest;   // (+infinity and -infinity)
        int ahead = 0;
        for (int g = 0; g < s.num_groups; g++) {
            const C o = __shfl(value, g);
            ahead += o > value || (o == value && g < lane);
        }
        const unsigned long long stay = __ballot(lane < s.num_groups && ahead < s.top_groups);
#pragma unroll
        for (int v = 0; v < V; v++)
            if (e0 + v < E && !((stay >> ((e0 + v) / size)) & 1)) out_of |= 1ull << v;
    }

    int my_id = 0;
    float my_logit = 0.f;
    for (int k = 0; k < s.top_k; k++) {
        C best = lowest;
        int at = -1;
#pragma unroll
        for (int v = V - 1; v >= 0; v--)
            if (!((out_of >> v) & 1) && (at < 0 || c[v] >= best)) best = c[v], at = v;
        const C m = wave_max(best);
        const int src = __builtin_ctzll(__ballot(at >= 0 && best == m));   // (top_k experts stay: there is one)
        float x = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v == at) x = l[v];
        const int id = __shfl(e0 + at, src);
        x = __shfl(x, src);
        if (lane == src) out_of |= 1ull << at;
        if (lane == k) my_id = id, my_logit = x;
    }

    double w = lane < s.top_k ? score(my_logit) : 0.0;
    if (s.renormalize) {
        const double sum = wave_sum(w);
        w = sum != 0.0 ? w / sum : 0.0;
    }
    const int kept = s.top_k + s.shared;
    const size_t out = (size_t)blockIdx.x * kept;
    if (lane < s.top_k) {
        s.weights[out + lane] = any_nan ? __builtin_nanf("") : (float)w;
        s.ids[out + lane] = my_id;
    }
    for (int i = lane; i < s.shared; i += 64) {
        s.weights[out + s.top_k + i] = s.shared_weight;
        s.ids[out + s.top_k + i] = E + i;
    }
}

typedef void (*RouteFn)(const RouteParams);
template <typename T, typename C>
RouteFn route_variant(int E)
{
    if (E <= 64) return route_kernel<T, C, 1>;
    if (E <= 128) return route_kernel<T, C, 2>;
    if (E <= 256) return route_kernel<T, C, 4>;
    if (E <= 512) return route_kernel<T, C, 8>;
    if (E <= 1024) return route_kernel<T, C, 16>;
    return route_kernel<T, C, 64>;
}

}  // namespace
}  // namespace alpha_moe

extern "C" int alpha_moe_route_topk(const void *logits, int is_f32, const float *bias, float *topk_weights, int32_t *topk_ids,
                                    int M, int E, int top_k, int sigmoid, int num_groups, int top_groups, int renormalize,
                                    int shared_experts, float shared_weight, void *stream)
{
    using namespace alpha_moe;
    if (M < 0 || E <= 0 || E > kRouteMaxExperts || top_k <= 0 || top_k > kRouteMaxTopK || num_groups <= 0 ||
        num_groups > kRouteMaxGroups || E % num_groups != 0 || top_groups <= 0 || top_groups > num_groups ||
        top_k > top_groups * (E / num_groups) || shared_experts < 0 || shared_experts > kRouteMaxExperts)
        return ALPHA_MOE_ERR_SHAPE;
    if (M == 0) return ALPHA_MOE_OK;
    if (!logits || !topk_weights || !topk_ids) return ALPHA_MOE_ERR_NULL_POINTER;
    const RouteParams s = {logits, bias, topk_weights, topk_ids, M, E, top_k, num_groups, top_groups, shared_experts,
                           shared_weight, sigmoid != 0, renormalize != 0};
    const RouteFn fn = is_f32 ? (bias ? route_variant<float, double>(E) : route_variant<float, float>(E))
                              : (bias ? route_variant<uint16_t, double>(E) : route_variant<uint16_t, float>(E));
    const size_t lds = num_groups > 1 ? (size_t)E * (bias ? 8 : 4) : 0;
    void *args[] = {const_cast<RouteParams *>(&s)};
    return hipLaunchKernel(reinterpret_cast<const void *>(fn), dim3((unsigned)M), dim3(64), args, lds,
                           static_cast<hipStream_t>(stream)) == hipSuccess ? ALPHA_MOE_OK : ALPHA_MOE_ERR_LAUNCH;
}
