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
// A NaN choice ranks as -infinity.  Every id is a valid one whatever the logits hold; a row with a NaN logit, or with +infinity in a
// softmax, has NaN weights, a row without scores (every chosen logit -infinity) weights of 0.  Scores up to e^-700, which masks make
// rather than routers, are 0.  Above, renormalised weights keep their ratio also where fp32 has no numbers for the scores: where the
// chosen ones' sum is below 2^-24 they are exp(l - the largest chosen l), which is a softmax's ratio exactly and a sigmoid's but for its
// factor 1 + exp(l) < 1 + 2^-24.
//
// One wavefront to a token.  Lane l holds the V experts l V .. l V + V - 1, so that the lowest lane of several with the same value
// has the lowest expert.  What bounds it is instructions, one dependent chain of them per token, so:
//   * choices become unsigned keys of the same order (an expert that is out has key 0, below every other), whose maximum over the
//     wavefront is six data-parallel steps of one instruction each;
//   * a group's lanes put their two best together in as many steps as their number has bits;
//   * with a bias, choices are taken in fp32 first.  Where the last group that stays, or any two neighbours of the result, are
//     closer than fp32 can be off, the groups or the neighbours are decided again in 64 bits (in some ten of 8192 tokens).
// MI355X, 8192 tokens of 256 experts, the 8 best of 4 of 8 groups, fp32 logits, sigmoid and bias 9.7 us (softmax without a bias or
// groups 5.8; 2.2 are an empty call's); one token 4.3.  With all choices in 64 bits 15.1; with maxima of doubles through LDS as well
// and one lane's walk over each group 24 and, for one token, 8.9.
// Many experts are served, but not fast: 1025 to 4096 take one variant with 64 of them a lane, which with a bias fills 256 registers, keeps
// 300 bytes a lane in scratch memory and runs one wavefront a SIMD.  8192 tokens, the 8 best of all: 1024 experts softmax with a bias 35 us;
// 2048 softmax with a bias 295, sigmoid with a bias 212; 4096 softmax with a bias 290, without 170; one token of 2048 20.
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
    int vector;       // rows of logits and bias can be loaded in pieces of a lane's experts
    int group_lanes;  // lanes that hold a group between them, a power of two; 0: a group does not begin and end with lanes
};

constexpr int kRouteMaxExperts = 4096;
constexpr int kRouteMaxTopK = 64;     // a lane each
constexpr int kRouteMaxGroups = 64;
constexpr int kRouteWaves = 4;        // most tokens of a workgroup
constexpr float kNoScore = -700.f;    // a score of its exponential, or less, is 0

// The largest value of the wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#define ROUTE_STEP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    ROUTE_STEP(0x111, 0xf);   // from 1, 2, 4, 8 lanes below in the row
    ROUTE_STEP(0x112, 0xf);
    ROUTE_STEP(0x114, 0xf);
    ROUTE_STEP(0x118, 0xf);
    ROUTE_STEP(0x142, 0xa);   // lane 15 of rows 0 and 2 to rows 1 and 3
    ROUTE_STEP(0x143, 0xc);   // lane 31 to rows 2 and 3
#undef ROUTE_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// The sum of f(0) .. f(V - 1), halves first: none of them passes more than log2 V additions.
template <int V, int FROM = 0, typename F>
__device__ __forceinline__ float tree_sum(F f)
{
    if constexpr (V == 1) return f(FROM);
    else return tree_sum<V / 2, FROM>(f) + tree_sum<V / 2, FROM + V / 2>(f);
}

// An unsigned number of the same order; a NaN is -infinity, and the two zeros are one.
__device__ __forceinline__ uint32_t order_key(float v)
{
    v = v == v ? v + 0.0f : -__builtin_inff();
    const int b = __builtin_bit_cast(int, v);
    return (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v)
{
    v = v == v ? v + 0.0 : -__builtin_inf();
    const int64_t b = __builtin_bit_cast(int64_t, v);
    return (uint64_t)b ^ ((uint64_t)(b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double from_key(uint64_t k)   // (key 0: NaN)
{
    return __builtin_bit_cast(double, k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull));
}

// What the lane at a distance of d (a power of two) holds, where the lanes of each run of d hold the same.
__device__ __forceinline__ uint32_t other_half(uint32_t v, int d)
{
    if (d == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false);    // lanes 1, 0, 3, 2
    if (d == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false);    // lanes 2, 3, 0, 1
    if (d == 4) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false);   // mirrored in eight
    if (d == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false);   // mirrored in sixteen
    return (uint32_t)__shfl_xor((int)v, d);
}
__device__ __forceinline__ uint64_t other_half(uint64_t v, int d)
{
    return (uint64_t)other_half((uint32_t)(v >> 32), d) << 32 | other_half((uint32_t)v, d);
}
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int l)
{
    return (uint64_t)of_lane((uint32_t)(v >> 32), l) << 32 | of_lane((uint32_t)v, l);
}

template <typename T>
__device__ __forceinline__ float logit_at(const void *p, size_t at)
{
    if constexpr (sizeof(T) == 4) return static_cast<const float *>(p)[at];
    else return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t *>(p)[at] << 16);
}

// V values from element `at` on; those from `end` on are -infinity.
template <typename T, int V>
__device__ __forceinline__ void load_run(const void *p, size_t at, int e0, int end, bool vector, float (&v)[V])
{
    const T *from = static_cast<const T *>(p) + at;
    alignas(16) T raw[V];
    if (vector) {
        if (e0 < end) {   // (then all V are there, at a multiple of their size)
            constexpr int bytes = V * (int)sizeof(T);
            typedef uint32_t Piece __attribute__((ext_vector_type(bytes >= 16 ? 4 : bytes >= 8 ? 2 : 1)));
            if constexpr (bytes >= 4) {
#pragma unroll
                for (int i = 0; i < bytes; i += sizeof(Piece))
                    *reinterpret_cast<Piece *>(reinterpret_cast<char *>(raw) + i) =
                        *reinterpret_cast<const Piece *>(reinterpret_cast<const char *>(from) + i);
            } else {
                raw[0] = from[0];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (e0 + i < end) raw[i] = from[i];
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        float f;
        if constexpr (sizeof(T) == 4) f = __builtin_bit_cast(float, raw[i]);
        else f = __builtin_bit_cast(float, (uint32_t)raw[i] << 16);
        v[i] = e0 + i < end ? f : -__builtin_inff();
    }
}

// LDS accesses of one wavefront complete in order; this keeps the compiler to the written order
__device__ __forceinline__ void lds_order()
{
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ float from_key(uint32_t k) { return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : ~0u)); }

// exp(x) within (1.25 |x| + 2) roundings, relatively: the product's counts |x|, the constant's own 0.22 |x|, the exponential two.
// s = 1 / (1 + exp(-x)) within (1.25 |x| + 5); absolutely within 4 of 1, since the exponential's error counts (1 - s) s times, and
// (1 - s) s (1.25 |x| + 2) is below 0.8.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-x)); }

// How far two choices in fp32 have to be from each other for their order to be that in 64 bits, in roundings (2^-24) of 1 + the largest
// finite bias.  A sigmoid is at most 4 off, a choice one of its size more, and there are two of them: 12.  The sum of two choices that a
// group is worth is off by both and its own rounding, and there are two of these: 24.
// A softmax score e^x / sum, x <= 0: the subtraction that makes x and the exponential are (2.25 |x| + 2) off, which the score's size turns
// into less than 2.1; the division is one of its size.  The sum is off by its terms' errors, each with the share p of its term - at
// most sum p (2.25 |x| + 2), which with the score's own share is below 6 for 4096 experts -, and by log2 V + 6 <= 12 additions, whose
// parts are none of them larger than the sum (one behind the other V = 64 would be 69, and loses that much where one score is near 1 and
// the others of its lane are just below 2^-24).  The sum's 18 are common to both scores, whose difference is below 1.  So two choices:
// 2 (2.1 + 1) + 18 and their own roundings 2, less than 36; two groups, of two scores each that together are below 1: 4 (2.1 + 1) + 18
// and additions 4 + 4, less than 76.  (Equal infinities are never far enough.)
struct Margin {
    float choice, group;
    __device__ __forceinline__ Margin(float largest_bias, bool sigmoid)
        : choice((sigmoid ? 12.f : 36.f) * 0x1p-24f * (1.0f + largest_bias)),
          group((sigmoid ? 24.f : 76.f) * 0x1p-24f * (1.0f + largest_bias))
    {
    }
};
__device__ __forceinline__ bool far(float a, float b, float margin) { return fabsf(a - b) > margin; }

// The keys of experts outside the top_groups best groups become 0.  SUMS: a group is worth the sum of its two best choices.  CHECK
// (keys of fp32 choices): returns whether the same groups stay in 64 bits; if not, the keys are left as they are.
template <typename Key, bool SUMS, bool CHECK, int V>
__device__ __forceinline__ bool keep_groups(const RouteParams &s, Key (&key)[V], Key *scratch, int lane, float margin)
{
    const int E = s.E, e0 = lane * V;
    bool sure = true;
    auto worth = [&](Key first, Key second, bool alone) {
        if constexpr (SUMS) return alone ? first : order_key(from_key(first) + from_key(second));
        else return first;
    };
    auto stays = [&](Key mine, int group, int stride) {   // whether fewer than top_groups groups are ahead of the lane's
        int ahead = 0;
        for (int g = 0; g < s.num_groups; g++) {
            const Key o = of_lane(mine, g * stride);   // (no valid key is 0: one less is still a key)
            ahead += o > mine - (g < group ? 1 : 0);
        }
        const bool in = ahead < s.top_groups, is = group < s.num_groups;
        if constexpr (CHECK) {   // the last group that stays and the first that does not
            const uint32_t last = ~wave_max(is && in ? ~(uint32_t)mine : 0u), out = wave_max(is && !in ? (uint32_t)mine : 0u);
            sure = out == 0 || far(from_key(last), from_key(out), margin);
        }
        return is && in;
    };
    if (s.group_lanes > 0) {
        Key first = 0, second = 0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            second = max(second, min(first, key[v]));
            first = max(first, key[v]);
        }
        for (int d = 1; d < s.group_lanes; d <<= 1) {
            const Key of = other_half(first, d);
            if constexpr (SUMS) second = max(max(second, other_half(second, d)), min(first, of));
            first = max(first, of);
        }
        // (lanes behind the last group hold no experts)
        const bool in = stays(worth(first, second, V == 1 && s.group_lanes == 1), lane >> __builtin_ctz(s.group_lanes), s.group_lanes);
        if (!sure) return false;
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = in ? key[v] : 0;
    } else {   // lane g walks over group g
        lds_order();
#pragma unroll
        for (int v = 0; v < V; v++)
            if (e0 + v < E) scratch[e0 + v] = key[v];
        lds_order();
        const int size = E / s.num_groups;
        Key first = 0, second = 0;
        if (lane < s.num_groups)
            for (int i = 0; i < size; i++) {
                const Key x = scratch[lane * size + i];
                second = max(second, min(first, x));
                first = max(first, x);
            }
        lds_order();
        const unsigned long long stay = __ballot(stays(worth(first, second, size == 1), lane, 1));
        if (!sure) return false;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (e0 + v < E && !((stay >> ((e0 + v) / size)) & 1)) key[v] = 0;
    }
    return true;
}

// Lane k gets the k-th best expert of the keys.  CHECK (keys of fp32 choices): returns whether that is the order in 64 bits, too.
// Experts that are too close to tell are put in order by exact(expert), the key of its choice in 64 bits - one evaluation, of all
// lanes at once -, as long as it is sure which top_k + 1 experts are the best.
template <typename Key, bool CHECK, int V, typename Exact>
__device__ __forceinline__ bool pick(const RouteParams &s, Key (&key)[V], int lane, int &my_id, float margin, Exact exact)
{
    // A lane's few experts are put in order once, neighbours changing places so that equal ones do not; of more, the best is looked
    // for again when it has been taken.
    constexpr bool kSorted = V <= 4;
    int expert[V];
#pragma unroll
    for (int v = 0; v < V; v++) expert[v] = lane * V + v;
    if constexpr (kSorted) {
#pragma unroll
        for (int end = V - 1; end > 0; end--)
#pragma unroll
            for (int v = 0; v < end; v++) {
                const bool swap = key[v + 1] > key[v];
                const Key high = max(key[v], key[v + 1]), low = min(key[v], key[v + 1]);
                const int a = expert[v], b = expert[v + 1];
                key[v] = high, key[v + 1] = low;
                expert[v] = swap ? b : a, expert[v + 1] = swap ? a : b;
            }
    }
    Key best = key[0];
    int at = lane * V;
    auto find_best = [&]() {   // the lane's own, the lowest of equal ones
        best = key[0];
        at = expert[0];
        if constexpr (!kSorted) {
#pragma unroll
            for (int v = 1; v < V; v++)
                if (key[v] > best) best = key[v], at = expert[v];
        }
    };
    auto take_best = [&]() {
        if constexpr (kSorted) {
#pragma unroll
            for (int v = 0; v + 1 < V; v++) key[v] = key[v + 1], expert[v] = expert[v + 1];
            key[V - 1] = 0;
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) key[v] = expert[v] == at ? 0 : key[v];
        }
        find_best();
    };
    find_best();
    int chosen = 0;   // the key of the lane's expert
    my_id = 0;
    // (At least top_k experts are not out, so the largest key is not 0 before.  CHECK looks at the one behind them as well.)
    for (int k = 0; k < s.top_k + (CHECK ? 1 : 0); k++) {
        unsigned long long equal;
        if constexpr (sizeof(Key) == 8) {
            const uint32_t high = wave_max((uint32_t)(best >> 32));
            bool is = (uint32_t)(best >> 32) == high;
            equal = __ballot(is);
            if (equal & (equal - 1)) {
                const uint32_t low = wave_max(is ? (uint32_t)best : 0u);
                is = is && (uint32_t)best == low;
                equal = __ballot(is);
            }
        } else {
            const uint32_t high = wave_max(best);
            equal = __ballot(best == high);
            if constexpr (CHECK) chosen = lane == k ? (int)high : chosen;
        }
        const int src = __builtin_ctzll(equal);
        const int id = __builtin_amdgcn_readlane(at, src);
        my_id = lane == k ? id : my_id;
        if (lane == src) take_best();
    }
    if constexpr (CHECK) {
        if (s.top_k > 62) return false;
        const uint32_t mine32 = (uint32_t)chosen, next = (uint32_t)__shfl_down(chosen, 1);   // (0: there is no other expert)
        if (__all(lane >= s.top_k || next == 0 || far(from_key(mine32), from_key(next), margin))) return true;
        const uint32_t beyond = wave_max(best), last = of_lane(mine32, s.top_k - 1);
        if (s.sigmoid == 0 || !(beyond == 0 || far(from_key(last), from_key(beyond), margin))) return false;
        const int n = s.top_k + (of_lane(mine32, s.top_k) != 0 ? 1 : 0);
        const uint64_t mine = lane < n ? exact(my_id) : 0;
        int ahead = 0;
        for (int k = 0; k < n; k++) {
            const uint64_t o = of_lane(mine, k);
            ahead += o > mine || (o == mine && __builtin_amdgcn_readlane(my_id, k) < my_id);
        }
        my_id = __builtin_amdgcn_ds_permute(4 * (lane < n ? ahead : lane), my_id);
    }
    return true;
}

template <typename T, bool BIAS, int V>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(const RouteParams s)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token = blockIdx.x * (blockDim.x >> 6) + wave;
    if (token >= s.M) return;   // (no barriers: a wavefront's part of LDS is its own)
    const int E = s.E, e0 = lane * V;

    float l[V];
    load_run<T, V>(s.logits, (size_t)token * E + e0, e0, E, s.vector, l);
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; v++) nan |= l[v] != l[v];
    bool lost = __ballot(nan) != 0;   // whether the row has no weights

    float top = 0.f;   // the softmax's largest logit
    if (!s.sigmoid) {
        uint32_t m = 0;
#pragma unroll
        for (int v = 0; v < V; v++) m = max(m, order_key(l[v]));
        top = from_key(wave_max(m));
        lost |= top == __builtin_inff();
    }
    auto part = [&](float x) { return x == -__builtin_inff() ? 0.f : exp_of(x - top); };
    int my_id;
    float w = 0.f;     // the score of the lane's expert
    uint32_t key[V];
    if constexpr (BIAS) {
        float bias[V], score[V];
        load_run<float, V>(s.bias, (size_t)e0, e0, E, s.vector, bias);
        if (s.sigmoid) {
#pragma unroll
            for (int v = 0; v < V; v++) score[v] = sigmoid_of(l[v]);
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) score[v] = part(l[v]);
            const float sum = wave_sum(tree_sum<V>([&](int v) { return l[v] == l[v] ? score[v] : 0.f; }));   // (a NaN logit has no part in it)
#pragma unroll
            for (int v = 0; v < V; v++) score[v] = l[v] == -__builtin_inff() ? 0.f : score[v] / sum;
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            const uint32_t of = order_key(score[v] + bias[v]);
            key[v] = e0 + v < E ? of : 0;
        }
        uint32_t largest = 0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const uint32_t b = __builtin_bit_cast(uint32_t, bias[v]) & 0x7fffffffu;
            largest = b < 0x7f800000u ? max(largest, b) : largest;
        }
        const Margin margin(__builtin_bit_cast(float, wave_max(largest)), s.sigmoid);
        auto exact = [&](int e) {
            const double x = (double)logit_at<T>(s.logits, (size_t)token * E + e);
            return order_key((x <= kNoScore ? 0.0 : 1.0 / (1.0 + exp(-x))) + (double)s.bias[e]);
        };
        auto exact_keys = [&](uint64_t (&wide)[V]) {
            double sum = 1.0;
            const float lowest = s.sigmoid ? kNoScore : top < __builtin_inff() ? top + kNoScore : -__builtin_inff();
            if (!s.sigmoid) {
                sum = 0.0;
#pragma unroll
                for (int v = 0; v < V; v++)
                    if (l[v] > -__builtin_inff()) sum += exp((double)l[v] - (double)top);
                sum = wave_sum(sum);
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                double d = s.sigmoid ? 1.0 / (1.0 + exp(-(double)l[v])) : exp((double)l[v] - (double)top) / sum;
                if (l[v] <= lowest) d = 0.0;
                const uint64_t of = order_key(d + (double)bias[v]);
                wide[v] = e0 + v < E ? of : 0;
            }
            if (s.num_groups > 1)
                keep_groups<uint64_t, true, false, V>(s, wide, reinterpret_cast<uint64_t *>(lds + (size_t)wave * E * 8), lane, 0.f);
        };
        uint64_t wide[V];
        if (s.num_groups > 1 &&
            !keep_groups<uint32_t, true, true, V>(s, key, reinterpret_cast<uint32_t *>(lds + (size_t)wave * E * 8), lane, margin.group)) {
            exact_keys(wide);
#pragma unroll
            for (int v = 0; v < V; v++) key[v] = wide[v] != 0 ? key[v] : 0;
        }
        if (!pick<uint32_t, true, V>(s, key, lane, my_id, margin.choice, exact)) {
            exact_keys(wide);
            pick<uint64_t, false, V>(s, wide, lane, my_id, 0.f, exact);
        }
        const int from = my_id / V, which = my_id % V;   // lane k fetches what its expert's lane holds
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float o = __shfl(score[v], from);
            w = v == which ? o : w;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const uint32_t of = order_key(l[v]);
            key[v] = e0 + v < E ? of : 0;
        }
        if (s.num_groups > 1)
            keep_groups<uint32_t, false, false, V>(s, key, reinterpret_cast<uint32_t *>(lds + (size_t)wave * E * 4), lane, 0.f);
        pick<uint32_t, false, V>(s, key, lane, my_id, 0.f, [](int) { return uint64_t(0); });
        const int from = my_id / V, which = my_id % V;
        float x = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float o = __shfl(l[v], from);
            x = v == which ? o : x;
        }
        if (s.sigmoid) {
            w = sigmoid_of(x);
        } else {
            w = part(x);
            if (!s.renormalize) {
                const float sum = wave_sum(tree_sum<V>([&](int v) { return part(l[v]); }));
                w = sum != 0.f ? w / sum : 0.f;
            }
        }
    }
    w = lane < s.top_k ? w : 0.f;
    if (s.renormalize) {
        float sum = wave_sum(w);
        if (sum < 0x1p-24f) {   // (one value in all lanes)
            const float x = lane < s.top_k ? logit_at<T>(s.logits, (size_t)token * E + my_id) : -__builtin_inff();
            const float best = from_key(wave_max(order_key(x)));
            w = x == -__builtin_inff() || (s.sigmoid ? x : x - top) <= kNoScore ? 0.f : exp_of(x - best);
            sum = wave_sum(w);
        }
        w = sum != 0.f ? w / sum : 0.f;
    }
    const int kept = s.top_k + s.shared;
    const size_t out = (size_t)token * kept;
    if (lane < s.top_k) {
        s.weights[out + lane] = lost ? __builtin_nanf("") : w;
        s.ids[out + lane] = my_id;
    }
    for (int i = lane; i < s.shared; i += 64) {
        s.weights[out + s.top_k + i] = s.shared_weight;
        s.ids[out + s.top_k + i] = E + i;
    }
}

typedef void (*RouteFn)(const RouteParams);
struct RouteVariant {
    RouteFn fn;
    int per_lane;
};
template <typename T, bool BIAS>
RouteVariant route_variant(int E)
{
    if (E <= 64) return {route_kernel<T, BIAS, 1>, 1};
    if (E <= 128) return {route_kernel<T, BIAS, 2>, 2};
    if (E <= 256) return {route_kernel<T, BIAS, 4>, 4};
    if (E <= 512) return {route_kernel<T, BIAS, 8>, 8};
    if (E <= 1024) return {route_kernel<T, BIAS, 16>, 16};
    return {route_kernel<T, BIAS, 64>, 64};
}

}  // namespace
}  // namespace alpha_moe

extern "C" int alpha_moe_route_topk(const void *logits, int is_f32, const float *bias, float *topk_weights, int32_t *topk_ids,
                                    int M, int E, int top_k, int sigmoid, int num_groups, int top_groups, int renormalize,
                                    int shared_experts, float shared_weight, void *stream)
{
    using namespace alpha_moe;
    if (M < 0 || M >= 1 << 26 || E <= 0 || E > kRouteMaxExperts || top_k <= 0 || top_k > kRouteMaxTopK || num_groups <= 0 ||
        num_groups > kRouteMaxGroups || E % num_groups != 0 || top_groups <= 0 || top_groups > num_groups ||
        top_k > top_groups * (E / num_groups) || shared_experts < 0 || shared_experts > kRouteMaxExperts)
        return ALPHA_MOE_ERR_SHAPE;   // (2^26 tokens: 2^32 threads a launch)
    if (M == 0) return ALPHA_MOE_OK;
    if (!logits || !topk_weights || !topk_ids) return ALPHA_MOE_ERR_NULL_POINTER;
    const RouteVariant variant = is_f32 ? (bias ? route_variant<uint32_t, true>(E) : route_variant<uint32_t, false>(E))
                                        : (bias ? route_variant<uint16_t, true>(E) : route_variant<uint16_t, false>(E));
    const int V = variant.per_lane, size = E / num_groups;
    auto in_runs = [&](const void *p, int bytes) {
        const int run = V * bytes < 16 ? V * bytes : 16;
        return (reinterpret_cast<uintptr_t>(p) & (run - 1)) == 0;
    };
    const bool vector = E % V == 0 && in_runs(logits, is_f32 ? 4 : 2) && (!bias || in_runs(bias, 4));
    const int lanes = size % V == 0 && ((size / V) & (size / V - 1)) == 0 ? size / V : 0;
    const RouteParams s = {logits, bias, topk_weights, topk_ids, M, E, top_k, num_groups, top_groups, shared_experts,
                           shared_weight, sigmoid != 0, renormalize != 0, vector, lanes};
    const int lds = num_groups > 1 && lanes == 0 ? E * (bias ? 8 : 4) : 0;   // of a token
    int waves = M < kRouteWaves ? M : kRouteWaves;
    while (waves > 1 && waves * lds > 64 * 1024) waves--;
    void *args[] = {const_cast<RouteParams *>(&s)};
    return hipLaunchKernel(reinterpret_cast<const void *>(variant.fn), dim3((unsigned)((M + waves - 1) / waves)),
                           dim3(64 * (unsigned)waves), args, (size_t)(waves * lds), static_cast<hipStream_t>(stream)) == hipSuccess
               ? ALPHA_MOE_OK : ALPHA_MOE_ERR_LAUNCH;
}
