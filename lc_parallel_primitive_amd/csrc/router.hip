// router.hip — the experts of every token and their weights, and the gradient of the
// router's logits.
//
//   key = logit + bias (one rounding; bias 0 where there is none)
//   the k largest keys, in falling order, ties to the lowest index, a NaN before all
//   others; experts whose logit or key is -infinity are never chosen: -1, weight 0
//   weight = scale p, with p over the row of logits l and the chosen ones C
//     softmax              exp(l_j) / sum over all of exp(l)
//     softmax, normalised  exp(l_j) / sum over C of exp(l)
//     sigmoid              1 / (1 + exp(-l_j))
//     sigmoid, normalised  exp(t_j) / sum over C of exp(t), t = log(1 / (1 + exp(-l)))
//
// With w the weights, g their gradients (of those chosen), m = sum over C of g w:
//     softmax              dl = p ((chosen: scale g) - m)          for all experts
//     softmax, normalised  dl = w (g - m / scale)                  for the chosen ones
//     sigmoid              dl = scale g p (1 - p)
//     sigmoid, normalised  dl = w (g - m / scale) (1 / (1 + exp(l)))
//
// A row lies in the registers of 16, 32 or 64 lanes, eight or sixteen neighbouring
// experts each.  The choice is k rounds of a maximum over the lane's keys and one over
// the lanes, in 32 bits: keys of 2-byte logits without a bias have the expert's number in
// their lower half, so that the largest one names its expert; others are ties in so far as
// they are equal, and the lowest lane that holds the largest has the lowest expert.
//
// Bound by these rounds' instructions: 28 or 45 each.  32768 x 256, 8 chosen: float32 16 us
// forward (35 MB, 7 us of a copy), 12 backward (4.7 TB/s); bfloat16 13 without a bias (3.4 of a
// copy) and 15.5 with one, 7 backward; 48 x 128: 3.1, the launch.
#include <algorithm>

#include "tensor.hpp"

namespace lcpp {
namespace {

constexpr int kMaxChoices = 64;
constexpr uint32_t kMaxExperts = 1024;
constexpr int kRouteThreads = 256;

struct RouterArgs {
    const void *logits;
    uint64_t logits_stride, grad_stride;
    const float *bias;
    int32_t *experts;         // [token][choice]
    const int32_t *chosen;    // the same, read by the backward pass
    float *weights;           // [token][choice]
    const float *grad_weights;
    void *grad_logits;
    uint32_t tokens, num_experts, choices;
    float scale;
    bool sigmoid, normalize;
};

struct FMax {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct UMax {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
// Fold over the GL lanes of a row's group, in each of them: inside 16 lanes by DPP, between
// them by exchanging rows of 16 and halves of 32.
template <int GL, class T, class Op>
__device__ __forceinline__ T lanes_fold(T x, Op op)
{
    static_assert(GL == 16 || GL == 32 || GL == kWave, "rows of a wave");
    x = op(x, dpp_perm<kDppQuadXor1>(x));
    x = op(x, dpp_perm<kDppQuadXor2>(x));
    x = op(x, dpp_perm<kDppRowHalfMirror>(x));
    x = op(x, dpp_perm<kDppRowMirror>(x));
    if constexpr (GL > 16) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x);
        const auto w = __builtin_amdgcn_permlane16_swap(b, b, false, false);
        x = op(__builtin_bit_cast(T, (uint32_t)w[0]), __builtin_bit_cast(T, (uint32_t)w[1]));
    }
    if constexpr (GL > 32) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x);
        const auto w = __builtin_amdgcn_permlane32_swap(b, b, false, false);
        x = op(__builtin_bit_cast(T, (uint32_t)w[0]), __builtin_bit_cast(T, (uint32_t)w[1]));
    }
    return x;
}

// Bits ordered like the value, NaN last of all; both zeros are one.
__device__ __forceinline__ uint32_t order_bits(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 0xFFFFFFFFu : b >> 31 ? ~b : b | 0x80000000u;
}
constexpr uint32_t kLowest = 0x007FFFFFu;  // order_bits(-infinity)
// The same of a 2-byte type, in 16 bits: never 0.
template <class T>
__device__ __forceinline__ uint32_t order_bits16(T x)
{
    const float f = (float)x;
    uint32_t b = __builtin_bit_cast(uint16_t, x);
    b = f == 0.0f ? 0u : b;
    return f != f ? 0xFFFFu : b >> 15 ? 0xFFFFu ^ b : b | 0x8000u;
}

__device__ __forceinline__ float sigmoid(float x)
{
    // exp(-|x|) cannot overflow
    const float e = __expf(-fabsf(x)), r = 1.0f / (1.0f + e);
    return x >= 0.0f ? r : e * r;
}
// (what rounding 1 + exp(-|x|) loses is a rounding of 1, and so of the exponential that follows)
__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.0f) - __logf(1.0f + __expf(-fabsf(x))); }

// V logits of a lane, or what stands for them, `past` past the row's end.
template <class T, int V>
__device__ __forceinline__ void load_logits(const T *row, uint32_t first, uint32_t n, float past, float (&l)[V])
{
#pragma unroll
    for (int h = 0; h < V; h += kOctet) {
        const uint32_t col = first + h;
        if (col + kOctet <= n) {
            const Octet<T> o = load_pack<kOctet>(row + col);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) l[h + i] = o[i];
        } else {
#pragma unroll
            for (int i = 0; i < kOctet; ++i)
                l[h + i] = col + i < n ? (float)row[col + i] : past;
        }
    }
}

// The largest logit of a row and the sum of exp(logit - largest); 0 and 1 for a row of
// -infinity alone, so that its shares are 0.
template <int GL, int V>
__device__ __forceinline__ void soft_sum(const float (&l)[V], float &most, float &sum)
{
    most = l[0];
#pragma unroll
    for (int i = 1; i < V; ++i) most = fmaxf(most, l[i]);
    most = lanes_fold<GL>(most, FMax());
    if (most == -std::numeric_limits<float>::infinity()) most = 0.0f;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum += __expf(l[i] - most);
    sum = lanes_fold<GL>(sum, SumOp());
    if (sum == 0.0f) sum = 1.0f;
}

// The weights (without the scale) of the choices that a lane of the group has, KV at most:
// choice t + i GL.  `l`: their logits, `has`: whether there is one.
template <int GL, int KV>
__device__ __forceinline__ void choice_weights(const RouterArgs &a, const float (&l)[KV], const bool (&has)[KV], float most,
                                               float sum, float (&p)[KV])
{
    if (a.normalize) {
        float t[KV], top = -std::numeric_limits<float>::infinity();
#pragma unroll
        for (int i = 0; i < KV; ++i) {
            t[i] = a.sigmoid ? log_sigmoid(l[i]) : l[i];
            if (has[i]) top = fmaxf(top, t[i]);
        }
        top = lanes_fold<GL>(top, FMax());
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
            p[i] = has[i] ? __expf(t[i] - top) : 0.0f;
            total += p[i];
        }
        total = lanes_fold<GL>(total, SumOp());
#pragma unroll
        for (int i = 0; i < KV; ++i) p[i] = has[i] ? p[i] / total : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < KV; ++i) p[i] = !has[i] ? 0.0f : a.sigmoid ? sigmoid(l[i]) : __expf(l[i] - most) / sum;
    }
}

// NAMED: 2-byte logits without a bias, whose keys name their expert.
template <class T, int GL, int V, int KV, bool NAMED>
__global__ __launch_bounds__(kRouteThreads) void router_forward_kernel(RouterArgs a)
{
    constexpr int RG = kRouteThreads / GL;
    constexpr float kNone = -std::numeric_limits<float>::infinity();
    __shared__ int32_t ids[NAMED ? 1 : RG][KV * GL];
    const uint32_t t = threadIdx.x % GL, group = threadIdx.x / GL;
    const uint64_t row = (uint64_t)blockIdx.x * RG + group;
    const bool live = row < a.tokens;
    const uint32_t first = t * V;
    const T *in = static_cast<const T *>(a.logits) + (live ? row : 0) * a.logits_stride;
    float l[V];
    load_logits<T, V>(in, first, a.num_experts, kNone, l);
    float most = 0.0f, sum = 1.0f;
    if (!a.sigmoid && !a.normalize) soft_sum<GL, V>(l, most, sum);
    float bias[V] = {};
    if (!NAMED && a.bias) load_logits<float, V>(a.bias, first, a.num_experts, 0.0f, bias);
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (NAMED) {
            const uint32_t k = order_bits16((T)l[i]);  // (back to the type it came from: exact)
            key[i] = l[i] == kNone ? 0u : k << 16 | (0xFFFFu - (first + i));
        } else {
            const uint32_t k = order_bits(a.bias ? l[i] + bias[i] : l[i]);
            key[i] = l[i] == kNone || k <= kLowest ? 0u : k;
        }
    }
    int32_t id[KV];
#pragma unroll
    for (int i = 0; i < KV; ++i) id[i] = -1;
    for (uint32_t j = 0; j < a.choices; ++j) {
        uint32_t mine = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) mine = UMax()(mine, key[i]);
        const uint32_t best = lanes_fold<GL>(mine, UMax());
        if constexpr (NAMED) {
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = key[i] == best ? 0u : key[i];
#pragma unroll
            for (int i = 0; i < KV; ++i)
                if (t + i * GL == j) id[i] = best ? (int32_t)(0xFFFFu - (best & 0xFFFFu)) : -1;
        } else {
            uint64_t holds = ballot(mine == best) >> (lane_id() / GL * GL);
            if constexpr (GL < kWave) holds &= (1ull << (GL % kWave)) - 1;
            bool own = (uint32_t)__builtin_ctzll(holds) == t && best;
            uint32_t at = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool take = own && key[i] == best;
                key[i] = take ? 0u : key[i];
                at = take ? first + i : at;
                own = own && !take;
            }
            if ((uint32_t)__builtin_ctzll(holds) == t) ids[group][j] = best ? (int32_t)at : -1;
        }
    }
    if constexpr (!NAMED) {
        wave_lds_sync();  // (a group is within a wave)
#pragma unroll
        for (int i = 0; i < KV; ++i)
            if (t + i * GL < a.choices) id[i] = ids[group][t + i * GL];
    }
    float x[KV], p[KV];
    bool has[KV];
#pragma unroll
    for (int i = 0; i < KV; ++i) {
        has[i] = id[i] >= 0;
        x[i] = has[i] ? (float)in[id[i]] : 0.0f;  // (from the caches)
    }
    choice_weights<GL, KV>(a, x, has, most, sum, p);
    if (!live) return;
#pragma unroll
    for (int i = 0; i < KV; ++i) {
        const uint32_t j = t + i * GL;
        if (j >= a.choices) continue;
        a.experts[row * a.choices + j] = id[i];
        a.weights[row * a.choices + j] = p[i] * a.scale;
    }
}

// The gradient's coefficients of the chosen experts meet the row in LDS.
template <class T, int GL, int V, int KV>
__global__ __launch_bounds__(kRouteThreads) void router_backward_kernel(RouterArgs a)
{
    constexpr int RG = kRouteThreads / GL;
    __shared__ float coef[RG][GL * V];
    const uint32_t t = threadIdx.x % GL, group = threadIdx.x / GL;
    const uint64_t row = (uint64_t)blockIdx.x * RG + group;
    const bool live = row < a.tokens;
    const uint32_t first = t * V;
    const T *in = static_cast<const T *>(a.logits) + (live ? row : 0) * a.logits_stride;
    const bool dense = !a.sigmoid && !a.normalize;  // every expert has a gradient
    float l[V], most = 0.0f, sum = 1.0f;
    if (dense) {
        load_logits<T, V>(in, first, a.num_experts, -std::numeric_limits<float>::infinity(), l);
        soft_sum<GL, V>(l, most, sum);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) coef[group][i * GL + t] = 0.0f;
    float x[KV], p[KV], g[KV];
    bool has[KV];
    int32_t id[KV];
#pragma unroll
    for (int i = 0; i < KV; ++i) {
        const uint32_t j = t + i * GL;
        const bool there = live && j < a.choices;
        id[i] = there ? a.chosen[row * a.choices + j] : -1;
        has[i] = id[i] >= 0 && (uint32_t)id[i] < a.num_experts;
        x[i] = has[i] ? (float)in[id[i]] : 0.0f;
        g[i] = has[i] ? a.grad_weights[row * a.choices + j] : 0.0f;
    }
    choice_weights<GL, KV>(a, x, has, most, sum, p);
    float m = 0.0f;  // the sum of g p
#pragma unroll
    for (int i = 0; i < KV; ++i) m += has[i] ? g[i] * p[i] : 0.0f;
    m = lanes_fold<GL>(m, SumOp());
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < KV; ++i) {
        if (!has[i]) continue;
        float d = a.scale * g[i];
        if (a.normalize) d = a.scale * p[i] * (g[i] - m);
        else if (a.sigmoid) d *= p[i];
        if (a.sigmoid) d *= sigmoid(-x[i]);
        const uint32_t e = (uint32_t)id[i];
        // (an expert that the caller's choices name twice has the sum)
        __hip_atomic_fetch_add(&coef[group][e % V * GL + e / V], d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    wave_lds_sync();
    if (!live) return;
    T *out = static_cast<T *>(a.grad_logits) + row * a.grad_stride;
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        d[i] = coef[group][i * GL + t];
        if (dense) d[i] = __expf(l[i] - most) / sum * (d[i] - a.scale * m);
    }
#pragma unroll
    for (int h = 0; h < V; h += kOctet) {
        const uint32_t col = first + h;
        if (col >= a.num_experts) continue;
        float v[kOctet];
#pragma unroll
        for (int i = 0; i < kOctet; ++i) v[i] = d[h + i];
        store_octet(out, col, a.num_experts, v);
    }
}

// A launch of 2^32 threads or more reports success and leaves most of them out, so more rows than these workgroups have
// take several launches, f(first row, rows).
constexpr uint64_t kMaxRouteGroups = 1u << 23;
template <class F>
int router_launches(uint64_t tokens, int rows_of_group, F f)
{
    const uint64_t most = kMaxRouteGroups * rows_of_group;
    for (uint64_t first = 0; first < tokens; first += most) {
        const int status = f(first, std::min(tokens - first, most));
        if (status) return status;
    }
    return LCPP_OK;
}

// f(lanes of a row, experts of a lane, choices of a lane) as integral constants: the fewest
// lanes that hold the row, and one choice a lane where that is enough.
template <class F>
int router_shape(uint32_t experts, uint32_t choices, F f)
{
    auto of = [&](auto lanes, auto values) {
        constexpr int GL = decltype(lanes)::value;
        if (choices <= GL) return f(lanes, values, std::integral_constant<int, 1>{});
        return f(lanes, values, std::integral_constant<int, kMaxChoices / GL>{});
    };
    if (experts <= 128) return of(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{});
    if (experts <= 256) return of(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
    if (experts <= 512) return of(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    return of(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
}

int router_args(lcpp_dtype t, lcpp_score score, int normalize, float scale, uint64_t tokens, uint64_t experts, uint64_t choices,
                RouterArgs *a)
{
    if (!float_size(t)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (score != LCPP_SCORE_SOFTMAX && score != LCPP_SCORE_SIGMOID) return LCPP_ERR_INVALID_ARG;
    // (tokens * choices numbers the pairs in 31 bits)
    if (experts > kMaxExperts || choices > kMaxChoices || choices > experts || tokens > 0x7FFFFFFFull) return LCPP_ERR_INVALID_ARG;
    if (tokens * choices > 0x7FFFFFFFull || !(scale == scale)) return LCPP_ERR_INVALID_ARG;
    a->tokens = (uint32_t)tokens, a->num_experts = (uint32_t)experts, a->choices = (uint32_t)choices;
    a->scale = scale;
    a->sigmoid = score == LCPP_SCORE_SIGMOID;
    a->normalize = normalize != 0;
    return LCPP_OK;
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_router_forward(lcpp_dtype t, lcpp_score score, int normalize, float scale, const void *logits,
                                   uint64_t logits_stride, const float *bias, int32_t *experts, float *weights,
                                   uint64_t tokens, uint64_t num_experts, uint64_t choices, void *stream)
{
    RouterArgs a = {};
    const int status = router_args(t, score, normalize, scale, tokens, num_experts, choices, &a);
    if (status) return status;
    if (tokens == 0 || choices == 0) return LCPP_OK;
    if (!elem_ok(logits, float_size(t)) || !elem_ok(experts, 4) || !elem_ok(weights, 4)) return LCPP_ERR_INVALID_ARG;
    if ((bias && !elem_ok(bias, 4)) || same_place(experts, weights)) return LCPP_ERR_INVALID_ARG;
    a.logits = logits, a.logits_stride = logits_stride, a.bias = bias;
    a.experts = experts, a.weights = weights;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return router_shape(a.num_experts, a.choices, [&](auto gl, auto v, auto kv) -> int {
            constexpr int GL = decltype(gl)::value, V = decltype(v)::value, KV = decltype(kv)::value;
            return router_launches(tokens, kRouteThreads / GL, [&](uint64_t first, uint64_t n) -> int {
                RouterArgs b = a;
                b.logits = static_cast<const T *>(logits) + first * logits_stride;
                b.experts = experts + first * choices, b.weights = weights + first * choices;
                b.tokens = (uint32_t)n;
                const uint32_t grid = (uint32_t)ceil_div(n, kRouteThreads / GL);
                if constexpr (sizeof(T) == 2) {
                    if (!b.bias) {
                        LCPP_LAUNCH("router_forward", s, router_forward_kernel<T, GL, V, KV, true><<<grid, kRouteThreads, 0, s>>>(b));
                        LCPP_CHECK_LAUNCH();
                        return LCPP_OK;
                    }
                }
                LCPP_LAUNCH("router_forward", s, router_forward_kernel<T, GL, V, KV, false><<<grid, kRouteThreads, 0, s>>>(b));
                LCPP_CHECK_LAUNCH();
                return LCPP_OK;
            });
        });
    });
}

extern "C" int lcpp_router_backward(lcpp_dtype t, lcpp_score score, int normalize, float scale, const void *logits,
                                    uint64_t logits_stride, const int32_t *experts, const float *grad_weights,
                                    void *grad_logits, uint64_t grad_stride, uint64_t tokens, uint64_t num_experts,
                                    uint64_t choices, void *stream)
{
    RouterArgs a = {};
    const int status = router_args(t, score, normalize, scale, tokens, num_experts, choices, &a);
    if (status) return status;
    if (tokens == 0 || num_experts == 0) return LCPP_OK;
    const size_t e = float_size(t);
    if (!elem_ok(logits, e) || !elem_ok(grad_logits, e) || !rows_apart(grad_stride, tokens, num_experts)) return LCPP_ERR_INVALID_ARG;
    if (choices && (!elem_ok(experts, 4) || !elem_ok(grad_weights, 4))) return LCPP_ERR_INVALID_ARG;
    a.logits = logits, a.logits_stride = logits_stride, a.chosen = experts, a.grad_weights = grad_weights;
    a.grad_logits = grad_logits, a.grad_stride = grad_stride;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return router_shape(a.num_experts, a.choices, [&](auto gl, auto v, auto kv) -> int {
            constexpr int GL = decltype(gl)::value, V = decltype(v)::value, KV = decltype(kv)::value;
            return router_launches(tokens, kRouteThreads / GL, [&](uint64_t first, uint64_t n) -> int {
                RouterArgs b = a;
                b.logits = static_cast<const T *>(logits) + first * logits_stride;
                b.chosen = experts + first * choices, b.grad_weights = grad_weights + first * choices;
                b.grad_logits = static_cast<T *>(grad_logits) + first * grad_stride;
                b.tokens = (uint32_t)n;
                const uint32_t grid = (uint32_t)ceil_div(n, kRouteThreads / GL);
                LCPP_LAUNCH("router_backward", s, router_backward_kernel<T, GL, V, KV><<<grid, kRouteThreads, 0, s>>>(b));
                LCPP_CHECK_LAUNCH();
                return LCPP_OK;
            });
        });
    });
}
