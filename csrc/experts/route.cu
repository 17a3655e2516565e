/**
 * The choice of a token's experts and their weights, and its gradient
 *
 *     s = softmax(z), or sigmoid(z) of each;  c = s + bias;  of groups of experts those with the best score stay;  the k best c of those, ties to the lowest index
 *     w_j = scale * s_j, or scale * s_j / sum of the chosen s
 *     g = scale * dw;  renormalised: dz_j = r_j (g_j - sum g_i r_i) * (1, or 1 - s_j) with r the weights without scale, else
 *     softmax: dz_e = s_e (g_e - sum of the chosen s_i g_i),  sigmoid: dz_j = g_j s_j (1 - s_j)
 *
 * One warp per token, its logits in registers. Which expert is chosen must not hang on the rounding of an exponential. Without a bias both
 * scores grow with the logit, and logits are compared. With one, scores are compared in fp32; where two that matter lie closer
 * than fp32 can tell (about one token in two thousand of random fp32 logits), the warp does its token again in 64 bits.
 */
#include "expert_ops.hpp"
#include "../kernels/launch_early.cuh"
#include "../decoder/row_access.cuh"

namespace dccl {

constexpr int kRouteWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
    const void* logits;
    const float* bias;
    float* weights;
    int* chosen;
    const float* dweights;
    void* dlogits;
    unsigned tokens, experts;
    DcclRouting how;
    Divisor group;              // by the experts of a group
};

/** fp32 as a number whose order is that of the values. No NaN comes here. */
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);       // of the two zeros the positive one
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

/** The largest value of the warp, and the lowest of the numbers that come with it; minus infinity and some number where all are. */
__device__ __forceinline__ void best_of_warp(float& v, int& at) {
    const unsigned key = ordered(v), top = __reduce_max_sync(kAll, key);
    at = (int)__reduce_min_sync(kAll, key == top ? (unsigned)at : 0x7fffffffu);
    v = from_ordered(top);
}
__device__ __forceinline__ void best_of_warp(double& v, int& at) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double w = __shfl_xor_sync(kAll, v, o);
        const int b = __shfl_xor_sync(kAll, at, o);
        if (w > v || (w == v && b < at)) { v = w; at = b; }
    }
}
template <typename S> __device__ __forceinline__ S warp_sum(S v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

template <typename S> __device__ __forceinline__ S nothing() { return -(S)INFINITY; }

template <typename T> __device__ __forceinline__ float logit(const RouteArgs& a, size_t token, int e) {
    return Traits<T>::up(reinterpret_cast<const T*>(a.logits)[token * a.experts + e]);
}

/**
 * The choice by scores c[i] of the experts lane + 32 i (minus infinity: none): lane j < k gets the j-th expert, or -1. False where two that decide lie
 * within `unsure` (below zero: nobody asks) of each other, two groups within twice that, and are not the same numbers.
 */
template <typename T, typename S, int PER> __device__ __forceinline__ bool choose(const RouteArgs& a, size_t token, S (&c)[PER], S unsure, int& mine) {
    const int lane = threadIdx.x % 32;
    bool sure = true;
    if (a.how.groups > 1) {
        S of_group = nothing<S>();
        const int size = (int)a.group.d;
        for (int g = 0; g < a.how.groups; g++) {
            S first = nothing<S>(), second = nothing<S>();
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = lane + 32 * i;
                const S v = e >= g * size && e < (g + 1) * size ? c[i] : nothing<S>();
                second = v > first ? first : v > second ? v : second;
                first = v > first ? v : first;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const S f = __shfl_xor_sync(kAll, first, o), s = __shfl_xor_sync(kAll, second, o);
                const S low = f > first ? first : f;
                first = f > first ? f : first;
                second = s > second ? s : second;
                second = low > second ? low : second;
            }
            if (lane == g) of_group = a.how.top2 && second > nothing<S>() ? first + second : first;
        }
        unsigned kept = 0;
        S last = 0;
        for (int j = 0; j <= a.how.top_groups && j < a.how.groups; j++) {
            S v = kept >> lane & 1 ? nothing<S>() : of_group;
            int at = lane;
            best_of_warp(v, at);
            if (!(v > nothing<S>())) break;
            if (j == a.how.top_groups) {        // the first that does not stay
                sure = last - v > 2 * unsure;
                break;
            }
            kept |= 1u << at;
            last = v;
        }
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 32 * i;
            if (e < (int)a.experts && !(kept >> a.group.quotient(e) & 1)) c[i] = nothing<S>();
        }
    }
    mine = -1;
    S last = 0;
    int last_at = -1;
    for (int j = 0; j <= a.how.k; j++) {
        if (j == a.how.k && unsure < 0) break;          // nobody asks for the first that is not chosen
        S v = c[0];
        int at = lane;
#pragma unroll
        for (int i = 1; i < PER; i++)
            if (c[i] > v) { v = c[i]; at = lane + 32 * i; }
        best_of_warp(v, at);
        if (!(v > nothing<S>())) break;
        if (unsure >= 0 && j > 0 && !(last - v > unsure)
            && !(logit<T>(a, token, last_at) == logit<T>(a, token, at) && (!a.bias || a.bias[last_at] == a.bias[at])))
            sure = false;
        if (j == a.how.k) break;
        if (lane == j) mine = at;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 32 * i == at) c[i] = nothing<S>();
        last = v;
        last_at = at;
    }
    return sure;
}

/** The choice in 64 bits. */
template <typename T, int PER> __device__ __noinline__ int choose_exactly(const RouteArgs& a, size_t token) {
    const int lane = threadIdx.x % 32;
    double c[PER], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 32 * i;
        c[i] = e < (int)a.experts ? (double)logit<T>(a, token, e) : -INFINITY;
        top = c[i] > top ? c[i] : top;
    }
    double sum = 1;
    if (!a.how.sigmoid) {
        int at = 0;
        best_of_warp(top, at);
        double part = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) part += c[i] > -INFINITY ? exp(c[i] - top) : 0.0;
        sum = warp_sum(part);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 32 * i;
        if (!(c[i] > -INFINITY)) { c[i] = -INFINITY; continue; }
        c[i] = (a.how.sigmoid ? 1.0 / (1.0 + exp(-c[i])) : exp(c[i] - top) / sum) + (a.bias ? (double)a.bias[e] : 0.0);
        if (!(c[i] > -INFINITY)) c[i] = -INFINITY;          // NaN as well
    }
    int mine;
    choose<T, double, PER>(a, token, c, -1.0, mine);
    return mine;
}

/**
 * How close two scores of at most `largest`, with biases up to `bias`, may lie for their order not to be known, in units of 2^-23. A sigmoid is off by two
 * (exponential one, sum and quotient half each). A softmax by its own exponential, difference and quotient likewise, and by the sum that all of the row
 * share: one of its terms, and half for each of the PER + 5 additions. Twice that for two, and half of the result's size for the sum with the bias.
 * Two groups lie within twice all this: two scores each, and the rounding of their sum.
 */
template <int PER> __device__ __forceinline__ float unsure_within(bool sigmoid, float largest, float bias) {
    return ((sigmoid ? 8 : PER + 16) * largest + 2 * (largest + bias)) * (1.0f / (1 << 23));
}

/** sigmoid(z) and a common factor of all that makes up for z far below zero: 1 / (e^-c + e^(-z - c)), c = max(0, -largest z). */
__device__ __forceinline__ float sigmoid_beside(float z, float largest) {
    const float c = largest < 0.0f ? -largest : 0.0f;
    return 1.0f / (expf(-c) + expf(-z - c));
}

/** Lane j's share r_j of the chosen, from its logit z (none: -infinity); 0 where there is none. */
__device__ __forceinline__ float share_of(const DcclRouting& how, bool there, float z) {
    int at = 0;
    float top = there ? z : -INFINITY;
    best_of_warp(top, at);
    const float s = !there ? 0.0f : how.sigmoid ? sigmoid_beside(z, top) : expf(z - top);
    const float sum = warp_sum(s);
    return there ? s / sum : 0.0f;
}

/**
 * Bytes are few (16384 tokens of 256 fp32 logits: 17 MB, 2.6 us); the choice is what takes time: k + 1 rounds of a comparison per register and two reductions
 * of the warp.
 */
template <typename T, int PER> __global__ void __launch_bounds__(32 * kRouteWarps) k_route(const __grid_constant__ RouteArgs a) {
    wait_for_stream();
    const int lane = threadIdx.x % 32;
    const size_t token = (size_t)blockIdx.x * kRouteWarps + threadIdx.x / 32;
    if (token >= a.tokens) return;
    float z[PER], c[PER], top = -INFINITY;
    bool poisoned = false;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 32 * i;
        z[i] = e < (int)a.experts ? logit<T>(a, token, e) : -INFINITY;
        poisoned |= z[i] != z[i];
        top = z[i] > top ? z[i] : top;
    }
    poisoned = __any_sync(kAll, poisoned);
    // whether the order of the scores is that of the logits
    const bool plain = !a.bias && (a.how.groups == 1 || !a.how.top2);
    float sum = 1.0f, bias = 0.0f;
    if (!a.how.sigmoid && (!plain || !a.how.renormalize)) {
        int at = 0;
        best_of_warp(top, at);
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            c[i] = z[i] > -INFINITY ? expf(z[i] - top) : 0.0f;
            part += c[i];
        }
        sum = warp_sum(part);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 32 * i;
        float s = z[i];
        if (!plain && z[i] > -INFINITY) {
            const float b = a.bias ? a.bias[e] : 0.0f;
            s = (a.how.sigmoid ? 1.0f / (1.0f + expf(-z[i])) : c[i] / sum) + b;
            if (fabsf(b) < INFINITY) bias = fmaxf(bias, fabsf(b));
        }
        c[i] = s > -INFINITY ? s : -INFINITY;           // NaN is not chosen
    }
    if (a.bias) bias = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(bias)));
    int mine;
    // of a softmax the largest score is 1 / sum
    const float unsure = plain ? -1.0f : unsure_within<PER>(a.how.sigmoid, a.how.sigmoid ? 1.0f : 1.0f / sum, bias);
    if (!choose<T, float, PER>(a, token, c, unsure, mine) && !plain) mine = choose_exactly<T, PER>(a, token);
    const bool there = mine >= 0;
    const float zm = there ? logit<T>(a, token, mine) : -INFINITY;
    float w;
    if (a.how.renormalize) w = share_of(a.how, there, zm);
    else w = !there ? 0.0f : a.how.sigmoid ? 1.0f / (1.0f + expf(-zm)) : expf(zm - top) / sum;
    if (poisoned && there && !a.how.sigmoid) w = NAN;
    if (lane < a.how.k) {
        a.weights[token * a.how.k + lane] = a.how.scale * w;
        a.chosen[token * a.how.k + lane] = mine;
    }
}

template <typename T, int PER> __global__ void __launch_bounds__(32 * kRouteWarps) k_route_grad(const __grid_constant__ RouteArgs a) {
    wait_for_stream();
    const int lane = threadIdx.x % 32, k = a.how.k;
    const size_t token = (size_t)blockIdx.x * kRouteWarps + threadIdx.x / 32;
    if (token >= a.tokens) return;
    const int mine = lane < k ? a.chosen[token * k + lane] : -1;
    const bool there = mine >= 0 && mine < (int)a.experts;
    const float zm = there ? logit<T>(a, token, mine) : -INFINITY;
    const float g = there ? a.how.scale * a.dweights[token * k + lane] : 0.0f;
    T* to = reinterpret_cast<T*>(a.dlogits) + token * a.experts;
    float d[PER] = {}, dm = 0.0f;
    if (a.how.renormalize) {
        const float r = share_of(a.how, there, zm);
        dm = r * (g - warp_sum(there ? g * r : 0.0f));
        if (a.how.sigmoid) dm *= 1.0f / (1.0f + expf(zm));
    } else if (a.how.sigmoid) {
        const float s = 1.0f / (1.0f + expf(-zm));
        dm = g * s * (1.0f / (1.0f + expf(zm)));
    } else {
        float top = -INFINITY, part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 32 * i;
            d[i] = e < (int)a.experts ? logit<T>(a, token, e) : -INFINITY;
            top = d[i] > top ? d[i] : top;
        }
        int at = 0;
        best_of_warp(top, at);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            d[i] = d[i] == -INFINITY ? 0.0f : expf(d[i] - top);
            part += d[i];
        }
        const float sum = warp_sum(part), s = there ? expf(zm - top) / sum : 0.0f, common = warp_sum(there ? s * g : 0.0f);
#pragma unroll
        for (int i = 0; i < PER; i++) d[i] = d[i] == 0.0f ? 0.0f : -(d[i] / sum) * common;
        dm = s * (g - common);
    }
    for (int j = 0; j < k; j++) {
        const int e = __shfl_sync(kAll, there ? mine : -1, j);
        const float v = __shfl_sync(kAll, dm, j);
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 32 * i == e) d[i] = v;
    }
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (lane + 32 * i < (int)a.experts) to[lane + 32 * i] = Traits<T>::down(d[i]);
}

template <typename T> static cudaError_t run_route(const RouteArgs& a, bool backward, cudaStream_t stream) {
    const unsigned grid = (a.tokens + kRouteWarps - 1) / kRouteWarps, per = (a.experts + 31) / 32;
    const auto go = [&](auto kernel) { return launch_early(kernel, grid, 32 * kRouteWarps, stream, a); };
    if (per <= 1) return go(backward ? k_route_grad<T, 1> : k_route<T, 1>);
    if (per <= 2) return go(backward ? k_route_grad<T, 2> : k_route<T, 2>);
    if (per <= 4) return go(backward ? k_route_grad<T, 4> : k_route<T, 4>);
    if (per <= 8) return go(backward ? k_route_grad<T, 8> : k_route<T, 8>);
    if (per <= 16) return go(backward ? k_route_grad<T, 16> : k_route<T, 16>);
    return go(backward ? k_route_grad<T, 32> : k_route<T, 32>);
}

static int route(const char* who, int device, int dtype, size_t tokens, int experts, RouteArgs a, const DcclRouting* how, bool backward, void* stream) {
    if (!tokens) return 0;
    if (!how || experts < 1 || experts > DCCL_EXPERTS_MAX || how->k < 1 || how->k > DCCL_EXPERTS_MAX_CHOSEN || how->k > experts || how->groups < 1 || how->groups > DCCL_EXPERTS_MAX_GROUPS
        || experts % how->groups || how->top_groups < 1 || how->top_groups > how->groups || tokens * how->k > DCCL_EXPERTS_MAX_PLACES || (dtype != 6 && dtype != 7 && dtype != 9)
        || !a.logits || !a.chosen || (backward ? !a.dweights || !a.dlogits : !a.weights))
        return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    a.tokens = (unsigned)tokens;
    a.experts = (unsigned)experts;
    a.how = *how;
    a.group = Divisor((unsigned)(experts / how->groups));
    const cudaStream_t s = (cudaStream_t)stream;
    return report(who, dtype == 6 ? run_route<__half>(a, backward, s) : dtype == 7 ? run_route<float>(a, backward, s) : run_route<__nv_bfloat16>(a, backward, s));
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_route(int device, int dtype, size_t tokens, int experts, const void* logits, const float* bias, const DcclRouting* how, float* weights, int* chosen, void* stream) {
    RouteArgs a = {};
    a.logits = logits;
    a.bias = bias;
    a.weights = weights;
    a.chosen = chosen;
    return route("dccl_route", device, dtype, tokens, experts, a, how, false, stream);
}

extern "C" int dccl_route_backward(int device, int dtype, size_t tokens, int experts, const void* logits, const int* chosen, const float* dweights, const DcclRouting* how,
                                   void* dlogits, void* stream) {
    RouteArgs a = {};
    a.logits = logits;
    a.chosen = const_cast<int*>(chosen);
    a.dweights = dweights;
    a.dlogits = dlogits;
    return route("dccl_route_backward", device, dtype, tokens, experts, a, how, true, stream);
}
