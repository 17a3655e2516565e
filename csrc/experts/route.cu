/**
 * The choice of a token's experts and their weights, and its gradient
 *
 *     s = softmax(z), or sigmoid(z) of each;  c = s + bias;  of groups of experts those with the best score stay;  the k best c of those, ties to the lowest index
 *     w_j = scale * s_j, or scale * s_j / sum of the chosen s
 *     g = scale * dw;  renormalised: dz_j = r_j (g_j - sum g_i r_i) * (1, or 1 - s_j) with r the weights without scale, else
 *     softmax: dz_e = s_e (g_e - sum of the chosen s_i g_i),  sigmoid: dz_j = g_j s_j (1 - s_j)
 *
 * One warp per token, its logits in registers. Which expert is chosen must not hang on the rounding of an exponential: without a bias both
 * scores grow with the logit, and logits are compared. With one scores are, in fp32; where two that matter lie closer
 * than fp32 can tell, the warp does its token again in 64 bits. How many tokens that are depends on the logits: about one in a thousand of random fp32 ones with a
 * deviation of 1.5, most where sigmoids are all but 1. 16384 tokens of 64 experts, bf16, sigmoid with a bias, the best 6: 10.0 us with a deviation of 1.5, 15.3
 * with 6 and 19.3 with 10; logits that are all equal 12.1.
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
    unsigned ends;              // registers with which a group of whole registers ends
    bool vec;                   // rows of the gradient start on 16 bytes
};

/** fp32 as a number whose order is that of the values. No NaN comes here. */
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);       // of the two zeros the positive one
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned k) { return __uint_as_float(k ^ (~(unsigned)((int)k >> 31) | 0x80000000u)); }
constexpr unsigned kNothing = 0x007fffffu;             // ordered(-infinity)

__device__ __forceinline__ float largest_of_warp(float v) { return from_ordered(__reduce_max_sync(kAll, ordered(v))); }
template <typename S> __device__ __forceinline__ S warp_sum(S v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

template <typename T> __device__ __forceinline__ float logit(const RouteArgs& a, size_t token, int e) {
    return Traits<T>::up(reinterpret_cast<const T*>(a.logits)[token * a.experts + e]);
}

/** The logits of the experts lane + 32 i; minus infinity behind the last. */
template <typename T, int PER> __device__ __forceinline__ void load_logits(const RouteArgs& a, size_t token, float (&z)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = threadIdx.x % 32 + 32 * i;
        z[i] = e < (int)a.experts ? logit<T>(a, token, e) : -INFINITY;
    }
}

/** The two best of a set, and of another one that has none of its elements, or of one more element. */
__device__ __forceinline__ void join_best(float& first, float& second, float f, float s) {
    second = fmaxf(fminf(first, f), fmaxf(second, s));
    first = fmaxf(first, f);
}
__device__ __forceinline__ void join_best(float& first, float& second, float c) {
    second = fmaxf(second, fminf(first, c));
    first = fmaxf(first, c);
}

/**
 * The two best over the warp of each register: lane l gets those of register l / (32 / PER). With every step half of the registers go to the lanes that will keep
 * them, and the others come.
 */
template <int PER> __device__ __forceinline__ void best_of_registers(float (&first)[PER], float (&second)[PER]) {
    int o = 16;
#pragma unroll
    for (int n = PER / 2; n >= 1; n /= 2, o /= 2) {
        const bool up = threadIdx.x & o;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float f = __shfl_xor_sync(kAll, up ? first[i] : first[i + n], o), s = __shfl_xor_sync(kAll, up ? second[i] : second[i + n], o);
            first[i] = up ? first[i + n] : first[i];
            second[i] = up ? second[i + n] : second[i];
            join_best(first[i], second[i], f, s);
        }
    }
    for (; o; o /= 2) join_best(first[0], second[0], __shfl_xor_sync(kAll, first[0], o), __shfl_xor_sync(kAll, second[0], o));
}

/** A sorted list of a lane's keys, the largest first: Batcher's odd-even merge sort. */
template <int PER> __device__ __forceinline__ void sort_keys(unsigned (&key)[PER]) {
#pragma unroll
    for (int p = 1; p < PER; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < PER; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < PER && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const unsigned x = key[i + j], y = key[i + j + k];
                        key[i + j] = max(x, y);
                        key[i + j + k] = min(x, y);
                    }
}

/**
 * The choice by scores c[i] of the experts lane + 32 i (minus infinity: none): lane j < k gets the j-th expert, or -1. False where two that decide lie so close
 * that their order is not known: within `unsure`, or within `part` of their sizes, and are not the same numbers; two groups within twice that. Those that decide are each of
 * the chosen and the one behind it, and, where the last one and the first that is not chosen are the same numbers, the last one and all that are left.
 *
 * The lowest bits of a score's key give way to the number of its register, lower ones first, so that a key says all: of equal ones the lowest i, and of those the
 * first lane, is the lowest expert. What those bits told is in `part`.
 */
template <typename T, int PER> __device__ __forceinline__ bool choose(const RouteArgs& a, size_t token, float (&c)[PER], float unsure, int& mine) {
    const int lane = threadIdx.x % 32;
    unsigned beyond = kNothing;         // of k = 32
    int beyond_lane = 0;
    constexpr float part = (PER + 2) * (1.0f / (1 << 23));
    bool sure = true;
    if (a.how.groups > 1) {
        constexpr int spread = 32 / PER;
        const int size = (int)a.group.d, whole = size % 32 ? 0 : size / 32;       // registers of a group, where it has whole ones
        float first[PER], second[PER];          // where it has, of the group that ends with this register; otherwise in the first
        if (whole) {
            float f = -INFINITY, t = -INFINITY;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                join_best(f, t, c[i]);
                first[i] = second[i] = -INFINITY;
                if (a.ends >> i & 1) {
                    first[i] = f;
                    second[i] = t;
                    f = t = -INFINITY;
                }
            }
            best_of_registers(first, second);
        } else {
            float f = -INFINITY, t = -INFINITY;
            for (int g = 0; g < a.how.groups; g++) {
                float one = -INFINITY, two = -INFINITY;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int e = lane + 32 * i - g * size;
                    join_best(one, two, e >= 0 && e < size ? c[i] : -INFINITY);
                }
                const unsigned key = ordered(one), top = __reduce_max_sync(kAll, key);
                const int winner = __ffs(__ballot_sync(kAll, key == top)) - 1;
                const unsigned next = __reduce_max_sync(kAll, lane == winner ? ordered(two) : key);
                if (lane == g) { f = from_ordered(top); t = from_ordered(next); }
            }
            first[0] = f;
            second[0] = t;
        }
        const bool two = a.how.top2 && second[0] > -INFINITY;
        unsigned kept = 0, key = ordered(two ? first[0] + second[0] : first[0]);
        const float sizes = first[0] > -INFINITY ? fabsf(first[0]) + (two ? fabsf(second[0]) : 0.0f) : 0.0f;
        const float largest = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(sizes)));
        if (whole && lane % spread) key = kNothing;         // one lane speaks for a register
        float last = 0.0f;
        for (int j = 0; j <= a.how.top_groups && j < a.how.groups; j++) {
            const unsigned top = __reduce_max_sync(kAll, key);
            if (top <= kNothing) break;
            if (j == a.how.top_groups) {        // the first that does not stay
                sure = last - from_ordered(top) > 2 * (unsure + part * largest);
                break;
            }
            const int at = __ffs(__ballot_sync(kAll, key == top)) - 1;
            kept |= 1u << at;
            if (lane == at) key = kNothing;
            last = from_ordered(top);
        }
        if (whole) {
            bool stays = false;
#pragma unroll
            for (int i = PER - 1; i >= 0; i--) {
                if (a.ends >> i & 1) stays = kept >> (i * spread) & 1;
                if (!stays) c[i] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (lane + 32 * i < (int)a.experts && !(kept >> a.group.quotient(lane + 32 * i) & 1)) c[i] = -INFINITY;
        }
    }
    const auto expert_of = [](unsigned key, int lane) { return lane + 32 * (PER - 1 - (int)(key & (PER - 1))); };
    unsigned key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) key[i] = (ordered(c[i]) & ~(unsigned)(PER - 1)) | (PER - 1 - i);
    if constexpr (PER <= 8) sort_keys(key);
    unsigned mine_key = kNothing;
    int mine_lane = 0;
    for (int j = 0; j <= a.how.k; j++) {            // one more to see how far the first is that is not chosen
        unsigned best = key[0];
        if constexpr (PER > 8) {
#pragma unroll
            for (int i = 1; i < PER; i++) best = max(best, key[i]);
        }
        const unsigned top = __reduce_max_sync(kAll, best);
        if (top <= kNothing) break;
        const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
        if constexpr (PER > 8) {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (lane == winner && key[i] == top) key[i] = 0;
        } else if (lane == winner) {
#pragma unroll
            for (int i = 0; i + 1 < PER; i++) key[i] = key[i + 1];
            key[PER - 1] = 0;
        }
        if (lane == j) { mine_key = top; mine_lane = winner; }
        if (j == a.how.k) { beyond = top; beyond_lane = winner; }
    }
    // lane j against lane j + 1; the last of 32 against what came after it
    const bool there = mine_key > kNothing;
    mine = there ? expert_of(mine_key, mine_lane) : -1;
    unsigned next_key = __shfl_down_sync(kAll, mine_key, 1);
    int next = __shfl_down_sync(kAll, mine, 1);
    if (lane == 31) {
        next_key = beyond;
        next = expert_of(beyond, beyond_lane);
    }
    const auto apart = [&](float v, float w) { return v - w > unsure + part * fmaxf(fabsf(v), fabsf(w)); };
    const auto same = [&](int e, int f) { return logit<T>(a, token, e) == logit<T>(a, token, f) && (!a.bias || a.bias[e] == a.bias[f]); };
    bool tied = false;
    if (there && lane < a.how.k && next_key > kNothing && !apart(from_ordered(mine_key), from_ordered(next_key))) {
        tied = same(mine, next);
        sure &= tied;
    }
    // a tie of the last one is not settled by the first that is not chosen: any of the rest may be above both, where fp32 cannot tell it from them
    if (__shfl_sync(kAll, tied, a.how.k - 1)) {
        const float v = from_ordered(__shfl_sync(kAll, mine_key, a.how.k - 1));
        const int e = __shfl_sync(kAll, mine, a.how.k - 1);
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (key[i] > kNothing && !apart(v, from_ordered(key[i])) && !same(e, expert_of(key[i], lane))) sure = false;
    }
    sure = __all_sync(kAll, sure);
    if (lane >= a.how.k) mine = -1;
    return sure;
}

/** The same for 64 bits, in two halves: the largest value of the warp, and the first lane that has it. */
__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double largest_of_warp(double v, int& lane) {
    const unsigned long long key = ordered(v);
    const unsigned high = (unsigned)(key >> 32), top = __reduce_max_sync(kAll, high), low = __reduce_max_sync(kAll, high == top ? (unsigned)key : 0u);
    lane = __ffs(__ballot_sync(kAll, high == top && (unsigned)key == low)) - 1;
    return __shfl_sync(kAll, v, lane);
}

/** The choice in 64 bits. plain: by the logits. */
template <typename T, int PER> __device__ __noinline__ int choose_exactly(const RouteArgs& a, size_t token, bool plain) {
    const int lane = threadIdx.x % 32;
    double c[PER], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 32 * i;
        c[i] = e < (int)a.experts ? (double)logit<T>(a, token, e) : -INFINITY;
        top = c[i] > top ? c[i] : top;
    }
    double sum = 1;
    if (!plain && !a.how.sigmoid) {
        int at;
        top = largest_of_warp(top, at);
        double part = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) part += c[i] > -INFINITY ? exp(c[i] - top) : 0.0;
        sum = warp_sum(part);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (!(c[i] > -INFINITY)) { c[i] = -INFINITY; continue; }
        if (!plain) c[i] = (a.how.sigmoid ? 1.0 / (1.0 + exp(-c[i])) : exp(c[i] - top) / sum) + (a.bias ? (double)a.bias[lane + 32 * i] : 0.0);
        if (!(c[i] > -INFINITY)) c[i] = -INFINITY;          // NaN as well
    }
    if (a.how.groups > 1) {
        const int size = (int)a.group.d;
        double of_group = -INFINITY;
        for (int g = 0; g < a.how.groups; g++) {
            double first = -INFINITY, second = -INFINITY;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = lane + 32 * i - g * size;
                const double v = e >= 0 && e < size ? c[i] : -INFINITY;
                second = v > first ? first : v > second ? v : second;
                first = v > first ? v : first;
            }
            int at;
            const double f = largest_of_warp(first, at);
            if (a.how.top2) second = largest_of_warp(lane == at ? second : first, at);
            first = f;
            if (lane == g) of_group = a.how.top2 && second > -INFINITY ? first + second : first;
        }
        unsigned kept = 0;
        for (int j = 0; j < a.how.top_groups; j++) {
            int at;
            if (!(largest_of_warp(kept >> lane & 1 ? -INFINITY : of_group, at) > -INFINITY)) break;
            kept |= 1u << at;
        }
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 32 * i < (int)a.experts && !(kept >> a.group.quotient(lane + 32 * i) & 1)) c[i] = -INFINITY;
    }
    int mine = -1;
    for (int j = 0; j < a.how.k; j++) {
        double v = c[0];
        int of = 0, at;
#pragma unroll
        for (int i = 1; i < PER; i++)
            if (c[i] > v) { v = c[i]; of = i; }
        // equal ones in two lanes: the lower register, then the lower lane
        const double top = largest_of_warp(v, at);
        if (!(top > -INFINITY)) break;
        const int low = (int)__reduce_min_sync(kAll, v == top ? (unsigned)(32 * of + lane) : ~0u);
        if (lane == j) mine = low;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 32 * i == low) c[i] = -INFINITY;
    }
    return mine;
}

/**
 * What two scores of at most `largest` before their biases may be off against each other, in units of 2^-23. __expf is off by 2 + 1.173 |x| of e^x. A sigmoid,
 * s (1 - s) (2 + 1.173 |x|) < 0.8 from it, 0.5 from the sum and 2 from __fdividef; a softmax 2 from it (largest at x = 0), 0.2 from the difference, and 1.5 from
 * the quotient and the product. Twice that for two. All of a softmax share their sum: 2.2 of its terms and half for each of the PER + 5 additions. (The rounding of the
 * sum with the bias is in choose's `part`.)
 */
template <int PER> __device__ __forceinline__ float unsure_within(bool sigmoid, float largest) { return (sigmoid ? 8 : PER + 16) * largest * (1.0f / (1 << 23)); }

/** sigmoid(z) and a common factor of all that makes up for z far below zero: 1 / (e^-c + e^(-z - c)), c = max(0, -largest z). */
__device__ __forceinline__ float sigmoid_beside(float z, float largest) {
    const float c = largest < 0.0f ? -largest : 0.0f;
    return 1.0f / (expf(-c) + expf(-z - c));
}

/** Lane j's share r_j of the chosen, from its logit z (none: -infinity); 0 where there is none. */
__device__ __forceinline__ float share_of(const DcclRouting& how, bool there, float z) {
    const float top = largest_of_warp(there ? z : -INFINITY);
    const float s = !there ? 0.0f : how.sigmoid ? sigmoid_beside(z, top) : expf(z - top);
    const float sum = warp_sum(s);
    return there ? s / sum : 0.0f;
}

/**
 * Bytes are few (16384 tokens of 256 fp32 logits: 17 MB, 2.6 us); the instructions of the choice take the time. Groups of whole registers get their scores all at once,
 * and each of the k + 1 rounds is one reduction of the lists' heads. 16384 tokens of 256 fp32 logits, sigmoid with a bias, the best 4 of 8 groups by their two best, 8 experts: 30.0 us, and
 * 6.7 for the gradient; with a warp that had its next token's logits in flight, and so fewer warps of an SM, 34. 16 tokens take 2.6 us, of which the launch is most.
 */
template <typename T, int PER> __global__ void __launch_bounds__(32 * kRouteWarps, PER <= 8 ? 8 : 1) k_route(const __grid_constant__ RouteArgs a) {
    wait_for_stream();
    const int lane = threadIdx.x % 32;
    // whether the order of the scores is that of the logits
    const bool plain = !a.bias && (a.how.groups == 1 || !a.how.top2);
    const size_t token = (size_t)blockIdx.x * kRouteWarps + threadIdx.x / 32;
    if (token >= a.tokens) return;
    float c[PER], top = -INFINITY, sum = 1.0f;
    load_logits<T, PER>(a, token, c);
    bool poisoned = false;
    if (!a.how.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            poisoned |= c[i] != c[i];
            top = fmaxf(top, c[i]);
        }
        poisoned = __any_sync(kAll, poisoned);
        if (!plain || !a.how.renormalize) top = largest_of_warp(top);
    }
    if (!a.how.renormalize && !a.how.sigmoid) {         // the weights will take this sum
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) part += c[i] == -INFINITY ? 0.0f : expf(c[i] - top);
        sum = warp_sum(part);
    }
    float unsure = 1e-37f;          // of logits: below the normal numbers, steps are not parts of a size
    if (!plain) {
        if (a.how.sigmoid) {
#pragma unroll
            for (int i = 0; i < PER; i++) c[i] = c[i] == -INFINITY ? c[i] : __fdividef(1.0f, 1.0f + __expf(-c[i]));
            unsure = 1.0f;
        } else {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const float e = __expf(c[i] - top);
                part += c[i] == -INFINITY ? 0.0f : e;
                c[i] = c[i] == -INFINITY ? c[i] : e;
            }
            unsure = __fdividef(1.0f, warp_sum(part));          // of a softmax the largest score
#pragma unroll
            for (int i = 0; i < PER; i++) c[i] *= unsure;
        }
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (lane + 32 * i < (int)a.experts) c[i] += a.bias[lane + 32 * i];
        }
        unsure = unsure_within<PER>(a.how.sigmoid, unsure);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) c[i] = fmaxf(c[i], -INFINITY);          // NaN is not chosen
    int mine;
    if (!choose<T, PER>(a, token, c, unsure, mine)) mine = choose_exactly<T, PER>(a, token, plain);
    const bool there = mine >= 0;
    const float zm = there ? logit<T>(a, token, mine) : -INFINITY;
    float w;
    if (a.how.renormalize) w = share_of(a.how, there, zm);
    else w = !there ? 0.0f : a.how.sigmoid ? 1.0f / (1.0f + expf(-zm)) : expf(zm - top) / sum;
    if (poisoned && there) w = NAN;
    if (lane < a.how.k) {
        a.weights[token * a.how.k + lane] = a.how.scale * w;
        a.chosen[token * a.how.k + lane] = mine;
    }
}

/** The row goes through shared memory: what every expert gets first, then what the chosen get. */
template <typename T, int PER> __global__ void __launch_bounds__(32 * kRouteWarps) k_route_grad(const __grid_constant__ RouteArgs a) {
    wait_for_stream();
    __shared__ alignas(16) float rows[kRouteWarps][32 * PER];
    const int lane = threadIdx.x % 32, k = a.how.k;
    const size_t token = (size_t)blockIdx.x * kRouteWarps + threadIdx.x / 32;
    if (token >= a.tokens) return;
    float* const row = rows[threadIdx.x / 32];
    const int mine = lane < k ? a.chosen[token * k + lane] : -1;
    const bool there = mine >= 0 && mine < (int)a.experts;
    const float zm = there ? logit<T>(a, token, mine) : -INFINITY;
    const float g = there ? a.how.scale * a.dweights[token * k + lane] : 0.0f;
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
        load_logits<T, PER>(a, token, d);
#pragma unroll
        for (int i = 0; i < PER; i++) top = fmaxf(top, d[i]);
        top = largest_of_warp(top);
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
#pragma unroll
    for (int i = 0; i < PER; i++) row[lane + 32 * i] = d[i];
    __syncwarp();
    if (there) row[mine] = dm;
    __syncwarp();
    T* to = reinterpret_cast<T*>(a.dlogits) + token * a.experts;
    constexpr int M = 16 / sizeof(T);
    if (a.vec) {
        for (int e = lane * M; e < (int)a.experts; e += 32 * M) {
            float f[M];
#pragma unroll
            for (int q = 0; q < M; q += 4) {
                const Run<float, 4> r = ld_run<float, 4>(row + e + q);
#pragma unroll
                for (int p = 0; p < 4; p++) f[q + p] = r.e[p];
            }
            st_run<T, M>(to + e, round_run<T, M>(f));
        }
    } else {
        for (int e = lane; e < (int)a.experts; e += 32) to[e] = Traits<T>::down(row[e]);
    }
}

template <typename T, int PER> static cudaError_t run_route(const RouteArgs& a, bool backward, cudaStream_t stream) {
    const unsigned ctas = (a.tokens + kRouteWarps - 1) / kRouteWarps;
    return launch_early(backward ? k_route_grad<T, PER> : k_route<T, PER>, ctas, 32 * kRouteWarps, stream, a);
}
template <typename T> static cudaError_t run_route(RouteArgs a, bool backward, cudaStream_t stream) {
    a.vec = a.experts % (16 / sizeof(T)) == 0 && aligned_to(16, {a.dlogits});
    const unsigned per = (a.experts + 31) / 32;
    if (per <= 1) return run_route<T, 1>(a, backward, stream);
    if (per <= 2) return run_route<T, 2>(a, backward, stream);
    if (per <= 4) return run_route<T, 4>(a, backward, stream);
    if (per <= 8) return run_route<T, 8>(a, backward, stream);
    if (per <= 16) return run_route<T, 16>(a, backward, stream);
    return run_route<T, 32>(a, backward, stream);
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
    for (unsigned i = 0, whole = experts / how->groups / 32; i < 32 && experts / how->groups % 32 == 0; i++) a.ends |= (unsigned)((i + 1) % whole == 0) << i;
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
