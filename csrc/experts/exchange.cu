/**
 * What stands between a router and the experts' products: where each token goes in the order of the experts (a stable counting sort), its row copied there
 * once for each of its experts, and the experts' results added up where the tokens came from,
 *
 *     out[r(t, j)] = x[t]             dx[t] = sum_j dout[r(t, j)]
 *     y[t] = sum_j w_tj in[r(t, j)]   din[r(t, j)] = w_tj dy[t],  dw_tj = in[r(t, j)] . dy[t]
 *
 * All four go token by token: a token's own row is read or written once, and no two add to the same place, so that sums need no atomics and come in the order of
 * j. HBM bounds them.
 */
#include "expert_ops.hpp"
#include "../kernels/launch_early.cuh"
#include "../decoder/row_access.cuh"

namespace dccl {

/* ---- the order of the experts ---- */

constexpr int kPlanCtas = 8;            // a cluster of the portable size

struct PlanArgs {
    const void* chosen;
    int *rows, *counts, *starts;
    unsigned places, experts;
    bool wide;                          // 64-bit numbers
};

__device__ __forceinline__ unsigned plan_expert(const PlanArgs& a, unsigned i) {
    // a number that is none of an expert, whatever its size, becomes one that is none either
    if (!a.wide) return (unsigned)reinterpret_cast<const int*>(a.chosen)[i];
    const unsigned long long e = reinterpret_cast<const unsigned long long*>(a.chosen)[i];
    return e < a.experts ? (unsigned)e : 0xffffffffu;
}

__device__ __forceinline__ void plan_cluster_sync(bool many) {
    if (many) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}
__device__ __forceinline__ unsigned of_other_cta(const unsigned* mine, unsigned rank) {
    uint32_t at, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

/**
 * One launch of one CTA, or of a cluster of eight that exchange their counts through shared memory. Every warp has a run of consecutive places; the ranks of
 * equal experts among 32 places come from a match, and one lane of each kind counts on. Two walks over the places: how many there are, and where they go.
 */
template <bool MANY> __device__ __forceinline__ void plan(const PlanArgs& a) {
    extern __shared__ unsigned counted[];           // [warps][experts], then [experts] of the CTA, then [32]
    const unsigned warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32, E = a.experts;
    unsigned* const mine = counted + warp * E;
    unsigned* const total = counted + warps * E;
    unsigned* const sums = total + E;
    unsigned rank = 0;
    if constexpr (MANY) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const unsigned ctas = MANY ? kPlanCtas : 1, runs = ctas * warps, per = (((a.places + runs - 1) / runs) + 31) / 32 * 32;
    // in 64 bits: the last warps' runs may start behind everything
    const unsigned long long begin = (unsigned long long)(rank * warps + warp) * per;
    const unsigned from = begin < a.places ? (unsigned)begin : a.places, to = a.places - from < per ? a.places : from + per;
    for (unsigned i = threadIdx.x; i < warps * E; i += blockDim.x) counted[i] = 0;
    __syncthreads();
    wait_for_stream();
    for (unsigned base = from; base < to; base += 32) {
        const unsigned e = base + lane < to ? plan_expert(a, base + lane) : 0xffffffffu;
        const unsigned alike = __match_any_sync(0xffffffffu, e);
        if (e < E && lane == (unsigned)__ffs(alike) - 1) mine[e] += __popc(alike);
        __syncwarp();
    }
    __syncthreads();
    for (unsigned e = threadIdx.x; e < E; e += blockDim.x) {
        unsigned sum = 0;
        for (unsigned w = 0; w < warps; w++) {
            const unsigned n = counted[w * E + e];
            counted[w * E + e] = sum;
            sum += n;
        }
        total[e] = sum;
    }
    plan_cluster_sync(MANY);
    // starts of the experts: threads take runs of consecutive ones
    const unsigned each = (E + blockDim.x - 1) / blockDim.x, first = min(threadIdx.x * each, E), last = min(first + each, E);
    unsigned own = 0;
    for (unsigned e = first; e < last; e++)
        for (unsigned c = 0; c < ctas; c++) own += MANY ? of_other_cta(total + e, c) : total[e];
    unsigned before = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= (unsigned)o) before += v;
    }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    unsigned start = before - own;
    for (unsigned w = 0; w < warp; w++) start += sums[w];
    for (unsigned e = first; e < last; e++) {
        unsigned n = 0, here = 0;
        for (unsigned c = 0; c < ctas; c++) {
            const unsigned v = MANY ? of_other_cta(total + e, c) : total[e];
            here += c < rank ? v : 0;
            n += v;
        }
        if (rank == 0) {
            a.starts[e] = (int)start;
            a.counts[e] = (int)n;
            if (e == E - 1) a.starts[E] = (int)(start + n);
        }
        for (unsigned w = 0; w < warps; w++) counted[w * E + e] += start + here;
        start += n;
    }
    plan_cluster_sync(MANY);        // nobody's totals go before the others have read them, either
    for (unsigned base = from; base < to; base += 32) {
        const unsigned i = base + lane, e = i < to ? plan_expert(a, i) : 0xffffffffu;
        const unsigned alike = __match_any_sync(0xffffffffu, e);
        const unsigned at = e < E ? mine[e] : 0;
        __syncwarp();
        if (e < E && lane == (unsigned)__ffs(alike) - 1) mine[e] = at + __popc(alike);
        if (i < to) a.rows[i] = e < E ? (int)(at + __popc(alike & ((1u << lane) - 1))) : -1;
        __syncwarp();
    }
}
__global__ void __launch_bounds__(1024) k_plan(const __grid_constant__ PlanArgs a) { plan<false>(a); }
__global__ void __launch_bounds__(1024) __cluster_dims__(kPlanCtas, 1, 1) k_plan_cluster(const __grid_constant__ PlanArgs a) { plan<true>(a); }

/* ---- rows ---- */

struct RowsArgs {
    const void *x, *in, *weights;       // of a token, and of rows in the experts' order
    void *out, *out2;
    const int *rows, *used;
    unsigned tokens, k;
    size_t width;
    bool weights32;
};

constexpr int kRowThreads = 128;

/** Where the row of a place is, or -1: a number that is none of a row is not followed. */
__device__ __forceinline__ int row_of(const RowsArgs& a, size_t place) {
    const int row = a.rows[place];
    return (unsigned)row < a.tokens * a.k ? row : -1;
}

template <typename T> __device__ __forceinline__ float weight_of(const RowsArgs& a, size_t place) {
    return !a.weights ? 1.0f : a.weights32 ? reinterpret_cast<const float*>(a.weights)[place] : Traits<T>::up(reinterpret_cast<const T*>(a.weights)[place]);
}

/** Zeros in those of the rows that stand at this token's places in `to` which nobody uses. */
template <typename T, int N> __device__ __forceinline__ void clear_unused(const RowsArgs& a, T* to, size_t token) {
    const unsigned used = (unsigned)*a.used;
    if ((token + 1) * a.k <= used) return;
    for (unsigned j = 0; j < a.k; j++) {
        const size_t row = token * a.k + j;
        if (row < used) continue;
        for (size_t i = threadIdx.x * N; i < a.width; i += kRowThreads * N) st_run<T, N>(to + row * a.width + i, Run<T, N>{});
    }
}

/** Rows are bytes here: T is an unsigned integer of the elements' size. */
template <typename T, int N> __global__ void __launch_bounds__(kRowThreads) k_dispatch(const __grid_constant__ RowsArgs a) {
    wait_for_stream();
    const size_t token = blockIdx.x;
    const T* from = reinterpret_cast<const T*>(a.x) + token * a.width;
    T* out = reinterpret_cast<T*>(a.out);
    for (size_t i = threadIdx.x * N; i < a.width; i += kRowThreads * N) {
        const Run<T, N> v = ld_run<T, N>(from + i);
        for (unsigned j = 0; j < a.k; j++) {
            const int row = row_of(a, token * a.k + j);
            if (row >= 0) st_run<T, N>(out + (size_t)row * a.width + i, v);
        }
    }
    clear_unused<T, N>(a, out, token);
}

template <typename T, int N> __global__ void __launch_bounds__(kRowThreads) k_combine(const __grid_constant__ RowsArgs a) {
    wait_for_stream();
    const size_t token = blockIdx.x;
    const T* in = reinterpret_cast<const T*>(a.in);
    for (size_t i = threadIdx.x * N; i < a.width; i += kRowThreads * N) {
        float sum[N] = {};
        for (unsigned j = 0; j < a.k; j++) {
            const int row = row_of(a, token * a.k + j);
            if (row < 0) continue;
            const float w = weight_of<T>(a, token * a.k + j);
            const Run<T, N> v = ld_run<T, N>(in + (size_t)row * a.width + i);
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] = fmaf(w, Traits<T>::up(v.e[e]), sum[e]);
        }
        st_run<T, N>(reinterpret_cast<T*>(a.out) + token * a.width + i, round_run<T, N>(sum));
    }
}

template <typename T, int N> __global__ void __launch_bounds__(kRowThreads) k_combine_grad(const __grid_constant__ RowsArgs a) {
    wait_for_stream();
    __shared__ float dots[kRowThreads / 32][DCCL_EXPERTS_MAX_CHOSEN];
    const size_t token = blockIdx.x;
    const T* dy = reinterpret_cast<const T*>(a.x) + token * a.width;
    const T* in = reinterpret_cast<const T*>(a.in);
    T* din = reinterpret_cast<T*>(a.out);
    for (unsigned j = 0; j < a.k; j++) {
        const size_t place = token * a.k + j;
        const int row = row_of(a, place);
        float dot = 0.0f;
        if (row >= 0) {
            const float w = weight_of<T>(a, place);
            for (size_t i = threadIdx.x * N; i < a.width; i += kRowThreads * N) {
                const Run<T, N> g = ld_run<T, N>(dy + i);
                float to[N];
                if (a.out2) {
                    const Run<T, N> v = ld_run<T, N>(in + (size_t)row * a.width + i);
#pragma unroll
                    for (int e = 0; e < N; e++) dot = fmaf(Traits<T>::up(g.e[e]), Traits<T>::up(v.e[e]), dot);
                }
                if (din) {
#pragma unroll
                    for (int e = 0; e < N; e++) to[e] = w * Traits<T>::up(g.e[e]);
                    st_run<T, N>(din + (size_t)row * a.width + i, round_run<T, N>(to));
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (threadIdx.x % 32 == 0) dots[threadIdx.x / 32][j] = dot;
    }
    if (din) clear_unused<T, N>(a, din, token);
    if (!a.out2) return;
    __syncthreads();
    if (threadIdx.x < a.k) {
        float dot = 0.0f;
        for (int w = 0; w < kRowThreads / 32; w++) dot += dots[w][threadIdx.x];
        const size_t place = token * a.k + threadIdx.x;
        if (a.weights32) reinterpret_cast<float*>(a.out2)[place] = dot;
        else reinterpret_cast<T*>(a.out2)[place] = Traits<T>::down(dot);
    }
}

/* ---- host side ---- */

static bool rows_fit(size_t tokens, int k, size_t width) {
    return k >= 1 && k <= DCCL_EXPERTS_MAX_CHOSEN && width >= 1 && width <= DCCL_EXPERTS_MAX_WIDTH && tokens <= DCCL_EXPERTS_MAX_PLACES && tokens * k <= DCCL_EXPERTS_MAX_PLACES;
}

/** The widest access of whole runs that the rows allow: 16 bytes, 4, or single elements. */
template <typename T> static int run_of(size_t width, std::initializer_list<const void*> ps) {
    const int most = 16 / sizeof(T), few = 4 / sizeof(T);
    return width % most == 0 && aligned_to(16, ps) ? most : width % few == 0 && aligned_to(4, ps) ? few : 1;
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_expert_plan(int device, size_t places, int experts, const void* chosen, int chosen64, int* rows, int* counts, int* starts, void* stream) {
    const char* who = "dccl_expert_plan";
    if (places > DCCL_EXPERTS_MAX_PLACES || experts < 1 || experts > DCCL_EXPERTS_MAX || !counts || !starts || (places && (!chosen || !rows))) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const PlanArgs a = {chosen, rows, counts, starts, (unsigned)places, (unsigned)experts, chosen64 != 0};
    // one warp for 32 places, up to 32 of them, and from there on a cluster
    const bool many = places > 2048;
    const unsigned warps = many ? 32 : places > 32 ? (unsigned)((places + 31) / 32 > 32 ? 32 : (places + 31) / 32) : 1;
    const size_t shared = ((size_t)warps * experts + experts + 32) * sizeof(unsigned);
    const auto kernel = many ? k_plan_cluster : k_plan;
    static std::atomic<bool> ready[2][64];
    if (device < 0 || device >= 64) return report(who, cudaErrorInvalidDevice);
    if (shared > 48 * 1024 && !ready[many][device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (33 * DCCL_EXPERTS_MAX + 32) * (int)sizeof(unsigned));
        if (e != cudaSuccess) return report(who, e);
        ready[many][device].store(true, std::memory_order_relaxed);
    }
    return report(who, launch_early_shared(kernel, many ? kPlanCtas : 1, warps * 32, shared, (cudaStream_t)stream, a));
}

extern "C" int dccl_dispatch(int device, int dtype, size_t tokens, int k, size_t width, const void* x, const int* rows, const int* used, void* out, void* stream) {
    const char* who = "dccl_dispatch";
    if (!tokens) return 0;
    if (!rows_fit(tokens, k, width) || !x || !rows || !used || !out || (dtype != 6 && dtype != 7 && dtype != 9)) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    RowsArgs a = {};
    a.x = x;
    a.out = out;
    a.rows = rows;
    a.used = used;
    a.tokens = (unsigned)tokens;
    a.k = (unsigned)k;
    a.width = width;
    const auto go = [&](auto kernel) { return launch_early(kernel, a.tokens, kRowThreads, (cudaStream_t)stream, a); };
    if (dtype == 7) {
        const int n = run_of<uint32_t>(width, {x, out});
        return report(who, n == 4 ? go(k_dispatch<uint32_t, 4>) : go(k_dispatch<uint32_t, 1>));
    }
    const int n = run_of<uint16_t>(width, {x, out});
    return report(who, n == 8 ? go(k_dispatch<uint16_t, 8>) : n == 2 ? go(k_dispatch<uint16_t, 2>) : go(k_dispatch<uint16_t, 1>));
}

template <typename T> static cudaError_t run_combine(const RowsArgs& a, cudaStream_t stream) {
    const auto go = [&](auto kernel) { return launch_early(kernel, a.tokens, kRowThreads, stream, a); };
    const int n = run_of<T>(a.width, {a.in, a.out});
    if (n == 16 / (int)sizeof(T)) return go(k_combine<T, 16 / sizeof(T)>);
    if (sizeof(T) == 2 && n == 2) return go(k_combine<T, 2>);
    return go(k_combine<T, 1>);
}

template <typename T> static cudaError_t run_combine_grad(const RowsArgs& a, cudaStream_t stream) {
    const auto go = [&](auto kernel) { return launch_early(kernel, a.tokens, kRowThreads, stream, a); };
    const int n = run_of<T>(a.width, {a.x, a.in, a.out});
    if (n == 16 / (int)sizeof(T)) return go(k_combine_grad<T, 16 / sizeof(T)>);
    if (sizeof(T) == 2 && n == 2) return go(k_combine_grad<T, 2>);
    return go(k_combine_grad<T, 1>);
}

extern "C" int dccl_combine(int device, int dtype, size_t tokens, int k, size_t width, const void* in, const int* rows, const void* weights, int weights32, void* y, void* stream) {
    const char* who = "dccl_combine";
    if (!tokens) return 0;
    if (!rows_fit(tokens, k, width) || !in || !rows || !y || (dtype != 6 && dtype != 7 && dtype != 9)) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    RowsArgs a = {};
    a.in = in;
    a.weights = weights;
    a.weights32 = weights32 != 0;
    a.out = y;
    a.rows = rows;
    a.tokens = (unsigned)tokens;
    a.k = (unsigned)k;
    a.width = width;
    const cudaStream_t s = (cudaStream_t)stream;
    return report(who, dtype == 6 ? run_combine<__half>(a, s) : dtype == 7 ? run_combine<float>(a, s) : run_combine<__nv_bfloat16>(a, s));
}

extern "C" int dccl_combine_backward(int device, int dtype, size_t tokens, int k, size_t width, const void* dy, const void* in, const int* rows, const int* used, const void* weights,
                                     int weights32, void* din, void* dweights, void* stream) {
    const char* who = "dccl_combine_backward";
    if (!tokens || (!din && !dweights)) return 0;
    if (!rows_fit(tokens, k, width) || !dy || !rows || !used || (dweights && !in) || (dtype != 6 && dtype != 7 && dtype != 9)) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    RowsArgs a = {};
    a.x = dy;
    a.in = in;
    a.weights = weights;
    a.weights32 = weights32 != 0;
    a.out = din;
    a.out2 = dweights;
    a.rows = rows;
    a.used = used;
    a.tokens = (unsigned)tokens;
    a.k = (unsigned)k;
    a.width = width;
    const cudaStream_t s = (cudaStream_t)stream;
    return report(who, dtype == 6 ? run_combine_grad<__half>(a, s) : dtype == 7 ? run_combine_grad<float>(a, s) : run_combine_grad<__nv_bfloat16>(a, s));
}
