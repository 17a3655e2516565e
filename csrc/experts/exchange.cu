/**
 * What stands between a router and the experts' products: where each token goes in the order of the experts (a stable counting sort), its row copied there
 * once for each of its experts, and the experts' results added up where the tokens came from,
 *
 *     out[r(t, j)] = x[t]             dx[t] = sum_j dout[r(t, j)]
 *     y[t] = sum_j w_tj in[r(t, j)]   din[r(t, j)] = w_tj dy[t],  dw_tj = in[r(t, j)] . dy[t]
 *
 * All four go token by token: a token's own row is read or written once, and no two add to the same place, so that sums need no atomics and come in the order of
 * j. HBM bounds them: 16384 tokens of 2048 bf16 by four experts, dispatch 51 us (335 MB, 6.5 TB/s), combine 59 (335 MB, 5.7), its gradient 112 (604 MB, 5.4); by one
 * expert 32 us and 51. Rows of an odd width go one element at a time: nothing wider starts where they do, and aligned pieces would have to
 * be shifted by what the starts of two rows differ.
 */
#include "expert_ops.hpp"
#include "../kernels/launch_early.cuh"
#include "../decoder/row_access.cuh"

namespace dccl {

/* ---- the order of the experts ---- */

constexpr int kPlanCtas = 8;            // a cluster of the portable size
constexpr int kPlanKept = 8;            // places of a lane that stay in registers

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

/** Lanes with the same number as this one, of `bits` bits that decide: as many ballots. With a match of 32-bit numbers the plan of 65536 places took 20 us, with these 11. */
__device__ __forceinline__ unsigned lanes_alike(unsigned e, int bits) {
    unsigned alike = 0xffffffffu;
    for (int b = 0; b < bits; b++) {
        const unsigned set = __ballot_sync(0xffffffffu, e >> b & 1);
        alike &= e >> b & 1 ? set : ~set;
    }
    return alike;
}

/**
 * One launch of one CTA, or of a cluster of eight that exchange their counts through shared memory. Every warp has a run of consecutive places, and counts of its
 * own. Two walks over the places: how many there are of each expert, and where they go; among 32 places one lane of each kind counts on. The chain from one 32
 * places to the next bounds it: 48 places 2.8 us, 1024 of 64 experts 5.6, 16384 by the cluster 6.7, 65536 10.4. More SMs would need a second launch, or a barrier over the device,
 * of 3 us: nothing to be gained up to some 16384 places, and more and more beyond.
 */
template <bool MANY> __device__ __forceinline__ void plan(const PlanArgs& a) {
    extern __shared__ unsigned counted[];           // [warps][experts], then [experts] of the CTA, then [32]
    const unsigned warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32, E = a.experts;
    unsigned* const mine = counted + warp * E;
    unsigned* const total = counted + warps * E;
    unsigned* const sums = total + E;
    unsigned rank = 0;
    if constexpr (MANY) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    constexpr unsigned ctas = MANY ? kPlanCtas : 1;
    const unsigned runs = ctas * warps, per = (((a.places + runs - 1) / runs) + 31) / 32 * 32;
    // in 64 bits: the last warps' runs may start behind everything
    const unsigned long long begin = (unsigned long long)(rank * warps + warp) * per;
    const unsigned from = begin < a.places ? (unsigned)begin : a.places, to = a.places - from < per ? a.places : from + per;
    for (unsigned i = threadIdx.x; i < warps * E; i += blockDim.x) counted[i] = 0;
    __syncthreads();
    wait_for_stream();
    unsigned kept[kPlanKept];                       // the first of the run, for the second walk
#pragma unroll
    for (int k = 0; k < kPlanKept; k++) kept[k] = from + 32 * k + lane < to ? plan_expert(a, from + 32 * k + lane) : 0xffffffffu;
#pragma unroll
    for (int k = 0; k < kPlanKept; k++)
        if (kept[k] < E) atomicAdd(mine + kept[k], 1);
    for (unsigned i = from + 32 * kPlanKept + lane; i < to; i += 32) {
        const unsigned e = plan_expert(a, i);
        if (e < E) atomicAdd(mine + e, 1);
    }
    __syncthreads();
    for (unsigned e = threadIdx.x; e < E; e += blockDim.x) {
        unsigned sum = 0;
#pragma unroll 8
        for (unsigned w = 0; w < warps; w++) {
            const unsigned n = counted[w * E + e];
            counted[w * E + e] = sum;
            sum += n;
        }
        total[e] = sum;
    }
    plan_cluster_sync(MANY);
    // every thread of a round has one expert: what the CTAs before have of it, and all
    unsigned start = 0;                             // of the round's first expert
    for (unsigned round = 0; round < E; round += blockDim.x) {
        const unsigned e = round + threadIdx.x;
        unsigned n = 0, here = 0;
        if (e < E) {
            unsigned v[ctas];
#pragma unroll
            for (unsigned c = 0; c < ctas; c++) v[c] = MANY ? of_other_cta(total + e, c) : total[e];
#pragma unroll
            for (unsigned c = 0; c < ctas; c++) {
                here += c < rank ? v[c] : 0;
                n += v[c];
            }
        }
        unsigned upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (unsigned)o) upto += v;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        unsigned before = start, all = 0;
        for (unsigned w = 0; w < warps; w++) {
            before += w < warp ? sums[w] : 0;
            all += sums[w];
        }
        before += upto - n;
        if (e < E) {
            if (rank == 0) {
                a.starts[e] = (int)before;
                a.counts[e] = (int)n;
                if (e == E - 1) a.starts[E] = (int)(before + n);
            }
#pragma unroll 8
            for (unsigned w = 0; w < warps; w++) counted[w * E + e] += before + here;
        }
        start += all;
        __syncthreads();
    }
    plan_cluster_sync(MANY);        // nobody's totals go before the others have read them, either
    const int bits = 32 - __clz(E);                 // a number of no expert is E
    const auto place = [&](unsigned i, unsigned e) {
        e = e < E ? e : E;
        const unsigned alike = lanes_alike(e, bits);
        const unsigned at = e < E ? mine[e] : 0;
        __syncwarp();
        if (e < E && lane == (unsigned)__ffs(alike) - 1) mine[e] = at + __popc(alike);
        if (i < to) a.rows[i] = e < E ? (int)(at + __popc(alike & ((1u << lane) - 1))) : -1;
        __syncwarp();
    };
#pragma unroll
    for (int k = 0; k < kPlanKept; k++)
        if (from + 32 * k < to) place(from + 32 * k + lane, kept[k]);
    for (unsigned base = from + 32 * kPlanKept; base < to; base += 32) place(base + lane, base + lane < to ? plan_expert(a, base + lane) : E);
}
__global__ void __launch_bounds__(1024) k_plan(const __grid_constant__ PlanArgs a) { plan<false>(a); }
__global__ void __launch_bounds__(1024) __cluster_dims__(kPlanCtas, 1, 1) k_plan_cluster(const __grid_constant__ PlanArgs a) { plan<true>(a); }

/* ---- rows ---- */

struct RowsArgs {
    const void *x, *in, *weights;       // of a token, and of rows in the experts' order
    void *out, *out2;
    const int *rows, *used;
    unsigned tokens, k, across;
    size_t width;
    bool weights32;
};

/**
 * A token belongs to `across` threads (whole warps), which take U runs of N elements each at a time, so far apart that a warp's accesses are of neighbours. A CTA has as
 * many tokens as fit; H of a token's rows are read at once. Lane j of every warp has the token's j-th row and weight, and hands them round: loads of them between those of the rows, under conditions of their
 * own, kept the latter from being in flight together (combine of 16384 x 2048 bf16 by 4: 84 us, and 58 without).
 */
constexpr int kRowThreads = 128;
constexpr unsigned kNoRow = 0xffffffffu;

struct Token { size_t index; unsigned thread, row; float weight; bool there; };
template <typename T> __device__ __forceinline__ Token token_of(const RowsArgs& a) {
    Token t;
    t.index = (size_t)blockIdx.x * (kRowThreads / a.across) + threadIdx.x / a.across;
    t.thread = threadIdx.x % a.across;
    t.there = t.index < a.tokens && threadIdx.x / a.across < kRowThreads / a.across;
    t.row = kNoRow;
    t.weight = 1.0f;
    const unsigned lane = threadIdx.x % 32;
    if (t.there && lane < a.k) {
        const size_t place = t.index * a.k + lane;
        t.row = (unsigned)a.rows[place];
        if (t.row >= a.tokens * a.k) t.row = kNoRow;        // a number that is none of a row is not followed
        if (a.weights) t.weight = a.weights32 ? reinterpret_cast<const float*>(a.weights)[place] : Traits<T>::up(reinterpret_cast<const T*>(a.weights)[place]);
        if (t.row == kNoRow) t.weight = 0.0f;
    }
    return t;
}

/** Zeros in those of the rows that stand at this token's places in `to` which nobody uses, where somebody says how many are used. */
template <typename T, int N> __device__ __forceinline__ void clear_unused(const RowsArgs& a, T* to, const Token& t) {
    if (!a.used) return;
    const unsigned used = (unsigned)*a.used;
    if ((t.index + 1) * a.k <= used) return;
    for (unsigned j = 0; j < a.k; j++) {
        const size_t row = t.index * a.k + j;
        if (row < used) continue;
        for (unsigned i = t.thread * N; i < a.width; i += a.across * N) st_run<T, N>(to + row * a.width + i, Run<T, N>{});
    }
}

/** Rows are bytes here: T is an unsigned integer of the elements' size. */
template <typename T, int N, int U> __global__ void __launch_bounds__(kRowThreads) k_dispatch(const __grid_constant__ RowsArgs a) {
    wait_for_stream();
    const Token t = token_of<T>(a);
    if (!t.there) return;
    const T* from = reinterpret_cast<const T*>(a.x) + t.index * a.width;
    T* const out = reinterpret_cast<T*>(a.out);
    const unsigned step = a.across * N;
    for (unsigned first = (t.thread & ~31u) * N; first < a.width; first += U * step) {       // of the warp, which goes on as one
        const unsigned i = first + (t.thread & 31) * N;
        Run<T, N> v[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * step < a.width) v[u] = ld_run<T, N>(from + i + u * step);
        for (unsigned j = 0; j < a.k; j++) {
            const unsigned row = __shfl_sync(0xffffffffu, t.row, j);
            if (row == kNoRow) continue;
            T* const to = out + (size_t)row * a.width + i;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i + u * step < a.width) st_run<T, N>(to + u * step, v[u]);
        }
    }
    clear_unused<T, N>(a, out, t);
}

/** H of a token's rows from the j0-th on, zeros where there is none. */
template <typename T, int N, int U, int H> __device__ __forceinline__ void hold_rows(const RowsArgs& a, const Token& t, unsigned j0, unsigned i, unsigned step, Run<T, N> (&v)[H][U]) {
#pragma unroll
    for (int j = 0; j < H; j++) {
        const unsigned row = __shfl_sync(0xffffffffu, t.row, j0 + j);
        const T* const from = reinterpret_cast<const T*>(a.in) + (size_t)row * a.width + i;
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[j][u] = Run<T, N>{};
            if (row != kNoRow && i + u * step < a.width) v[j][u] = ld_run<T, N>(from + u * step);
        }
    }
}

template <typename T, int N, int U, int H> __global__ void __launch_bounds__(kRowThreads, 9) k_combine(const __grid_constant__ RowsArgs a) {
    wait_for_stream();
    const Token t = token_of<T>(a);
    if (!t.there) return;
    const unsigned step = a.across * N;
    for (unsigned first = (t.thread & ~31u) * N; first < a.width; first += U * step) {
        const unsigned i = first + (t.thread & 31) * N;
        float sum[U][N] = {};
        for (unsigned j0 = 0; j0 < a.k; j0 += H) {          // at most 32, and lanes behind the last have none
            Run<T, N> v[H][U];
            hold_rows<T, N, U, H>(a, t, j0, i, step, v);
#pragma unroll
            for (int j = 0; j < H; j++) {
                const float w = __shfl_sync(0xffffffffu, t.weight, j0 + j);
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < N; e++) sum[u][e] = fmaf(w, Traits<T>::up(v[j][u].e[e]), sum[u][e]);
            }
        }
        T* const to = reinterpret_cast<T*>(a.out) + t.index * a.width + i;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * step < a.width) st_run<T, N>(to + u * step, round_run<T, N>(sum[u]));
    }
}

template <typename T, int N, int U, int H> __global__ void __launch_bounds__(kRowThreads, 9) k_combine_grad(const __grid_constant__ RowsArgs a) {
    wait_for_stream();
    __shared__ float dots[kRowThreads / 32][DCCL_EXPERTS_MAX_CHOSEN];
    const Token t = token_of<T>(a);
    T* const din = reinterpret_cast<T*>(a.out);
    const unsigned step = a.across * N;
    if (t.there) {
        const T* dy = reinterpret_cast<const T*>(a.x) + t.index * a.width;
        for (unsigned j0 = 0; j0 < a.k; j0 += H) {
            float dot[H] = {};
            for (unsigned first = (t.thread & ~31u) * N; first < a.width; first += U * step) {
                const unsigned i = first + (t.thread & 31) * N;
                Run<T, N> g[U], v[H][U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    g[u] = Run<T, N>{};
                    if (i + u * step < a.width) g[u] = ld_run<T, N>(dy + i + u * step);
                }
                if (a.out2) hold_rows<T, N, U, H>(a, t, j0, i, step, v);
#pragma unroll
                for (int j = 0; j < H; j++) {
                    if (a.out2) {
#pragma unroll
                        for (int u = 0; u < U; u++)
#pragma unroll
                            for (int e = 0; e < N; e++) dot[j] = fmaf(Traits<T>::up(g[u].e[e]), Traits<T>::up(v[j][u].e[e]), dot[j]);
                    }
                    const unsigned row = __shfl_sync(0xffffffffu, t.row, j0 + j);
                    const float w = __shfl_sync(0xffffffffu, t.weight, j0 + j);
                    if (!din || row == kNoRow) continue;
                    T* const to = din + (size_t)row * a.width + i;
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        float f[N];
#pragma unroll
                        for (int e = 0; e < N; e++) f[e] = w * Traits<T>::up(g[u].e[e]);
                        if (i + u * step < a.width) st_run<T, N>(to + u * step, round_run<T, N>(f));
                    }
                }
            }
            if (a.out2) {
#pragma unroll
                for (int j = 0; j < H; j++) {
                    float d = dot[j];
#pragma unroll
                    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                    if (threadIdx.x % 32 == 0 && j0 + j < a.k) dots[threadIdx.x / 32][j0 + j] = d;
                }
            }
        }
        if (din) clear_unused<T, N>(a, din, t);
    }
    if (!a.out2) return;
    __syncthreads();
    if (t.there && t.thread < a.k) {            // the first warp of the token, whose lane j has place j
        float dot = 0.0f;
        for (unsigned w = 0; w < a.across / 32; w++) dot += dots[threadIdx.x / 32 + w][t.thread];
        const size_t place = t.index * a.k + t.thread;
        if (t.row == kNoRow) dot = 0.0f;        // of a gradient that is not finite
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

/** Threads of a token: as many as one round of accesses needs, up to a CTA of them. */
static cudaError_t run_rows(void (*kernel)(const RowsArgs), int n, int u, RowsArgs& a, cudaStream_t stream) {
    const size_t warps = (a.width + 32 * n * u - 1) / (32 * n * u);
    a.across = warps >= kRowThreads / 32 ? kRowThreads : (unsigned)warps * 32;
    const unsigned tokens = kRowThreads / a.across;
    return launch_early_shared(kernel, (a.tokens + tokens - 1) / tokens, kRowThreads, 0, stream, a);
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_expert_plan(int device, size_t places, int experts, const void* chosen, int chosen64, int* rows, int* counts, int* starts, void* stream) {
    const char* who = "dccl_expert_plan";
    if (places > DCCL_EXPERTS_MAX_PLACES || experts < 1 || experts > DCCL_EXPERTS_MAX || !counts || !starts || (places && (!chosen || !rows))) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const PlanArgs a = {chosen, rows, counts, starts, (unsigned)places, (unsigned)experts, chosen64 != 0};
    // one warp for 32 places, up to 32 of them, and from two each on a cluster: 3063 places 5.8 us, by one CTA 6.7; 8192 places 6.3, by one 10
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
    if (!rows_fit(tokens, k, width) || !x || !rows || !out || (dtype != 6 && dtype != 7 && dtype != 9)) return report(who, cudaErrorInvalidValue);
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
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == 7) return report(who, run_of<uint32_t>(width, {x, out}) == 4 ? run_rows(k_dispatch<uint32_t, 4, 1>, 4, 1, a, s) : run_rows(k_dispatch<uint32_t, 1, 4>, 1, 4, a, s));
    const int n = run_of<uint16_t>(width, {x, out});
    return report(who, n == 8 ? run_rows(k_dispatch<uint16_t, 8, 1>, 8, 1, a, s) : n == 2 ? run_rows(k_dispatch<uint16_t, 2, 2>, 2, 2, a, s) : run_rows(k_dispatch<uint16_t, 1, 4>, 1, 4, a, s));
}

template <typename T> static cudaError_t run_combine(RowsArgs& a, cudaStream_t stream) {
    constexpr int most = 16 / sizeof(T), few = 4 / sizeof(T);
    const int n = run_of<T>(a.width, {a.in, a.out});
    // of one row two runs of a thread, of several a run each of two: 38 us by the latter for 16384 x 2048 bf16 by one, 32 by the former
    if (n == most && a.k == 1) return run_rows(k_combine<T, most, 2, 1>, most, 2, a, stream);
    if (n == most) return run_rows(k_combine<T, most, 1, 2>, most, 1, a, stream);
    if constexpr (few > 1)
        if (n == few) return run_rows(k_combine<T, few, 2, 2>, few, 2, a, stream);
    return run_rows(k_combine<T, 1, 4, 2>, 1, 4, a, stream);
}

template <typename T> static cudaError_t run_combine_grad(RowsArgs& a, cudaStream_t stream) {
    constexpr int most = 16 / sizeof(T), few = 4 / sizeof(T);
    const int n = run_of<T>(a.width, {a.x, a.in, a.out});
    // of one row two runs of a thread, of several a run each of two: 62 us by the latter for 16384 x 2048 bf16 by one, 51 by the former
    if (n == most && a.k == 1) return run_rows(k_combine_grad<T, most, 2, 1>, most, 2, a, stream);
    if (n == most) return run_rows(k_combine_grad<T, most, 1, 2>, most, 1, a, stream);
    if constexpr (few > 1)
        if (n == few) return run_rows(k_combine_grad<T, few, 2, 2>, few, 2, a, stream);
    return run_rows(k_combine_grad<T, 1, 4, 2>, 1, 4, a, stream);
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
    if (!rows_fit(tokens, k, width) || !dy || !rows || (dweights && !in) || (dtype != 6 && dtype != 7 && dtype != 9)) return report(who, cudaErrorInvalidValue);
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
