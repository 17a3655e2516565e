/**
 * A product of each expert's rows with that expert's weights, h_r = act(x_r W_e^T) for the rows r of expert e, and its gradients
 *
 *     dz = dh .* act'(z)      dx_r = dz_r W_e      dW_e = sum over the rows of e of dz_r x_r^T
 *
 * 2 N D F operations each for N rows of D elements and F results: the tensor cores bound it, for few rows the reading of the weights. Where an expert's rows start
 * is in device memory, and the host never reads it: each CTA makes the list of tiles from it. Operands keep the layout that they have in memory, as in
 * gated_linear.cu. A tile of one expert may load rows of the next behind its own; nobody stores what becomes of them, and where rows are what is summed
 * over, those behind the last are cleared in shared memory.
 */
#include "expert_ops.hpp"
#include "../kernels/launch_early.cuh"
#include "../decoder/activation.cuh"
#include "../decoder/products.cuh"
#include "grouped_tiles.hpp"

namespace dccl {

constexpr int kGroupedWarps = 8, kGroupedThreads = 32 * (kGroupedWarps + 2);      // that store; and one that loads, one that multiplies
constexpr unsigned kGroupedLoader = kGroupedWarps, kGroupedMultiplier = kGroupedWarps + 1;
constexpr int kNoActivation = -1;

/**
 * The normal distribution's cdf(z) and e^(-z^2 / 2), which its density needs as well. erfc(x) = t (c1 + ... + c7 t^6) e^(-x^2) with t = 1 / (1 + p x), the form of
 * Abramowitz and Stegun, "Handbook of Mathematical Functions", 7.1.26, with one more term pair and coefficients fitted on [0, 8] for an error that stays small against
 * erfc itself: 2e-8 near 0, 3e-6 of erfc at 4; in fp32 the cdf is off by 1.5e-7 at most. With erff the epilogue of a tile took longer than its
 * products, and k_act_grad, bound by its arithmetic, 177 us for 16384 x 5632 bf16 instead of 124 (each alone; see there).
 */
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    constexpr float root = 0.70710678118654752f;
    e = __expf(-0.5f * z * z);
    const float t = __fdividef(1.0f, fmaf(0.36f * root, fabsf(z), 1.0f));
    float c = fmaf(t, -0.1658067272f, 0.5732104218f);
    c = fmaf(t, c, -0.3708126889f);
    c = fmaf(t, c, 0.4417887144f);
    c = fmaf(t, c, 0.1015090368f);
    c = fmaf(t, c, 0.2180343121f);
    c = fmaf(t, c, 0.2020769013f);
    const float tail = 0.5f * t * c * e;
    return z < 0.0f ? tail : 1.0f - tail;
}
template <int ACT> __device__ __forceinline__ float value_of(float z) {
    if constexpr (ACT == DCCL_ACT_GELU) {
        float e;
        return z * normal_cdf(z, e);
    } else {
        return activate<ACT>(z);
    }
}
template <int ACT> __device__ __forceinline__ float slope_of(float z) {
    if constexpr (ACT == DCCL_ACT_GELU) {
        float e;
        const float cdf = normal_cdf(z, e);
        return fmaf(z * 0.3989422804014327f, e, cdf);
    } else {
        float value, slope;
        activate_grad<ACT>(z, value, slope);
        return slope;
    }
}

struct GroupedArgs : Grouped, GroupedResults {
    CUtensorMap a, b;
    const int* starts;
    int* ordered;                   // room for the starts in order, where the list has not one entry for each
    unsigned descriptor;            // of one product
    int act;
    bool whole_a, whole_b;          // one box holds all blocks of 64 columns of an operand
    int* gave_up;
};

/**
 * Tiles of M x N. A product reads 128 rows of the first operand from shared memory: behind M of them lies something else, and nobody reads what becomes of it. Tiles of more
 * are those of a pair of CTAs, each of which holds 128 of the rows and half of what makes the columns.
 */
template <int M, int N> struct GroupedShape {
    static constexpr bool kPair = M > kTileM;
    static constexpr int kHeldM = kPair ? kTileM : M, kHeldN = kPair ? N / 2 : N;
    static constexpr int kCtas = M < kTileM ? 2 : 1;        // of an SM: for small tiles, what one thread takes to give products out is what bounds a CTA
    static constexpr int kBytesA = kHeldM * kTileK * 2, kBytesB = kHeldN * kTileK * 2, kBytes = kBytesA + kBytesB, kStages = 192 * 1024 / kCtas / kBytes;
    static constexpr int kStagings = M < kTileM ? 2 : kGroupedWarps;                    // warps that have rows to store
    static constexpr int kShared = kStages * kBytes + kStagings * 4096 + 1024;          // 1024: the tiles' alignment
    static_assert(kCtas * (kShared + 2 * 1024) <= 227 * 1024, "with the list of tiles and the barriers");
    static_assert(kTileM * kTileK * 2 - kBytes <= kStagings * 4096, "what the last stage's product reads");
};

/**
 * The list of tiles, by one warp: first[i], the rows of tiles before expert i * stride, and all of them. own: the starts, where every expert is listed. False where a start lies before
 * those ahead of it.
 */
__device__ __forceinline__ bool list_tiles(const Grouped& a, const int* starts, unsigned* first, int* own) {
    const unsigned lane = threadIdx.x % 32, entries = listed_of(a);
    unsigned before = 0;
    bool back = false;
    for (unsigned base = 0; base < entries; base += 32) {
        const unsigned i = base + lane;
        unsigned n = 0;
        for (unsigned e = i * a.stride; e < (i + 1) * a.stride && e <= a.experts; e++) {
            n += tall_of(starts, e, a);
            back |= goes_back(starts, e, a);
        }
        if (a.stride == 1 && i < entries) own[i] = starts[i];
        const unsigned mine = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= (unsigned)o) n += v;
        }
        if (i < entries) first[i] = before + n - mine;
        before += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) first[entries] = before;
    return !__any_sync(0xffffffffu, back);
}

/** The starts in order, each as far as those ahead of it. By one warp; several CTAs may write the same numbers to the same place. */
__device__ __noinline__ void order_starts(const Grouped& a, const int* starts, volatile int* ordered) {
    const unsigned lane = threadIdx.x % 32;
    unsigned reached = 0;
    for (unsigned base = 0; base <= a.experts; base += 32) {
        unsigned reach = base + lane <= a.experts ? max(reached, row_within(starts[base + lane], a.rows)) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, reach, o);
            if (lane >= (unsigned)o) reach = max(reach, v);
        }
        if (base + lane <= a.experts) ordered[base + lane] = (int)reach;
        reached = __reduce_max_sync(0xffffffffu, reach);
    }
    __syncwarp();
}

/**
 * Zeros in the rows of a block of k behind `left` of them, for both operands, which stand in LINES / 64 blocks of 64 rows of 128 bytes: rows of the next expert, and whatever
 * they are; as many as the last product of 16 would add. By one warp.
 */
template <int LINES> __device__ __forceinline__ void clear_rows(char* at, unsigned left, unsigned lane) {
    const unsigned pieces = ((left + 15) / 16 * 16 - left) * 8;
    for (unsigned i = lane; i < pieces * LINES / 64; i += 32) *reinterpret_cast<uint4*>(at + i / pieces * 64 * 128 + left * 128 + i % pieces * 16) = uint4{};
    shared_writes_before_products();
    __syncwarp();
}

/**
 * One CTA per SM walks over tiles of M rows and N columns; one warp loads, one multiplies, eight store: a warp reaches the quarter of the tile's rows that its
 * number gives, so two share one and take half of the columns each. The sums of two tiles fit into tensor memory, so that one is stored while the next is
 * multiplied.
 *
 * What an SM can load bounds a single CTA: the 48 KB of a block of 64 in k for 128 x 256 take 450 ns (57 bytes a clock), their products 270; for 128 x 128, 32 KB and 275 ns. As a
 * pair, two CTAs share tiles of 256 x 256 and load 32 KB each. The leader's barriers count the bytes of both, and the leader multiplies; only where rows behind the last are
 * cleared, each does that to its own, and the other one tells the leader (by an arrival for every block it took 900 ns a block). 16384 rows of 8 experts, 2048 x 5632,
 * bf16, pairs (and single CTAs): h 249 us (288), dx 247 (273), dW 278 (289), 1.36 to 1.53 PFLOP/s, where power bounds them as it does the library's products.
 * The loader must never pause: it finds its place in a tile from shared memory and without divisions, and as a load takes it some 60 clocks to give out, one box holds all
 * blocks of an operand where rows allow (dW of single CTAs 333 us with a box per block of 64 columns, 286 with one).
 * Tiles of 128 x 128 and 128 x 256 serve where the larger would leave SMs without work; tiles of 32 x 64, two CTAs of an SM, where experts have few rows and reading the weights
 * takes the time (two rows of each of those experts: 41 us, 4.5 TB/s; four of each of four: 25); there, what one thread takes to give products out counts: 60 us with descriptors made anew for each, 44 with
 * their low words counted up.
 */
template <typename T, int FORM, int M, int N> __device__ __forceinline__ void grouped(const GroupedArgs& a) {
    using Shape = GroupedShape<M, N>;
    constexpr int kStages = Shape::kStages;
    constexpr bool PAIR = Shape::kPair;
    extern __shared__ char shared[];
    __shared__ uint64_t bars[(PAIR ? 3 : 2) * kStages + 5];
    __shared__ unsigned first[kListed + 1];
    __shared__ int own[kListed + 1];
    __shared__ uint32_t tmem_base;
    __shared__ int failed, in_order;
    char* const tiles = shared + (1024 - shared_addr(shared) % 1024) % 1024;
    char* const staging = tiles + kStages * Shape::kBytes;
    const uint32_t full = shared_addr(bars), empty = full + 8 * kStages, sums_full = empty + 8 * kStages, sums_empty = sums_full + 16, drained = sums_empty + 16, landed = drained + 8;
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = PAIR ? cluster_rank() : 0;
    const unsigned worker = PAIR ? blockIdx.x / 2 : blockIdx.x, workers = PAIR ? gridDim.x / 2 : gridDim.x;
    if (warp == kGroupedMultiplier) {
        if constexpr (PAIR) pair_tmem_alloc(shared_addr(&tmem_base), 2 * N);
        else tmem_alloc(shared_addr(&tmem_base), 2 * N);
    }
    if (threadIdx.x == 0) {
        failed = 0;
        for (int i = 0; i < kStages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; PAIR && i < kStages; i++) bar_init(landed + 8 * i, 1);
        for (int i = 0; i < 2; i++) { bar_init(sums_full + 8 * i, 1); bar_init(sums_empty + 8 * i, (PAIR ? 2 : 1) * kGroupedWarps); }
        bar_init(drained, 1);
        bar_init_fence();
    }
    if (threadIdx.x == 32 * kGroupedLoader) {
        prefetch_map(&a.a);
        prefetch_map(&a.b);
    }
    wait_for_stream();
    if (warp == 1) {
        const bool sound = list_tiles(a, a.starts, first, own);
        in_order = sound;
        if (!sound) {
            order_starts(a, a.starts, a.stride == 1 ? own : a.ordered);
            list_tiles(a, a.stride == 1 ? own : a.ordered, first, own);
        }
    }
    tc_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    tc_after_sync();
    const int* const starts = a.stride == 1 ? own : in_order ? a.starts : a.ordered;
    const uint32_t sums = tmem_base;
    const unsigned total = grouped_tiles(FORM, a, first);
    InFlight loads;                 // of the loader
    if (warp == kGroupedLoader && lane == 0) {
        unsigned s = 0, parity = 1;
        const auto load = [](auto... box) {
            if constexpr (PAIR) pair_load_box(box...);
            else load_box(box...);
        };
        for (unsigned tile = worker; tile < total; tile += workers) {
            const GroupedPlace p = grouped_place(FORM, tile, a, first, starts);
            const unsigned row = p.row + rank * Shape::kHeldM, column = p.column + rank * Shape::kHeldN;
            const unsigned blocks = (p.k_count + kTileK - 1) / kTileK;
            unsigned kb = 0;
            for (; kb < blocks; kb++) {
                if (!bar_wait(empty + 8 * s, parity, &failed)) break;
                const bool tail = PAIR && FORM == EXPERTS_WEIGHT && kb + 1 == blocks && p.k_count % kTileK;          // where each CTA clears rows first
                const uint32_t to_a = shared_addr(tiles) + s * Shape::kBytes, to_b = to_a + Shape::kBytesA, bar = tail ? in_cta(landed + 8 * s, rank) : PAIR ? in_cta(full + 8 * s, 0) : full + 8 * s;
                const int k = p.k_from + kb * kTileK;
                loads.load(s, tail);
                if (tail) bar_expect(landed + 8 * s, Shape::kBytes);
                else if (rank == 0) bar_expect(full + 8 * s, (PAIR ? 2 : 1) * Shape::kBytes);         // the leader counts both CTAs' bytes
                if constexpr (FORM == EXPERTS_FORWARD) {
                    load(to_a, &a.a, k, row, bar);
                    load(to_b, &a.b, k, column, p.expert, bar);
                } else if constexpr (FORM == EXPERTS_INPUT) {
                    load(to_a, &a.a, k, row, bar);
                    if (a.whole_b) load(to_b, &a.b, 0, k, column / 64, p.expert, bar);
                    else
#pragma unroll
                        for (int i = 0; i < Shape::kHeldN / 64; i++) load(to_b + i * 64 * 128, &a.b, column + 64 * i, k, p.expert, bar);
                } else {
                    if (a.whole_a) load(to_a, &a.a, 0, k, row / 64, bar);
                    else
#pragma unroll
                        for (int i = 0; i < Shape::kHeldM / 64; i++) load(to_a + i * 64 * 128, &a.a, row + 64 * i, k, bar);
                    if (a.whole_b) load(to_b, &a.b, 0, k, column / 64, bar);
                    else
#pragma unroll
                        for (int i = 0; i < Shape::kHeldN / 64; i++) load(to_b + i * 64 * 128, &a.b, column + 64 * i, k, bar);
                }
                if (++s == kStages) { s = 0; parity ^= 1; }
            }
            if (kb < blocks) break;
        }
    } else if (warp == kGroupedMultiplier && rank != 0) {       // the leader multiplies
        if constexpr (FORM == EXPERTS_WEIGHT) {
            unsigned used = 0, parities = 0;
            for (unsigned tile = worker; tile < total; tile += workers) {
                const GroupedPlace p = grouped_place(FORM, tile, a, first, starts);
                used += (p.k_count + kTileK - 1) / kTileK;
                const unsigned left = p.k_count % kTileK;
                if (!left) continue;
                const unsigned s = (used - 1) % kStages;
                if (!bar_wait_warp(landed + 8 * s, parities >> s & 1, &failed)) break;
                parities ^= 1u << s;
                clear_rows<Shape::kHeldM + Shape::kHeldN>(tiles + s * Shape::kBytes, left, lane);
                if (elect_one()) bar_arrive_remote(in_cta(full + 8 * s, 0));
            }
        }
    } else if (warp == kGroupedMultiplier) {
        unsigned done = 0, s = 0, parity = 0, parities = 0;
        const uint64_t of_a = tile_descriptor(shared_addr(tiles), FORM == EXPERTS_WEIGHT ? 64 * 128 : 16);
        const uint64_t of_b = tile_descriptor(shared_addr(tiles) + Shape::kBytesA, FORM == EXPERTS_FORWARD ? 16 : 64 * 128);
        const uint32_t first_a = (uint32_t)of_a, high_a = (uint32_t)(of_a >> 32), first_b = (uint32_t)of_b, high_b = (uint32_t)(of_b >> 32);
        for (unsigned tile = worker; tile < total; tile += workers) {
            const GroupedPlace p = grouped_place(FORM, tile, a, first, starts);
            const unsigned blocks = (p.k_count + kTileK - 1) / kTileK;
            if (!blocks) continue;
            const unsigned buffer = done & 1;
            if (!bar_wait_warp(sums_empty + 8 * buffer, (done / 2 & 1) ^ 1, &failed)) break;
            tc_after_sync();
            const uint32_t d = sums + buffer * N;
            unsigned kb = 0;
            for (; kb < blocks; kb++) {
                if (!bar_wait_warp(full + 8 * s, parity, &failed)) break;
                tc_after_sync();
                char* const at = tiles + s * Shape::kBytes;
                unsigned steps = kTileK / 16;
                if constexpr (FORM == EXPERTS_WEIGHT) {
                    const unsigned left = p.k_count - kb * kTileK;
                    if (left < (unsigned)kTileK) {      // rows of the next expert, and whatever they are: as many as the last product of 16 would add
                        steps = (left + 15) / 16;
                        if constexpr (PAIR) {
                            if (!bar_wait_warp(landed + 8 * s, parities >> s & 1, &failed)) break;
                            parities ^= 1u << s;
                        }
                        clear_rows<Shape::kHeldM + Shape::kHeldN>(at, left, lane);
                    }
                }
                if (elect_one()) {
                    const uint32_t da = first_a + s * (Shape::kBytes >> 4), db = first_b + s * (Shape::kBytes >> 4);
#pragma unroll
                    for (unsigned k = 0; k < kTileK / 16; k++) {
                        if (FORM == EXPERTS_WEIGHT && k >= steps) break;
                        // 16 k: 32 bytes further along K-major rows, or 16 rows of 128 bytes further
                        const uint32_t at_a = da + k * (FORM == EXPERTS_WEIGHT ? 128 : 2), at_b = db + k * (FORM == EXPERTS_FORWARD ? 2 : 128);
                        if constexpr (PAIR) pair_product(d, at_a, high_a, at_b, high_b, a.descriptor, kb || k);
                        else product(d, at_a, high_a, at_b, high_b, a.descriptor, kb || k);
                    }
                    if constexpr (PAIR) pair_commit(empty + 8 * s);
                    else commit(empty + 8 * s);
                }
                __syncwarp();
                if (++s == kStages) { s = 0; parity ^= 1; }
            }
            if (kb < blocks) break;
            if (elect_one()) {
                if constexpr (PAIR) pair_commit(sums_full + 8 * buffer);
                else commit(sums_full + 8 * buffer);
            }
            done++;
        }
    } else if (warp < kGroupedWarps) {
        char* const stage = staging + (M < kTileM ? warp / 4 : warp) * 4096;
        unsigned done = 0;
        const bool vec = a.n % 8 == 0 && aligned16(a.c);
        const unsigned quarter = warp % 4, half = warp / 4, above = rank * kTileM + quarter * 32;
        for (unsigned tile = worker; tile < total; tile += workers) {
            const GroupedPlace p = grouped_place(FORM, tile, a, first, starts);
            const int rows = above < p.rows ? (int)(p.rows - above < 32 ? p.rows - above : 32) : 0;
            const size_t row = grouped_row(FORM, p, above, a);
            const bool summed = p.k_count != 0;         // otherwise nothing was: rows of nobody, an expert without rows
            const unsigned buffer = done & 1;
            if (summed) {
                if (!bar_wait_warp(sums_full + 8 * buffer, done / 2 & 1, &failed)) break;
                tc_after_sync();
            }
            const uint32_t d = sums + buffer * N + (quarter * 32u << 16);
#pragma unroll 1
            for (int c = half * (N / 2); c < (int)(half + 1) * (N / 2); c += 32) {
                const size_t column = (size_t)p.column + c;
                if (column >= a.n || !rows) break;
                const int columns = (int)(a.n - column < 32 ? a.n - column : 32);
                float v[32] = {};
                if (summed) {
                    uint32_t r[32];
                    tmem_load32(r, d + c);
                    tmem_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = __uint_as_float(r[e]);
                }
                if (a.splits.d > 1) {
                    stage_rows(stage, v);
                    store_fp32(stage, a.partial + (p.split * grouped_rows(FORM, a) + row) * a.partial_stride + column, a.partial_stride, rows, columns);
                    continue;
                }
                if constexpr (FORM == EXPERTS_FORWARD) {
                    if (summed && a.act != kNoActivation) {
                        if (a.z) {
                            stage_rows(stage, v);
                            store_fp32(stage, a.z + row * a.z_stride + column, a.z_stride, rows, columns);
                        }
                        with_activation(a.act, [&](auto act) {
#pragma unroll
                            for (int e = 0; e < 32; e++) v[e] = value_of<decltype(act)::value>(v[e]);
                        });
                    }
                }
                stage_rows(stage, v);
                store_as<T>(stage, reinterpret_cast<T*>(a.c) + row * a.n + column, a.n, rows, columns, vec);
            }
            if (!summed) continue;
            done++;
            tc_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) bar_arrive_remote(in_cta(sums_empty + 8 * buffer, 0));
                else bar_arrive(sums_empty + 8 * buffer);
            }
        }
    }
    __syncthreads();
    if (failed) {       // no wait is expected to run out: copies in flight still have to land, and products to end, before the memory is given back
        int late = 0;
        grouped_mark(FORM, a, a, first, starts, worker, workers, threadIdx.x, kGroupedThreads);
        if (warp == kGroupedLoader && lane == 0 && rank != 0)       // its copies count on the leader's barriers: here only time tells that they have landed
            for (const long long start = clock64(); clock64() - start < kLandClocks;) {}
        if (warp == kGroupedLoader && lane == 0 && rank == 0)
            for (unsigned i = loads.oldest(kStages); i < loads.filled; i++)
                bar_wait((loads.on_landed(i, kStages) ? landed : full) + 8 * (i % kStages), loads.parity(i, kStages), &late);
        if (rank == 0 && warp == kGroupedMultiplier && elect_one()) {        // the lane whose products they are
            if constexpr (PAIR) pair_commit(drained);
            else commit(drained);
            bar_wait(drained, 0, &late);
        }
        if (threadIdx.x == 0 && a.gave_up) *reinterpret_cast<volatile int*>(a.gave_up) = 1;
        __syncthreads();
    }
    if constexpr (PAIR) cluster_sync();      // neither CTA's memory goes before the other is done with it
    tc_after_sync();
    if (warp == kGroupedMultiplier) {
        if constexpr (PAIR) pair_tmem_free(sums, 2 * N);
        else tmem_free(sums, 2 * N);
    }
}
template <typename T, int FORM, int M, int N> __global__ void __launch_bounds__(kGroupedThreads, GroupedShape<M, N>::kCtas) k_grouped(const __grid_constant__ GroupedArgs a) {
    grouped<T, FORM, M, N>(a);
}
template <typename T, int FORM, int N> __global__ void __launch_bounds__(kGroupedThreads, 1) __cluster_dims__(2, 1, 1) k_grouped_pair(const __grid_constant__ GroupedArgs a) {
    grouped<T, FORM, 2 * kTileM, N>(a);
}

struct JoinPartsArgs { const float* partial; size_t rows, stride; unsigned n, splits, runs; int act; void* c; float* z; size_t z_stride; bool vec; };

/** Adds the parts that splits of k left, in the order of k, and finishes: four columns per thread. */
template <typename T> __global__ void __launch_bounds__(256) k_join_parts(const __grid_constant__ JoinPartsArgs a) {
    wait_for_stream();
    const size_t index = (size_t)blockIdx.x * 256 + threadIdx.x, row = index / a.runs;
    if (row >= a.rows) return;
    const unsigned column = (unsigned)(index - row * a.runs) * 4;
    const float* from = a.partial + row * a.stride + column;
    Run<float, 4> v = {};
#pragma unroll 4
    for (unsigned s = 0; s < a.splits; s++) {
        const Run<float, 4> p = ld_run<float, 4>(from + s * a.rows * a.stride);
#pragma unroll
        for (int e = 0; e < 4; e++) v.e[e] += p.e[e];
    }
    if (a.act != kNoActivation) {
        if (a.z) st_run<float, 4>(a.z + row * a.z_stride + column, v);      // rows of these end on four elements as well
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 4; e++) v.e[e] = value_of<decltype(act)::value>(v.e[e]);
        });
    }
    T* to = reinterpret_cast<T*>(a.c) + row * a.n + column;
    if (a.vec) st_run<T, 4>(to, round_run<T, 4>(v.e));
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (column + e < a.n) to[e] = Traits<T>::down(v.e[e]);
}

constexpr int kRowCta = 256;

struct PadRowsArgs { const uint16_t* from[2]; uint16_t* to[2]; size_t rows[2]; unsigned width, runs, across; };

/**
 * Rows that do not start on 16 bytes, copied to some that do, for the tiled loads; zeros behind a row. A thread writes eight elements at a time and reads the two
 * aligned pieces of 16 bytes that hold them, where those lie inside of the operand; the second is the neighbour's first, and comes from L1.
 */
__global__ void __launch_bounds__(kRowCta) k_pad_rows(const __grid_constant__ PadRowsArgs a) {
    wait_for_stream();
    size_t row = (size_t)blockIdx.x * (kRowCta / a.across) + threadIdx.x / a.across;
    if (threadIdx.x / a.across >= kRowCta / a.across) return;
    const int w = row >= a.rows[0];
    if (w) row -= a.rows[0];
    if (row >= a.rows[w]) return;
    const uint16_t *begin = a.from[w], *from = begin + row * a.width, *end = begin + a.rows[w] * a.width;
    const unsigned off = reinterpret_cast<uintptr_t>(from) % 16 / 2;        // elements behind a boundary
    for (unsigned i = threadIdx.x % a.across; i < a.runs; i += a.across) {
        const uint16_t* at = from + 8 * i;
        Run<uint16_t, 8> r = {};
        if (at - off >= begin && at - off + 16 <= end && 8 * i + 8 <= a.width) {
            uint32_t v[8];
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at - off);
            *reinterpret_cast<uint4*>(v + 4) = *reinterpret_cast<const uint4*>(at - off + 8);
            // first by whole words, then by half of one
#pragma unroll
            for (int by = 4; by >= 1; by /= 2)
                if (off / 2 & by) {
#pragma unroll
                    for (int q = 0; q + by < 8; q++) v[q] = v[q + by];
                }
            uint32_t* const o = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
            for (int q = 0; q < 4; q++) o[q] = off & 1 ? __funnelshift_r(v[q], v[q + 1], 16) : v[q];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (8 * i + e < a.width) r.e[e] = at[e];
        }
        st_run<uint16_t, 8>(a.to[w] + (row * a.runs + i) * 8, r);
    }
}

struct ActGradArgs { const void* dh; const float* z; void* dz; const int* starts; size_t z_stride, stride; unsigned rows, experts, n, from, threads; Divisor runs; int act; };

/** dz from dh and the saved products, eight elements per thread; rows behind the last expert's, whose products nobody wrote, are left out. Only the rows of dh may start
 *  anywhere (VEC: they do not). HBM bounds it: 8 bytes per element, 16384 x 5632 in 125 us alone (5.9 TB/s), in 142 between
 *  the products of a step, which take the clock down. */
template <typename T, bool VEC> __global__ void __launch_bounds__(kRowCta) k_act_grad(const __grid_constant__ ActGradArgs a) {
    wait_for_stream();
    __shared__ unsigned reach[kRowCta / 32];
    const unsigned index = blockIdx.x * kRowCta + threadIdx.x, last = min(blockIdx.x * kRowCta + kRowCta, a.threads) - 1;
    unsigned used = row_within(a.starts[a.experts], a.rows);
    if ((size_t)a.from + a.runs.quotient(last) >= used) {       // some of the CTA: a start ahead of the last may lie further
        unsigned most = 0;
        for (unsigned e = threadIdx.x; e < a.experts; e += kRowCta) most = max(most, row_within(a.starts[e], a.rows));
        most = __reduce_max_sync(0xffffffffu, most);
        if (threadIdx.x % 32 == 0) reach[threadIdx.x / 32] = most;
        __syncthreads();
        for (unsigned w = 0; w < kRowCta / 32; w++) used = max(used, reach[w]);
    }
    if (index >= a.threads) return;
    const unsigned line = a.runs.quotient(index), column = (index - line * a.runs.d) * 8;
    const size_t row = (size_t)a.from + line;
    if (row >= used) return;
    float z[8] = {}, d[8];
#pragma unroll
    for (int q = 0; q < 2; q++) {
        if (column + 4 * q >= a.n) break;           // rows of z end on four elements
        const Run<float, 4> x = ld_run<float, 4>(a.z + row * a.z_stride + column + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; e++) z[4 * q + e] = x.e[e];
    }
    const T* dh = reinterpret_cast<const T*>(a.dh) + row * a.n + column;
    if constexpr (VEC) {
        const Run<T, 8> r = ld_run<T, 8>(dh);
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] = Traits<T>::up(r.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] = column + e < a.n ? Traits<T>::up(dh[e]) : 0.0f;
    }
    with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] *= slope_of<decltype(act)::value>(z[e]);
    });
    st_run<T, 8>(reinterpret_cast<T*>(a.dz) + row * a.stride + column, round_run<T, 8>(d));
}

/* ------------------------------------------------------------------------------------------------ host side */

/** Where the parts of a call's workspace lie. */
struct GroupedLayout { size_t stride, x, w, padded, dz, d_stride, partial, ordered, total; GroupedPlan forward, input, weight; bool ok; };

static size_t parts_of(const GroupedPlan& p, size_t rows, size_t n) { return p.splits > 1 ? p.splits * rows * up_to(n, 4) * sizeof(float) : 0; }

static GroupedLayout grouped_layout(int device, size_t rows, int experts, size_t width, size_t out, bool aligned, bool backward) {
    GroupedLayout l = {};
    const int sms = sm_count(device);
    l.ok = sms > 0 && rows <= DCCL_EXPERTS_MAX_PLACES && experts >= 1 && experts <= DCCL_EXPERTS_MAX && width >= 1 && width <= DCCL_EXPERTS_MAX_WIDTH && out >= 1
           && out <= DCCL_EXPERTS_MAX_WIDTH;
    if (!l.ok) return l;
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t here = at; at += up_to(bytes, 256); return here; };
    // rows of whole lines: the tiled loads take twice as long for pieces of 128 bytes that lie in two
    const bool pad = !aligned || width % 8;
    l.stride = pad ? up_to(width, 64) : width;
    if (pad) {      // at the same places in both directions: the backward pass finds them in what the forward pass left
        l.x = take(rows * l.stride * 2);
        l.w = take((size_t)experts * out * l.stride * 2);
        l.padded = at;
        if (backward) at = 0;
    }
    l.d_stride = up_to(out, 64);
    l.forward = plan_grouped(EXPERTS_FORWARD, sms, rows, experts, 0, out, width);
    l.input = plan_grouped(EXPERTS_INPUT, sms, rows, experts, 0, width, out);
    l.weight = plan_grouped(EXPERTS_WEIGHT, sms, rows, experts, out, width, 0);
    if (backward) {
        l.dz = take(rows * l.d_stride * 2);
        const size_t input = parts_of(l.input, rows, width), weight = parts_of(l.weight, experts * out, width);
        l.partial = take(input > weight ? input : weight);
    } else {
        l.partial = take(parts_of(l.forward, rows, out));
    }
    if (listed_by(experts) > 1) l.ordered = take((experts + 1) * sizeof(int));
    l.total = at;
    return l;
}

template <typename T, int FORM, int M, int N> static auto grouped_kernel() {
    if constexpr (GroupedShape<M, N>::kPair) return k_grouped_pair<T, FORM, N>;
    else return k_grouped<T, FORM, M, N>;
}

template <typename T, int FORM, int M, int N> static cudaError_t run_grouped(int device, GroupedArgs& a, cudaStream_t stream) {
    using Shape = GroupedShape<M, N>;
    const auto kernel = grouped_kernel<T, FORM, M, N>();
    static std::atomic<bool> ready[64];
    if (!ready[device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kShared);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_relaxed);
    }
    a.descriptor = product_descriptor(std::is_same<T, __nv_bfloat16>::value, FORM == EXPERTS_WEIGHT, FORM != EXPERTS_FORWARD, Shape::kPair ? M : kTileM, N);
    const unsigned workers = Shape::kPair ? (unsigned)sm_count(device) / 2 : (unsigned)sm_count(device) * Shape::kCtas;
    return launch_early_shared(kernel, (a.most < workers ? a.most : workers) * (Shape::kPair ? 2 : 1), kGroupedThreads, Shape::kShared, stream, a);
}

template <typename T, int FORM> static cudaError_t run_grouped(int device, const GroupedPlan& p, GroupedArgs& a, cudaStream_t stream) {
    a.tile_rows = p.tile_rows;
    a.tile_columns = p.tile_columns;
    a.tiles_m = FORM == EXPERTS_WEIGHT ? blocks_of(a.m, p.tile_rows) : 0;
    a.tiles_n = By(blocks_of(a.n, p.tile_columns));
    a.group = By(16 * a.tiles_n.d);
    a.expert = By(FORM == EXPERTS_WEIGHT ? a.tiles_m * a.tiles_n.d : 1);
    a.splits = By(p.splits);
    // every expert may have a row of tiles that is not full, and the rows of nobody one at each end
    const unsigned long long most = (FORM == EXPERTS_WEIGHT ? (unsigned long long)a.experts * a.tiles_m : blocks_of(a.rows, p.tile_rows) + a.experts + 2ull) * a.tiles_n.d * p.splits;
    if (most > 1u << 30 || 16ull * a.tiles_n.d * (a.tiles_m ? a.tiles_m : 1) > 1u << 30) return cudaErrorInvalidValue;      // places are counted in 31 bits
    a.most = (unsigned)most;
    a.partial_stride = up_to(a.n, 4);
    a.gave_up = gave_up_flag(device);
    cudaError_t e;
    const auto large = [&] {
        return p.tile_rows > kTileM       ? run_grouped<T, FORM, 2 * kTileM, 256>(device, a, stream)
               : p.tile_columns == 128 ? run_grouped<T, FORM, 128, 128>(device, a, stream)
                                       : run_grouped<T, FORM, 128, 256>(device, a, stream);
    };
    if constexpr (FORM == EXPERTS_FORWARD) e = p.tile_rows == 32 ? run_grouped<T, FORM, 32, 64>(device, a, stream) : large();
    else e = large();
    if (e != cudaSuccess || p.splits == 1) return e;
    const JoinPartsArgs j = {a.partial, grouped_rows(FORM, a), a.partial_stride, a.n, p.splits, (unsigned)(a.partial_stride / 4), a.act, a.c, a.z, a.z_stride,
                             a.n % 4 == 0 && aligned_to(8, {a.c})};
    return launch_early(k_join_parts<T>, (unsigned)((j.rows * j.runs + 255) / 256), 256, stream, j);
}

/**
 * The map of an operand whose rows are summed over, [matrices][rows][columns], of which a tile takes `blocks` blocks of 64 columns. Where rows are whole blocks apart, the
 * blocks are a dimension of their own and one box holds them all: a load takes the loader some 60 clocks to give out, and six a block were as long as its products.
 */
static cudaError_t map_of_blocks(CUtensorMap* map, bool& whole, int dtype, const void* base, size_t matrices, size_t rows, size_t columns, size_t stride, unsigned blocks) {
    whole = stride % 64 == 0;
    if (whole && matrices) return make_map(map, dtype, base, 4, {64, rows, stride / 64, matrices}, {stride, 64, stride * rows}, {64, kTileK, blocks, 1});
    if (whole) return make_map(map, dtype, base, 3, {64, rows, stride / 64, 1}, {stride, 64, 0}, {64, kTileK, blocks, 1});
    if (matrices) return make_map(map, dtype, base, 3, {columns, rows, matrices, 1}, {stride, stride * rows, 0}, {64, kTileK, 1, 1});
    return make_map(map, dtype, base, columns, rows, stride, kTileK);
}

static cudaError_t pad_rows(const void*& x, const void*& w, size_t rows, size_t w_rows, size_t width, size_t stride, void* to_x, void* to_w, cudaStream_t stream) {
    PadRowsArgs a = {{(const uint16_t*)x, (const uint16_t*)w}, {(uint16_t*)to_x, (uint16_t*)to_w}, {rows, w_rows}, (unsigned)width, (unsigned)(stride / 8), kRowCta};
    if (a.runs < kRowCta) a.across = (a.runs + 31) / 32 * 32;
    x = to_x;
    w = to_w;
    const size_t per = kRowCta / a.across;
    return launch_early(k_pad_rows, (unsigned)((rows + w_rows + per - 1) / per), kRowCta, stream, a);
}

/** In launches of less than 2^31 threads. */
template <typename T> static cudaError_t run_act_grad(ActGradArgs a, bool vec, cudaStream_t stream) {
    a.runs = Divisor((a.n + 7) / 8);
    const unsigned most = ((1u << 31) - 1) / a.runs.d;
    cudaError_t e = cudaSuccess;
    for (size_t from = 0; from < a.rows && e == cudaSuccess; from += most) {
        a.from = (unsigned)from;
        a.threads = (unsigned)(a.rows - from < most ? a.rows - from : most) * a.runs.d;
        e = launch_early(vec ? k_act_grad<T, true> : k_act_grad<T, false>, (a.threads + kRowCta - 1) / kRowCta, kRowCta, stream, a);
    }
    return e;
}

struct GroupedCall {
    int device, dtype, experts, act;
    size_t rows, width, out;
    const int* starts;
    char* workspace;
    cudaStream_t stream;
};

static GroupedArgs grouped_args(const GroupedCall& k, const GroupedLayout& l) {
    GroupedArgs a = {};
    a.partial = (float*)(k.workspace + l.partial);
    a.rows = (unsigned)k.rows;
    a.experts = (unsigned)k.experts;
    a.starts = k.starts;
    a.act = kNoActivation;
    a.stride = listed_by(a.experts);
    if (a.stride > 1) a.ordered = (int*)(k.workspace + l.ordered);
    return a;
}

template <typename T> static cudaError_t grouped_forward(const GroupedCall& k, const GroupedLayout& l, const void* x, const void* w, void* h, float* z, size_t z_stride) {
    cudaError_t e = cudaSuccess;
    if (l.padded) e = pad_rows(x, w, k.rows, (size_t)k.experts * k.out, k.width, l.stride, k.workspace + l.x, k.workspace + l.w, k.stream);
    GroupedArgs a = grouped_args(k, l);
    a.n = (unsigned)k.out;
    a.k_blocks = blocks_of(k.width, kTileK);
    a.act = k.act;
    a.c = h;
    a.z = z;
    a.z_stride = z_stride;
    if (e == cudaSuccess) e = make_map(&a.a, k.dtype, x, k.width, k.rows, l.stride, l.forward.held_rows());
    if (e == cudaSuccess) e = make_map(&a.b, k.dtype, w, 3, {k.width, k.out, (size_t)k.experts, 1}, {l.stride, l.stride * k.out, 0}, {64, l.forward.held_columns(), 1, 1});
    return e == cudaSuccess ? run_grouped<T, EXPERTS_FORWARD>(k.device, l.forward, a, k.stream) : e;
}

template <typename T> static cudaError_t grouped_backward(const GroupedCall& k, const GroupedLayout& l, const void* dh, const float* z, size_t z_stride, const void* x, const void* w,
                                                          const char* padded, void* dx, void* dw) {
    cudaError_t e = cudaSuccess;
    const void* dz = dh;
    const bool vec = k.out % 8 == 0 && aligned_to(16, {dh});
    if (k.act != kNoActivation) {
        ActGradArgs d = {};
        d.dh = dh;
        d.z = z;
        d.dz = k.workspace + l.dz;
        d.starts = k.starts;
        d.z_stride = z_stride;
        d.stride = l.d_stride;
        d.rows = (unsigned)k.rows;
        d.experts = (unsigned)k.experts;
        d.n = (unsigned)k.out;
        d.act = k.act;
        e = run_act_grad<T>(d, vec, k.stream);
        dz = d.dz;
    } else if (!vec) {
        const void* none = nullptr;
        e = pad_rows(dz, none, k.rows, 0, k.out, l.d_stride, k.workspace + l.dz, nullptr, k.stream);
    }
    if (l.padded) {
        x = padded + l.x;
        w = padded + l.w;
    }
    const size_t d_stride = dz == dh ? k.out : l.d_stride;
    if (e == cudaSuccess && dx) {
        GroupedArgs a = grouped_args(k, l);
        a.n = (unsigned)k.width;
        a.k_blocks = blocks_of(k.out, kTileK);
        a.c = dx;
        e = make_map(&a.a, k.dtype, dz, k.out, k.rows, d_stride, kTileM);
        if (e == cudaSuccess) e = map_of_blocks(&a.b, a.whole_b, k.dtype, w, k.experts, k.out, k.width, l.stride, l.input.held_columns() / 64);
        if (e == cudaSuccess) e = run_grouped<T, EXPERTS_INPUT>(k.device, l.input, a, k.stream);
    }
    if (e == cudaSuccess && dw) {
        GroupedArgs a = grouped_args(k, l);
        a.m = (unsigned)k.out;
        a.n = (unsigned)k.width;
        a.c = dw;
        e = map_of_blocks(&a.a, a.whole_a, k.dtype, dz, 0, k.rows, k.out, d_stride, kTileM / 64);
        if (e == cudaSuccess) e = map_of_blocks(&a.b, a.whole_b, k.dtype, x, 0, k.rows, k.width, l.stride, l.weight.held_columns() / 64);
        if (e == cudaSuccess) e = run_grouped<T, EXPERTS_WEIGHT>(k.device, l.weight, a, k.stream);
    }
    return e;
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_expert_linear_pads(size_t width, int aligned) { return !aligned || width % 8; }

extern "C" long long dccl_expert_linear_workspace(int device, size_t rows, int experts, size_t width, size_t out, int aligned, int backward) {
    const GroupedLayout l = grouped_layout(device, rows, experts, width, out, aligned != 0, backward != 0);
    return l.ok ? (long long)l.total : -1;
}

extern "C" int dccl_expert_linear(int device, int dtype, size_t rows, int experts, size_t width, size_t out, const void* x, const void* w, const int* starts, int act, void* h, float* z,
                                  size_t z_stride, void* workspace, long long workspace_bytes, void* stream) {
    const char* who = "dccl_expert_linear";
    if (!rows) return 0;
    const GroupedLayout l = grouped_layout(device, rows, experts, width, out, aligned_to(16, {x, w}), false);
    if (!l.ok || workspace_bytes < (long long)l.total || (dtype != 6 && dtype != 9) || act < kNoActivation || act > DCCL_ACT_GELU_TANH || !x || !w || !starts || !h
        || (z && (z_stride < out || z_stride % 4)) || !aligned_to(16, {z, workspace}))
        return report(who, cudaErrorInvalidValue);
    if (gave_up(who, device)) return -1;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const GroupedCall k = {device, dtype, experts, act, rows, width, out, starts, (char*)workspace, (cudaStream_t)stream};
    return report(who, dtype == 6 ? grouped_forward<__half>(k, l, x, w, h, z, z_stride) : grouped_forward<__nv_bfloat16>(k, l, x, w, h, z, z_stride));
}

extern "C" int dccl_expert_linear_backward(int device, int dtype, size_t rows, int experts, size_t width, size_t out, const void* dh, const float* z, size_t z_stride, const void* x,
                                           const void* w, const int* starts, const void* forward_workspace, int act, void* dx, void* dw, void* workspace, long long workspace_bytes,
                                           void* stream) {
    const char* who = "dccl_expert_linear_backward";
    const GroupedLayout l = grouped_layout(device, rows, experts, width, out, aligned_to(16, {x, w}), true);
    if (!l.ok || !rows || workspace_bytes < (long long)l.total || (dtype != 6 && dtype != 9) || act < kNoActivation || act > DCCL_ACT_GELU_TANH || !dh || !x || !w || !starts
        || (act != kNoActivation && (!z || z_stride < out || z_stride % 4)) || !aligned_to(16, {z, workspace, forward_workspace}) || (l.padded && !forward_workspace))
        return report(who, cudaErrorInvalidValue);
    if (gave_up(who, device)) return -1;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const GroupedCall k = {device, dtype, experts, act, rows, width, out, starts, (char*)workspace, (cudaStream_t)stream};
    return report(who, dtype == 6 ? grouped_backward<__half>(k, l, dh, z, z_stride, x, w, (const char*)forward_workspace, dx, dw)
                                  : grouped_backward<__nv_bfloat16>(k, l, dh, z, z_stride, x, w, (const char*)forward_workspace, dx, dw));
}
