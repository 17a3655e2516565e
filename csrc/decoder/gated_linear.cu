/**
 * The gated half of a feed-forward layer, h = act(x Wg^T) .* (x Wu^T), and its gradients
 *
 *     dg = dh .* u .* act'(g)      dx  = dg Wg + du Wu
 *     du = dh .* act(g)            dWg = dg^T x,  dWu = du^T x
 *
 * 4 T F H operations forward and 8 T F H backward for T tokens: the tensor cores bound it, for few tokens the reading of the weights.
 * All products are one kernel in three forms, except for those of few tokens forward (k_gated_few). Operands keep the layout that they have in memory: whichever of their two
 * dimensions is the contiguous one, a box of 64 of it fills the 128-byte rows of a swizzled tile, and the product is told the
 * tile's orientation. Sums stay in tensor memory in fp32 until the end of a tile.
 */
#include "decoder_ops.hpp"
#include "../kernels/launch_early.cuh"
#include "row_access.cuh"
#include "../device/tcgen05.cuh"
#include "../gpu/driver_api.hpp"
#include "gated_tiles.hpp"
#include <cstring>

namespace dccl {

constexpr int kEpilogueWarps = 8, kGemmThreads = 32 * (kEpilogueWarps + 2);
constexpr unsigned kLoader = kEpilogueWarps, kMultiplier = kEpilogueWarps + 1;
constexpr int kStageRowsBytes = 128;                                // one row of a swizzled tile

struct GemmArgs : Tiling, Results {
    CUtensorMap a0, a1, b0, b1;
    unsigned k_half;                // INPUT_GRAD: blocks of ffn, after which the second pair of operands follows
    unsigned descriptor;            // of one product
    int act;
    int* gave_up;                   // host memory: a wait that did not end
};

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

constexpr float kTanhScale = 1.5957691216057308f, kTanhCubic = 0.044715f;      // 2 sqrt(2 / pi)

/** 0.5 g (1 + tanh(z)) = g sigmoid(2 z). */
template <int ACT> __device__ __forceinline__ float activate(float g) {
    if constexpr (ACT == DCCL_ACT_SILU) return g * sigmoid(g);
    else if constexpr (ACT == DCCL_ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
    else return g * sigmoid(kTanhScale * fmaf(kTanhCubic * g * g, g, g));
}

/** The activation and its derivative. */
template <int ACT> __device__ __forceinline__ void activate_grad(float g, float& a, float& da) {
    if constexpr (ACT == DCCL_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        da = s * fmaf(g, 1.0f - s, 1.0f);
    } else if constexpr (ACT == DCCL_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        a = g * cdf;
        da = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), cdf);
    } else {
        const float s = sigmoid(kTanhScale * fmaf(kTanhCubic * g * g, g, g));
        a = g * s;
        da = fmaf(g * s * (1.0f - s), kTanhScale * fmaf(3.0f * kTanhCubic * g, g, 1.0f), s);
    }
}

/** f with the activation as a constant: one choice for many elements. */
template <typename F> __device__ __forceinline__ void with_activation(int act, F&& f) {
    if (act == DCCL_ACT_SILU) f(std::integral_constant<int, DCCL_ACT_SILU>{});
    else if (act == DCCL_ACT_GELU) f(std::integral_constant<int, DCCL_ACT_GELU>{});
    else f(std::integral_constant<int, DCCL_ACT_GELU_TANH>{});
}

/** Rows of a tile's 32 columns pass through shared memory, so that a warp stores whole rows and not one line per lane. `stage`: 4 KB of
 *  this warp, 16-byte pieces of row r at piece ^ (r % 8). */
__device__ __forceinline__ void stage_rows(char* stage, const float (&v)[32]) {
    const int lane = threadIdx.x % 32;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; c++)
        *reinterpret_cast<float4*>(stage + lane * 128 + ((c ^ (lane & 7)) * 16)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    __syncwarp();
}
/** Stores the staged 32 x 32 values as fp32 at `to` (row 0, column 0), rows < rows and columns < columns. Rows start on 16 bytes. */
__device__ __forceinline__ void store_fp32(const char* stage, float* to, size_t stride, int rows, int columns) {
    const int lane = threadIdx.x % 32, c = lane % 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = i * 4 + lane / 8;
        const float4 v = *reinterpret_cast<const float4*>(stage + r * 128 + ((c ^ (r & 7)) * 16));
        if (r < rows && 4 * c < columns) *reinterpret_cast<float4*>(to + (size_t)r * stride + 4 * c) = v;      // up to three of the padding
    }
}
/** The same as T, whose rows may start anywhere. */
template <typename T> __device__ __forceinline__ void store_as(const char* stage, T* to, size_t stride, int rows, int columns, bool vec) {
    const int lane = threadIdx.x % 32;
    if (vec) {
        const int c = lane % 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = i * 8 + lane / 4;
            const float4 v = *reinterpret_cast<const float4*>(stage + r * 128 + (((2 * c) ^ (r & 7)) * 16));
            const float4 w = *reinterpret_cast<const float4*>(stage + r * 128 + (((2 * c + 1) ^ (r & 7)) * 16));
            Run<T, 8> o = {Traits<T>::down(v.x), Traits<T>::down(v.y), Traits<T>::down(v.z), Traits<T>::down(v.w),
                           Traits<T>::down(w.x), Traits<T>::down(w.y), Traits<T>::down(w.z), Traits<T>::down(w.w)};
            if (r < rows && 8 * c < columns) st_run<T, 8>(to + (size_t)r * stride + 8 * c, o);
        }
    } else if (lane < columns) {
#pragma unroll 4
        for (int r = 0; r < rows && r < 32; r++)
            to[(size_t)r * stride + lane] = Traits<T>::down(*reinterpret_cast<const float*>(stage + r * 128 + (((lane / 4) ^ (r & 7)) * 16) + lane % 4 * 4));
    }
}

template <int FORM, int N, bool PAIR> struct GemmShape {
    static constexpr int kRows = PAIR ? 2 * kTileM : kTileM, kHeldN = PAIR ? N / 2 : N;      // rows of a tile; columns whose operand one CTA holds
    static constexpr int kBytesA = kTileM * kTileK * 2, kBytesB = kHeldN * kTileK * 2, kBytes = kBytesA + kBytesB, kStages = 192 * 1024 / kBytes;
    static constexpr int kShared = kStages * kBytes + kEpilogueWarps * 4096 + 1024;      // 1024: the tiles' alignment
    static constexpr int kColumns = FORM == GATED ? N / 2 : N;                           // of the result
};

/**
 * One CTA per SM walks over tiles of 128 rows; one warp loads, one multiplies, eight store: a warp reaches the quarter of the tile's
 * rows that its number gives, so two share one and take half of the columns each. The sums of two tiles fit into tensor memory, so that
 * one is stored while the next is multiplied. As a PAIR, two CTAs share tiles of 256 rows, and each loads only half of the columns' operand.
 *
 * 16384 tokens x 2048 x 5632 bf16, pairs (and single CTAs): forward 503 us (535), with the products stored 556 (647), dx 471 (534), dW 527 (577):
 * 1.4 to 1.6 PFLOP/s in bursts, and what cuBLAS's product of the same shape takes in loops of a second, where power bounds both. Without
 * the stores the forward pass takes 473 us, without the products 314.
 */
template <typename T, int FORM, int N, bool PAIR> __device__ __forceinline__ void gemm(const GemmArgs& a) {
    using Shape = GemmShape<FORM, N, PAIR>;
    constexpr int kStages = Shape::kStages;
    extern __shared__ char shared[];
    __shared__ uint64_t bars[2 * kStages + 5];
    __shared__ uint32_t tmem_base;
    __shared__ int failed;
    char* const tiles = shared + (1024 - shared_addr(shared) % 1024) % 1024;
    char* const staging = tiles + kStages * Shape::kBytes;
    const uint32_t full = shared_addr(bars), empty = full + 8 * kStages, sums_full = empty + 8 * kStages, sums_empty = sums_full + 16, drained = sums_empty + 16;
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = PAIR ? cluster_rank() : 0;
    if (warp == kMultiplier) {
        if constexpr (PAIR) pair_tmem_alloc(shared_addr(&tmem_base), 2 * N);
        else tmem_alloc(shared_addr(&tmem_base), 2 * N);
    }
    if (threadIdx.x == 0) {
        failed = 0;
        for (int i = 0; i < kStages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { bar_init(sums_full + 8 * i, 1); bar_init(sums_empty + 8 * i, (PAIR ? 2 : 1) * kEpilogueWarps); }
        bar_init(drained, 1);
        bar_init_fence();
    }
    if (threadIdx.x == 32 * kLoader) {
        prefetch_map(&a.a0);
        prefetch_map(&a.b0);
        if (FORM == GATED) prefetch_map(&a.b1);
        if (FORM != GATED) prefetch_map(&a.a1);
    }
    tc_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    tc_after_sync();
    const uint32_t sums = tmem_base;
    wait_for_stream();
    const unsigned total = a.tiles_m * a.tiles_n * a.batch * a.splits, first = PAIR ? blockIdx.x / 2 : blockIdx.x, step = PAIR ? gridDim.x / 2 : gridDim.x;
    unsigned filled = 0;            // stages that the producer filled, or that the multiplier used
    if (warp == kLoader && lane == 0) {
        const auto load = [&](uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
            if constexpr (PAIR) pair_load_box(to, map, x, y, bar);
            else load_box(to, map, x, y, bar);
        };
        for (unsigned tile = first; tile < total; tile += step) {
            const Place p = place_of(tile, a);
            const unsigned from = (unsigned)((unsigned long long)a.k_blocks * p.split / a.splits), to = (unsigned)((unsigned long long)a.k_blocks * (p.split + 1) / a.splits);
            const int row = p.m * Shape::kRows + rank * kTileM, column = p.n * Shape::kColumns + (FORM == GATED ? 0 : rank * Shape::kHeldN);
            unsigned kb = from;
            for (; kb < to; kb++, filled++) {
                const unsigned s = filled % kStages;
                if (!bar_wait(empty + 8 * s, (filled / kStages & 1) ^ 1, &failed)) break;
                const uint32_t to_a = shared_addr(tiles) + s * Shape::kBytes, to_b = to_a + Shape::kBytesA, bar = PAIR ? in_cta(full + 8 * s, 0) : full + 8 * s;
                if (rank == 0) bar_expect(full + 8 * s, (PAIR ? 2 : 1) * Shape::kBytes);       // the leader counts both CTAs' bytes
                if constexpr (FORM == GATED) {
                    load(to_a, &a.a0, kb * kTileK, row, bar);
                    if constexpr (PAIR) load(to_b, rank ? &a.b1 : &a.b0, kb * kTileK, column, bar);
                    else {
                        load(to_b, &a.b0, kb * kTileK, column, bar);
                        load(to_b + Shape::kBytesB / 2, &a.b1, kb * kTileK, column, bar);
                    }
                } else if constexpr (FORM == INPUT_GRAD) {
                    const bool second = kb >= a.k_half;
                    const int k = (second ? kb - a.k_half : kb) * kTileK;
                    load(to_a, second ? &a.a1 : &a.a0, k, row, bar);
#pragma unroll
                    for (int i = 0; i < Shape::kHeldN / 64; i++) load(to_b + i * 64 * kStageRowsBytes, second ? &a.b1 : &a.b0, column + 64 * i, k, bar);
                } else {
                    const CUtensorMap* map = p.batch ? &a.a1 : &a.a0;
#pragma unroll
                    for (int i = 0; i < kTileM / 64; i++) load(to_a + i * 64 * kStageRowsBytes, map, row + 64 * i, kb * kTileK, bar);
#pragma unroll
                    for (int i = 0; i < Shape::kHeldN / 64; i++) load(to_b + i * 64 * kStageRowsBytes, &a.b0, column + 64 * i, kb * kTileK, bar);
                }
            }
            if (kb < to) break;
        }
    } else if (warp == kMultiplier && lane == 0 && rank == 0) {
        unsigned done = 0;
        for (unsigned tile = first; tile < total; tile += step, done++) {
            const Place p = place_of(tile, a);
            const unsigned from = (unsigned)((unsigned long long)a.k_blocks * p.split / a.splits), to = (unsigned)((unsigned long long)a.k_blocks * (p.split + 1) / a.splits);
            const unsigned buffer = done & 1;
            if (!bar_wait(sums_empty + 8 * buffer, (done / 2 & 1) ^ 1, &failed)) break;
            tc_after_sync();
            const uint32_t d = sums + buffer * N;
            unsigned kb = from;
            for (; kb < to; kb++, filled++) {
                const unsigned s = filled % kStages;
                if (!bar_wait(full + 8 * s, filled / kStages & 1, &failed)) break;
                tc_after_sync();
                const uint32_t at_a = shared_addr(tiles) + s * Shape::kBytes, at_b = at_a + Shape::kBytesA;
#pragma unroll
                for (int k = 0; k < kTileK / 16; k++) {
                    // 16 k: 32 bytes further along K-major rows, or 16 rows of 128 bytes further
                    const uint64_t da = FORM == WEIGHT_GRAD ? tile_descriptor(at_a + k * 2048, 64 * kStageRowsBytes) : tile_descriptor(at_a + k * 32, 16);
                    const uint64_t db = FORM == GATED ? tile_descriptor(at_b + k * 32, 16) : tile_descriptor(at_b + k * 2048, 64 * kStageRowsBytes);
                    if constexpr (PAIR) pair_product(d, da, db, a.descriptor, kb > from || k);
                    else product(d, da, db, a.descriptor, kb > from || k);
                }
                if constexpr (PAIR) pair_commit(empty + 8 * s);
                else commit(empty + 8 * s);
            }
            if (kb < to) break;
            if constexpr (PAIR) pair_commit(sums_full + 8 * buffer);
            else commit(sums_full + 8 * buffer);
        }
    } else if (warp < kEpilogueWarps) {
        char* const stage = staging + warp * 4096;
        unsigned done = 0;
        const bool vec = a.n % 8 == 0 && aligned16(a.c0) && aligned16(a.c1);
        for (unsigned tile = first; tile < total; tile += step, done++) {
            const Place p = place_of(tile, a);
            const unsigned buffer = done & 1;
            if (!bar_wait_warp(sums_full + 8 * buffer, done / 2 & 1, &failed)) break;
            tc_after_sync();
            const unsigned quarter = warp % 4, half = warp / 4;
            const uint32_t d = sums + buffer * N + (quarter * 32u << 16);
            const size_t row = (size_t)p.m * Shape::kRows + rank * kTileM + quarter * 32;
            const int rows = row < a.m ? (int)(a.m - row < 32 ? a.m - row : 32) : 0;
#pragma unroll 1
            for (int c = half * (Shape::kColumns / 2); c < (int)(half + 1) * (Shape::kColumns / 2); c += 32) {
                const size_t column = (size_t)p.n * Shape::kColumns + c;
                if (column >= a.n || !rows) break;
                const int columns = (int)(a.n - column < 32 ? a.n - column : 32);
                uint32_t r[32];
                tmem_load32(r, d + c);
                if constexpr (FORM == GATED) {
                    uint32_t r2[32];
                    tmem_load32(r2, d + N / 2 + c);
                    tmem_wait();
                    float g[32], u[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) { g[e] = __uint_as_float(r[e]); u[e] = __uint_as_float(r2[e]); }
                    float* gate_to = a.splits > 1 ? a.partial + ((size_t)p.split * 2 * a.m + row) * a.partial_stride + column : a.g ? a.g + row * a.pre_stride + column : nullptr;
                    float* up_to = a.splits > 1 ? a.partial + (((size_t)p.split * 2 + 1) * a.m + row) * a.partial_stride + column : a.u ? a.u + row * a.pre_stride + column : nullptr;
                    const size_t stride = a.splits > 1 ? a.partial_stride : a.pre_stride;
                    if (gate_to) {
                        stage_rows(stage, g);
                        store_fp32(stage, gate_to, stride, rows, columns);
                        stage_rows(stage, u);
                        store_fp32(stage, up_to, stride, rows, columns);
                    }
                    if (a.splits == 1) {
                        with_activation(a.act, [&](auto act) {
#pragma unroll
                            for (int e = 0; e < 32; e++) g[e] = activate<decltype(act)::value>(g[e]) * u[e];
                        });
                        stage_rows(stage, g);
                        store_as<T>(stage, reinterpret_cast<T*>(a.c0) + row * a.n + column, a.n, rows, columns, vec);
                    }
                } else {
                    tmem_wait();
                    float v[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = __uint_as_float(r[e]);
                    stage_rows(stage, v);
                    if (a.splits > 1) store_fp32(stage, a.partial + (((size_t)p.split * a.batch + p.batch) * a.m + row) * a.partial_stride + column, a.partial_stride, rows, columns);
                    else store_as<T>(stage, reinterpret_cast<T*>(p.batch ? a.c1 : a.c0) + row * a.n + column, a.n, rows, columns, vec);
                }
            }
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
        mark_incomplete(FORM, a, a, Shape::kRows, Shape::kColumns, rank, first, step, threadIdx.x, kGemmThreads);
        if (warp == kLoader && lane == 0 && rank != 0)      // its copies count on the leader's barriers: here only time tells that they have landed
            for (const long long start = clock64(); clock64() - start < kLandClocks;) {}
        if (warp == kLoader && lane == 0 && rank == 0)
            for (unsigned i = filled > kStages ? filled - kStages : 0; i < filled; i++) bar_wait(full + 8 * (i % kStages), i / kStages & 1, &late);
        if (warp == kMultiplier && lane == 0 && rank == 0) {
            if constexpr (PAIR) pair_commit(drained);
            else commit(drained);
            bar_wait(drained, 0, &late);
        }
        if (threadIdx.x == 0 && a.gave_up) *reinterpret_cast<volatile int*>(a.gave_up) = 1;
        __syncthreads();
    }
    if constexpr (PAIR) cluster_sync();      // neither CTA's memory goes before the other is done with it
    tc_after_sync();
    if (warp == kMultiplier) {
        if constexpr (PAIR) pair_tmem_free(sums, 2 * N);
        else tmem_free(sums, 2 * N);
    }
}

template <typename T, int FORM, int N> __global__ void __launch_bounds__(kGemmThreads, 1) k_gemm(const __grid_constant__ GemmArgs a) { gemm<T, FORM, N, false>(a); }
template <typename T, int FORM, int N> __global__ void __launch_bounds__(kGemmThreads, 1) __cluster_dims__(2, 1, 1) k_gemm_pair(const __grid_constant__ GemmArgs a) { gemm<T, FORM, N, true>(a); }

/* ---- few tokens ---- */

constexpr int kFewStages = 16;          // at most
constexpr int kFewShared = 112 * 1024, kFewThreads = 192;

struct FewArgs {
    CUtensorMap x, w_gate, w_up;
    unsigned tokens, ffn, k_blocks, descriptor;
    unsigned rows, stages;              // rows of each weight for one CTA, a multiple of eight up to 64
    int act;
    void* h;
    float *g, *u;
    size_t pre_stride;
    int* gave_up;
};

/**
 * Up to 128 tokens: reading the weights bounds it. Here they are the rows of the product and the tokens its columns, so that the work of the
 * tensor cores shrinks with the tokens. Each CTA takes some rows of both weights over all of k, and nothing is left to join. The rows of Wg come first in a tile, then those of Wu. A product has 128 rows: the others are whatever lies behind in
 * shared memory, and nobody reads what becomes of them.
 */
template <typename T, int N> __global__ void __launch_bounds__(kFewThreads, 2) k_gated_few(const __grid_constant__ FewArgs a) {
    constexpr int kColumns = N < 32 ? 32 : N;
    extern __shared__ char shared[];
    __shared__ uint64_t bars[2 * kFewStages + 2];
    __shared__ uint32_t tmem_base;
    __shared__ int failed;
    char* const tiles = shared + (1024 - shared_addr(shared) % 1024) % 1024;
    const uint32_t full = shared_addr(bars), empty = full + 8 * kFewStages, sums_full = empty + 8 * kFewStages, drained = sums_full + 8;
    const uint32_t bytes_w = a.rows * 2 * kStageRowsBytes, bytes = bytes_w + N * kStageRowsBytes;
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32, first = blockIdx.x * a.rows;
    if (warp == 5) tmem_alloc(shared_addr(&tmem_base), kColumns);
    if (threadIdx.x == 0) {
        failed = 0;
        for (unsigned i = 0; i < a.stages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        bar_init(sums_full, 1);
        bar_init(drained, 1);
        bar_init_fence();
    }
    if (threadIdx.x == 32 * 4) {
        prefetch_map(&a.x);
        prefetch_map(&a.w_gate);
        prefetch_map(&a.w_up);
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t sums = tmem_base;
    wait_for_stream();
    unsigned filled = 0, stage = 0, parity = 0;
    if (warp == 4 && lane == 0) {
        unsigned kb = blockIdx.x * 5 % a.k_blocks;
        for (; filled < a.k_blocks; filled++) {
            if (!bar_wait(empty + 8 * stage, parity ^ 1, &failed)) break;
            const uint32_t bar = full + 8 * stage, to = shared_addr(tiles) + stage * bytes;
            bar_expect(bar, bytes);
            load_box(to, &a.w_gate, kb * kTileK, first, bar);
            load_box(to + bytes_w / 2, &a.w_up, kb * kTileK, first, bar);
            load_box(to + bytes_w, &a.x, kb * kTileK, 0, bar);
            if (++kb == a.k_blocks) kb = 0;
            if (++stage == a.stages) { stage = 0; parity ^= 1; }
        }
    } else if (warp == 5 && lane == 0) {
        for (unsigned kb = 0; kb < a.k_blocks; kb++) {
            if (!bar_wait(full + 8 * stage, parity, &failed)) break;
            tc_after_sync();
            const uint32_t at = shared_addr(tiles) + stage * bytes;
#pragma unroll
            for (int k = 0; k < kTileK / 16; k++) product(sums, tile_descriptor(at + k * 32, 16), tile_descriptor(at + bytes_w + k * 32, 16), a.descriptor, kb || k);
            commit(empty + 8 * stage);
            if (++stage == a.stages) { stage = 0; parity ^= 1; }
        }
        commit(sums_full);
    }
    __syncwarp();
    // [gate, up][token][row]: the loads are over and the products done once the sums are
    float* const values = reinterpret_cast<float*>(tiles);
    if (warp < 4 && warp * 32 < 2 * a.rows && bar_wait_warp(sums_full, 0, &failed)) {
        tc_after_sync();
#pragma unroll 1
        for (int c = 0; c < N && c < (int)a.tokens; c += 32) {
            uint32_t r[32];
            tmem_load32(r, sums + (warp * 32u << 16) + c);
            tmem_wait();
            if (threadIdx.x < 2 * a.rows) {
                float* const to = values + (threadIdx.x < a.rows ? threadIdx.x : N * a.rows + threadIdx.x - a.rows) + c * a.rows;
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (c + e < (int)a.tokens) to[e * a.rows] = __uint_as_float(r[e]);
            }
        }
        tc_before_sync();
    }
    __syncthreads();
    if (failed) {       // as in k_gemm
        int late = 0;
        if (warp == 4 && lane == 0)
            for (unsigned i = filled > a.stages ? filled - a.stages : 0; i < filled; i++) bar_wait(full + 8 * (i % a.stages), i / a.stages & 1, &late);
        if (warp == 5 && lane == 0) {
            commit(drained);
            bar_wait(drained, 0, &late);
        }
        for (unsigned i = threadIdx.x; i < a.tokens * a.rows; i += kFewThreads) {
            const unsigned t = i / a.rows, row = first + i % a.rows;
            if (row < a.ffn) mark_incomplete(a.h, a.g, a.u, (size_t)t * a.ffn + row, t * a.pre_stride + row);
        }
        if (threadIdx.x == 0 && a.gave_up) *reinterpret_cast<volatile int*>(a.gave_up) = 1;
        __syncthreads();
    } else {
        const unsigned rows = a.ffn - first < a.rows ? a.ffn - first : a.rows;
        with_activation(a.act, [&](auto act) {
            for (unsigned t = warp; t < a.tokens; t += kFewThreads / 32)
                for (unsigned r = lane; r < rows; r += 32) {
                    const float g = values[t * a.rows + r], u = values[(N + t) * a.rows + r];
                    if (a.g) {
                        a.g[t * a.pre_stride + first + r] = g;
                        a.u[t * a.pre_stride + first + r] = u;
                    }
                    reinterpret_cast<T*>(a.h)[(size_t)t * a.ffn + first + r] = Traits<T>::down(activate<decltype(act)::value>(g) * u);
                }
        });
    }
    __syncwarp();
    tc_after_sync();
    if (warp == 5) tmem_free(sums, kColumns);
}

struct JoinArgs {
    const float* partial;
    size_t m, stride;               // rows, and elements between rows of a partial result
    unsigned n, splits, batch;
    int act;
    void *c0, *c1;
    float *g, *u;
    size_t pre_stride;
    bool vec;                       // rows of the results start on four elements
};

/** Adds the parts that splits of k left, in the order of k, and finishes: four columns per thread. */
template <typename T, bool GATE> __global__ void __launch_bounds__(256) k_join(const __grid_constant__ JoinArgs a) {
    wait_for_stream();
    const size_t plane = a.m * a.stride;
    const unsigned runs = (unsigned)(a.stride / 4);
    const size_t index = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (index >= a.m * runs * (GATE ? 1 : a.batch)) return;
    const size_t line = index / runs, row = GATE ? line : line % a.m, batch = GATE ? 0 : line / a.m;
    const unsigned column = (unsigned)(index % runs) * 4;
    const float* from = a.partial + batch * plane + row * a.stride + column;
    const size_t next = plane * (GATE ? 2 : a.batch);
    Run<float, 4> g = {}, u = {};
#pragma unroll 4
    for (unsigned s = 0; s < a.splits; s++) {
        const Run<float, 4> p = ld_run<float, 4>(from + s * next);
#pragma unroll
        for (int e = 0; e < 4; e++) g.e[e] += p.e[e];
        if constexpr (GATE) {
            const Run<float, 4> q = ld_run<float, 4>(from + s * next + plane);
#pragma unroll
            for (int e = 0; e < 4; e++) u.e[e] += q.e[e];
        }
    }
    if constexpr (GATE) {
        if (a.g) {      // rows of these end on four elements as well
            st_run<float, 4>(a.g + row * a.pre_stride + column, g);
            st_run<float, 4>(a.u + row * a.pre_stride + column, u);
        }
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 4; e++) g.e[e] = activate<decltype(act)::value>(g.e[e]) * u.e[e];
        });
    }
    T* to = reinterpret_cast<T*>(batch ? a.c1 : a.c0) + row * a.n + column;
    if (a.vec) st_run<T, 4>(to, round_run<T, 4>(g.e));
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (column + e < a.n) to[e] = Traits<T>::down(g.e[e]);
}

struct PadArgs { const void* from[3]; void* to[3]; size_t rows[3]; unsigned width, stride; };

/** Rows that do not start on 16 bytes, copied to some that do, for the tiled loads: eight elements per thread. Nobody reads what is behind a row. */
__global__ void __launch_bounds__(256) k_pad(const __grid_constant__ PadArgs a) {
    wait_for_stream();
    const unsigned runs = a.stride / 8;
    size_t index = (size_t)blockIdx.x * 256 + threadIdx.x;
    int w = 0;
    while (w < 3 && index >= a.rows[w] * runs) index -= a.rows[w++] * runs;
    if (w == 3) return;
    const size_t row = index / runs;
    const unsigned column = (unsigned)(index % runs) * 8;
    const uint16_t* from = reinterpret_cast<const uint16_t*>(a.from[w]) + row * a.width + column;
    Run<uint16_t, 8> r = {};
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (column + e < a.width) r.e[e] = from[e];
    st_run<uint16_t, 8>(reinterpret_cast<uint16_t*>(a.to[w]) + row * a.stride + column, r);
}

struct GateGradArgs { const void* dh; const float *g, *u; void *dg, *du; size_t pre_stride, stride; unsigned rows, n; int act; };

/** dg and du from dh and the saved products, eight elements per thread. Only the rows of dh may start anywhere (VEC: they do not). */
template <typename T, bool VEC> __global__ void __launch_bounds__(256) k_gate_grad(const __grid_constant__ GateGradArgs a) {
    wait_for_stream();
    const unsigned runs = (a.n + 7) / 8;
    const size_t index = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (index >= (size_t)a.rows * runs) return;
    const size_t row = index / runs;
    const unsigned column = (unsigned)(index % runs) * 8;
    const bool second = column + 4 < a.n;       // rows of g and u end on four elements
    float g[8], u[8], d[8];
#pragma unroll
    for (int q = 0; q < 2; q++) {
        if (q && !second) break;
        const Run<float, 4> x = ld_run<float, 4>(a.g + row * a.pre_stride + column + 4 * q), y = ld_run<float, 4>(a.u + row * a.pre_stride + column + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; e++) { g[4 * q + e] = x.e[e]; u[4 * q + e] = y.e[e]; }
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
        for (int e = 0; e < 8; e++) {
            float value, slope;
            activate_grad<decltype(act)::value>(g[e], value, slope);
            g[e] = d[e] * u[e] * slope;
            u[e] = d[e] * value;
        }
    });
    st_run<T, 8>(reinterpret_cast<T*>(a.dg) + row * a.stride + column, round_run<T, 8>(g));
    st_run<T, 8>(reinterpret_cast<T*>(a.du) + row * a.stride + column, round_run<T, 8>(u));
}

/* ------------------------------------------------------------------------------------------------ host side */

/** Set by a kernel whose wait ran out, which leaves NaN in what it was to store; looked at by the next call on the device. Host memory that the device
 *  writes, for the life of the process. */
static int* gave_up_flag(int device) {
    static int* const flags = [] {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);       // a first call may come while a stream is being captured
        void* p = nullptr;
        if (cudaHostAlloc(&p, 64 * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess) { cudaGetLastError(); p = nullptr; }
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (p) memset(p, 0, 64 * sizeof(int));
        return reinterpret_cast<int*>(p);
    }();
    return flags ? flags + device : nullptr;        // of the 64 devices that sm_count knows
}

/** The two dimensions of an operand by which one is contiguous, and the box of it. */
static cudaError_t make_map(CUtensorMap* map, int dtype, const void* base, size_t inner, size_t outer, size_t stride, unsigned box_outer) {
    const DriverApi* d = driver_api(nullptr);
    if (!d || !d->TensorMapEncodeTiled) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {inner, outer}, strides[1] = {stride * 2};
    const cuuint32_t box[2] = {64, box_outer}, steps[2] = {1, 1};
    const CUresult r = d->TensorMapEncodeTiled(map, dtype == 6 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps,
                                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int FORM, int N, bool PAIR> static cudaError_t run_gemm(int device, const GemmPlan& p, GemmArgs& a, cudaStream_t stream) {
    using Shape = GemmShape<FORM, N, PAIR>;
    void (*const kernel)(const GemmArgs) = PAIR ? k_gemm_pair<T, FORM, N> : k_gemm<T, FORM, N>;
    static std::atomic<bool> ready[64];
    if (!ready[device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kShared);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_relaxed);
    }
    a.tiles_m = p.tiles_m;
    a.tiles_n = p.tiles_n;
    a.batch = p.batch;
    a.splits = p.splits;
    a.k_blocks = p.k_blocks;
    a.partial_stride = up_to(a.n, 4);
    a.descriptor = product_descriptor(std::is_same<T, __nv_bfloat16>::value, FORM == WEIGHT_GRAD, FORM != GATED, Shape::kRows, N);
    a.gave_up = gave_up_flag(device);
    const size_t tiles = (size_t)p.tiles_m * p.tiles_n * p.batch * p.splits, workers = PAIR ? sm_count(device) / 2 : sm_count(device);
    cudaError_t e = launch_early_shared(kernel, (unsigned)(tiles < workers ? tiles : workers) * (PAIR ? 2 : 1), kGemmThreads, Shape::kShared, stream, a);
    if (e != cudaSuccess || p.splits == 1) return e;
    const JoinArgs j = {a.partial, a.m, a.partial_stride, a.n, p.splits, p.batch, a.act, a.c0, a.c1, a.g, a.u, a.pre_stride, a.n % 4 == 0 && aligned_to(8, {a.c0, a.c1})};
    const size_t threads = (size_t)a.m * (a.partial_stride / 4) * p.batch;
    return launch_early(k_join<T, FORM == GATED>, (unsigned)((threads + 255) / 256), 256, stream, j);
}

template <typename T, int FORM> static cudaError_t run_gemm(int device, const GemmPlan& p, GemmArgs& a, cudaStream_t stream) {
    if (p.pair) return p.columns == 128 ? run_gemm<T, FORM, 128, true>(device, p, a, stream) : run_gemm<T, FORM, 256, true>(device, p, a, stream);
    return p.columns == 128 ? run_gemm<T, FORM, 128, false>(device, p, a, stream) : run_gemm<T, FORM, 256, false>(device, p, a, stream);
}

/** Where the parts of a call's workspace lie. */
struct GatedLayout { size_t stride, x, gate, up, padded, dg, du, d_stride, partial, total; GemmPlan forward, input, weight; bool ok; };

static GatedLayout layout_of(int device, size_t tokens, size_t width, size_t ffn, bool aligned, bool backward) {
    GatedLayout l = {};
    const int sms = sm_count(device);
    l.ok = sms > 0 && tokens < DCCL_GATED_MAX_DIMENSION && width < DCCL_GATED_MAX_DIMENSION && ffn < DCCL_GATED_MAX_DIMENSION;
    if (!l.ok) return l;
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t here = at; at += up_to(bytes, 256); return here; };
    const bool pad = !aligned || width % 8;
    l.stride = pad ? up_to(width, 8) : width;
    if (pad) {      // at the same places in both directions: the backward pass finds them in what the forward pass left
        l.x = take(tokens * l.stride * 2);
        l.gate = take(ffn * l.stride * 2);
        l.up = take(ffn * l.stride * 2);
        l.padded = at;
        if (backward) at = 0;
    }
    l.d_stride = up_to(ffn, 8);
    size_t partial = 0;
    if (backward) {
        l.dg = take(tokens * l.d_stride * 2);
        l.du = take(tokens * l.d_stride * 2);
        l.input = plan_gemm(sms, INPUT_GRAD, tokens, width, ffn);
        l.weight = plan_gemm(sms, WEIGHT_GRAD, ffn, width, tokens);
        partial = l.input.partial_bytes > l.weight.partial_bytes ? l.input.partial_bytes : l.weight.partial_bytes;
    } else {
        l.forward = plan_gemm(sms, GATED, tokens, ffn, width);
        if (!few_tokens(sms, tokens, width, ffn)) partial = l.forward.partial_bytes;
    }
    l.partial = take(partial);
    l.total = at;
    return l;
}

/** x, Wg and Wu as the tiled loads take them: in place, or padded into the workspace. */
static cudaError_t pad_operands(const GatedLayout& l, size_t tokens, size_t width, size_t ffn, const void*& x, const void*& w_gate, const void*& w_up, char* workspace,
                                cudaStream_t stream) {
    if (!l.padded) return cudaSuccess;
    const PadArgs a = {{x, w_gate, w_up}, {workspace + l.x, workspace + l.gate, workspace + l.up}, {tokens, ffn, ffn}, (unsigned)width, (unsigned)l.stride};
    x = a.to[0];
    w_gate = a.to[1];
    w_up = a.to[2];
    const size_t threads = (a.rows[0] + a.rows[1] + a.rows[2]) * (l.stride / 8);
    return launch_early(k_pad, (unsigned)((threads + 255) / 256), 256, stream, a);
}

template <typename T, int N> static cudaError_t run_few(int device, FewArgs& a, cudaStream_t stream) {
    static std::atomic<bool> ready[64];
    if (!ready[device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(k_gated_few<T, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_relaxed);
    }
    a.descriptor = product_descriptor(std::is_same<T, __nv_bfloat16>::value, false, false, 128, N);
    // the product of the last stage reads 128 rows of it, and what behind them is inside of the allocation
    const unsigned bytes = (2 * a.rows + N) * kStageRowsBytes, room = kFewShared - 1024 - 128 * kStageRowsBytes;
    a.stages = room / bytes < (unsigned)kFewStages ? room / bytes : kFewStages;
    return launch_early_shared(k_gated_few<T, N>, blocks_of(a.ffn, a.rows), kFewThreads, kFewShared, stream, a);
}

template <typename T> static cudaError_t gated_forward(int device, int dtype, const GatedLayout& l, size_t tokens, size_t width, size_t ffn, const void* x, const void* w_gate, const void* w_up,
                                                       int act, void* h, float* g, float* u, size_t pre_stride, char* workspace, cudaStream_t stream) {
    cudaError_t e = pad_operands(l, tokens, width, ffn, x, w_gate, w_up, workspace, stream);
    if (few_tokens(sm_count(device), tokens, width, ffn)) {
        const int columns = tokens <= 16 ? 16 : tokens <= 32 ? 32 : tokens <= 64 ? 64 : 128;
        FewArgs f = {};
        if (e == cudaSuccess) e = make_map(&f.x, dtype, x, width, tokens, l.stride, columns);
        f.rows = few_rows(sm_count(device), ffn);
        if (e == cudaSuccess) e = make_map(&f.w_gate, dtype, w_gate, width, ffn, l.stride, f.rows);
        if (e == cudaSuccess) e = make_map(&f.w_up, dtype, w_up, width, ffn, l.stride, f.rows);
        if (e != cudaSuccess) return e;
        f.tokens = (unsigned)tokens;
        f.ffn = (unsigned)ffn;
        f.k_blocks = blocks_of(width, kTileK);
        f.act = act;
        f.h = h;
        f.g = g;
        f.u = u;
        f.pre_stride = pre_stride;
        f.gave_up = gave_up_flag(device);
        return columns == 16 ? run_few<T, 16>(device, f, stream) : columns == 32 ? run_few<T, 32>(device, f, stream) : columns == 64 ? run_few<T, 64>(device, f, stream)
                                                                                                                                    : run_few<T, 128>(device, f, stream);
    }
    GemmArgs a = {};
    if (e == cudaSuccess) e = make_map(&a.a0, dtype, x, width, tokens, l.stride, kTileM);
    if (e == cudaSuccess) e = make_map(&a.b0, dtype, w_gate, width, ffn, l.stride, l.forward.columns / 2);
    if (e == cudaSuccess) e = make_map(&a.b1, dtype, w_up, width, ffn, l.stride, l.forward.columns / 2);
    if (e != cudaSuccess) return e;
    a.m = (unsigned)tokens;
    a.n = (unsigned)ffn;
    a.act = act;
    a.c0 = a.c1 = h;
    a.g = g;
    a.u = u;
    a.pre_stride = pre_stride;
    a.partial = (float*)(workspace + l.partial);
    return run_gemm<T, GATED>(device, l.forward, a, stream);
}

template <typename T> static cudaError_t gated_backward(int device, int dtype, const GatedLayout& l, size_t tokens, size_t width, size_t ffn, const void* dh, const float* g, const float* u,
                                                        size_t pre_stride, const void* x, const void* w_gate, const void* w_up, const char* padded, int act, void* dx, void* dw_gate,
                                                        void* dw_up, char* workspace, cudaStream_t stream) {
    const GateGradArgs d = {dh, g, u, workspace + l.dg, workspace + l.du, pre_stride, l.d_stride, (unsigned)tokens, (unsigned)ffn, act};
    const size_t threads = tokens * ((ffn + 7) / 8);
    cudaError_t e = launch_early(ffn % 8 == 0 && aligned_to(16, {dh}) ? k_gate_grad<T, true> : k_gate_grad<T, false>, (unsigned)((threads + 255) / 256), 256, stream, d);
    if (l.padded) {
        x = padded + l.x;
        w_gate = padded + l.gate;
        w_up = padded + l.up;
    }
    GemmArgs a = {};
    a.partial = (float*)(workspace + l.partial);
    if (e == cudaSuccess && dx) {
        e = make_map(&a.a0, dtype, d.dg, ffn, tokens, l.d_stride, kTileM);
        if (e == cudaSuccess) e = make_map(&a.a1, dtype, d.du, ffn, tokens, l.d_stride, kTileM);
        if (e == cudaSuccess) e = make_map(&a.b0, dtype, w_gate, width, ffn, l.stride, kTileK);
        if (e == cudaSuccess) e = make_map(&a.b1, dtype, w_up, width, ffn, l.stride, kTileK);
        if (e != cudaSuccess) return e;
        a.m = (unsigned)tokens;
        a.n = (unsigned)width;
        a.k_half = blocks_of(ffn, kTileK);
        a.c0 = a.c1 = dx;
        e = run_gemm<T, INPUT_GRAD>(device, l.input, a, stream);
    }
    if (e == cudaSuccess && dw_gate) {
        e = make_map(&a.a0, dtype, d.dg, ffn, tokens, l.d_stride, kTileK);
        if (e == cudaSuccess) e = make_map(&a.a1, dtype, d.du, ffn, tokens, l.d_stride, kTileK);
        if (e == cudaSuccess) e = make_map(&a.b0, dtype, x, width, tokens, l.stride, kTileK);
        if (e != cudaSuccess) return e;
        a.m = (unsigned)ffn;
        a.n = (unsigned)width;
        a.c0 = dw_gate;
        a.c1 = dw_up;
        e = run_gemm<T, WEIGHT_GRAD>(device, l.weight, a, stream);
    }
    return e;
}

static bool gave_up(const char* who, int device) {
    const int* flag = gave_up_flag(device);
    if (!flag || !*reinterpret_cast<const volatile int*>(flag)) return false;
    fprintf(stderr, "%s: an earlier product of this process on device %d did not end in time; what it did not finish is NaN, and no other is started there\n", who, device);
    return true;
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_gated_linear_pads(size_t width, int aligned) { return !aligned || width % 8; }

extern "C" long long dccl_gated_linear_workspace(int device, size_t tokens, size_t width, size_t ffn, int aligned, int backward) {
    const GatedLayout l = layout_of(device, tokens, width, ffn, aligned != 0, backward != 0);
    return l.ok ? (long long)l.total : -1;
}

extern "C" int dccl_gated_linear(int device, int dtype, size_t tokens, size_t width, size_t ffn, const void* x, const void* w_gate, const void* w_up, int act, void* h,
                                 float* g, float* u, size_t pre_stride, void* workspace, long long workspace_bytes, void* stream) {
    const char* who = "dccl_gated_linear";
    if (!tokens || !ffn) return 0;
    const GatedLayout l = layout_of(device, tokens, width, ffn, aligned_to(16, {x, w_gate, w_up}), false);
    if (!l.ok || !width || workspace_bytes < (long long)l.total || (dtype != 6 && dtype != 9) || act < 0 || act > DCCL_ACT_GELU_TANH || (!g != !u) || (g && pre_stride < ffn)
        || pre_stride % 4 || !aligned_to(16, {g, u, workspace}))
        return report(who, cudaErrorInvalidValue);
    if (gave_up(who, device)) return -1;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const auto run = dtype == 6 ? gated_forward<__half> : gated_forward<__nv_bfloat16>;
    return report(who, run(device, dtype, l, tokens, width, ffn, x, w_gate, w_up, act, h, g, u, pre_stride, (char*)workspace, (cudaStream_t)stream));
}

extern "C" int dccl_gated_linear_backward(int device, int dtype, size_t tokens, size_t width, size_t ffn, const void* dh, const float* g, const float* u, size_t pre_stride,
                                          const void* x, const void* w_gate, const void* w_up, const void* forward_workspace, int act, void* dx, void* dw_gate,
                                          void* dw_up, void* workspace, long long workspace_bytes, void* stream) {
    const char* who = "dccl_gated_linear_backward";
    const GatedLayout l = layout_of(device, tokens, width, ffn, aligned_to(16, {x, w_gate, w_up}), true);
    if (!l.ok || !tokens || !width || !ffn || workspace_bytes < (long long)l.total || (dtype != 6 && dtype != 9) || act < 0 || act > DCCL_ACT_GELU_TANH || !g || !u
        || pre_stride < ffn || pre_stride % 4 || !aligned_to(16, {g, u, workspace, forward_workspace}) || (!dw_gate != !dw_up)
        || (l.padded && !forward_workspace))
        return report(who, cudaErrorInvalidValue);
    if (gave_up(who, device)) return -1;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const auto run = dtype == 6 ? gated_backward<__half> : gated_backward<__nv_bfloat16>;
    return report(who, run(device, dtype, l, tokens, width, ffn, dh, g, u, pre_stride, x, w_gate, w_up, (const char*)forward_workspace, act, dx, dw_gate, dw_up, (char*)workspace,
                           (cudaStream_t)stream));
}
