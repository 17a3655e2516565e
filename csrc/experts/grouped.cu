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

struct GroupedArgs : Grouped {
    CUtensorMap a, b;
    const int* starts;
    unsigned descriptor;            // of one product
    int act;
    void* c;
    float* z;
    size_t z_stride;
    int* gave_up;
};

template <int N> struct GroupedShape {
    static constexpr int kBytesA = kTileM * kTileK * 2, kBytesB = N * kTileK * 2, kBytes = kBytesA + kBytesB, kStages = 192 * 1024 / kBytes;
    static constexpr int kShared = kStages * kBytes + kGroupedWarps * 4096 + 1024;      // 1024: the tiles' alignment
    static_assert(kShared + 2 * 1024 <= 227 * 1024, "with the list of tiles and the barriers");
};

/** The list of tiles, by one warp: first[i], the rows of tiles before expert i * stride, and all of them. */
__device__ __forceinline__ void list_tiles(const Grouped& a, const int* starts, unsigned* first) {
    const unsigned lane = threadIdx.x % 32, entries = listed_of(a);
    unsigned before = 0;
    for (unsigned base = 0; base < entries; base += 32) {
        const unsigned i = base + lane;
        unsigned n = 0;
        for (unsigned e = i * a.stride; e < (i + 1) * a.stride && e <= a.experts; e++) n += tall_of(starts, e, a.experts, a.rows);
        const unsigned own = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= (unsigned)o) n += v;
        }
        if (i < entries) first[i] = before + n - own;
        before += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) first[entries] = before;
}

/**
 * One CTA per SM walks over tiles of 128 rows and N columns; one warp loads, one multiplies, eight store: a warp reaches the quarter of the tile's rows that its
 * number gives, so two share one and take half of the columns each. The sums of two tiles fit into tensor memory, so that one is stored while the next is
 * multiplied.
 */
template <typename T, int FORM, int N> __global__ void __launch_bounds__(kGroupedThreads, 1) k_grouped(const __grid_constant__ GroupedArgs a) {
    using Shape = GroupedShape<N>;
    constexpr int kStages = Shape::kStages;
    extern __shared__ char shared[];
    __shared__ uint64_t bars[2 * kStages + 5];
    __shared__ unsigned first[FORM == EXPERTS_WEIGHT ? 1 : kListed + 1];
    __shared__ uint32_t tmem_base;
    __shared__ int failed;
    char* const tiles = shared + (1024 - shared_addr(shared) % 1024) % 1024;
    char* const staging = tiles + kStages * Shape::kBytes;
    const uint32_t full = shared_addr(bars), empty = full + 8 * kStages, sums_full = empty + 8 * kStages, sums_empty = sums_full + 16, drained = sums_empty + 16;
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (warp == kGroupedMultiplier) tmem_alloc(shared_addr(&tmem_base), 2 * N);
    if (threadIdx.x == 0) {
        failed = 0;
        for (int i = 0; i < kStages; i++) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { bar_init(sums_full + 8 * i, 1); bar_init(sums_empty + 8 * i, kGroupedWarps); }
        bar_init(drained, 1);
        bar_init_fence();
    }
    if (threadIdx.x == 32 * kGroupedLoader) {
        prefetch_map(&a.a);
        prefetch_map(&a.b);
    }
    wait_for_stream();
    if (FORM != EXPERTS_WEIGHT && warp == 1) list_tiles(a, a.starts, first);
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t sums = tmem_base;
    const unsigned long long total = grouped_tiles(FORM, a, first);
    unsigned filled = 0;            // stages that the producer filled, or that the multiplier used
    if (warp == kGroupedLoader && lane == 0) {
        for (unsigned long long tile = blockIdx.x; tile < total; tile += gridDim.x) {
            const GroupedPlace p = grouped_place(FORM, tile, N, a, first, a.starts);
            const unsigned blocks = (p.k_count + kTileK - 1) / kTileK;
            unsigned kb = 0;
            for (; kb < blocks; kb++, filled++) {
                const unsigned s = filled % kStages;
                if (!bar_wait(empty + 8 * s, (filled / kStages & 1) ^ 1, &failed)) break;
                const uint32_t to_a = shared_addr(tiles) + s * Shape::kBytes, to_b = to_a + Shape::kBytesA, bar = full + 8 * s;
                bar_expect(bar, Shape::kBytes);
                if constexpr (FORM == EXPERTS_FORWARD) {
                    load_box(to_a, &a.a, kb * kTileK, p.row, bar);
                    load_box(to_b, &a.b, kb * kTileK, p.column, p.expert, bar);
                } else if constexpr (FORM == EXPERTS_INPUT) {
                    load_box(to_a, &a.a, kb * kTileK, p.row, bar);
#pragma unroll
                    for (int i = 0; i < N / 64; i++) load_box(to_b + i * 64 * 128, &a.b, p.column + 64 * i, kb * kTileK, p.expert, bar);
                } else {
                    const int row = p.k_from + kb * kTileK;
#pragma unroll
                    for (int i = 0; i < kTileM / 64; i++) load_box(to_a + i * 64 * 128, &a.a, p.row + 64 * i, row, bar);
#pragma unroll
                    for (int i = 0; i < N / 64; i++) load_box(to_b + i * 64 * 128, &a.b, p.column + 64 * i, row, bar);
                }
            }
            if (kb < blocks) break;
        }
    } else if (warp == kGroupedMultiplier) {
        unsigned done = 0;
        for (unsigned long long tile = blockIdx.x; tile < total; tile += gridDim.x) {
            const GroupedPlace p = grouped_place(FORM, tile, N, a, first, a.starts);
            const unsigned blocks = (p.k_count + kTileK - 1) / kTileK;
            if (!blocks) continue;
            const unsigned buffer = done & 1;
            if (!bar_wait_warp(sums_empty + 8 * buffer, (done / 2 & 1) ^ 1, &failed)) break;
            tc_after_sync();
            const uint32_t d = sums + buffer * N;
            unsigned kb = 0;
            for (; kb < blocks; kb++, filled++) {
                const unsigned s = filled % kStages;
                if (!bar_wait_warp(full + 8 * s, filled / kStages & 1, &failed)) break;
                tc_after_sync();
                char* const at = tiles + s * Shape::kBytes;
                unsigned steps = kTileK / 16;
                if constexpr (FORM == EXPERTS_WEIGHT) {
                    const unsigned left = p.k_count - kb * kTileK;
                    if (left < (unsigned)kTileK) {      // rows of the next expert, and whatever they are: as many as the last product of 16 would add
                        steps = (left + 15) / 16;
                        const unsigned pieces = (steps * 16 - left) * 8;
                        for (unsigned i = lane; i < pieces * (kTileM + N) / 64; i += 32)
                            *reinterpret_cast<uint4*>(at + i / pieces * 64 * 128 + left * 128 + i % pieces * 16) = uint4{};
                        shared_writes_before_products();
                        __syncwarp();
                    }
                }
                const uint32_t at_a = shared_addr(at), at_b = at_a + Shape::kBytesA;
                if (lane == 0) {
#pragma unroll
                    for (unsigned k = 0; k < kTileK / 16; k++) {
                        if (FORM == EXPERTS_WEIGHT && k >= steps) break;
                        // 16 k: 32 bytes further along K-major rows, or 16 rows of 128 bytes further
                        const uint64_t da = FORM == EXPERTS_WEIGHT ? tile_descriptor(at_a + k * 2048, 64 * 128) : tile_descriptor(at_a + k * 32, 16);
                        const uint64_t db = FORM == EXPERTS_FORWARD ? tile_descriptor(at_b + k * 32, 16) : tile_descriptor(at_b + k * 2048, 64 * 128);
                        product(d, da, db, a.descriptor, kb || k);
                    }
                    commit(empty + 8 * s);
                }
                __syncwarp();
            }
            if (kb < blocks) break;
            if (lane == 0) commit(sums_full + 8 * buffer);
            done++;
        }
    } else if (warp < kGroupedWarps) {
        char* const stage = staging + warp * 4096;
        unsigned done = 0;
        const bool vec = a.n % 8 == 0 && aligned16(a.c);
        const unsigned quarter = warp % 4, half = warp / 4;
        for (unsigned long long tile = blockIdx.x; tile < total; tile += gridDim.x) {
            const GroupedPlace p = grouped_place(FORM, tile, N, a, first, a.starts);
            const int rows = quarter * 32 < p.rows ? (int)(p.rows - quarter * 32 < 32 ? p.rows - quarter * 32 : 32) : 0;
            T* const to = reinterpret_cast<T*>(a.c) + (rows ? grouped_row(FORM, p, quarter * 32, a) : 0);
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
                if constexpr (FORM == EXPERTS_FORWARD) {
                    if (summed && a.act != kNoActivation) {
                        if (a.z) {
                            stage_rows(stage, v);
                            store_fp32(stage, a.z + (p.row + quarter * 32) * a.z_stride + column, a.z_stride, rows, columns);
                        }
                        with_activation(a.act, [&](auto act) {
#pragma unroll
                            for (int e = 0; e < 32; e++) v[e] = activate<decltype(act)::value>(v[e]);
                        });
                    }
                }
                stage_rows(stage, v);
                store_as<T>(stage, to + column, a.n, rows, columns, vec);
            }
            if (!summed) continue;
            done++;
            tc_before_sync();
            __syncwarp();
            if (lane == 0) bar_arrive(sums_empty + 8 * buffer);
        }
    }
    __syncthreads();
    if (failed) {       // no wait is expected to run out: copies in flight still have to land, and products to end, before the memory is given back
        int late = 0;
        grouped_mark(FORM, a, N, first, a.starts, reinterpret_cast<uint16_t*>(a.c), a.z, a.z_stride, blockIdx.x, gridDim.x, threadIdx.x, kGroupedThreads);
        if (warp == kGroupedLoader && lane == 0)
            for (unsigned i = filled > kStages ? filled - kStages : 0; i < filled; i++) bar_wait(full + 8 * (i % kStages), i / kStages & 1, &late);
        if (warp == kGroupedMultiplier && lane == 0) {
            commit(drained);
            bar_wait(drained, 0, &late);
        }
        if (threadIdx.x == 0 && a.gave_up) *reinterpret_cast<volatile int*>(a.gave_up) = 1;
        __syncthreads();
    }
    tc_after_sync();
    if (warp == kGroupedMultiplier) tmem_free(sums, 2 * N);
}

struct PadRowsArgs { const void* from[2]; void* to[2]; size_t rows[2]; unsigned width, stride; };

/** Rows that do not start on 16 bytes, copied to some that do, for the tiled loads: eight elements per thread. Nobody reads what is behind a row. */
__global__ void __launch_bounds__(256) k_pad_rows(const __grid_constant__ PadRowsArgs a) {
    wait_for_stream();
    const unsigned runs = a.stride / 8;
    size_t index = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int w = index >= a.rows[0] * runs;
    if (w) index -= a.rows[0] * runs;
    if (index >= a.rows[w] * runs) return;
    const size_t row = index / runs;
    const unsigned column = (unsigned)(index % runs) * 8;
    const uint16_t* from = reinterpret_cast<const uint16_t*>(a.from[w]) + row * a.width + column;
    Run<uint16_t, 8> r = {};
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (column + e < a.width) r.e[e] = from[e];
    st_run<uint16_t, 8>(reinterpret_cast<uint16_t*>(a.to[w]) + row * a.stride + column, r);
}

struct ActGradArgs { const void* dh; const float* z; void* dz; const int* starts; size_t z_stride, stride; unsigned rows, experts, n; int act; };

/** dz from dh and the saved products, eight elements per thread; rows of nobody, whose products nobody wrote, are left out. Only the rows of dh may start
 *  anywhere (VEC: they do not). */
template <typename T, bool VEC> __global__ void __launch_bounds__(256) k_act_grad(const __grid_constant__ ActGradArgs a) {
    wait_for_stream();
    const unsigned runs = (a.n + 7) / 8;
    const size_t index = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t row = index / runs;
    if (row >= a.rows || row >= row_within(a.starts[a.experts], a.rows)) return;
    const unsigned column = (unsigned)(index % runs) * 8;
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
        for (int e = 0; e < 8; e++) {
            float value, slope;
            activate_grad<decltype(act)::value>(z[e], value, slope);
            d[e] *= slope;
        }
    });
    st_run<T, 8>(reinterpret_cast<T*>(a.dz) + row * a.stride + column, round_run<T, 8>(d));
}

/* ------------------------------------------------------------------------------------------------ host side */

/** Where the parts of a call's workspace lie. */
struct GroupedLayout { size_t stride, x, w, padded, dz, d_stride, total; bool ok; };

static GroupedLayout grouped_layout(int device, size_t rows, int experts, size_t width, size_t out, bool aligned, bool backward) {
    GroupedLayout l = {};
    l.ok = sm_count(device) > 0 && rows <= DCCL_EXPERTS_MAX_PLACES && experts >= 1 && experts <= DCCL_EXPERTS_MAX && width >= 1 && width <= DCCL_EXPERTS_MAX_WIDTH && out >= 1
           && out <= DCCL_EXPERTS_MAX_WIDTH;
    if (!l.ok) return l;
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t here = at; at += up_to(bytes, 256); return here; };
    const bool pad = !aligned || width % 8;
    l.stride = pad ? up_to(width, 8) : width;
    if (pad) {      // at the same places in both directions: the backward pass finds them in what the forward pass left
        l.x = take(rows * l.stride * 2);
        l.w = take((size_t)experts * out * l.stride * 2);
        l.padded = at;
        if (backward) at = 0;
    }
    l.d_stride = up_to(out, 8);
    if (backward) l.dz = take(rows * l.d_stride * 2);
    l.total = at;
    return l;
}

template <typename T, int FORM, int N> static cudaError_t run_grouped(int device, GroupedArgs& a, size_t most_tiles, cudaStream_t stream) {
    static std::atomic<bool> ready[64];
    if (!ready[device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(k_grouped<T, FORM, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, GroupedShape<N>::kShared);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_relaxed);
    }
    a.descriptor = product_descriptor(std::is_same<T, __nv_bfloat16>::value, FORM == EXPERTS_WEIGHT, FORM != EXPERTS_FORWARD, kTileM, N);
    a.gave_up = gave_up_flag(device);
    const size_t workers = sm_count(device);
    return launch_early_shared(k_grouped<T, FORM, N>, (unsigned)(most_tiles < workers ? most_tiles : workers), kGroupedThreads, GroupedShape<N>::kShared, stream, a);
}

/** Tiles of 128 columns where those of 256 would leave SMs without one, with the rows spread evenly. */
static int grouped_columns(int device, int form, const GroupedArgs& a) {
    const size_t rows_of_tiles = form == EXPERTS_WEIGHT ? (size_t)a.experts * blocks_of(a.m, kTileM)
                                 : a.experts < a.rows   ? a.experts * (size_t)blocks_of(blocks_of(a.rows, a.experts), kTileM)
                                                        : a.rows;
    return rows_of_tiles * blocks_of(a.n, 256) < (size_t)sm_count(device) ? 128 : 256;
}

template <typename T, int FORM> static cudaError_t run_grouped(int device, GroupedArgs& a, cudaStream_t stream) {
    const int columns = grouped_columns(device, FORM, a);
    a.tiles_m = FORM == EXPERTS_WEIGHT ? blocks_of(a.m, kTileM) : 0;
    a.tiles_n = blocks_of(a.n, columns);
    // every expert may have a row of tiles that is not full, and the rows of nobody another
    const size_t most = (FORM == EXPERTS_WEIGHT ? (size_t)a.experts * a.tiles_m : blocks_of(a.rows, kTileM) + (size_t)a.experts + 1) * a.tiles_n;
    return columns == 128 ? run_grouped<T, FORM, 128>(device, a, most, stream) : run_grouped<T, FORM, 256>(device, a, most, stream);
}

static cudaError_t pad_rows(const void*& x, const void*& w, size_t rows, size_t w_rows, size_t width, size_t stride, void* to_x, void* to_w, cudaStream_t stream) {
    const PadRowsArgs a = {{x, w}, {to_x, to_w}, {rows, w_rows}, (unsigned)width, (unsigned)stride};
    x = to_x;
    w = to_w;
    return launch_early(k_pad_rows, (unsigned)(((rows + w_rows) * (stride / 8) + 255) / 256), 256, stream, a);
}

struct GroupedCall {
    int device, dtype, experts, act;
    size_t rows, width, out;
    const int* starts;
    char* workspace;
    cudaStream_t stream;
};

static GroupedArgs grouped_args(const GroupedCall& k) {
    GroupedArgs a = {};
    a.rows = (unsigned)k.rows;
    a.experts = (unsigned)k.experts;
    a.starts = k.starts;
    a.act = k.act;
    a.stride = (a.experts + kListed) / kListed;       // experts and rows of nobody in at most kListed entries
    return a;
}

template <typename T> static cudaError_t grouped_forward(const GroupedCall& k, const GroupedLayout& l, const void* x, const void* w, void* h, float* z, size_t z_stride) {
    cudaError_t e = cudaSuccess;
    if (l.padded) e = pad_rows(x, w, k.rows, (size_t)k.experts * k.out, k.width, l.stride, k.workspace + l.x, k.workspace + l.w, k.stream);
    GroupedArgs a = grouped_args(k);
    a.n = (unsigned)k.out;
    a.k_blocks = blocks_of(k.width, kTileK);
    a.c = h;
    a.z = z;
    a.z_stride = z_stride;
    if (e == cudaSuccess) e = make_map(&a.a, k.dtype, x, k.width, k.rows, l.stride, kTileM);
    if (e == cudaSuccess) e = make_map(&a.b, k.dtype, w, 3, {k.width, k.out, (size_t)k.experts}, {l.stride, l.stride * k.out}, grouped_columns(k.device, EXPERTS_FORWARD, a));
    return e == cudaSuccess ? run_grouped<T, EXPERTS_FORWARD>(k.device, a, k.stream) : e;
}

template <typename T> static cudaError_t grouped_backward(const GroupedCall& k, const GroupedLayout& l, const void* dh, const float* z, size_t z_stride, const void* x, const void* w,
                                                          const char* padded, void* dx, void* dw) {
    cudaError_t e = cudaSuccess;
    const void* dz = dh;
    const bool vec = k.out % 8 == 0 && aligned_to(16, {dh});
    if (k.act != kNoActivation) {
        const ActGradArgs d = {dh, z, k.workspace + l.dz, k.starts, z_stride, l.d_stride, (unsigned)k.rows, (unsigned)k.experts, (unsigned)k.out, k.act};
        e = launch_early(vec ? k_act_grad<T, true> : k_act_grad<T, false>, (unsigned)((k.rows * ((k.out + 7) / 8) + 255) / 256), 256, k.stream, d);
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
        GroupedArgs a = grouped_args(k);
        a.n = (unsigned)k.width;
        a.k_blocks = blocks_of(k.out, kTileK);
        a.c = dx;
        e = make_map(&a.a, k.dtype, dz, k.out, k.rows, d_stride, kTileM);
        if (e == cudaSuccess) e = make_map(&a.b, k.dtype, w, 3, {k.width, k.out, (size_t)k.experts}, {l.stride, l.stride * k.out}, kTileK);
        if (e == cudaSuccess) e = run_grouped<T, EXPERTS_INPUT>(k.device, a, k.stream);
    }
    if (e == cudaSuccess && dw) {
        GroupedArgs a = grouped_args(k);
        a.m = (unsigned)k.out;
        a.n = (unsigned)k.width;
        a.c = dw;
        e = make_map(&a.a, k.dtype, dz, k.out, k.rows, d_stride, kTileK);
        if (e == cudaSuccess) e = make_map(&a.b, k.dtype, x, k.width, k.rows, l.stride, kTileK);
        if (e == cudaSuccess) e = run_grouped<T, EXPERTS_WEIGHT>(k.device, a, k.stream);
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
