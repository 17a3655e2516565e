/**
 * The end of one sub-block of a decoder and the entry of the next in one pass:
 *
 *     p = b rb .* w2,  rb = 1 / sqrt(mean(b^2) + eps)      (or p = b)
 *     y = x + s g .* p
 *     n = y ry .* w,   ry = 1 / sqrt(mean(y^2) + eps)
 *
 * and its gradients. With yh = y ry, bh = b rb and t = dn .* w, the derivative of a row's norm is ry (t - yh mean(t .* yh)):
 *
 *     D = dy + ry (t - yh mean(t .* yh))        dx = D          dw  = sum over rows dn .* yh
 *     u = s g .* D .* w2                        db = rb (u - bh mean(u .* bh))
 *     dw2 = sum s g .* D .* bh                  dg  = sum s D .* p
 *
 * A few operations per element that is moved: HBM bounds both. A CTA holds a row in registers, so that x, b (forward) and
 * dy, dn, y, b (backward) are read once and the sums of a row cost one barrier each. Rows are summed in fp32, and n comes from the
 * y of fp32 and not from the rounded one that is stored. The backward pass of a plain sum starts from the stored y, which saves it one of
 * five arrays; the rounding of y reaches the gradients only through yh.
 */
#include "decoder_ops.hpp"
#include "launch_early.cuh"
#include "row_access.cuh"

namespace dccl {

struct NormArgs {
    const void *x, *branch, *weight, *post, *gate;
    void *y, *n;
    float *rstd, *rstd_post;
    size_t rows_per_gate;
    unsigned width;
    int f32;
    float eps, scale;
};

struct NormGradArgs {
    const void *dy, *dn, *y, *branch, *weight, *post, *gate;
    const float *rstd, *rstd_post;
    void *dx, *dbranch;
    float *weight_sums, *post_sums, *gate_sums;      // [CTA][width], [CTA][width], [unit][width]
    size_t rows_per_gate, chunks, units;
    unsigned width;
    int f32;
    float scale;
};

/** E elements per thread in runs of V, run k of thread t at (k * threads + t) * V. */
template <typename T, int V, int E>
__global__ void __launch_bounds__(E == 8 ? 256 : E == 16 ? 512 : 1024, 1) k_residual_norm(const __grid_constant__ NormArgs a) {
    wait_for_stream();
    constexpr int K = E / V;
    __shared__ float parts[2][32];
    const unsigned runs = a.width / V, step = blockDim.x, t = threadIdx.x;
    const size_t row = blockIdx.x, at = row * a.width;
    const T *x = reinterpret_cast<const T*>(a.x) + at, *b = reinterpret_cast<const T*>(a.branch) + at;
    const bool has_branch = a.branch != nullptr;
    Run<T, V> xr[K], br[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const unsigned i = t + k * step;
        if (i < runs) {
            xr[k] = ld_run<T, V>(x + (size_t)i * V);
            if (has_branch) br[k] = ld_run<T, V>(b + (size_t)i * V);
        }
    }
    float factor = a.scale;
    if (a.post) {
        float sum = 0;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (t + k * step < runs)
#pragma unroll
                for (int e = 0; e < V; e++) { const float v = Traits<T>::up(br[k].e[e]); sum = fmaf(v, v, sum); }
        const float rb = rsqrtf(cta_sum(sum, parts[0]) / a.width + a.eps);
        if (a.rstd_post && t == 0) a.rstd_post[row] = rb;
        factor = rb;
    }
    float y[E], sum = 0;
    const size_t gate_at = a.gate ? row / a.rows_per_gate * a.width : 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const unsigned i = t + k * step;
        if (i >= runs) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = has_branch ? factor * Traits<T>::up(br[k].e[e]) : 0.0f;
        if (a.post) {
            float w[V];
            ld_vector<T, V>(w, a.post, a.f32 & DCCL_NORM_POST_F32, (size_t)i * V);
#pragma unroll
            for (int e = 0; e < V; e++) v[e] *= w[e] * a.scale;
        }
        if (a.gate) {
            float g[V];
            ld_vector<T, V>(g, a.gate, a.f32 & DCCL_NORM_GATE_F32, gate_at + (size_t)i * V);
#pragma unroll
            for (int e = 0; e < V; e++) v[e] *= g[e];
        }
        Run<T, V> out;
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float s = has_branch ? Traits<T>::up(xr[k].e[e]) + v[e] : Traits<T>::up(xr[k].e[e]);
            y[k * V + e] = s;
            sum = fmaf(s, s, sum);
            out.e[e] = Traits<T>::down(s);
        }
        if (has_branch) st_run<T, V>(reinterpret_cast<T*>(a.y) + at + (size_t)i * V, out);
    }
    const float ry = rsqrtf(cta_sum(sum, parts[1]) / a.width + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = ry;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const unsigned i = t + k * step;
        if (i >= runs) continue;
        float w[V];
        ld_vector<T, V>(w, a.weight, a.f32 & DCCL_NORM_WEIGHT_F32, (size_t)i * V);
        Run<T, V> out;
#pragma unroll
        for (int e = 0; e < V; e++) out.e[e] = Traits<T>::down(y[k * V + e] * ry * w[e]);
        st_run<T, V>(reinterpret_cast<T*>(a.n) + at + (size_t)i * V, out);
    }
}

/** The arrays that a row of the backward pass reads. SUM: y = x + branch (or x), taken as it was stored. FULL: with post, a gate or a
 *  scale the branch is read in any case, and y comes from x and branch again, exact. */
enum NormForm { SUM, FULL };
enum { DN, Y, DY, B };      // Y: x in the FULL form

constexpr int kNormStages = 3;
/** Whether three rows fit into shared memory: 16-bit rows of up to 8192 elements, fp32 rows of up to 2048. */
template <typename T, int V, int E> constexpr bool kNormStaged = V * sizeof(T) == 16 && E * sizeof(T) <= 32;

/**
 * Each CTA takes units of rows that share a row of the gate and keeps the columns' sums (dw, dw2, dg) in registers: dg leaves at
 * the end of a unit, dw and dw2 at the end of the CTA, for k_norm_columns to add. Where accesses are 16 bytes wide a thread copies
 * its own elements of the next two rows into shared memory of its own while it works on this one: no register holds them and
 * no barrier guards them.
 */
template <typename T, int V, int E, NormForm F>
__global__ void __launch_bounds__(E == 8 ? 256 : E == 16 ? 512 : 1024, E == 8 ? (F == SUM ? 4 : 3) : 1) k_residual_norm_grad(const __grid_constant__ NormGradArgs a) {
    wait_for_stream();
    constexpr int K = E / V, kArrays = F == SUM ? 3 : 4;
    constexpr bool kStaged = kNormStaged<T, V, E>;
    extern __shared__ uint4 staged[];                   // [stage][array][run][thread]
    __shared__ float parts[2][2][32];
    const unsigned runs = a.width / V, step = blockDim.x, t = threadIdx.x;
    const float inv_width = 1.0f / a.width;
    const T* const arrays[4] = {reinterpret_cast<const T*>(a.dn), reinterpret_cast<const T*>(a.y), reinterpret_cast<const T*>(a.dy), reinterpret_cast<const T*>(a.branch)};
    const auto fetch = [&](size_t row, unsigned stage) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const unsigned i = t + k * step;
#pragma unroll
            for (int j = 0; j < kArrays; j++)
                if (i < runs && arrays[j]) {
                    const uint32_t to = (uint32_t)__cvta_generic_to_shared(staged + ((stage * kArrays + j) * K + k) * step + t);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(arrays[j] + row * a.width + (size_t)i * V) : "memory");
                }
        }
    };
    const auto load = [&](int j, int k, size_t row, unsigned stage, float (&f)[V]) {
        Run<T, V> r;
        if constexpr (kStaged) r = *reinterpret_cast<const Run<T, V>*>(staged + ((stage * kArrays + j) * K + k) * step + t);
        else r = ld_run<T, V>(arrays[j] + row * a.width + (size_t)(t + k * step) * V);
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = Traits<T>::up(r.e[e]);
    };
    float sum_w[E], sum_p[F == FULL ? E : 1], sum_g[F == FULL ? E : 1];
#pragma unroll
    for (int e = 0; e < E; e++) {
        sum_w[e] = 0;
        if constexpr (F == FULL) sum_p[e] = sum_g[e] = 0;
    }
    unsigned turn = 0;
    for (size_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const size_t gate = unit / a.chunks, chunk = unit % a.chunks;
        const size_t begin = gate * a.rows_per_gate + chunk * a.rows_per_gate / a.chunks, end = gate * a.rows_per_gate + (chunk + 1) * a.rows_per_gate / a.chunks;
        unsigned stage = 0;
        if constexpr (kStaged) {
#pragma unroll
            for (int s = 0; s < kNormStages - 1; s++) {
                if (begin + s < end) fetch(begin + s, s);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        }
        for (size_t row = begin; row < end; row++, turn ^= 1) {
            if constexpr (kStaged) {
                const unsigned ahead = stage == 0 ? kNormStages - 1 : stage - 1;
                if (row + kNormStages - 1 < end) fetch(row + kNormStages - 1, ahead);
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group %0;" ::"n"(kNormStages - 1) : "memory");
            }
            const float ry = a.dn ? a.rstd[row] : 0.0f, rb = F == FULL && a.post ? a.rstd_post[row] : 1.0f;
            float d[E], yh[E], dot = 0;
            if (a.dn) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const unsigned i = t + k * step;
                    if (i >= runs) continue;
                    float w[V], dn[V], y[V];
                    load(DN, k, row, stage, dn);
                    load(Y, k, row, stage, y);
                    if constexpr (F == FULL) {
                        float v[V], b[V];
                        load(B, k, row, stage, b);
#pragma unroll
                        for (int e = 0; e < V; e++) v[e] = (a.post ? rb : a.scale) * b[e];      // as the forward pass rounds
                        if (a.post) {
                            ld_vector<T, V>(w, a.post, a.f32 & DCCL_NORM_POST_F32, (size_t)i * V);
#pragma unroll
                            for (int e = 0; e < V; e++) v[e] *= w[e] * a.scale;
                        }
                        if (a.gate) {
                            ld_vector<T, V>(w, a.gate, a.f32 & DCCL_NORM_GATE_F32, gate * a.width + (size_t)i * V);
#pragma unroll
                            for (int e = 0; e < V; e++) v[e] *= w[e];
                        }
#pragma unroll
                        for (int e = 0; e < V; e++) y[e] += v[e];
                    }
                    ld_vector<T, V>(w, a.weight, a.f32 & DCCL_NORM_WEIGHT_F32, (size_t)i * V);
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const int j = k * V + e;
                        yh[j] = y[e] * ry;
                        d[j] = dn[e] * w[e];
                        dot = fmaf(d[j], yh[j], dot);
                        sum_w[j] = fmaf(dn[e], yh[j], sum_w[j]);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) d[e] = yh[e] = 0;
            }
            const float c = a.dn ? cta_sum(dot, parts[turn][0]) * inv_width : 0.0f;
            float dot_b = 0;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const unsigned i = t + k * step;
                if (i >= runs) continue;
                float dy[V];
                if (a.dy) load(DY, k, row, stage, dy);
                Run<T, V> dx, db;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const int j = k * V + e;
                    d[j] = fmaf(ry, d[j] - yh[j] * c, a.dy ? dy[e] : 0.0f);
                    dx.e[e] = Traits<T>::down(d[j]);
                }
                st_run<T, V>(reinterpret_cast<T*>(a.dx) + row * a.width + (size_t)i * V, dx);
                if constexpr (F == FULL) {
                    float w2[V], g[V], b[V];
                    load(B, k, row, stage, b);
                    if (a.post) ld_vector<T, V>(w2, a.post, a.f32 & DCCL_NORM_POST_F32, (size_t)i * V);
                    if (a.gate) ld_vector<T, V>(g, a.gate, a.f32 & DCCL_NORM_GATE_F32, gate * a.width + (size_t)i * V);
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const int j = k * V + e;
                        float v = d[j] * a.scale;
                        const float bh = b[e] * rb;
                        if (a.gate) {
                            sum_g[j] = fmaf(v, a.post ? bh * w2[e] : bh, sum_g[j]);
                            v *= g[e];
                        }
                        if (a.post) {
                            sum_p[j] = fmaf(v, bh, sum_p[j]);
                            v *= w2[e];
                            dot_b = fmaf(v, bh, dot_b);
                        }
                        d[j] = v;
                        db.e[e] = Traits<T>::down(v);
                    }
                    if (!a.post) st_run<T, V>(reinterpret_cast<T*>(a.dbranch) + row * a.width + (size_t)i * V, db);
                }
            }
            if constexpr (F == FULL) {
                if (a.post) {
                    const float cb = cta_sum(dot_b, parts[turn][1]) * inv_width;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        const unsigned i = t + k * step;
                        if (i >= runs) continue;
                        float b[V];
                        load(B, k, row, stage, b);
                        Run<T, V> db;
#pragma unroll
                        for (int e = 0; e < V; e++) db.e[e] = Traits<T>::down(rb * (d[k * V + e] - b[e] * rb * cb));
                        st_run<T, V>(reinterpret_cast<T*>(a.dbranch) + row * a.width + (size_t)i * V, db);
                    }
                }
            }
            stage = stage == kNormStages - 1 ? 0 : stage + 1;
        }
        if constexpr (F == FULL) {
            if (a.gate_sums) {
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (t + k * step < runs)
#pragma unroll
                        for (int e = 0; e < V; e++) {
                            a.gate_sums[unit * a.width + (size_t)(t + k * step) * V + e] = sum_g[k * V + e];
                            sum_g[k * V + e] = 0;
                        }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K; k++)
        if (t + k * step < runs)
#pragma unroll
            for (int e = 0; e < V; e++) {
                const size_t j = (size_t)blockIdx.x * a.width + (size_t)(t + k * step) * V + e;
                if (a.weight_sums) a.weight_sums[j] = sum_w[k * V + e];
                if constexpr (F == FULL)
                    if (a.post_sums) a.post_sums[j] = sum_p[k * V + e];
            }
}

struct NormColumnArgs {
    const float *weight_sums, *post_sums, *gate_sums;
    void *dweight, *dpost, *dgate;
    unsigned ctas, chunks, width, blocks;       // blocks: CTAs across the columns
    int f32;
};

constexpr int kColumnSlices = 16;

template <typename T> __device__ __forceinline__ void st_vector(void* p, bool f32, size_t i, float v) {
    if (f32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<T*>(p)[i] = Traits<T>::down(v);
}

/** Adds up what the CTAs left: 32 columns per CTA, 16 threads per column. The first blocks take the weight, then post, then each row of the gate. */
template <typename T> __global__ void __launch_bounds__(32 * kColumnSlices) k_norm_columns(const __grid_constant__ NormColumnArgs a) {
    wait_for_stream();
    __shared__ float parts[kColumnSlices][33];
    const unsigned what = blockIdx.x / a.blocks, lane = threadIdx.x % 32, slice = threadIdx.x / 32;
    const size_t column = (size_t)(blockIdx.x % a.blocks) * 32 + lane;
    const unsigned gate = what - (a.weight_sums != nullptr) - (a.post_sums != nullptr);
    const bool is_weight = a.weight_sums && what == 0, is_post = !is_weight && a.post_sums && what == (a.weight_sums != nullptr);
    const float* from = is_weight ? a.weight_sums : is_post ? a.post_sums : a.gate_sums + (size_t)gate * a.chunks * a.width;
    const unsigned n = is_weight || is_post ? a.ctas : a.chunks;
    float sum = 0;
    if (column < a.width)
        for (unsigned i = slice; i < n; i += kColumnSlices) sum += from[(size_t)i * a.width + column];
    parts[slice][lane] = sum;
    __syncthreads();
    if (slice || column >= a.width) return;
#pragma unroll
    for (int s = 1; s < kColumnSlices; s++) sum += parts[s][lane];
    if (is_weight) st_vector<T>(a.dweight, a.f32 & DCCL_NORM_WEIGHT_F32, column, sum);
    else if (is_post) st_vector<T>(a.dpost, a.f32 & DCCL_NORM_POST_F32, column, sum);
    else st_vector<T>(a.dgate, a.f32 & DCCL_NORM_GATE_F32, (size_t)gate * a.width + column, sum);
}

constexpr size_t kNormMaxWidth = 32768;

/** Elements per thread and threads of a CTA that hold a row. */
struct NormShape { int elements, threads; };
static NormShape norm_shape(size_t width) {
    const int e = width <= 2048 ? 8 : width <= 8192 ? 16 : 32;
    return {e, (int)((width + e * 32 - 1) / (e * 32)) * 32};
}

/** Elements per access: 16 bytes, else a pair of 16-bit elements, else one. */
static int norm_run(int dtype, size_t width, bool aligned16_all, bool aligned8_all) {
    const int wide = dtype == 7 ? 4 : 8;
    if (width % wide == 0 && aligned16_all) return wide;
    return dtype != 7 && width % 2 == 0 && aligned8_all ? 2 : 1;
}

/** CTAs of the backward pass, all resident at once, and how the rows of a gate are cut among them. */
struct NormCut { size_t chunks, units; unsigned ctas; };
static NormCut norm_cut(int device, size_t rows, size_t width, size_t gates, bool full) {
    const NormShape s = norm_shape(width);
    const size_t per_sm = s.elements == 8 ? (full ? 768 : 1024) / s.threads : s.elements == 16 ? 512 / s.threads : 1;
    const size_t want = (size_t)sm_count(device) * (per_sm ? per_sm : 1);
    if (!want) return {0, 0, 0};
    const size_t groups = gates ? gates : 1, rows_per = rows / groups;
    size_t chunks = (want + groups - 1) / groups;
    if (chunks > rows_per) chunks = rows_per;
    const size_t units = groups * chunks;
    return {chunks, units, (unsigned)(units < want ? units : want)};
}

template <typename T, int V, int E> static cudaError_t norm_launch(unsigned grid, unsigned block, cudaStream_t stream, const NormArgs& a, bool, int) {
    return launch_early(k_residual_norm<T, V, E>, grid, block, stream, a);
}
template <typename T, int V, int E, NormForm F> static cudaError_t norm_grad_launch(unsigned grid, unsigned block, cudaStream_t stream, const NormGradArgs& a, int device) {
    const size_t shared = kNormStaged<T, V, E> ? (size_t)kNormStages * (F == SUM ? 3 : 4) * E * sizeof(T) * block : 0;
    if (shared > 40 << 10) {        // 48 KB with the static part need no leave
        static std::atomic<bool> ready[64];
        if (!ready[device].load(std::memory_order_relaxed)) {
            const cudaError_t e = cudaFuncSetAttribute(k_residual_norm_grad<T, V, E, F>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024);
            if (e != cudaSuccess) return e;
            ready[device].store(true, std::memory_order_relaxed);
        }
    }
    return launch_early_shared(k_residual_norm_grad<T, V, E, F>, grid, block, shared, stream, a);
}
template <typename T, int V, int E> static cudaError_t norm_launch(unsigned grid, unsigned block, cudaStream_t stream, const NormGradArgs& a, bool full, int device) {
    return full ? norm_grad_launch<T, V, E, FULL>(grid, block, stream, a, device) : norm_grad_launch<T, V, E, SUM>(grid, block, stream, a, device);
}
template <typename T, int V, typename Args> static cudaError_t norm_launch(int elements, unsigned grid, unsigned block, cudaStream_t stream, const Args& a, bool full, int device) {
    return elements == 8 ? norm_launch<T, V, 8>(grid, block, stream, a, full, device) : elements == 16 ? norm_launch<T, V, 16>(grid, block, stream, a, full, device)
                                                                                                       : norm_launch<T, V, 32>(grid, block, stream, a, full, device);
}

template <typename Args> static cudaError_t norm_dispatch(int device, int dtype, int run, int elements, unsigned grid, unsigned block, cudaStream_t stream, const Args& a, bool full) {
    switch (dtype * 16 + run) {
        case 6 * 16 + 8: return norm_launch<__half, 8>(elements, grid, block, stream, a, full, device);
        case 6 * 16 + 2: return norm_launch<__half, 2>(elements, grid, block, stream, a, full, device);
        case 6 * 16 + 1: return norm_launch<__half, 1>(elements, grid, block, stream, a, full, device);
        case 9 * 16 + 8: return norm_launch<__nv_bfloat16, 8>(elements, grid, block, stream, a, full, device);
        case 9 * 16 + 2: return norm_launch<__nv_bfloat16, 2>(elements, grid, block, stream, a, full, device);
        case 9 * 16 + 1: return norm_launch<__nv_bfloat16, 1>(elements, grid, block, stream, a, full, device);
        case 7 * 16 + 4: return norm_launch<float, 4>(elements, grid, block, stream, a, full, device);
        case 7 * 16 + 1: return norm_launch<float, 1>(elements, grid, block, stream, a, full, device);
        default: return cudaErrorInvalidValue;
    }
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_residual_norm(int device, int dtype, size_t rows, size_t width, const void* x, const void* branch, const void* weight, const void* post,
                                  const void* gate, size_t rows_per_gate, int f32_vectors, double eps, double scale, void* y, void* n, void* rstd,
                                  void* rstd_post, void* stream) {
    if (!rows) return 0;
    if (!width || width > kNormMaxWidth || rows > 0x7fffffffu || (gate && !rows_per_gate) || (post && !branch) || (gate && !branch))
        return report("dccl_residual_norm", cudaErrorInvalidValue);
    const NormArgs a = {x, branch, weight, post, gate, y, n, (float*)rstd, (float*)rstd_post, rows_per_gate, (unsigned)width, f32_vectors, (float)eps, (float)scale};
    const auto all = {x, branch, weight, post, gate, (const void*)y, (const void*)n};
    const NormShape s = norm_shape(width);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report("dccl_residual_norm", on.e);
    return report("dccl_residual_norm", norm_dispatch(device, dtype, norm_run(dtype, width, aligned_to(16, all), aligned_to(8, all)), s.elements, (unsigned)rows, (unsigned)s.threads,
                                                      (cudaStream_t)stream, a, false));
}

extern "C" size_t dccl_residual_norm_workspace(int device, size_t rows, size_t width, size_t gates, int has_post, int full) {
    if (!rows || !width || (gates && rows % gates)) return 0;
    const NormCut cut = norm_cut(device, rows, width, gates, full != 0);
    return ((size_t)cut.ctas * (has_post ? 2 : 1) + (gates ? cut.units : 0)) * width * sizeof(float);
}

extern "C" int dccl_residual_norm_backward(int device, int dtype, size_t rows, size_t width, const void* dy, const void* dn, const void* y, const void* branch,
                                           const void* weight, const void* post, const void* gate, size_t rows_per_gate, int f32_vectors, double scale,
                                           const void* rstd, const void* rstd_post, void* dx, void* dbranch, void* dweight, void* dpost, void* dgate,
                                           void* workspace, size_t workspace_bytes, void* stream_v) {
    const char* who = "dccl_residual_norm_backward";
    const size_t gates = gate && rows_per_gate ? rows / rows_per_gate : 0;
    if (!rows || !width || width > kNormMaxWidth || (gate && (!gates || gates * rows_per_gate != rows)) || (post && (!branch || !rstd_post)) || (gate && !branch) || (dn && !rstd)
        || !branch != !dbranch)
        return report(who, cudaErrorInvalidValue);
    const bool full = branch != nullptr;
    const NormCut cut = norm_cut(device, rows, width, gates, full);
    const size_t blocks = (width + 31) / 32, vectors = (dn && dweight ? 1 : 0) + (post && dpost ? 1 : 0) + (gate && dgate ? gates : 0);
    if (!cut.units || blocks * vectors > 0x7fffffffu || workspace_bytes < dccl_residual_norm_workspace(device, rows, width, gates, post != nullptr, full))
        return report(who, cudaErrorInvalidValue);
    float* const weight_sums = (float*)workspace;
    float* const post_sums = post ? weight_sums + (size_t)cut.ctas * width : nullptr;
    float* const gate_sums = gate ? weight_sums + (size_t)cut.ctas * width * (post ? 2 : 1) : nullptr;
    const NormGradArgs a = {dy, dn, y, branch, weight, post, gate, (const float*)rstd, (const float*)rstd_post, dx, dbranch,
                            dn && dweight ? weight_sums : nullptr, post && dpost ? post_sums : nullptr, gate && dgate ? gate_sums : nullptr,
                            gate ? rows_per_gate : rows, cut.chunks, cut.units, (unsigned)width, f32_vectors, (float)scale};
    const auto all = {dy, dn, y, branch, weight, post, gate, (const void*)dx, (const void*)dbranch};
    const NormShape s = norm_shape(width);
    cudaStream_t stream = (cudaStream_t)stream_v;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    cudaError_t e = norm_dispatch(device, dtype, norm_run(dtype, width, aligned_to(16, all), aligned_to(8, all)), s.elements, cut.ctas, (unsigned)s.threads, stream, a, full);
    if (e == cudaSuccess && vectors) {
        const NormColumnArgs c = {a.weight_sums, a.post_sums, a.gate_sums, dweight, dpost, dgate, cut.ctas, (unsigned)cut.chunks, (unsigned)width, (unsigned)blocks, f32_vectors};
        const unsigned grid = (unsigned)(blocks * vectors);
        e = dtype == 6 ? launch_early(k_norm_columns<__half>, grid, 32 * kColumnSlices, stream, c) : dtype == 7 ? launch_early(k_norm_columns<float>, grid, 32 * kColumnSlices, stream, c)
                                                                                                               : launch_early(k_norm_columns<__nv_bfloat16>, grid, 32 * kColumnSlices, stream, c);
    }
    return report(who, e);
}
