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
 *     u = s g .* w2 .* D                        db = rb (u - bh mean(u .* bh))
 *     S   = sum over rows of a gate D .* bh     dg  = s w2 .* S,  dw2 = sum over gates s g .* S
 *
 * A few operations per element that is moved: HBM bounds both. A CTA holds a row in registers, so that x, b (forward) and
 * dy, dn, x, b (backward) are read once and the sums of a row cost one barrier each. Rows are summed in fp32, and n comes from the
 * y of fp32 and not from the rounded one that is stored. The backward pass makes y again from x and b: from the stored y, which
 * would save a plain sum one of five arrays, its rounding goes into every term of dw and makes that half again as inexact.
 *
 * A plain sum of 16384 x 2048 bf16: forward 41 us (6.5 TB/s of four arrays), backward 59 (5.7 TB/s of five) and 4 for the columns' sums. 8192 x 8192
 * bf16 with every part: 106 us (5.1 TB/s), 148 (5.4 TB/s of six) and 6; there sixteen warps with 112 registers each are all of an SM. 16384 x 2048 fp32: a
 * plain sum 81 us forward (6.6 TB/s) and 188 both ways, with every part 83 and 219.
 */
#include "decoder_ops.hpp"
#include "../kernels/launch_early.cuh"
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
    const void *dy, *dn, *x, *branch, *weight, *post, *gate;
    const float *rstd, *rstd_post;
    void *dx, *dbranch;
    float *weight_sums, *branch_sums;                // [CTA][width], [unit][width]
    size_t rows, rows_per_gate;
    Divisor chunks;                                  // of the rows of a gate
    unsigned chunk_rows, longer, units, width;
    int f32;
    float scale;
};

/** What a call has. The kernels are compiled for each: tests of pointers inside of the loops took a third of their instructions. */
enum { BRANCH = 1, POST = 2, GATE = 4, SCALE = 8 };

/** E elements per thread in runs of V, run k of thread t at (k * threads + t) * V. EXACT: rows fill the threads' elements, and no test stands between
 *  the loads of one run and the arithmetic of another (backward, 8192 elements: 227 -> 203 us). */
template <typename T, int V, int E, int F, bool EXACT>
__global__ void __launch_bounds__(E == 8 ? 256 : E == 16 ? 512 : 1024, E == 16 ? 2 : 1) k_residual_norm(const __grid_constant__ NormArgs a) {
    wait_for_stream();
    constexpr int K = E / V;
    __shared__ __align__(16) float parts[2][32];
    const unsigned runs = a.width / V, step = blockDim.x, t = threadIdx.x;
    const size_t row = blockIdx.x, at = row * a.width;
    const T *x = reinterpret_cast<const T*>(a.x) + at, *b = reinterpret_cast<const T*>(a.branch) + at;
    Run<T, V> xr[K], br[F & BRANCH ? K : 1];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const unsigned i = t + k * step;
        if (EXACT || i < runs) {
            xr[k] = ld_run<T, V>(x + (size_t)i * V);
            if constexpr (F & BRANCH) br[k] = ld_run<T, V>(b + (size_t)i * V);
        }
    }
    float factor = a.scale;
    if constexpr (F & POST) {
        float sum = 0;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (EXACT || t + k * step < runs)
#pragma unroll
                for (int e = 0; e < V; e++) { const float v = Traits<T>::up(br[k].e[e]); sum = fmaf(v, v, sum); }
        factor = rsqrtf(cta_sum(sum, parts[0]) / a.width + a.eps);
        if (a.rstd_post && t == 0) a.rstd_post[row] = factor;
        factor *= a.scale;
    }
    float y[E], sum = 0;
    const size_t gate_at = F & GATE ? row / a.rows_per_gate * a.width : 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const unsigned i = t + k * step;
        if (!EXACT && i >= runs) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = Traits<T>::up(xr[k].e[e]);
        if constexpr (F & BRANCH) {
            float p[V], w[V];
#pragma unroll
            for (int e = 0; e < V; e++) p[e] = Traits<T>::up(br[k].e[e]);
            if constexpr (F & POST) {
                ld_vector<T, V>(w, a.post, a.f32 & DCCL_NORM_POST_F32, (size_t)i * V);
#pragma unroll
                for (int e = 0; e < V; e++) p[e] *= w[e];
            }
            if constexpr (F & GATE) {
                ld_vector<T, V>(w, a.gate, a.f32 & DCCL_NORM_GATE_F32, gate_at + (size_t)i * V);
#pragma unroll
                for (int e = 0; e < V; e++) p[e] *= w[e];
            }
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = F & (POST | SCALE) ? fmaf(factor, p[e], v[e]) : v[e] + p[e];
            st_run<T, V>(reinterpret_cast<T*>(a.y) + at + (size_t)i * V, round_run<T, V>(v));
        }
#pragma unroll
        for (int e = 0; e < V; e++) {
            y[k * V + e] = v[e];
            sum = fmaf(v[e], v[e], sum);
        }
    }
    const float ry = rsqrtf(cta_sum(sum, parts[1]) / a.width + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = ry;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const unsigned i = t + k * step;
        if (!EXACT && i >= runs) continue;
        float w[V];
        ld_vector<T, V>(w, a.weight, a.f32 & DCCL_NORM_WEIGHT_F32, (size_t)i * V);
#pragma unroll
        for (int e = 0; e < V; e++) w[e] *= y[k * V + e] * ry;
        st_run<T, V>(reinterpret_cast<T*>(a.n) + at + (size_t)i * V, round_run<T, V>(w));
    }
}

/** The arrays that a row of the backward pass reads. */
enum { DN, X, DY, B };
enum { IN_WEIGHT, IN_BRANCH };          // the vectors, in shared memory as fp32: w, and s g .* w2, of which a row of the branch takes nothing else
constexpr int FULL = POST | GATE | SCALE;      // any of them, and the branch has a gradient that is not x's

/** Rows in shared memory at a time: three of up to 2048 elements, two of up to 8192 16-bit ones. */
template <typename T, int E> constexpr int kNormStages = E == 8 ? 3 : E == 16 && sizeof(T) == 2 ? 2 : 0;

/** Bytes of an array's row there: a place for each thread's accesses, or, where rows start anywhere, the aligned 16 bytes that a row touches. */
template <typename T, int V, int E> __host__ __device__ constexpr size_t norm_row_bytes(unsigned threads, unsigned width) {
    return V * sizeof(T) == 16 ? (size_t)threads * E * sizeof(T) : (width * sizeof(T) + 15) / 16 * 16 + 16;
}

template <typename T, int V, int E, int F> constexpr size_t norm_grad_shared(unsigned threads, unsigned width) {
    return kNormStages<T, E> * (F & BRANCH ? 4 : 3) * norm_row_bytes<T, V, E>(threads, width) + (E <= 16 ? (size_t)threads * E * (F & FULL ? 2 : 1) * sizeof(float) : 0);
}

/**
 * Each CTA takes units of rows that share a row of the gate and keeps the columns' sums (dw, S) in registers: S leaves at
 * the end of a unit, dw at the end of the CTA, for k_norm_columns to add. The next rows are copied into shared memory while
 * the CTA works on this one: where accesses are 16 bytes wide, each thread's own elements by itself, with no barrier to guard them. Rows
 * that start anywhere are copied in the aligned 16 bytes that they touch, which the threads share. (Read by element from global memory,
 * rows of 1451 fp16 took 36 us out of L2 and 60 out of HBM for 1551 rows.) The vectors are kept there in fp32.
 */
template <typename T, int V, int E, int F, bool EXACT>
__global__ void __launch_bounds__(E == 8 ? 256 : E == 16 ? 512 : 1024, E == 8 ? (F & FULL ? 3 : 4) : 1) k_residual_norm_grad(const __grid_constant__ NormGradArgs a) {
    wait_for_stream();
    constexpr int K = E / V, kArrays = F & BRANCH ? 4 : 3, kStages = kNormStages<T, E>, kPiece = V < 4 ? V : 4;
    constexpr bool kOwn = V * sizeof(T) == 16;          // a thread's elements are its own matter
    constexpr bool kVectors = E <= 16;                  // in shared memory
    extern __shared__ uint4 staged[];                   // [stage][array][run][thread], then [vector][run][piece][thread] of kPiece floats
    __shared__ __align__(16) float parts[2][2][32];
    const unsigned runs = a.width / V, step = blockDim.x, t = threadIdx.x;
    const float inv_width = 1.0f / a.width;
    const T* const arrays[4] = {reinterpret_cast<const T*>(a.dn), reinterpret_cast<const T*>(a.x), reinterpret_cast<const T*>(a.dy), reinterpret_cast<const T*>(a.branch)};
    const unsigned row_bytes = (unsigned)norm_row_bytes<T, V, E>(step, a.width);
    Run<float, kPiece>* const vectors = reinterpret_cast<Run<float, kPiece>*>(reinterpret_cast<char*>(staged) + (size_t)kStages * kArrays * row_bytes);
    const auto fetch = [&](size_t row, unsigned stage) {
        if constexpr (!kOwn) {
#pragma unroll
            for (int j = 0; j < kArrays; j++) {
                if (!arrays[j]) continue;
                const uintptr_t start = reinterpret_cast<uintptr_t>(arrays[j] + row * a.width), end = reinterpret_cast<uintptr_t>(arrays[j] + a.rows * a.width);
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(staged) + (stage * kArrays + j) * row_bytes;
                const unsigned pieces = (unsigned)(((start & 15) + a.width * sizeof(T) + 15) / 16);
                for (unsigned i = t; i < pieces; i += step) {
                    const uintptr_t from = (start & ~(uintptr_t)15) + 16 * (size_t)i;
                    const unsigned bytes = end - from < 16 ? (unsigned)(end - from) : 16;      // nothing is read behind the last row
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 16 * i), "l"(from), "r"(bytes) : "memory");
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const unsigned i = t + k * step;
#pragma unroll
                for (int j = 0; j < kArrays; j++)
                    if ((EXACT || i < runs) && arrays[j]) {
                        const uint32_t to = (uint32_t)__cvta_generic_to_shared(staged + ((stage * kArrays + j) * K + k) * step + t);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(arrays[j] + row * a.width + (size_t)i * V) : "memory");
                    }
            }
        }
    };
    const T* here[4];                   // this thread's first run of the current row, unless it is in its own part of shared memory
    T *dx_at, *db_at;
    const auto find = [&](size_t row, unsigned stage) {
        if constexpr (!kOwn || kStages == 0) {
#pragma unroll
            for (int j = 0; j < kArrays; j++) {
                const T* const start = arrays[j] + row * a.width;
                if constexpr (kStages > 0)
                    here[j] = reinterpret_cast<const T*>(reinterpret_cast<const char*>(staged) + (stage * kArrays + j) * row_bytes + (reinterpret_cast<uintptr_t>(start) & 15)) + t * V;
                else here[j] = start + t * V;
            }
            dx_at = reinterpret_cast<T*>(a.dx) + row * a.width + t * V;
            db_at = reinterpret_cast<T*>(a.dbranch) + row * a.width + t * V;
        }
    };
    const auto store = [&](bool branch, size_t row, int k, const float (&f)[V]) {
        T* to;
        if constexpr (!kOwn || kStages == 0) to = (branch ? db_at : dx_at) + k * step * V;
        else to = reinterpret_cast<T*>(branch ? a.dbranch : a.dx) + row * a.width + (size_t)(t + k * step) * V;
        st_run<T, V>(to, round_run<T, V>(f));
    };
    const auto load = [&](int j, int k, unsigned stage, float (&f)[V]) {
        Run<T, V> r;
        if constexpr (kOwn && kStages > 0) r = *reinterpret_cast<const Run<T, V>*>(staged + ((stage * kArrays + j) * K + k) * step + t);
        else r = ld_run<T, V>(here[j] + k * step * V);
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = Traits<T>::up(r.e[e]);
    };
    const auto put = [&](int which, int k, const float (&f)[V]) {
#pragma unroll
        for (int q = 0; q < V / kPiece; q++) {
            Run<float, kPiece> piece;
#pragma unroll
            for (int e = 0; e < kPiece; e++) piece.e[e] = f[q * kPiece + e];
            vectors[((which * K + k) * (V / kPiece) + q) * step + t] = piece;
        }
    };
    const auto weight_of = [&](int k, float (&f)[V]) { ld_vector<T, V>(f, a.weight, a.f32 & DCCL_NORM_WEIGHT_F32, (size_t)(t + k * step) * V); };
    const auto branch_of = [&](size_t gate_at, int k, float (&f)[V]) {
        const size_t i = (size_t)(t + k * step) * V;
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = a.scale;
        float w[V];
        if constexpr (F & POST) {
            ld_vector<T, V>(w, a.post, a.f32 & DCCL_NORM_POST_F32, i);
#pragma unroll
            for (int e = 0; e < V; e++) f[e] *= w[e];
        }
        if constexpr (F & GATE) {
            ld_vector<T, V>(w, a.gate, a.f32 & DCCL_NORM_GATE_F32, gate_at + i);
#pragma unroll
            for (int e = 0; e < V; e++) f[e] *= w[e];
        }
    };
    const auto vector = [&](int which, size_t gate_at, int k, float (&f)[V]) {
        if constexpr (kVectors) {
#pragma unroll
            for (int q = 0; q < V / kPiece; q++) {
                const Run<float, kPiece> piece = vectors[((which * K + k) * (V / kPiece) + q) * step + t];
#pragma unroll
                for (int e = 0; e < kPiece; e++) f[q * kPiece + e] = piece.e[e];
            }
        } else if (which == IN_WEIGHT) weight_of(k, f);
        else branch_of(gate_at, k, f);
    };
    if constexpr (kVectors) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (!EXACT && t + k * step >= runs) continue;
            float f[V];
            weight_of(k, f);
            put(IN_WEIGHT, k, f);
        }
    }
    float sum_w[E], sum_b[F & (POST | GATE) ? E : 1];
#pragma unroll
    for (int e = 0; e < E; e++) {
        sum_w[e] = 0;
        if constexpr (F & (POST | GATE)) sum_b[e] = 0;
    }
    unsigned turn = 0;
    for (unsigned unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const unsigned gate = a.chunks.quotient(unit), chunk = unit - gate * a.chunks.d;
        const size_t gate_at = (size_t)gate * a.width;
        // the first `longer` chunks have one row more than the others
        const size_t begin = (size_t)gate * a.rows_per_gate + (size_t)chunk * a.chunk_rows + (chunk < a.longer ? chunk : a.longer), end = begin + a.chunk_rows + (chunk < a.longer);
        unsigned stage = 0;
        if constexpr (kStages > 0) {
            if constexpr (!kOwn) __syncthreads();       // the last unit's rows
#pragma unroll
            for (int s = 0; s < kStages - 1; s++) {
                if (begin + s < end) fetch(begin + s, s);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        }
        if constexpr ((F & FULL) && kVectors) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (!EXACT && t + k * step >= runs) continue;
                float f[V];
                branch_of(gate_at, k, f);
                put(IN_BRANCH, k, f);
            }
        }
        float next_ry = a.dn && begin < end ? a.rstd[begin] : 0.0f, next_rb = 1.0f;
        if constexpr (F & POST) next_rb = begin < end ? a.rstd_post[begin] : 0.0f;
        for (size_t row = begin; row < end; row++, turn ^= 1) {
            if constexpr (kStages > 0) {
                const unsigned ahead = stage == 0 ? kStages - 1 : stage - 1;
                if constexpr (!kOwn) {      // this row is there, and every thread is done with the one before, whose place the next one takes
                    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
                    __syncthreads();
                }
                if (row + kStages - 1 < end) fetch(row + kStages - 1, ahead);
                asm volatile("cp.async.commit_group;" ::: "memory");
                if constexpr (kOwn) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            }
            const float ry = next_ry, rb = next_rb;
            if (row + 1 < end) {
                next_ry = a.dn ? a.rstd[row + 1] : 0.0f;
                if constexpr (F & POST) next_rb = a.rstd_post[row + 1];
            }
            find(row, stage);
            float d[E], yh[E], dot = 0;
            if (a.dn) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const unsigned i = t + k * step;
                    if (!EXACT && i >= runs) continue;
                    float w[V], dn[V], y[V];
                    load(DN, k, stage, dn);
                    load(X, k, stage, y);
                    if constexpr (F & BRANCH) {
                        float p[V];
                        load(B, k, stage, p);
                        if constexpr (F & FULL) {
                            vector(IN_BRANCH, gate_at, k, w);
#pragma unroll
                            for (int e = 0; e < V; e++) p[e] *= w[e];
                        }
#pragma unroll
                        for (int e = 0; e < V; e++) y[e] = F & POST ? fmaf(rb, p[e], y[e]) : y[e] + p[e];
                    }
                    vector(IN_WEIGHT, 0, k, w);
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
                if (!EXACT && i >= runs) continue;
                float dy[V];
                if (a.dy) load(DY, k, stage, dy);
                float out[V];
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const int j = k * V + e;
                    d[j] = fmaf(ry, d[j] - yh[j] * c, a.dy ? dy[e] : 0.0f);
                    out[e] = d[j];
                }
                store(false, row, k, out);
                if constexpr (F & FULL) {
                    float w[V], b[V];
                    load(B, k, stage, b);
                    vector(IN_BRANCH, gate_at, k, w);
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const int j = k * V + e;
                        const float bh = F & POST ? b[e] * rb : b[e];
                        if constexpr (F & (POST | GATE)) sum_b[j] = fmaf(d[j], bh, sum_b[j]);
                        d[j] = out[e] = d[j] * w[e];
                        if constexpr (F & POST) dot_b = fmaf(d[j], bh, dot_b);
                    }
                    if constexpr (!(F & POST)) store(true, row, k, out);
                }
            }
            if constexpr (F & POST) {
                const float cb = cta_sum(dot_b, parts[turn][1]) * inv_width * rb;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const unsigned i = t + k * step;
                    if (!EXACT && i >= runs) continue;
                    float b[V];
                    load(B, k, stage, b);
#pragma unroll
                    for (int e = 0; e < V; e++) b[e] = rb * (d[k * V + e] - b[e] * cb);
                    store(true, row, k, b);
                }
            }
            if constexpr (kStages > 0) stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        if constexpr (F & (POST | GATE)) {
            if (a.branch_sums) {
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (EXACT || t + k * step < runs)
#pragma unroll
                        for (int e = 0; e < V; e++) {
                            a.branch_sums[(size_t)unit * a.width + (t + k * step) * V + e] = sum_b[k * V + e];
                            sum_b[k * V + e] = 0;
                        }
            }
        }
    }
    if (!a.weight_sums) return;
#pragma unroll
    for (int k = 0; k < K; k++)
        if (EXACT || t + k * step < runs)
#pragma unroll
            for (int e = 0; e < V; e++) a.weight_sums[(size_t)blockIdx.x * a.width + (t + k * step) * V + e] = sum_w[k * V + e];
}

struct NormColumnArgs {
    const float *weight_sums, *branch_sums;
    const void *post, *gate;
    void *dweight, *dpost, *dgate;
    Divisor chunks, blocks;         // blocks: CTAs across the columns
    unsigned ctas, units, width;
    int f32;
    float scale;
};

template <typename T> __device__ __forceinline__ float ld_one(const void* p, bool f32, size_t i) {
    return f32 ? reinterpret_cast<const float*>(p)[i] : Traits<T>::up(reinterpret_cast<const T*>(p)[i]);
}
template <typename T> __device__ __forceinline__ void st_vector(void* p, bool f32, size_t i, float v) {
    if (f32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<T*>(p)[i] = Traits<T>::down(v);
}

/** Adds up what the CTAs left: 32 columns per CTA, SLICES threads per column. The first blocks take the weight, then post, then each row of the gate. */
template <typename T, int SLICES> __global__ void __launch_bounds__(32 * SLICES) k_norm_columns(const __grid_constant__ NormColumnArgs a) {
    wait_for_stream();
    __shared__ float parts[SLICES][33];
    const unsigned what = a.blocks.quotient(blockIdx.x), lane = threadIdx.x % 32, slice = threadIdx.x / 32;
    const size_t column = (size_t)(blockIdx.x - what * a.blocks.d) * 32 + lane;
    const bool is_weight = a.dweight && what == 0, is_post = !is_weight && a.dpost && what == (a.dweight != nullptr);
    const unsigned gate = what - (a.dweight != nullptr) - (a.dpost != nullptr);
    const float* from = is_weight ? a.weight_sums : is_post ? a.branch_sums : a.branch_sums + (size_t)gate * a.chunks.d * a.width;
    const unsigned n = is_weight ? a.ctas : is_post ? a.units : a.chunks.d;
    float sum = 0;
    if (column < a.width) {
        if (is_post && a.gate) {
#pragma unroll 8
            for (unsigned i = slice; i < n; i += SLICES)
                sum = fmaf(from[(size_t)i * a.width + column], ld_one<T>(a.gate, a.f32 & DCCL_NORM_GATE_F32, (size_t)a.chunks.quotient(i) * a.width + column), sum);
        } else {
#pragma unroll 8
            for (unsigned i = slice; i < n; i += SLICES) sum += from[(size_t)i * a.width + column];
        }
    }
    parts[slice][lane] = sum;
    __syncthreads();
    if (slice || column >= a.width) return;
#pragma unroll
    for (int s = 1; s < SLICES; s++) sum += parts[s][lane];
    if (is_weight) st_vector<T>(a.dweight, a.f32 & DCCL_NORM_WEIGHT_F32, column, sum);
    else if (is_post) st_vector<T>(a.dpost, a.f32 & DCCL_NORM_POST_F32, column, a.scale * sum);
    else {
        if (a.post) sum *= ld_one<T>(a.post, a.f32 & DCCL_NORM_POST_F32, column);
        st_vector<T>(a.dgate, a.f32 & DCCL_NORM_GATE_F32, (size_t)gate * a.width + column, a.scale * sum);
    }
}

/** Elements per thread and threads of a CTA that hold a row. Above 8192 elements a thread of 1024 has 64 registers for 32 elements, and every backward form
 *  spills: 2048 x 16384 bf16, a plain sum 44 us forward and 255 both ways, with every part 65 and 471 (floors 42 and 83; a plain sum
 *  of 16384 x 2048 takes 41 and 104). */
struct NormShape { int elements, threads; };
static NormShape norm_shape(size_t width) {
    const int e = width <= 2048 ? 8 : width <= 8192 ? 16 : 32;
    return {e, (int)((width + e * 32 - 1) / (e * 32)) * 32};
}

/** Elements per access: 16 bytes, else a pair of 16-bit elements, else one (both directions with every part, 16384 x 1450 fp16: pairs 164 us,
 *  single elements 254; 4096 x 6002 bf16, a plain sum: 118 and 180). */
static int norm_run(int dtype, size_t width, std::initializer_list<const void*> all) {
    const int wide = dtype == 7 ? 4 : 8;
    if (width % wide == 0 && aligned_to(16, all)) return wide;
    return dtype != 7 && width % 2 == 0 && aligned_to(8, all) ? 2 : 1;
}

/** CTAs of the backward pass, all resident at once, and how the rows of a gate are cut among them. */
struct NormCut { size_t chunks, units; unsigned ctas; };
static NormCut norm_cut(int device, int dtype, size_t rows, size_t width, size_t gates, bool full) {
    const NormShape s = norm_shape(width);
    const bool wide = dtype == 7;
    const size_t shared = s.elements == 8    ? (full ? wide ? norm_grad_shared<float, 4, 8, BRANCH | FULL>(s.threads, (unsigned)width) : norm_grad_shared<__half, 8, 8, BRANCH | FULL>(s.threads, (unsigned)width)
                                                     : wide ? norm_grad_shared<float, 4, 8, 0>(s.threads, (unsigned)width) : norm_grad_shared<__half, 8, 8, 0>(s.threads, (unsigned)width))
                          : s.elements == 16 ? (full ? wide ? norm_grad_shared<float, 4, 16, BRANCH | FULL>(s.threads, (unsigned)width) : norm_grad_shared<__half, 8, 16, BRANCH | FULL>(s.threads, (unsigned)width)
                                                     : wide ? norm_grad_shared<float, 4, 16, 0>(s.threads, (unsigned)width) : norm_grad_shared<__half, 8, 16, 0>(s.threads, (unsigned)width))
                                             : 0;
    size_t per_sm = s.elements == 8 ? (full ? 768 : 1024) / s.threads : s.elements == 16 ? 512 / s.threads : 1;      // by registers
    if (per_sm * (shared + 1536) > 227 * 1024) per_sm = 227 * 1024 / (shared + 1536);
    const size_t want = (size_t)sm_count(device) * (per_sm ? per_sm : 1);
    if (!want) return {0, 0, 0};
    const size_t groups = gates ? gates : 1, rows_per = rows / groups;
    size_t chunks = (want + groups - 1) / groups;
    if (chunks > rows_per) chunks = rows_per;
    const size_t units = groups * chunks;
    return {chunks, units, (unsigned)(units < want ? units : want)};
}

template <typename T, int V, int E, int F> static cudaError_t norm_launch(unsigned grid, unsigned block, cudaStream_t stream, const NormArgs& a, int) {
    if constexpr (V * sizeof(T) == 16 && E == 16)       // with fewer elements it takes more registers, and 1 us longer at 16384 x 2048
        if (a.width == block * E) return launch_early(k_residual_norm<T, V, E, F, true>, grid, block, stream, a);
    return launch_early(k_residual_norm<T, V, E, F, false>, grid, block, stream, a);
}
template <typename T, int V, int E, int F, bool EXACT> static cudaError_t norm_grad_launch(unsigned grid, unsigned block, cudaStream_t stream, const NormGradArgs& a, int device) {
    const size_t shared = norm_grad_shared<T, V, E, F>(block, a.width);
    if (shared > 40 << 10) {        // 48 KB with the static part need no leave
        static std::atomic<bool> ready[64];
        if (!ready[device].load(std::memory_order_relaxed)) {
            const cudaError_t e = cudaFuncSetAttribute(k_residual_norm_grad<T, V, E, F, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024);
            if (e != cudaSuccess) return e;
            ready[device].store(true, std::memory_order_relaxed);
        }
    }
    return launch_early_shared(k_residual_norm_grad<T, V, E, F, EXACT>, grid, block, shared, stream, a);
}
template <typename T, int V, int E, int F> static cudaError_t norm_launch(unsigned grid, unsigned block, cudaStream_t stream, const NormGradArgs& a, int device) {
    if constexpr (V * sizeof(T) == 16 && E <= 16)
        if (a.width == block * E) return norm_grad_launch<T, V, E, F, true>(grid, block, stream, a, device);
    return norm_grad_launch<T, V, E, F, false>(grid, block, stream, a, device);
}
template <typename T, int V, int E, typename Args> static cudaError_t norm_form(int form, unsigned grid, unsigned block, cudaStream_t stream, const Args& a, int device) {
    switch (form) {
        case BRANCH: return norm_launch<T, V, E, BRANCH>(grid, block, stream, a, device);
        case BRANCH | SCALE: return norm_launch<T, V, E, BRANCH | SCALE>(grid, block, stream, a, device);
        case BRANCH | POST: return norm_launch<T, V, E, BRANCH | POST>(grid, block, stream, a, device);
        case BRANCH | GATE | SCALE: return norm_launch<T, V, E, BRANCH | GATE | SCALE>(grid, block, stream, a, device);
        case BRANCH | POST | GATE: return norm_launch<T, V, E, BRANCH | POST | GATE>(grid, block, stream, a, device);
        default: return norm_launch<T, V, E, 0>(grid, block, stream, a, device);
    }
}
/** Few terms in many columns take small CTAs (148 terms of 3 x 8192 columns: 10.9 -> 6.4 us), many terms large ones. */
template <typename T> static cudaError_t norm_columns(unsigned grid, cudaStream_t stream, const NormColumnArgs& c) {
    return (c.ctas > c.units ? c.ctas : c.units) <= 256 ? launch_early(k_norm_columns<T, 8>, grid, 32 * 8, stream, c) : launch_early(k_norm_columns<T, 32>, grid, 32 * 32, stream, c);
}

/** BRANCH, POST, GATE and SCALE of a call; post takes the scale in. */
static int norm_form_of(const void* branch, const void* post, const void* gate, double scale) {
    if (!branch) return 0;
    return BRANCH | (post ? POST : 0) | (gate ? GATE : 0) | (!post && (gate || scale != 1.0) ? SCALE : 0);
}

template <typename T, int V, typename Args> static cudaError_t norm_elements(int elements, int form, unsigned grid, unsigned block, cudaStream_t stream, const Args& a, int device) {
    return elements == 8 ? norm_form<T, V, 8>(form, grid, block, stream, a, device) : elements == 16 ? norm_form<T, V, 16>(form, grid, block, stream, a, device)
                                                                                                     : norm_form<T, V, 32>(form, grid, block, stream, a, device);
}

template <typename Args> static cudaError_t norm_dispatch(int device, int dtype, int run, int elements, int form, unsigned grid, unsigned block, cudaStream_t stream, const Args& a) {
    switch (dtype * 16 + run) {
        case 6 * 16 + 8: return norm_elements<__half, 8>(elements, form, grid, block, stream, a, device);
        case 6 * 16 + 2: return norm_elements<__half, 2>(elements, form, grid, block, stream, a, device);
        case 6 * 16 + 1: return norm_elements<__half, 1>(elements, form, grid, block, stream, a, device);
        case 9 * 16 + 8: return norm_elements<__nv_bfloat16, 8>(elements, form, grid, block, stream, a, device);
        case 9 * 16 + 2: return norm_elements<__nv_bfloat16, 2>(elements, form, grid, block, stream, a, device);
        case 9 * 16 + 1: return norm_elements<__nv_bfloat16, 1>(elements, form, grid, block, stream, a, device);
        case 7 * 16 + 4: return norm_elements<float, 4>(elements, form, grid, block, stream, a, device);
        case 7 * 16 + 1: return norm_elements<float, 1>(elements, form, grid, block, stream, a, device);
        default: return cudaErrorInvalidValue;
    }
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_residual_norm(int device, int dtype, size_t rows, size_t width, const void* x, const void* branch, const void* weight, const void* post,
                                  const void* gate, size_t rows_per_gate, int f32_vectors, double eps, double scale, void* y, void* n, void* rstd,
                                  void* rstd_post, void* stream) {
    if (!rows) return 0;
    if (!width || width > DCCL_NORM_MAX_WIDTH || rows > 0x7fffffffu || !x || !weight || !n || (branch && !y) || (gate && !rows_per_gate) || (post && !branch) || (gate && !branch))
        return report("dccl_residual_norm", cudaErrorInvalidValue);
    const NormArgs a = {x, branch, weight, post, gate, y, n, (float*)rstd, (float*)rstd_post, rows_per_gate, (unsigned)width, f32_vectors, (float)eps, (float)scale};
    const auto all = {x, branch, weight, post, gate, (const void*)y, (const void*)n};
    const NormShape s = norm_shape(width);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report("dccl_residual_norm", on.e);
    return report("dccl_residual_norm", norm_dispatch(device, dtype, norm_run(dtype, width, all), s.elements, norm_form_of(branch, post, gate, scale),
                                                      (unsigned)rows, (unsigned)s.threads, (cudaStream_t)stream, a));
}

extern "C" size_t dccl_residual_norm_workspace(int device, int dtype, size_t rows, size_t width, size_t gates, int has_post, int full) {
    if (!rows || !width || (gates && rows % gates)) return 0;
    const NormCut cut = norm_cut(device, dtype, rows, width, gates, full != 0);
    return (cut.ctas + (has_post || gates ? cut.units : 0)) * width * sizeof(float);
}

extern "C" int dccl_residual_norm_backward(int device, int dtype, size_t rows, size_t width, const void* dy, const void* dn, const void* x, const void* branch,
                                           const void* weight, const void* post, const void* gate, size_t rows_per_gate, int f32_vectors, double scale,
                                           const void* rstd, const void* rstd_post, void* dx, void* dbranch, void* dweight, void* dpost, void* dgate,
                                           void* workspace, size_t workspace_bytes, void* stream_v) {
    const char* who = "dccl_residual_norm_backward";
    const size_t gates = gate && rows_per_gate ? rows / rows_per_gate : 0;
    if (!rows || rows > 0x7fffffffu || !width || width > DCCL_NORM_MAX_WIDTH || (gate && (!gates || gates * rows_per_gate != rows)) || (post && (!branch || !rstd_post)) || (gate && !branch) || (dn && !rstd)
        || !x || !weight || !dx || !workspace || (dbranch && !branch) || (!dbranch && branch && (post || gate || scale != 1.0)))
        return report(who, cudaErrorInvalidValue);
    const bool full = branch != nullptr;
    const NormCut cut = norm_cut(device, dtype, rows, width, gates, full);
    const size_t blocks = (width + 31) / 32, vectors = (dn && dweight ? 1 : 0) + (post && dpost ? 1 : 0) + (gate && dgate ? gates : 0);
    if (!cut.units || blocks * vectors > 0x7fffffffu || workspace_bytes < dccl_residual_norm_workspace(device, dtype, rows, width, gates, post != nullptr, full))
        return report(who, cudaErrorInvalidValue);
    float* const weight_sums = (float*)workspace;
    float* const branch_sums = (post && dpost) || (gate && dgate) ? weight_sums + (size_t)cut.ctas * width : nullptr;
    const NormGradArgs a = {dy, dn, x, branch, weight, post, gate, (const float*)rstd, (const float*)rstd_post, dx, dbranch,
                            dn && dweight ? weight_sums : nullptr, branch_sums,
                            rows, gate ? rows_per_gate : rows, Divisor((unsigned)cut.chunks), (unsigned)((gate ? rows_per_gate : rows) / cut.chunks),
                            (unsigned)((gate ? rows_per_gate : rows) % cut.chunks), (unsigned)cut.units, (unsigned)width, f32_vectors, (float)scale};
    const auto all = {dy, dn, x, branch, weight, post, gate, (const void*)dx, (const void*)dbranch};
    const NormShape s = norm_shape(width);
    cudaStream_t stream = (cudaStream_t)stream_v;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    const int form = norm_form_of(branch, post, gate, scale) | (dbranch && !post ? SCALE : 0);       // a plain sum has no array of its own for the branch
    cudaError_t e = norm_dispatch(device, dtype, norm_run(dtype, width, all), s.elements, form, cut.ctas, (unsigned)s.threads, stream, a);
    if (e == cudaSuccess && vectors) {
        const NormColumnArgs c = {weight_sums, branch_sums, post, gate, dn ? dweight : nullptr, post ? dpost : nullptr, gate ? dgate : nullptr, Divisor((unsigned)cut.chunks),
                                  Divisor((unsigned)blocks), cut.ctas, (unsigned)cut.units, (unsigned)width, f32_vectors, (float)scale};
        const unsigned grid = (unsigned)(blocks * vectors);
        e = dtype == 6 ? norm_columns<__half>(grid, stream, c) : dtype == 7 ? norm_columns<float>(grid, stream, c) : norm_columns<__nv_bfloat16>(grid, stream, c);
    }
    return report(who, e);
}
