/**
 * The norm of all gradients of a model, n = sqrt(sum of g^2 over all tensors), and the gradients times min(1, limit / (n + 1e-6))
 *
 * One launch reads every tensor: their addresses and sizes come as the kernel's parameters, which a graph keeps, and each CTA takes pieces of them in turn. A
 * second one adds the CTAs' sums, every CTA for itself, and scales; where the norm is within the limit and the gradients stay where they are, it ends
 * there. HBM bounds both: one pass to know the norm, then one in and one out. The second goes through the tensors backwards, as what was read last is still in L2.
 */
#include "grad_norm.hpp"
#include "../kernels/launch_early.cuh"
#include "../decoder/row_access.cuh"
#include <type_traits>

namespace dccl {

/**
 * The largest piece is what a CTA has in flight at once. 1.1 billion bf16 gradients, norm and scaled copy: 337 + 680 us (6.5 TB/s both). Pieces of 64 KB read in two steps
 * by four CTAs of an SM took 337 + 722, of 16 KB by 32 CTAs 392 + 696: reading alone likes few CTAs that go on, reading and writing many. Where all of it fits into L2,
 * and where nothing has to be written, what counts is how soon the last CTA has started: 17 M gradients within the limit, 12.5 us with four for both and 15.3 with 32.
 */
constexpr int kClipThreads = 256, kClipUnroll = 8, kFewCtas = 4, kManyCtas = 32;
constexpr unsigned long long kManyBytes = 64ull << 20;
constexpr size_t kMaxPiece = 32 * 1024, kMinPiece = 4 * 1024;
constexpr int kManyTensors = 512, kSomeTensors = 120, kFewTensors = 24;

enum { TYPE_HALF = 0, TYPE_BF16 = 1, TYPE_FLOAT = 2, TYPE_TO_FLOAT = 4 };      // of a tensor; TO_FLOAT: what is written is fp32

template <int MOST> struct Tensors {
    const void* in[MOST];
    void* out[MOST];
    unsigned long long elements[MOST];
    unsigned first[MOST + 1];               // the number of a tensor's first piece, and of all pieces
    unsigned char type[MOST];
    int count;
    unsigned piece;                         // bytes of one piece, as it is read
};

struct ClipArgs { const double* parts; size_t count; double limit; float* norm; };

/** The tensor that a piece belongs to. */
template <int MOST> __device__ __forceinline__ int tensor_of(const Tensors<MOST>& t, unsigned piece) {
    int low = 0, high = t.count;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (t.first[mid] <= piece) low = mid;
        else high = mid;
    }
    return low;
}

/** The sum over the CTA in thread 0, in a fixed order. */
__device__ __forceinline__ double cta_sum(double v, double* parts) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < kClipThreads / 32; w++) v += parts[w];
    return v;
}

/** Elements before the first 16-byte boundary behind p, at most n. */
template <typename T> __device__ __forceinline__ size_t before_boundary(const T* p, size_t n) {
    const size_t head = (16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T);
    return head < n ? head : n;
}

/** Squares of this thread's accesses in 64 bits. A function of its own: it is seldom called, and its registers are not the other's. */
template <typename T> __device__ __noinline__ double squares_exactly(const T* body, size_t runs) {
    constexpr int N = 16 / sizeof(T);
    double sum = 0;
    for (size_t i = threadIdx.x; i < runs; i += kClipThreads) {
        const Run<T, N> v = ld_run<T, N>(body + i * N);
#pragma unroll
        for (int e = 0; e < N; e++) sum = fma((double)Traits<T>::up(v.e[e]), (double)Traits<T>::up(v.e[e]), sum);
    }
    return sum;
}

/**
 * Squares of one access are added in fp32, and those sums in 64 bits. A square that overflowed shows in the thread's sum for the piece; what got lost below the normal numbers, 2^-150 of
 * each of at most 64 squares, may count where that sum is below 2^-110 (the 2^34th of it no longer does) without being of zeros alone, as many gradients are. Then the thread adds
 * all of its squares of the piece again, in 64 bits.
 * (1.1 billion bf16 gradients take 335 us; where each access was looked at 340, where it was decided there 404, and without any of it 330. Half as many, all of them to be added
 * again, 258 instead of 169.) Those of fp16 always fit.
 */
template <typename T> __device__ __forceinline__ double squares(const T* p, size_t n) {
    constexpr int N = 16 / sizeof(T);
    const size_t head = before_boundary(p, n), runs = (n - head) / N;
    double sum = 0;
    constexpr bool kMayNotFit = !std::is_same<T, __half>::value;
    uint32_t bits = 0;
    const T* body = p + head;
    size_t i = threadIdx.x;
    const auto some = [&](auto count) {         // as many at a time, while all of them are there
        constexpr int U = decltype(count)::value;
        for (; i + (U - 1) * kClipThreads < runs; i += U * kClipThreads) {
            Run<T, N> v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = ld_run<T, N>(body + (i + u * kClipThreads) * N);
#pragma unroll
            for (int u = 0; u < U; u++) {
                float s = 0;
#pragma unroll
                for (int e = 0; e < N; e++) s = fmaf(Traits<T>::up(v[u].e[e]), Traits<T>::up(v[u].e[e]), s);
                sum += s;
                if constexpr (kMayNotFit) {
                    const uint32_t* const w = reinterpret_cast<const uint32_t*>(&v[u]);
                    bits |= w[0] | w[1] | w[2] | w[3];
                }
            }
        }
    };
    some(std::integral_constant<int, kClipUnroll>{});
    some(std::integral_constant<int, kClipUnroll / 2>{});
    some(std::integral_constant<int, 1>{});
    if constexpr (kMayNotFit) {
        constexpr uint32_t sizes = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;         // without the signs
        if (!(sum < INFINITY) || (sum < 0x1p-110 && (bits & sizes))) sum = squares_exactly(body, runs);
    }
    if (threadIdx.x < head) {
        const float v = Traits<T>::up(p[threadIdx.x]);
        sum += (double)v * v;
    }
    for (size_t j = head + runs * N + threadIdx.x; j < n; j += kClipThreads) {
        const float v = Traits<T>::up(p[j]);
        sum += (double)v * v;
    }
    return sum;
}

template <int MOST> __global__ void __launch_bounds__(kClipThreads) k_grad_squares(const __grid_constant__ Tensors<MOST> t, double* parts) {
    wait_for_stream();
    __shared__ double shared[kClipThreads / 32];
    double sum = 0;
    for (unsigned piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
        const int i = tensor_of(t, piece);
        const int type = t.type[i] & 3;
        const size_t per = t.piece / (type == TYPE_FLOAT ? 4 : 2), from = (size_t)(piece - t.first[i]) * per, n = t.elements[i] - from < per ? t.elements[i] - from : per;
        if (type == TYPE_HALF) sum += squares(reinterpret_cast<const __half*>(t.in[i]) + from, n);
        else if (type == TYPE_BF16) sum += squares(reinterpret_cast<const __nv_bfloat16*>(t.in[i]) + from, n);
        else sum += squares(reinterpret_cast<const float*>(t.in[i]) + from, n);
    }
    sum = cta_sum(sum, shared);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

/** The sum of the parts, in every thread. */
__device__ __forceinline__ double total_of(const double* parts, size_t count) {
    __shared__ double shared[kClipThreads / 32];
    __shared__ double total;
    double sum = 0;
    for (size_t i = threadIdx.x; i < count; i += kClipThreads) sum += parts[i];
    sum = cta_sum(sum, shared);
    if (threadIdx.x == 0) total = sum;
    __syncthreads();
    return total;
}

__global__ void __launch_bounds__(kClipThreads) k_grad_total(const double* parts, size_t count, double* total, float* norm) {
    wait_for_stream();
    const double sum = total_of(parts, count);
    if (threadIdx.x) return;
    if (total) *total = sum;
    if (norm) *norm = (float)sqrt(sum);
}

template <typename T, typename O> __device__ __forceinline__ void scale(const T* p, O* out, size_t n, float factor) {
    constexpr int N = 16 / sizeof(T);
    const size_t head = before_boundary(p, n);
    size_t done = 0;
    if (reinterpret_cast<uintptr_t>(out + head) % 16 == 0) {
        const size_t runs = (n - head) / N;
        if (threadIdx.x < head) out[threadIdx.x] = Traits<O>::down(factor * Traits<T>::up(p[threadIdx.x]));
        const T* body = p + head;
        O* to = out + head;
        const auto store = [&](size_t i, const Run<T, N>& v) {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = factor * Traits<T>::up(v.e[e]);
            if constexpr (sizeof(O) == sizeof(T)) st_run<O, N>(to + i * N, round_run<O, N>(f));
            else
#pragma unroll
                for (int h = 0; h < N; h += 4) st_run<O, 4>(to + i * N + h, Run<O, 4>{f[h], f[h + 1], f[h + 2], f[h + 3]});
        };
        size_t i = threadIdx.x;
        const auto some = [&](auto count) {
            constexpr int U = decltype(count)::value;
            for (; i + (U - 1) * kClipThreads < runs; i += U * kClipThreads) {
                Run<T, N> v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = ld_run<T, N>(body + (i + u * kClipThreads) * N);
#pragma unroll
                for (int u = 0; u < U; u++) store(i + u * kClipThreads, v[u]);
            }
        };
        some(std::integral_constant<int, kClipUnroll>{});
        some(std::integral_constant<int, kClipUnroll / 2>{});
        some(std::integral_constant<int, 1>{});
        done = head + runs * N;
    }
    for (size_t j = done + threadIdx.x; j < n; j += kClipThreads) out[j] = Traits<O>::down(factor * Traits<T>::up(p[j]));
}

template <int MOST> __global__ void __launch_bounds__(kClipThreads) k_grad_clip(const __grid_constant__ Tensors<MOST> t, const __grid_constant__ ClipArgs a) {
    wait_for_stream();
    const double norm = sqrt(total_of(a.parts, a.count)), of = a.limit / (norm + 1e-6);
    const float factor = of >= 1.0 ? 1.0f : (float)of;          // NaN stays
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm) *a.norm = (float)norm;
    const unsigned pieces = t.first[t.count];
    for (unsigned k = blockIdx.x; k < pieces; k += gridDim.x) {
        const unsigned piece = pieces - 1 - k;
        const int i = tensor_of(t, piece);
        if (factor == 1.0f && t.in[i] == t.out[i]) continue;
        const int type = t.type[i];
        const size_t per = t.piece / ((type & 3) == TYPE_FLOAT ? 4 : 2), from = (size_t)(piece - t.first[i]) * per, n = t.elements[i] - from < per ? t.elements[i] - from : per;
        const void* in = t.in[i];
        void* out = t.out[i];
        if (type == TYPE_HALF) scale(reinterpret_cast<const __half*>(in) + from, reinterpret_cast<__half*>(out) + from, n, factor);
        else if (type == TYPE_BF16) scale(reinterpret_cast<const __nv_bfloat16*>(in) + from, reinterpret_cast<__nv_bfloat16*>(out) + from, n, factor);
        else if (type == (TYPE_HALF | TYPE_TO_FLOAT)) scale(reinterpret_cast<const __half*>(in) + from, reinterpret_cast<float*>(out) + from, n, factor);
        else if (type == (TYPE_BF16 | TYPE_TO_FLOAT)) scale(reinterpret_cast<const __nv_bfloat16*>(in) + from, reinterpret_cast<float*>(out) + from, n, factor);
        else scale(reinterpret_cast<const float*>(in) + from, reinterpret_cast<float*>(out) + from, n, factor);
    }
}

/* ---- host side ---- */

static size_t size_of(int dtype) { return dtype == 7 ? 4 : dtype == 6 || dtype == 9 ? 2 : 0; }

/** How one launch cuts its tensors: at most kManyTensors of them. */
struct ClipPlan { unsigned pieces, piece, read_ctas, scale_ctas; };

/** Pieces so small that every SM gets several, but not below 4 KB, which a CTA reads in one access per thread. */
static bool plan_clip(int device, size_t tensors, const DcclGradient* t, ClipPlan& p) {
    const int sms = sm_count(device);
    if (!sms || !tensors || tensors > kManyTensors) return false;
    unsigned long long bytes = 0;
    for (size_t i = 0; i < tensors; i++) {
        const size_t size = size_of(t[i].dtype);
        if (!size || (t[i].out_dtype != t[i].dtype && t[i].out_dtype != 7) || !t[i].in || t[i].elements >= DCCL_GRADIENTS_MAX
            || reinterpret_cast<uintptr_t>(t[i].in) % size || reinterpret_cast<uintptr_t>(t[i].out) % size_of(t[i].out_dtype))
            return false;
        bytes += t[i].elements * size;
    }
    size_t piece = kMaxPiece;
    while (piece > kMinPiece && bytes / piece < 8ull * sms) piece /= 2;
    while (bytes / piece > 1ull << 30) piece *= 2;
    unsigned long long pieces = 0;
    for (size_t i = 0; i < tensors; i++) pieces += (t[i].elements * size_of(t[i].dtype) + piece - 1) / piece;
    p.piece = (unsigned)piece;
    p.pieces = (unsigned)pieces;
    const auto within = [&](unsigned room) { return p.pieces < room ? (p.pieces ? p.pieces : 1) : room; };
    p.read_ctas = within(kFewCtas * sms);
    p.scale_ctas = within((bytes < kManyBytes ? kFewCtas : kManyCtas) * sms);
    return true;
}

template <int MOST> static void fill(Tensors<MOST>& s, size_t tensors, const DcclGradient* t, const ClipPlan& p) {
    unsigned at = 0;
    for (size_t i = 0; i < tensors; i++) {
        s.in[i] = t[i].in;
        s.out[i] = t[i].out;
        s.elements[i] = t[i].elements;
        s.first[i] = at;
        s.type[i] = (unsigned char)((t[i].dtype == 6 ? TYPE_HALF : t[i].dtype == 9 ? TYPE_BF16 : TYPE_FLOAT) | (t[i].dtype != 7 && t[i].out_dtype == 7 ? TYPE_TO_FLOAT : 0));
        at += (unsigned)((t[i].elements * size_of(t[i].dtype) + p.piece - 1) / p.piece);
    }
    s.first[tensors] = at;
    s.count = (int)tensors;
    s.piece = p.piece;
}

template <int MOST> static cudaError_t run_squares(size_t tensors, const DcclGradient* t, const ClipPlan& p, double* parts, cudaStream_t stream) {
    Tensors<MOST> s;
    fill(s, tensors, t, p);
    return launch_early_shared(k_grad_squares<MOST>, p.read_ctas, kClipThreads, 0, stream, s, parts);
}
template <int MOST> static cudaError_t run_clip(size_t tensors, const DcclGradient* t, const ClipPlan& p, const ClipArgs& a, cudaStream_t stream) {
    Tensors<MOST> s;
    fill(s, tensors, t, p);
    return launch_early_shared(k_grad_clip<MOST>, p.scale_ctas, kClipThreads, 0, stream, s, a);
}

} // namespace dccl

using namespace dccl;

extern "C" size_t dccl_grad_parts(int device, size_t tensors, const DcclGradient* t) {
    size_t parts = 0;
    for (size_t i = 0; i < tensors; i += kManyTensors) {
        ClipPlan p;
        if (!plan_clip(device, tensors - i < kManyTensors ? tensors - i : kManyTensors, t + i, p)) return 0;
        parts += p.read_ctas;
    }
    return parts;
}

extern "C" int dccl_grad_squares(int device, size_t tensors, const DcclGradient* t, double* parts, void* stream) {
    const char* who = "dccl_grad_squares";
    if (!tensors || !t || !parts) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    for (size_t i = 0; i < tensors; i += kManyTensors) {
        const size_t n = tensors - i < kManyTensors ? tensors - i : kManyTensors;
        ClipPlan p;
        if (!plan_clip(device, n, t + i, p)) return report(who, cudaErrorInvalidValue);
        const cudaError_t e = (n <= kFewTensors ? run_squares<kFewTensors> : n <= kSomeTensors ? run_squares<kSomeTensors> : run_squares<kManyTensors>)(n, t + i, p, parts, (cudaStream_t)stream);
        if (e != cudaSuccess) return report(who, e);
        parts += p.read_ctas;
    }
    return 0;
}

extern "C" int dccl_grad_total(int device, const double* parts, size_t count, double* total, float* norm, void* stream) {
    const char* who = "dccl_grad_total";
    if (!parts && count) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    return report(who, launch_early(k_grad_total, 1, kClipThreads, (cudaStream_t)stream, parts, count, total, norm));
}

extern "C" int dccl_grad_clip(int device, size_t tensors, const DcclGradient* t, const double* parts, size_t count, double limit, float* norm, void* stream) {
    const char* who = "dccl_grad_clip";
    if (!tensors || !t || !parts || !(limit >= 0)) return report(who, cudaErrorInvalidValue);
    OnDevice on(device);
    if (on.e != cudaSuccess) return report(who, on.e);
    for (size_t i = 0; i < tensors; i += kManyTensors) {
        const size_t n = tensors - i < kManyTensors ? tensors - i : kManyTensors;
        ClipPlan p;
        if (!plan_clip(device, n, t + i, p)) return report(who, cudaErrorInvalidValue);
        for (size_t j = 0; j < n; j++)
            if (!t[i + j].out) return report(who, cudaErrorInvalidValue);
        const ClipArgs a = {parts, count, limit, norm};
        const cudaError_t e = (n <= kFewTensors ? run_clip<kFewTensors> : n <= kSomeTensors ? run_clip<kSomeTensors> : run_clip<kManyTensors>)(n, t + i, p, a, (cudaStream_t)stream);
        if (e != cudaSuccess) return report(who, e);
    }
    return 0;
}
