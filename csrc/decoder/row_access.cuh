/**
 * What the kernels over rows of activations share: short runs of elements as one access, their conversion, sums over a CTA, and
 * launches on a device that need not be the current one.
 */
#pragma once
#include "../device/reduce_ops.cuh"
#include <atomic>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

namespace dccl {

/** N elements moved by one access. */
template <typename T, int N> struct alignas(sizeof(T) * N) Run { T e[N]; };

template <typename T, int N> __device__ __forceinline__ Run<T, N> ld_run(const T* p) { return *reinterpret_cast<const Run<T, N>*>(p); }
template <typename T, int N> __device__ __forceinline__ void st_run(T* p, const Run<T, N>& v) { *reinterpret_cast<Run<T, N>*>(p) = v; }

/** Elements [i, i + N) of a vector that is of type T, or fp32. */
template <typename T, int N> __device__ __forceinline__ void ld_vector(float (&f)[N], const void* p, bool f32, size_t i) {
    if (f32) {
        if constexpr (N * sizeof(float) <= 16) {
            const Run<float, N> r = ld_run<float, N>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = r.e[e];
        } else {
#pragma unroll
            for (int k = 0; k < N; k += 4) {
                const Run<float, 4> r = ld_run<float, 4>(reinterpret_cast<const float*>(p) + i + k);
#pragma unroll
                for (int e = 0; e < 4; e++) f[k + e] = r.e[e];
            }
        }
    } else {
        const Run<T, N> r = ld_run<T, N>(reinterpret_cast<const T*>(p) + i);
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = Traits<T>::up(r.e[e]);
    }
}

/** N fp32 values, rounded to T: 16-bit types two at a time. */
template <typename T, int N> __device__ __forceinline__ Run<T, N> round_run(const float (&f)[N]) {
    Run<T, N> r;
    if constexpr (N % 2 == 0 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int e = 0; e < N; e += 2) *reinterpret_cast<__nv_bfloat162*>(&r.e[e]) = __floats2bfloat162_rn(f[e], f[e + 1]);
    } else if constexpr (N % 2 == 0 && std::is_same<T, __half>::value) {
#pragma unroll
        for (int e = 0; e < N; e += 2) *reinterpret_cast<__half2*>(&r.e[e]) = __floats2half2_rn(f[e], f[e + 1]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) r.e[e] = Traits<T>::down(f[e]);
    }
    return r;
}

/** The sum over the CTA, in every thread and in a fixed order. `parts`: 32 aligned words of shared memory that no other call uses until
 *  every thread has passed a barrier after this one. */
__device__ __forceinline__ float cta_sum(float v, float* parts) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const unsigned warps = blockDim.x / 32;
    if (warps == 1) return v;
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = v;
    if (threadIdx.x < 4 && warps % 4 && threadIdx.x >= warps % 4) parts[warps / 4 * 4 + threadIdx.x] = 0.0f;      // up to a multiple of four
    __syncthreads();
    v = 0;
    for (unsigned w = 0; w < warps; w += 4) {
        const float4 p = *reinterpret_cast<const float4*>(parts + w);
        v += (p.x + p.y) + (p.z + p.w);
    }
    return v;
}

/**
 * Division of n < 2^31 by a number that the host knows: n / d = (n m) >> (32 + s) with m = ceil(2^(32 + s) / d) and 2^s >= d > 2^(s - 1), which is
 * right as n times the excess of m over the quotient (below d / d) stays under 2^31 (Granlund and Montgomery, "Division by Invariant Integers using
 * Multiplication"). m takes 33 bits; its highest is added as n.
 */
struct Divisor {
    unsigned d, m, s;
    Divisor() = default;
    explicit Divisor(unsigned divisor) : d(divisor), s(0) {
        while (s < 31 && (1u << s) < d) s++;
        m = (unsigned)((((uint64_t)1 << (32 + s)) + d - 1) / d - ((uint64_t)1 << 32));
    }
    __host__ __device__ __forceinline__ unsigned quotient(unsigned n) const {
#ifdef __CUDA_ARCH__
        return (__umulhi(n, m) + n) >> s;
#else
        return ((unsigned)((uint64_t)n * m >> 32) + n) >> s;
#endif
    }
};

/** Makes `device` current for as long as it lives. */
class OnDevice {
public:
    explicit OnDevice(int device) : device_(device) {
        e = cudaGetDevice(&prev_);
        if (e == cudaSuccess && prev_ != device) e = cudaSetDevice(device);
    }
    ~OnDevice() { if (prev_ >= 0 && prev_ != device_) cudaSetDevice(prev_); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    cudaError_t e;

private:
    int device_, prev_ = -1;
};

/** SMs of a device, asked once; 0 after an error. */
inline int sm_count(int device) {
    static std::atomic<int> known[64];
    if (device < 0 || device >= 64) return 0;
    int n = known[device].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { cudaGetLastError(); return 0; }
        known[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

inline int report(const char* who, cudaError_t e) {
    if (e == cudaSuccess) return 0;
    fprintf(stderr, "%s: %s\n", who, cudaGetErrorString(e));
    cudaGetLastError();
    return -1;
}

inline bool aligned_to(size_t bytes, std::initializer_list<const void*> ps) {
    uintptr_t low = 0;
    for (const void* p : ps) low |= reinterpret_cast<uintptr_t>(p);
    return low % bytes == 0;
}

} // namespace dccl
