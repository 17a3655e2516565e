/**
 * What the kernels of products on the tensor cores share: how the sums of a tile go from registers to rows in memory, the maps of their operands, and the flag
 * of a wait that ran out.
 */
#pragma once
#include "row_access.cuh"
#include "../device/tcgen05.cuh"
#include "../gpu/driver_api.hpp"
#include <cstring>

namespace dccl {

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
            const float f[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
            if (r < rows && 8 * c < columns) st_run<T, 8>(to + (size_t)r * stride + 8 * c, round_run<T, 8>(f));
        }
    } else if (lane < columns) {
#pragma unroll 4
        for (int r = 0; r < rows && r < 32; r++)
            to[(size_t)r * stride + lane] = Traits<T>::down(*reinterpret_cast<const float*>(stage + r * 128 + (((lane / 4) ^ (r & 7)) * 16) + lane % 4 * 4));
    }
}

/** Set by a kernel whose wait ran out, which leaves NaN in what it was to store; looked at by the next call on the device. Host memory that the device
 *  writes, for the life of the process. */
inline int* gave_up_flag(int device) {
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

/** An operand by its dimensions, the contiguous one first, the strides of the others in elements, and the box of it. */
inline cudaError_t make_map(CUtensorMap* map, int dtype, const void* base, int rank, const size_t (&size)[4], const size_t (&stride)[3], const unsigned (&box_of)[4]) {
    const DriverApi* d = driver_api(nullptr);
    if (!d || !d->TensorMapEncodeTiled) return cudaErrorNotSupported;
    const cuuint64_t dims[4] = {size[0], size[1], size[2], size[3]}, strides[3] = {stride[0] * 2, stride[1] * 2, stride[2] * 2};
    const cuuint32_t box[4] = {box_of[0], box_of[1], box_of[2], box_of[3]}, steps[4] = {1, 1, 1, 1};
    const auto encode = [&] {
        return d->TensorMapEncodeTiled(map, dtype == 6 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, steps,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {      // the thread's first call of CUDA: the runtime has its device, but no context current yet
        int device = 0;
        if (cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = encode();
    }
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
inline cudaError_t make_map(CUtensorMap* map, int dtype, const void* base, size_t inner, size_t outer, size_t stride, unsigned box_outer) {
    return make_map(map, dtype, base, 2, {inner, outer, 1, 1}, {stride, 0, 0}, {64, box_outer, 1, 1});
}

inline bool gave_up(const char* who, int device) {
    const int* flag = gave_up_flag(device);
    if (!flag || !*reinterpret_cast<const volatile int*>(flag)) return false;
    fprintf(stderr, "%s: an earlier product of this process on device %d did not end in time; what it did not finish is NaN, and no other is started there\n", who, device);
    return true;
}

} // namespace dccl
