/**
 * Entry points of the norm of many tensors and of their scaling to a limit (grad_norm.cu). Pointers inside are device memory of `device`, and the work goes to
 * `stream`. They return 0, or -1 after a message on stderr.
 */
#pragma once
#include <cstddef>

/** A dense tensor: `in` is read, `out` written (the same, or another one that does not overlap any); dtype and out_dtype are ncclDataType_t (float16, float32 or
 *  bfloat16), out_dtype dtype or float32. */
struct DcclGradient { const void* in; void* out; size_t elements; int dtype, out_dtype; };

/** All elements of a call, over all its tensors. */
enum : unsigned long long { DCCL_GRADIENTS_MAX = 1ull << 44 };

extern "C" {

/** Sums of squares (double) that dccl_grad_squares leaves for these tensors; 0 after an error. */
size_t dccl_grad_parts(int device, size_t tensors, const DcclGradient* t);

/** Sums of squares of all elements, parts [dccl_grad_parts] of them, in an order that depends on sizes, types and addresses only. */
int dccl_grad_squares(int device, size_t tensors, const DcclGradient* t, double* parts, void* stream);

/** total (double) and norm (float) of the parts; either may be null. */
int dccl_grad_total(int device, const double* parts, size_t count, double* total, float* norm, void* stream);

/** out = in * min(1, limit / (norm + 1e-6)), rounded once, with the norm that the parts give, which `norm` (float, may be null) receives. Where nothing changes, an
 *  `out` that is its `in` is not touched. */
int dccl_grad_clip(int device, size_t tensors, const DcclGradient* t, const double* parts, size_t count, double limit, float* norm, void* stream);

} // extern "C"
