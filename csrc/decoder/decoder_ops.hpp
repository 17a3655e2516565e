/**
 * Entry points of the operators of a decoder block (residual_norm.cu, rotary.cu, gated_linear.cu). All pointers are device
 * memory of `device`, dtype is an ncclDataType_t (float16, float32 or bfloat16), and the work goes to `stream`. They return 0, or
 * -1 after a message on stderr.
 */
#pragma once
#include <cstddef>
#include <cstdint>

/** What the entry points take, and with them dccl_b200/ops/decoder.py: elements of a row, pairs of a head, elements of a token, and each dimension of
 *  a gated layer below. */
enum { DCCL_NORM_MAX_WIDTH = 32768, DCCL_ROTARY_MAX_PAIRS = 1024, DCCL_ROTARY_MAX_TOKEN = 1 << 24, DCCL_GATED_MAX_DIMENSION = 1 << 30 };

/** Which of the vectors of a norm are fp32 and not of the activations' type. */
enum { DCCL_NORM_WEIGHT_F32 = 1, DCCL_NORM_POST_F32 = 2, DCCL_NORM_GATE_F32 = 4 };

extern "C" {

/**
 * y = x + scale * gate .* p with p = branch, or rms_norm(branch) .* post where post is given; n = rms_norm(y) .* weight. rows x width,
 * rows in a row. Row r uses row r / rows_per_gate of the gate. Without a branch, n = rms_norm(x) .* weight and y is not
 * written. rstd and rstd_post (fp32, one per row) may be null, gate and post too.
 */
int dccl_residual_norm(int device, int dtype, size_t rows, size_t width, const void* x, const void* branch, const void* weight, const void* post,
                       const void* gate, size_t rows_per_gate, int f32_vectors, double eps, double scale, void* y, void* n, void* rstd, void* rstd_post,
                       void* stream);

/** Bytes of workspace that the backward pass of `gates` rows of gates (0: without a gate) takes; 0 after an error. full: with a branch. */
size_t dccl_residual_norm_workspace(int device, int dtype, size_t rows, size_t width, size_t gates, int has_post, int full);

/**
 * Gradients of dccl_residual_norm: from dy and dn (either may be null) those of x and branch, and in the vectors' own types those of
 * weight, post and gate. dbranch may be null where it equals dx (scale 1, no post, no gate), and is written wherever it is not. No atomics:
 * the same inputs give the same gradients.
 */
int dccl_residual_norm_backward(int device, int dtype, size_t rows, size_t width, const void* dy, const void* dn, const void* x, const void* branch,
                                const void* weight, const void* post, const void* gate, size_t rows_per_gate, int f32_vectors, double scale,
                                const void* rstd, const void* rstd_post, void* dx, void* dbranch, void* dweight, void* dpost, void* dgate,
                                void* workspace, size_t workspace_bytes, void* stream);

/** A tensor [batch, seq, heads, head dim] by its strides in elements; the head dim is dense. */
struct DcclHeads { const void* in; void* out; long long in_batch, in_seq, in_head, out_batch, out_seq, out_head; int heads; };

/**
 * Turns pair j of every head of q and k (heads 0: not given) by positions * freqs[j] radians, or back where `back`, and scales it; what
 * lies behind the pairs is copied. Pair j is (j, pairs + j), or (2j, 2j + 1) where `interleaved`. positions: int64 or int32 with
 * the strides pos_batch and pos_seq, or null for first + index in the sequence.
 */
int dccl_rotary(int device, int dtype, size_t batch, size_t seq, int head_dim, int pairs, int interleaved, int back, const DcclHeads* q, const DcclHeads* k,
                const double* freqs, const void* positions, int positions64, long long pos_batch, long long pos_seq, long long first, double scale, void* stream);

/** Activations of a gated linear layer. */
enum { DCCL_ACT_SILU = 0, DCCL_ACT_GELU = 1, DCCL_ACT_GELU_TANH = 2 };

/** Bytes of workspace that a call of these sizes takes (0 as well); -1 after an error. `aligned`: every operand starts on 16 bytes. */
long long dccl_gated_linear_workspace(int device, size_t tokens, size_t width, size_t ffn, int aligned, int backward);

/**
 * h = act(x Wg^T) .* (x Wu^T): x [tokens][width], Wg and Wu [ffn][width], h [tokens][ffn], all dense and of dtype float16 or bfloat16.
 * Where g and u are not null they receive the two products in fp32, in rows of pre_stride elements (a multiple of four). A product that does
 * not end in time leaves NaN, and no later call on its device starts one.
 */
int dccl_gated_linear(int device, int dtype, size_t tokens, size_t width, size_t ffn, const void* x, const void* w_gate, const void* w_up, int act, void* h,
                      float* g, float* u, size_t pre_stride, void* workspace, long long workspace_bytes, void* stream);

/** Whether the backward pass of these operands needs the workspace of the forward pass, which holds copies of them in rows that start on 16 bytes. */
int dccl_gated_linear_pads(size_t width, int aligned);

/** Its gradients from dh and the products that it left. Each of dx, and dw_gate with dw_up, may be null. No atomics. */
int dccl_gated_linear_backward(int device, int dtype, size_t tokens, size_t width, size_t ffn, const void* dh, const float* g, const float* u, size_t pre_stride,
                               const void* x, const void* w_gate, const void* w_up, const void* forward_workspace, int act, void* dx, void* dw_gate, void* dw_up,
                               void* workspace, long long workspace_bytes, void* stream);

} // extern "C"
