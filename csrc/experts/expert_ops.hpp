/**
 * Entry points of the operators of a mixture of experts (route.cu, exchange.cu, grouped.cu). All pointers are device memory of `device`, dtype is an
 * ncclDataType_t (float16, float32 or bfloat16), and the work goes to `stream`. They return 0, or -1 after a message on stderr.
 */
#pragma once
#include <cstddef>
#include <cstdint>

/** What the entry points take, and with them dccl_b200/ops/experts.py: experts, experts of one token, groups of experts, elements of a row, and all
 *  places of a call (tokens x experts of a token). */
enum { DCCL_EXPERTS_MAX = 1024, DCCL_EXPERTS_MAX_CHOSEN = 32, DCCL_EXPERTS_MAX_GROUPS = 32, DCCL_EXPERTS_MAX_WIDTH = 1 << 20, DCCL_EXPERTS_MAX_PLACES = 1 << 30 };

/** How a token's experts are chosen, and their weights. */
struct DcclRouting {
    int sigmoid;                // scores: softmax over the experts, or a sigmoid of each
    int k, groups, top_groups;
    int top2;                   // a group's score: the sum of its two best, or its best
    int renormalize;
    float scale;
};

extern "C" {

/** weights and experts [tokens][k] from logits [tokens][experts] and, where it is not null, bias [experts]. */
int dccl_route(int device, int dtype, size_t tokens, int experts, const void* logits, const float* bias, const DcclRouting* how, float* weights, int* chosen, void* stream);

/** dlogits from dweights and what the forward pass chose. */
int dccl_route_backward(int device, int dtype, size_t tokens, int experts, const void* logits, const int* chosen, const float* dweights, const DcclRouting* how, void* dlogits,
                        void* stream);

/** Where each of `places` chosen experts (int32, or int64) goes in the order of the experts, places of one expert in their own order: rows [places] (-1 where
 *  the number is none of an expert), counts [experts], starts [experts + 1]. */
int dccl_expert_plan(int device, size_t places, int experts, const void* chosen, int chosen64, int* rows, int* counts, int* starts, void* stream);

/** out[rows[t][j]] = x[t], and zeros in the rows from *used up to tokens * k: each of those before has a place. With a null `used`, rows without a place are left as they are. */
int dccl_dispatch(int device, int dtype, size_t tokens, int k, size_t width, const void* x, const int* rows, const int* used, void* out, void* stream);

/** y[t] = sum over j of weights[t][j] * in[rows[t][j]], those with a row; weights (null: ones) are fp32, or of dtype. */
int dccl_combine(int device, int dtype, size_t tokens, int k, size_t width, const void* in, const int* rows, const void* weights, int weights32, void* y, void* stream);

/** Its gradients: din[rows[t][j]] = weights[t][j] * dy[t], zeros in the rows from *used on (null: as above), and dweights[t][j] = in[rows[t][j]] . dy[t]. Each may be null. */
int dccl_combine_backward(int device, int dtype, size_t tokens, int k, size_t width, const void* dy, const void* in, const int* rows, const int* used, const void* weights,
                          int weights32, void* din, void* dweights, void* stream);

/** Bytes of workspace that a call of these sizes takes (0 as well); -1 after an error. `aligned`: every operand starts on 16 bytes. */
long long dccl_expert_linear_workspace(int device, size_t rows, int experts, size_t width, size_t out, int aligned, int backward);

/** Whether the backward pass of these operands needs the workspace of the forward pass, which holds copies of them in rows that start on 16 bytes. */
int dccl_expert_linear_pads(size_t width, int aligned);

/**
 * h[r] = act(x[r] W[e]^T) for the rows r from starts[e] to starts[e + 1], and zeros in the rows before starts[0] and from starts[experts] on: x [rows][width], W [experts][out][width],
 * h [rows][out], all dense and of dtype float16 or bfloat16; act: DCCL_ACT_* or -1 for none. Where z is not null it receives the products in fp32, in rows of
 * z_stride elements (a multiple of four). Starts are taken inside of [0, rows], and none before those ahead of it. A product that does not end in time leaves NaN, and no later call on its device starts one.
 */
int dccl_expert_linear(int device, int dtype, size_t rows, int experts, size_t width, size_t out, const void* x, const void* w, const int* starts, int act, void* h, float* z,
                       size_t z_stride, void* workspace, long long workspace_bytes, void* stream);

/** Its gradients from dh, and from z where there is an activation. Each of dx and dw may be null. No atomics. */
int dccl_expert_linear_backward(int device, int dtype, size_t rows, int experts, size_t width, size_t out, const void* dh, const float* z, size_t z_stride, const void* x,
                                const void* w, const int* starts, const void* forward_workspace, int act, void* dx, void* dw, void* workspace, long long workspace_bytes,
                                void* stream);

} // extern "C"
