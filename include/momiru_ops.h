/*
 * momiru_ops.h -- C ABI of the operators around the MatMul node: the linear
 * layer (bias, activation and residual in the product's epilogue, 16-bit or
 * f32 operands) and its gradient, tokens sorted by expert and back with their
 * gradients, and the experts' products over the sorted rows with theirs.
 *
 * The conventions are those of momiru_gemm.h: int32 statuses, mmr_last_error()
 * for the message, caller-owned buffers that stay alive until quiesce or
 * destroy, everything decided at bind (validation, kernel choice, TMA
 * descriptors, workspaces), and a run that only enqueues on its stream. One
 * handle type serves every operator here.
 *
 *   mmr_<operator>_bind  ->  mmr_op_run / mmr_op_run_on  ->  mmr_op_quiesce  ->  mmr_op_destroy
 *
 * A handle's runs are ordered one after another whichever streams they are
 * given, cudaStreamPerThread among them (a workspace belongs to its handle), and
 * may come from several host threads, as may quiesce; destroy follows them all.
 * Under stream capture the caller orders the graph's launches; quiesce then
 * reports only the error word.
 */
#ifndef MOMIRU_OPS_H
#define MOMIRU_OPS_H

#include "momiru_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- element types */
enum {
  MMR_DTYPE_F32 = 0,
  MMR_DTYPE_BF16 = 1,
  MMR_DTYPE_F16 = 2,
  MMR_DTYPE_I32 = 3
};

/* ---- activations: the functions of the MMR_EPI_* codes. f32 operands in
 * MMR_MATH_EXACT evaluate them as the MatMul node does, bit for bit; the other
 * modes and 16-bit operands in f32 arithmetic of their own */
enum {
  MMR_ACT_NONE = 0,
  MMR_ACT_RELU = 1,
  MMR_ACT_RELU6 = 2,
  MMR_ACT_GELU_ERF = 3,
  MMR_ACT_GELU_TANH = 4,
  MMR_ACT_SILU = 5
};

/* A view whose strides count elements of `dtype` (base_offset_bytes is in
 * bytes, as in mmr_view). An absent operand has view.address 0 and rank 0. */
typedef struct mmr_tensor {
  mmr_view view;
  int32_t dtype;              /* MMR_DTYPE_*                                  */
  int32_t reserved;           /* 0                                            */
} mmr_tensor;

typedef struct mmr_op_handle mmr_op_handle;

/* ---- linear:  pre = lhs rhs + bias;  out = act(pre) + residual
 * lhs [m, k], rhs [k, n] (each given transposed with its flag), out, pre and
 * residual [m, n], bias [n]; all of one type, bf16, f16 or f32. `pre` (an
 * output), bias and residual are optional. 16-bit operands: f32 sums, every
 * result rounded once, math_mode MMR_MATH_STRICT_FP32 only. f32 operands: the
 * MatMul node's modes. Views may have any strides; those that TMA does not
 * take are packed into a workspace by each run. residual may be out's own view;
 * any other overlap of an output is refused. */
typedef struct mmr_linear_desc {
  mmr_tensor lhs, rhs, out, bias, residual, pre;
  int32_t transpose_lhs, transpose_rhs;
  int32_t activation;         /* MMR_ACT_*                                    */
  int32_t math_mode;          /* MMR_MATH_*                                   */
  int32_t device_ordinal;
  int32_t reserved;           /* 0                                            */
  void *stream;
} mmr_linear_desc;

/* ---- its gradient:  d_pre = d_out act'(pre);  d_lhs = d_pre rhs^T;
 * d_rhs = lhs^T d_pre;  d_bias = column sums of d_pre (f32 sums). The
 * residual's gradient is d_out itself. d_lhs, d_rhs (in the layouts of lhs and
 * rhs) and d_bias are each optional, one at least present; `pre` is needed
 * where there is an activation. d_pre is held in the operands' type between it
 * and the two products: rounded once more, and with that type's range (an f16
 * d_pre above 65504 is infinite). */
typedef struct mmr_linear_grad_desc {
  mmr_tensor d_out, lhs, rhs, pre, d_lhs, d_rhs, d_bias;
  int32_t transpose_lhs, transpose_rhs;
  int32_t activation;
  int32_t math_mode;
  int32_t device_ordinal;
  int32_t reserved;
  void *stream;
} mmr_linear_grad_desc;

/* ---- tokens sorted by expert
 * Assignment i = t * top_k + j sends token t to expert ids[t, j]; an id outside
 * [0, experts) drops it. Expert e's segment of the sorted rows starts at
 * offsets[e], a multiple of row_align, and holds counts[e] assignments in
 * increasing i. slots[t, j] is the assignment's row or -1; sources[r] the row's
 * assignment or -1; offsets has experts + 1 entries, the last one the end of
 * the last segment. `rows` is mmr_expert_rows(...): enough for any ids. In
 * every sorted buffer a row that holds no token is zero; the operators write
 * it so and the gradients rely on it. All four are contiguous i32. */
typedef struct mmr_expert_layout {
  int64_t tokens, top_k, experts, row_align; /* experts <= 1024; row_align a power of two <= 128 */
  mmr_tensor slots, sources, offsets, counts;
} mmr_expert_layout;

/* Rows of the sorted buffers (host arithmetic). */
MMR_API int32_t mmr_expert_rows(int64_t tokens, int64_t top_k, int64_t experts, int64_t row_align, int64_t *rows);

/* Writes the layout and rows[r] = x[sources[r] / top_k] (zero without a token).
 * ids [tokens, top_k] i32; x [tokens, h], rows [rows, h] of one type, f32, bf16
 * or f16, with unit column strides. */
typedef struct mmr_dispatch_desc {
  mmr_expert_layout layout;   /* outputs                                      */
  mmr_tensor ids, x, rows;
  int32_t device_ordinal;
  int32_t reserved;
  void *stream;
} mmr_dispatch_desc;

/* out[t] = sum_j weights[t, j] rows[slots[t, j]] (+ residual[t]): f32 sums in
 * increasing j, dropped assignments left out (whatever rows holds). weights
 * [tokens, top_k] f32, or absent for all ones: that form is the dispatch's
 * gradient. residual may be out's own view. */
typedef struct mmr_combine_desc {
  mmr_expert_layout layout;
  mmr_tensor rows, weights, residual, out;
  int32_t device_ordinal;
  int32_t reserved;
  void *stream;
} mmr_combine_desc;

/* d_rows[slots[t, j]] = weights[t, j] d_out[t], zero without a token;
 * d_weights[t, j] = <d_out[t], rows[slots[t, j]]> in f32, 0 where dropped. One
 * of d_rows and d_weights may be absent. */
typedef struct mmr_combine_grad_desc {
  mmr_expert_layout layout;
  mmr_tensor d_out, rows, weights, d_rows, d_weights;
  int32_t device_ordinal;
  int32_t reserved;
  void *stream;
} mmr_combine_grad_desc;

/* ---- the experts' products: for the rows of expert e
 * pre = rows weights[e] + bias[e];  out = act(pre); bf16 or f16.
 * rows [rows, k], weights [experts, k, n] ([experts, n, k] with
 * transpose_rhs), bias [experts, n], out and pre [rows, n]. */
typedef struct mmr_expert_linear_desc {
  mmr_expert_layout layout;
  mmr_tensor rows, weights, bias, out, pre;
  int32_t transpose_rhs;
  int32_t activation;
  int32_t device_ordinal;
  int32_t reserved;
  void *stream;
} mmr_expert_linear_desc;

/* Gradient: d_rows, d_weights (in the layout of weights; zeros for an expert
 * without tokens), d_bias, each optional, one at least present. d_weights and
 * d_bias need row_align to be a multiple of 64. */
typedef struct mmr_expert_linear_grad_desc {
  mmr_expert_layout layout;
  mmr_tensor d_out, rows, weights, pre, d_rows, d_weights, d_bias;
  int32_t transpose_rhs;
  int32_t activation;
  int32_t device_ordinal;
  int32_t reserved;
  void *stream;
} mmr_expert_linear_grad_desc;

MMR_API int32_t mmr_linear_bind(const mmr_linear_desc *desc, mmr_op_handle **out);
MMR_API int32_t mmr_linear_grad_bind(const mmr_linear_grad_desc *desc, mmr_op_handle **out);
MMR_API int32_t mmr_dispatch_bind(const mmr_dispatch_desc *desc, mmr_op_handle **out);
MMR_API int32_t mmr_combine_bind(const mmr_combine_desc *desc, mmr_op_handle **out);
MMR_API int32_t mmr_combine_grad_bind(const mmr_combine_grad_desc *desc, mmr_op_handle **out);
MMR_API int32_t mmr_expert_linear_bind(const mmr_expert_linear_desc *desc, mmr_op_handle **out);
MMR_API int32_t mmr_expert_linear_grad_bind(const mmr_expert_linear_grad_desc *desc, mmr_op_handle **out);

MMR_API int32_t mmr_op_run(mmr_op_handle *h);
MMR_API int32_t mmr_op_run_on(mmr_op_handle *h, void *stream);
MMR_API int32_t mmr_op_quiesce(mmr_op_handle *h, uint64_t timeout_ns);
MMR_API int32_t mmr_op_destroy(mmr_op_handle *h);

/* What a handle launches, in order: kernel names and shapes, one per line. The
 * string lives as long as the handle. */
MMR_API const char *mmr_op_plan(const mmr_op_handle *h);

#ifdef __cplusplus
}
#endif

#endif /* MOMIRU_OPS_H */
