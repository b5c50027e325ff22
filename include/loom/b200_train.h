#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The training-step operators of the Loom B200 (sm_100a) backend: hand-written kernels beside the compiled entries.
   They have no counterpart in the reference, whose entries take fp32 vectors one by one.

   Conventions of every entry:
   - tensors are caller-owned device memory on the current device; the library allocates nothing and holds no state;
   - <symbol> runs on the legacy default stream and waits for it; <symbol>_stream runs on the given stream, never waits, and may be captured into a graph;
   - <symbol>_packed is <symbol>_stream with the arguments in one structure, in the same order: for callers to whom each argument of a call costs;
   - a workspace of <symbol>_workspace_size(...) bytes belongs to one call at a time: calls that may overlap on the GPU, two captured graphs among them, each need their own;
   - the return value is one of the status codes of the compiled packages; arguments are checked before anything is launched;
   - a list has at most 2^40 values in all;
   - arrays of pointers and of sizes are host memory, read during the call only (a captured launch keeps its own copy);
   - tensors that are written may not overlap each other or any that is read. */
#ifndef LOOM_STATUS_OK
#define LOOM_STATUS_OK 0
#define LOOM_STATUS_INVALID_ARGUMENT 1
#define LOOM_STATUS_WORKSPACE_TOO_SMALL 2
#define LOOM_STATUS_CUDA_ERROR 3
#endif

/* Element types. */
#define LOOM_DTYPE_F32 0
#define LOOM_DTYPE_BF16 1
#define LOOM_DTYPE_F16 2

/* grad_norm: out[0] = the 2-norm of all values of `count` tensors (sizes[i] values each), out[1] = the factor that brings it down to max_norm (> 0):
   max_norm / norm where the norm is larger, 1 where it is not, NaN where the sum of squares is not finite (a square beyond the fp32 range counts as infinite; smaller ones add up as they are, however small). */
size_t loom_train_grad_norm_workspace_size(int64_t count);
int loom_train_grad_norm(int64_t count, const void* const* grads, const int64_t* sizes, int grad_dtype, float max_norm, float* out, void* workspace, size_t workspace_size);
int loom_train_grad_norm_stream(int64_t count, const void* const* grads, const int64_t* sizes, int grad_dtype, float max_norm, float* out, void* workspace, size_t workspace_size, void* stream);
typedef struct loom_train_grad_norm_args {
  int64_t count;
  const void* const* grads;
  const int64_t* sizes;
  int grad_dtype;
  float max_norm;
  float* out;
  void* workspace;
  size_t workspace_size;
} loom_train_grad_norm_args;
int loom_train_grad_norm_packed(const loom_train_grad_norm_args* args, void* stream);

/* adamw: one step, in place, of `count` tensors.  With t = *step + 1, g = *grad_scale * grad (grad_scale may be null: 1), fp32 moments m and v:
     m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;
     p = p (1 - lr weight_decay[i]) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps);  *step = t.
   step and lr are device memory, so that a captured step can be replayed.  master (or null): fp32 copies that the step reads and writes; params then only receive them, rounded.
   A grad_scale that is not finite skips the step: nothing is changed, *step included.
   Every call counts a step: lists that make up one step in several calls (parameters of two types, two learning rates) each need a step of their own. */
size_t loom_train_adamw_workspace_size(int64_t count);
int loom_train_adamw(int64_t count, void* const* params, const void* const* grads, float* const* exp_avg, float* const* exp_avg_sq, float* const* master, const int64_t* sizes, const double* weight_decay, int param_dtype, int grad_dtype, const float* lr, double beta1, double beta2, double eps, const float* grad_scale, int64_t* step, void* workspace, size_t workspace_size);
int loom_train_adamw_stream(int64_t count, void* const* params, const void* const* grads, float* const* exp_avg, float* const* exp_avg_sq, float* const* master, const int64_t* sizes, const double* weight_decay, int param_dtype, int grad_dtype, const float* lr, double beta1, double beta2, double eps, const float* grad_scale, int64_t* step, void* workspace, size_t workspace_size, void* stream);
typedef struct loom_train_adamw_args {
  int64_t count;
  void* const* params;
  const void* const* grads;
  float* const* exp_avg;
  float* const* exp_avg_sq;
  float* const* master;
  const int64_t* sizes;
  const double* weight_decay;
  int param_dtype;
  int grad_dtype;
  const float* lr;
  double beta1;
  double beta2;
  double eps;
  const float* grad_scale;
  int64_t* step;
  void* workspace;
  size_t workspace_size;
} loom_train_adamw_args;
int loom_train_adamw_packed(const loom_train_adamw_args* args, void* stream);

/* adamw8: the same step with both moments in 8 bits.  Blocks of 256 values of a tensor (the last one may be short) share an fp32 top, the block's largest magnitude;
   a value is e4m3 code * top / 256.  exp_avg_top[i] and exp_avg_sq_top[i] hold ceil(sizes[i] / 256) tops.  The step computes in fp32 and rounds each new moment up or down
   with the probability of its distance, by random bits of (seed, t, place in the list); a second moment above zero never becomes zero.  A block with a moment that is not
   finite reads back as not finite throughout; one whose largest is below 2^-100 holds zeros.
   The sign of a code that stands for zero is not specified.  eps is at least FLT_MIN. */
size_t loom_train_adamw8_workspace_size(int64_t count);
int loom_train_adamw8(int64_t count, void* const* params, const void* const* grads, uint8_t* const* exp_avg, uint8_t* const* exp_avg_sq, float* const* exp_avg_top, float* const* exp_avg_sq_top, float* const* master, const int64_t* sizes, const double* weight_decay, int param_dtype, int grad_dtype, const float* lr, double beta1, double beta2, double eps, const float* grad_scale, int64_t* step, uint64_t seed, void* workspace, size_t workspace_size);
int loom_train_adamw8_stream(int64_t count, void* const* params, const void* const* grads, uint8_t* const* exp_avg, uint8_t* const* exp_avg_sq, float* const* exp_avg_top, float* const* exp_avg_sq_top, float* const* master, const int64_t* sizes, const double* weight_decay, int param_dtype, int grad_dtype, const float* lr, double beta1, double beta2, double eps, const float* grad_scale, int64_t* step, uint64_t seed, void* workspace, size_t workspace_size, void* stream);
typedef struct loom_train_adamw8_args {
  int64_t count;
  void* const* params;
  const void* const* grads;
  uint8_t* const* exp_avg;
  uint8_t* const* exp_avg_sq;
  float* const* exp_avg_top;
  float* const* exp_avg_sq_top;
  float* const* master;
  const int64_t* sizes;
  const double* weight_decay;
  int param_dtype;
  int grad_dtype;
  const float* lr;
  double beta1;
  double beta2;
  double eps;
  const float* grad_scale;
  int64_t* step;
  uint64_t seed;
  void* workspace;
  size_t workspace_size;
} loom_train_adamw8_args;
int loom_train_adamw8_packed(const loom_train_adamw8_args* args, void* stream);

/* block_norm: the norms after and before a block, with its gate and the residual's scale, over rows of 1 <= width <= 32768 values:
     u = h post_rstd (post_weight + weight_offset), post_rstd = 1 / sqrt(mean(h^2) + eps)   (post_norm 0: u = h)
     y = residual_scale x + branch_scale gate u
     z = y pre_rstd (pre_weight + weight_offset), pre_rstd = 1 / sqrt(mean(y^2) + eps)      (pre_norm 0: no z)
   x, y are of x_dtype; h, gate, the weights and z of h_dtype (x_dtype, or 16-bit beside a 32-bit x).  rows and strides are below 2^31.  h null: y is x (residual_scale has no part in it, nor in dx), is not written and may be null.
   gate (or null): gate_rows rows, each for rows / gate_rows consecutive rows.  A null weight is all ones (no offset).  Strides are in elements, outputs contiguous;
   post_rstd and pre_rstd ([rows], for the backward pass) may be null.  Sums are fp32: a row whose sum of squares passes its range has a statistic of 0, and squares below it count as zero (with eps 0 a row of these has an infinite one). */
int loom_train_block_norm(const void* x, int64_t x_stride, const void* h, int64_t h_stride, const void* gate, int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight, int64_t rows, int64_t width, int x_dtype, int h_dtype, int post_norm, int pre_norm, float eps, float weight_offset, float residual_scale, float branch_scale, void* y, void* z, float* post_rstd, float* pre_rstd);
int loom_train_block_norm_stream(const void* x, int64_t x_stride, const void* h, int64_t h_stride, const void* gate, int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight, int64_t rows, int64_t width, int x_dtype, int h_dtype, int post_norm, int pre_norm, float eps, float weight_offset, float residual_scale, float branch_scale, void* y, void* z, float* post_rstd, float* pre_rstd, void* stream);
typedef struct loom_train_block_norm_args {
  const void* x;
  int64_t x_stride;
  const void* h;
  int64_t h_stride;
  const void* gate;
  int64_t gate_stride;
  int64_t gate_rows;
  const void* post_weight;
  const void* pre_weight;
  int64_t rows;
  int64_t width;
  int x_dtype;
  int h_dtype;
  int post_norm;
  int pre_norm;
  float eps;
  float weight_offset;
  float residual_scale;
  float branch_scale;
  void* y;
  void* z;
  float* post_rstd;
  float* pre_rstd;
} loom_train_block_norm_args;
int loom_train_block_norm_packed(const loom_train_block_norm_args* args, void* stream);

/* block_norm_backward: the gradients of block_norm from y (x where h is null), h, gate, the weights and the statistics, for dy (null: zero) and dz (with pre_norm).
   dx is written; dh with h; dgate with gate; dpost_weight and dpre_weight where not null.  Each has the type of what it is the gradient of, rounded once from fp32 sums. */
size_t loom_train_block_norm_backward_workspace_size(int64_t rows, int64_t width, int64_t gate_rows);
int loom_train_block_norm_backward(const void* y, int64_t y_stride, const void* h, int64_t h_stride, const void* gate, int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight, const float* post_rstd, const float* pre_rstd, const void* dy, int64_t dy_stride, const void* dz, int64_t dz_stride, int64_t rows, int64_t width, int x_dtype, int h_dtype, int post_norm, int pre_norm, float weight_offset, float residual_scale, float branch_scale, void* dx, void* dh, void* dgate, void* dpost_weight, void* dpre_weight, void* workspace, size_t workspace_size);
int loom_train_block_norm_backward_stream(const void* y, int64_t y_stride, const void* h, int64_t h_stride, const void* gate, int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight, const float* post_rstd, const float* pre_rstd, const void* dy, int64_t dy_stride, const void* dz, int64_t dz_stride, int64_t rows, int64_t width, int x_dtype, int h_dtype, int post_norm, int pre_norm, float weight_offset, float residual_scale, float branch_scale, void* dx, void* dh, void* dgate, void* dpost_weight, void* dpre_weight, void* workspace, size_t workspace_size, void* stream);
typedef struct loom_train_block_norm_backward_args {
  const void* y;
  int64_t y_stride;
  const void* h;
  int64_t h_stride;
  const void* gate;
  int64_t gate_stride;
  int64_t gate_rows;
  const void* post_weight;
  const void* pre_weight;
  const float* post_rstd;
  const float* pre_rstd;
  const void* dy;
  int64_t dy_stride;
  const void* dz;
  int64_t dz_stride;
  int64_t rows;
  int64_t width;
  int x_dtype;
  int h_dtype;
  int post_norm;
  int pre_norm;
  float weight_offset;
  float residual_scale;
  float branch_scale;
  void* dx;
  void* dh;
  void* dgate;
  void* dpost_weight;
  void* dpre_weight;
  void* workspace;
  size_t workspace_size;
} loom_train_block_norm_backward_args;
int loom_train_block_norm_backward_packed(const loom_train_block_norm_backward_args* args, void* stream);

#ifdef __cplusplus
}
#endif
