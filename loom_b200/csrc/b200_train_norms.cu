// C entries of the norms around a block (include/loom/b200_train.h): argument
// checks, the choice of the kernel by the element types, launches.
// Build: -gencode arch=compute_100a,code=sm_100a -fmad=false.
#include "loom/b200_train.h"

#include "loom_b200_block_norm.cuh"

namespace loomb {
#define LOOM_ROWS_ELSEWHERE(TX, TB)                                                             \
  extern template int launch_block_norm<TX, TB>(const BlockNorm&, const BlockNormOut&,          \
                                                cudaStream_t);                                  \
  extern template int launch_block_norm_grad<TX, TB>(const BlockNorm&, BlockNormGrad, int64_t,  \
                                                     void*, void*, void*, cudaStream_t);
LOOM_ROW_TYPES(LOOM_ROWS_ELSEWHERE)
#undef LOOM_ROWS_ELSEWHERE
}  // namespace loomb

namespace {

using loomb::BlockNorm;
using loomb::BlockNormGrad;
using loomb::BlockNormOut;

bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

bool stride_ok(int64_t s) { return s >= 0 && s < ((int64_t)1 << 31); }

bool types_ok(int x_dtype, int h_dtype) {
  return loomb::valid_dtype(x_dtype) && loomb::valid_dtype(h_dtype) &&
         (x_dtype == h_dtype || x_dtype == loomb::kF32);
}

// Calls f with a value of each of the two element types.
template <class F>
int with_types(int x_dtype, int h_dtype, const F& f) {
  if (x_dtype == loomb::kBF16) return f(__nv_bfloat16(), __nv_bfloat16());
  if (x_dtype == loomb::kF16) return f(__half(), __half());
  if (h_dtype == loomb::kBF16) return f(float(), __nv_bfloat16());
  if (h_dtype == loomb::kF16) return f(float(), __half());
  return f(float(), float());
}

// What both directions ask of their common arguments.
bool common_ok(const BlockNorm& a, int64_t gate_rows, int64_t width, int x_dtype, int h_dtype) {
  if (!types_ok(x_dtype, h_dtype) || a.rows < 0 || a.rows > ((int64_t)1 << 31) - 1 || width < 1 ||
      width > loomb::kRowMaxWidth)
    return false;
  if (a.post_norm != 0 && a.post_norm != 1) return false;
  if (a.pre_norm != 0 && a.pre_norm != 1) return false;
  // tensors without rows may come as null pointers
  if (a.rows > 0 && a.h == nullptr && (a.gate != nullptr || a.post_weight != nullptr ||
                                        !a.pre_norm))
    return false;
  if (!a.post_norm && a.post_weight != nullptr) return false;
  if (!a.pre_norm && a.pre_weight != nullptr) return false;
  if (a.gate != nullptr && (gate_rows < 1 || a.rows % gate_rows != 0)) return false;
  if (!(fabsf(a.offset) < INFINITY) || !(fabsf(a.residual_scale) < INFINITY) ||
      !(fabsf(a.branch_scale) < INFINITY))
    return false;
  const int bx = loomb::dtype_bytes(x_dtype), bh = loomb::dtype_bytes(h_dtype);
  return aligned_to(a.x, bx) && aligned_to(a.h, bh) && aligned_to(a.gate, bh) &&
         aligned_to(a.post_weight, bh) && aligned_to(a.pre_weight, bh) && stride_ok(a.x_stride) &&
         stride_ok(a.h_stride) && stride_ok(a.gate_stride);
}

int forward(BlockNorm a, int64_t gate_rows, int64_t width, int x_dtype, int h_dtype,
            const BlockNormOut& o, cudaStream_t stream) {
  if (!common_ok(a, gate_rows, width, x_dtype, h_dtype) || !(a.eps >= 0.0f && a.eps < INFINITY))
    return LOOM_STATUS_INVALID_ARGUMENT;
  const int bx = loomb::dtype_bytes(x_dtype), bh = loomb::dtype_bytes(h_dtype);
  if (!aligned_to(o.y, bx) || !aligned_to(o.z, bh) || !aligned_to(o.post_rstd, 4) ||
      !aligned_to(o.pre_rstd, 4))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if (a.rows == 0) return LOOM_STATUS_OK;
  if (a.x == nullptr || (a.h != nullptr && o.y == nullptr) || (a.pre_norm && o.z == nullptr))
    return LOOM_STATUS_INVALID_ARGUMENT;
  a.rows_per_gate = a.gate != nullptr ? a.rows / gate_rows : a.rows;
  return with_types(x_dtype, h_dtype, [&](auto tx, auto th) {
    return loomb::launch_block_norm<decltype(tx), decltype(th)>(a, o, stream);
  });
}

int backward(const BlockNorm& a, int64_t gate_rows, int64_t width, int x_dtype, int h_dtype,
             const BlockNormGrad& b, void* dpost_weight, void* dpre_weight, void* workspace,
             size_t workspace_size, cudaStream_t stream) {
  if (!common_ok(a, gate_rows, width, x_dtype, h_dtype)) return LOOM_STATUS_INVALID_ARGUMENT;
  const int bx = loomb::dtype_bytes(x_dtype), bh = loomb::dtype_bytes(h_dtype);
  if (!aligned_to(b.dy, bx) || !aligned_to(b.dz, bh) || !aligned_to(b.dx, bx) ||
      !aligned_to(b.dh, bh) || !aligned_to(b.dgate, bh) || !aligned_to(dpost_weight, bh) ||
      !aligned_to(dpre_weight, bh) || !aligned_to(b.post_rstd, 4) || !aligned_to(b.pre_rstd, 4) ||
      !stride_ok(b.dy_stride) || !stride_ok(b.dz_stride))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if ((dpost_weight != nullptr && a.post_weight == nullptr) ||
      (dpre_weight != nullptr && a.pre_weight == nullptr))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if ((a.gate != nullptr) != (b.dgate != nullptr)) return LOOM_STATUS_INVALID_ARGUMENT;
  if (a.rows > 0 &&
      (b.dx == nullptr || (a.h != nullptr) != (b.dh != nullptr) ||
       (a.pre_norm && (a.x == nullptr || b.dz == nullptr || b.pre_rstd == nullptr)) ||
       (a.h != nullptr && a.post_norm && b.post_rstd == nullptr)))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if (workspace == nullptr ||
      workspace_size < loomb::block_norm_grad_workspace_bytes(a.rows, width,
                                                              a.gate != nullptr ? gate_rows : 0))
    return LOOM_STATUS_WORKSPACE_TOO_SMALL;
  if (a.rows == 0 && b.dgate != nullptr &&
      cudaMemsetAsync(b.dgate, 0, (size_t)gate_rows * (size_t)width * bh, stream) != cudaSuccess) {
    cudaGetLastError();
    return LOOM_STATUS_CUDA_ERROR;
  }
  return with_types(x_dtype, h_dtype, [&](auto tx, auto th) {
    return loomb::launch_block_norm_grad<decltype(tx), decltype(th)>(
        a, b, gate_rows, dpost_weight, dpre_weight, workspace, stream);
  });
}

int finish(int status) {
  return status == LOOM_STATUS_OK ? loomb::finish_sync() : status;
}

}  // namespace

extern "C" int loom_train_block_norm_stream(
    const void* x, int64_t x_stride, const void* h, int64_t h_stride, const void* gate,
    int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight,
    int64_t rows, int64_t width, int x_dtype, int h_dtype, int post_norm, int pre_norm, float eps,
    float weight_offset, float residual_scale, float branch_scale, void* y, void* z,
    float* post_rstd, float* pre_rstd, void* stream) {
  const BlockNorm a = {x, h, gate, post_weight, pre_weight, x_stride, h_stride, gate_stride,
                       rows, 1, (int)width, post_norm, pre_norm, eps, weight_offset,
                       residual_scale, branch_scale};
  const BlockNormOut o = {y, z, post_rstd, pre_rstd};
  return forward(a, gate_rows, width, x_dtype, h_dtype, o, static_cast<cudaStream_t>(stream));
}

extern "C" int loom_train_block_norm(
    const void* x, int64_t x_stride, const void* h, int64_t h_stride, const void* gate,
    int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight,
    int64_t rows, int64_t width, int x_dtype, int h_dtype, int post_norm, int pre_norm, float eps,
    float weight_offset, float residual_scale, float branch_scale, void* y, void* z,
    float* post_rstd, float* pre_rstd) {
  return finish(loom_train_block_norm_stream(
      x, x_stride, h, h_stride, gate, gate_stride, gate_rows, post_weight, pre_weight, rows, width,
      x_dtype, h_dtype, post_norm, pre_norm, eps, weight_offset, residual_scale, branch_scale, y,
      z, post_rstd, pre_rstd, nullptr));
}

extern "C" size_t loom_train_block_norm_backward_workspace_size(int64_t rows, int64_t width,
                                                                int64_t gate_rows) {
  return loomb::block_norm_grad_workspace_bytes(rows, width, gate_rows);
}

extern "C" int loom_train_block_norm_backward_stream(
    const void* y, int64_t y_stride, const void* h, int64_t h_stride, const void* gate,
    int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight,
    const float* post_rstd, const float* pre_rstd, const void* dy, int64_t dy_stride,
    const void* dz, int64_t dz_stride, int64_t rows, int64_t width, int x_dtype, int h_dtype,
    int post_norm, int pre_norm, float weight_offset, float residual_scale, float branch_scale,
    void* dx, void* dh, void* dgate, void* dpost_weight, void* dpre_weight, void* workspace,
    size_t workspace_size, void* stream) {
  const BlockNorm a = {y, h, gate, post_weight, pre_weight, y_stride, h_stride, gate_stride,
                       rows, 1, (int)width, post_norm, pre_norm, 0.0f, weight_offset,
                       residual_scale, branch_scale};
  const BlockNormGrad b = {post_rstd, pre_rstd, dy, dz, dy_stride, dz_stride, dx, dh, dgate,
                           nullptr, nullptr, nullptr, 0, 1};
  return backward(a, gate_rows, width, x_dtype, h_dtype, b, dpost_weight, dpre_weight, workspace,
                  workspace_size, static_cast<cudaStream_t>(stream));
}

extern "C" int loom_train_block_norm_backward(
    const void* y, int64_t y_stride, const void* h, int64_t h_stride, const void* gate,
    int64_t gate_stride, int64_t gate_rows, const void* post_weight, const void* pre_weight,
    const float* post_rstd, const float* pre_rstd, const void* dy, int64_t dy_stride,
    const void* dz, int64_t dz_stride, int64_t rows, int64_t width, int x_dtype, int h_dtype,
    int post_norm, int pre_norm, float weight_offset, float residual_scale, float branch_scale,
    void* dx, void* dh, void* dgate, void* dpost_weight, void* dpre_weight, void* workspace,
    size_t workspace_size) {
  return finish(loom_train_block_norm_backward_stream(
      y, y_stride, h, h_stride, gate, gate_stride, gate_rows, post_weight, pre_weight, post_rstd,
      pre_rstd, dy, dy_stride, dz, dz_stride, rows, width, x_dtype, h_dtype, post_norm, pre_norm,
      weight_offset, residual_scale, branch_scale, dx, dh, dgate, dpost_weight, dpre_weight,
      workspace, workspace_size, nullptr));
}

extern "C" int loom_train_block_norm_packed(const loom_train_block_norm_args* a, void* stream) {
  if (a == nullptr) return LOOM_STATUS_INVALID_ARGUMENT;
  return loom_train_block_norm_stream(a->x, a->x_stride, a->h, a->h_stride, a->gate,
      a->gate_stride, a->gate_rows, a->post_weight, a->pre_weight, a->rows, a->width, a->x_dtype,
      a->h_dtype, a->post_norm, a->pre_norm, a->eps, a->weight_offset, a->residual_scale,
      a->branch_scale, a->y, a->z, a->post_rstd, a->pre_rstd, stream);
}

extern "C" int loom_train_block_norm_backward_packed(const loom_train_block_norm_backward_args* a,
      void* stream) {
  if (a == nullptr) return LOOM_STATUS_INVALID_ARGUMENT;
  return loom_train_block_norm_backward_stream(a->y, a->y_stride, a->h, a->h_stride, a->gate,
      a->gate_stride, a->gate_rows, a->post_weight, a->pre_weight, a->post_rstd, a->pre_rstd,
      a->dy, a->dy_stride, a->dz, a->dz_stride, a->rows, a->width, a->x_dtype, a->h_dtype,
      a->post_norm, a->pre_norm, a->weight_offset, a->residual_scale, a->branch_scale, a->dx,
      a->dh, a->dgate, a->dpost_weight, a->dpre_weight, a->workspace, a->workspace_size, stream);
}
