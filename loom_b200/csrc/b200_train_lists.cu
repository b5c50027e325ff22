// C entries of the operators over lists of tensors (include/loom/b200_train.h):
// argument checks, the choice of the kernel by the element types, launches.
// Build: -gencode arch=compute_100a,code=sm_100a -fmad=false.
#include <float.h>

#include "loom/b200_train.h"

#include "loom_b200_lists.cuh"

namespace {

using loomb::AdamLists;
using loomb::StepConst;
using loomb::StepValues;

bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// A list argument: an array of `count` pointers, each non-null and aligned to
// its elements where its tensor has any.
bool list_ok(int64_t count, const void* const* p, const int64_t* sizes, int bytes) {
  if (count == 0) return true;
  if (p == nullptr) return false;
  for (int64_t i = 0; i < count; ++i)
    if (sizes[i] > 0 && (p[i] == nullptr || !aligned_to(p[i], bytes))) return false;
  return true;
}

// At most kListMost values in all, so that the tiles of any launch can be counted
// in 31 bits: nothing is left to refuse once a step has begun.
bool sizes_ok(int64_t count, const int64_t* sizes) {
  if (count < 0 || (count > 0 && sizes == nullptr)) return false;
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] > loomb::kListMost - all) return false;
    all += sizes[i];
  }
  return true;
}

int grad_norm_impl(int64_t count, const void* const* grads, const int64_t* sizes, int grad_dtype,
                   float max_norm, float* out, void* workspace, size_t workspace_size,
                   cudaStream_t stream) {
  if (!sizes_ok(count, sizes) || !loomb::valid_dtype(grad_dtype) || !(max_norm > 0.0f) ||
      out == nullptr || !aligned_to(out, 4) ||
      !list_ok(count, grads, sizes, loomb::dtype_bytes(grad_dtype)))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if (workspace == nullptr || workspace_size < loomb::list_norm_workspace_bytes(count))
    return LOOM_STATUS_WORKSPACE_TOO_SMALL;
  switch (grad_dtype) {
    case loomb::kF32:
      return loomb::launch_list_norm<float>(count, grads, sizes, max_norm, out, workspace, stream);
    case loomb::kBF16:
      return loomb::launch_list_norm<__nv_bfloat16>(count, grads, sizes, max_norm, out, workspace,
                                                    stream);
    default:
      return loomb::launch_list_norm<__half>(count, grads, sizes, max_norm, out, workspace,
                                             stream);
  }
}

template <bool kEight, class Tp, class Tg>
int launch_step(const AdamLists& l, const StepConst& c, const StepValues* v, cudaStream_t stream) {
  if constexpr (sizeof(Tp) == 4) {
    if constexpr (kEight) return loomb::launch_adamw8_lists<Tp, Tg, false>(l, c, v, stream);
    return loomb::launch_adamw_lists<Tp, Tg, false>(l, c, v, stream);
  } else if constexpr (kEight) {
    return l.master != nullptr ? loomb::launch_adamw8_lists<Tp, Tg, true>(l, c, v, stream)
                               : loomb::launch_adamw8_lists<Tp, Tg, false>(l, c, v, stream);
  } else {
    return l.master != nullptr ? loomb::launch_adamw_lists<Tp, Tg, true>(l, c, v, stream)
                               : loomb::launch_adamw_lists<Tp, Tg, false>(l, c, v, stream);
  }
}

template <bool kEight, class Tp>
int launch_by_grad(const AdamLists& l, int grad_dtype, const StepConst& c, const StepValues* v,
                   cudaStream_t stream) {
  switch (grad_dtype) {
    case loomb::kF32: return launch_step<kEight, Tp, float>(l, c, v, stream);
    case loomb::kBF16: return launch_step<kEight, Tp, __nv_bfloat16>(l, c, v, stream);
    default: return launch_step<kEight, Tp, __half>(l, c, v, stream);
  }
}

template <bool kEight>
int adamw_impl(const AdamLists& l, int param_dtype, int grad_dtype, const float* lr, double beta1,
               double beta2, double eps, const float* grad_scale, int64_t* step, uint64_t seed,
               void* workspace, size_t workspace_size, cudaStream_t stream) {
  if (!sizes_ok(l.count, l.sizes) || !loomb::valid_dtype(param_dtype) ||
      !loomb::valid_dtype(grad_dtype) || !(beta1 >= 0.0 && beta1 < 1.0) ||
      !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0 && eps < (double)INFINITY) ||
      (kEight && !((float)eps >= FLT_MIN)) || lr == nullptr || !aligned_to(lr, 4) ||
      !aligned_to(grad_scale, 4) || step == nullptr || !aligned_to(step, 8))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if (!list_ok(l.count, l.params, l.sizes, loomb::dtype_bytes(param_dtype)) ||
      !list_ok(l.count, l.grads, l.sizes, loomb::dtype_bytes(grad_dtype)) ||
      !list_ok(l.count, l.exp_avg, l.sizes, kEight ? 1 : 4) ||
      !list_ok(l.count, l.exp_avg_sq, l.sizes, kEight ? 1 : 4) ||
      (l.count > 0 && l.weight_decay == nullptr))
    return LOOM_STATUS_INVALID_ARGUMENT;
  if (kEight && (!list_ok(l.count, (const void* const*)l.exp_avg_top, l.sizes, 4) ||
                 !list_ok(l.count, (const void* const*)l.exp_avg_sq_top, l.sizes, 4)))
    return LOOM_STATUS_INVALID_ARGUMENT;
  // masters beside 16-bit parameters only: fp32 parameters are their own
  if (l.master != nullptr && (param_dtype == loomb::kF32 ||
                              !list_ok(l.count, (const void* const*)l.master, l.sizes, 4)))
    return LOOM_STATUS_INVALID_ARGUMENT;
  for (int64_t i = 0; i < l.count; ++i)
    if (!(fabs(l.weight_decay[i]) < (double)INFINITY)) return LOOM_STATUS_INVALID_ARGUMENT;
  if (workspace == nullptr || workspace_size < loomb::adamw_workspace_bytes())
    return LOOM_STATUS_WORKSPACE_TOO_SMALL;
  StepConst c;
  c.beta1 = (float)beta1;
  c.rest1 = (float)(1.0 - beta1);
  c.beta2 = (float)beta2;
  c.rest2 = (float)(1.0 - beta2);
  // an eps below the fp32 range stays above zero: 0 / eps is 0
  c.eps = eps > 0.0 && (float)eps == 0.0f ? FLT_TRUE_MIN : (float)eps;
  c.zero = -0.0f;
  c.sixteen = 16u;
  StepValues* values = reinterpret_cast<StepValues*>(loomb::workspace_base(workspace));
  const int st = loomb::launch_dependent(loomb::adamw_begin_kernel, dim3(1), dim3(32), stream,
                                         (size_t)0, values, lr, grad_scale, step, beta1, beta2, seed);
  if (st != LOOM_STATUS_OK) return st;
  switch (param_dtype) {
    case loomb::kF32: return launch_by_grad<kEight, float>(l, grad_dtype, c, values, stream);
    case loomb::kBF16:
      return launch_by_grad<kEight, __nv_bfloat16>(l, grad_dtype, c, values, stream);
    default: return launch_by_grad<kEight, __half>(l, grad_dtype, c, values, stream);
  }
}

int finish(int status) {
  return status == LOOM_STATUS_OK ? loomb::finish_sync() : status;
}

}  // namespace

extern "C" size_t loom_train_grad_norm_workspace_size(int64_t count) {
  return loomb::list_norm_workspace_bytes(count);
}

extern "C" int loom_train_grad_norm_stream(int64_t count, const void* const* grads,
                                           const int64_t* sizes, int grad_dtype, float max_norm,
                                           float* out, void* workspace, size_t workspace_size,
                                           void* stream) {
  return grad_norm_impl(count, grads, sizes, grad_dtype, max_norm, out, workspace, workspace_size,
                        static_cast<cudaStream_t>(stream));
}

extern "C" int loom_train_grad_norm(int64_t count, const void* const* grads, const int64_t* sizes,
                                    int grad_dtype, float max_norm, float* out, void* workspace,
                                    size_t workspace_size) {
  return finish(grad_norm_impl(count, grads, sizes, grad_dtype, max_norm, out, workspace,
                               workspace_size, nullptr));
}

extern "C" size_t loom_train_adamw_workspace_size(int64_t count) {
  return count < 0 ? 0 : loomb::adamw_workspace_bytes();
}

extern "C" int loom_train_adamw_stream(
    int64_t count, void* const* params, const void* const* grads, float* const* exp_avg,
    float* const* exp_avg_sq, float* const* master, const int64_t* sizes,
    const double* weight_decay, int param_dtype, int grad_dtype, const float* lr, double beta1,
    double beta2, double eps, const float* grad_scale, int64_t* step, void* workspace,
    size_t workspace_size, void* stream) {
  const AdamLists l = {count, params, grads, (void* const*)exp_avg, (void* const*)exp_avg_sq,
                       nullptr, nullptr, master, sizes, weight_decay};
  return adamw_impl<false>(l, param_dtype, grad_dtype, lr, beta1, beta2, eps, grad_scale, step, 0,
                           workspace, workspace_size, static_cast<cudaStream_t>(stream));
}

extern "C" int loom_train_adamw(
    int64_t count, void* const* params, const void* const* grads, float* const* exp_avg,
    float* const* exp_avg_sq, float* const* master, const int64_t* sizes,
    const double* weight_decay, int param_dtype, int grad_dtype, const float* lr, double beta1,
    double beta2, double eps, const float* grad_scale, int64_t* step, void* workspace,
    size_t workspace_size) {
  return finish(loom_train_adamw_stream(count, params, grads, exp_avg, exp_avg_sq, master, sizes,
                                        weight_decay, param_dtype, grad_dtype, lr, beta1, beta2,
                                        eps, grad_scale, step, workspace, workspace_size,
                                        nullptr));
}

extern "C" size_t loom_train_adamw8_workspace_size(int64_t count) {
  return count < 0 ? 0 : loomb::adamw_workspace_bytes();
}

extern "C" int loom_train_adamw8_stream(
    int64_t count, void* const* params, const void* const* grads, uint8_t* const* exp_avg,
    uint8_t* const* exp_avg_sq, float* const* exp_avg_top, float* const* exp_avg_sq_top,
    float* const* master, const int64_t* sizes, const double* weight_decay, int param_dtype,
    int grad_dtype, const float* lr, double beta1, double beta2, double eps,
    const float* grad_scale, int64_t* step, uint64_t seed, void* workspace,
    size_t workspace_size, void* stream) {
  const AdamLists l = {count, params, grads, (void* const*)exp_avg, (void* const*)exp_avg_sq,
                       exp_avg_top, exp_avg_sq_top, master, sizes, weight_decay};
  return adamw_impl<true>(l, param_dtype, grad_dtype, lr, beta1, beta2, eps, grad_scale, step,
                          seed, workspace, workspace_size, static_cast<cudaStream_t>(stream));
}

extern "C" int loom_train_adamw8(
    int64_t count, void* const* params, const void* const* grads, uint8_t* const* exp_avg,
    uint8_t* const* exp_avg_sq, float* const* exp_avg_top, float* const* exp_avg_sq_top,
    float* const* master, const int64_t* sizes, const double* weight_decay, int param_dtype,
    int grad_dtype, const float* lr, double beta1, double beta2, double eps,
    const float* grad_scale, int64_t* step, uint64_t seed, void* workspace,
    size_t workspace_size) {
  return finish(loom_train_adamw8_stream(
      count, params, grads, exp_avg, exp_avg_sq, exp_avg_top, exp_avg_sq_top, master, sizes,
      weight_decay, param_dtype, grad_dtype, lr, beta1, beta2, eps, grad_scale, step, seed,
      workspace, workspace_size, nullptr));
}

extern "C" int loom_train_grad_norm_packed(const loom_train_grad_norm_args* a, void* stream) {
  if (a == nullptr) return LOOM_STATUS_INVALID_ARGUMENT;
  return loom_train_grad_norm_stream(a->count, a->grads, a->sizes, a->grad_dtype, a->max_norm,
      a->out, a->workspace, a->workspace_size, stream);
}

extern "C" int loom_train_adamw_packed(const loom_train_adamw_args* a, void* stream) {
  if (a == nullptr) return LOOM_STATUS_INVALID_ARGUMENT;
  return loom_train_adamw_stream(a->count, a->params, a->grads, a->exp_avg, a->exp_avg_sq,
      a->master, a->sizes, a->weight_decay, a->param_dtype, a->grad_dtype, a->lr, a->beta1,
      a->beta2, a->eps, a->grad_scale, a->step, a->workspace, a->workspace_size, stream);
}

extern "C" int loom_train_adamw8_packed(const loom_train_adamw8_args* a, void* stream) {
  if (a == nullptr) return LOOM_STATUS_INVALID_ARGUMENT;
  return loom_train_adamw8_stream(a->count, a->params, a->grads, a->exp_avg, a->exp_avg_sq,
      a->exp_avg_top, a->exp_avg_sq_top, a->master, a->sizes, a->weight_decay, a->param_dtype,
      a->grad_dtype, a->lr, a->beta1, a->beta2, a->eps, a->grad_scale, a->step, a->seed,
      a->workspace, a->workspace_size, stream);
}
