/* A plain C (C11) caller of the training-step operator package: one AdamW
 * step of two tensors with the factor that grad_norm left on the device.
 * Prints "train_smoke ok" and exits 0 when it agrees with a host computation. */
#include <cuda_runtime.h>
#include <math.h>
#include <stdio.h>

#include "loom/b200_train.h"

#define N0 1000
#define N1 33
#define N (N0 + N1)

static int bad(int line) {
  fprintf(stderr, "failed at line %d: %s\n", line, cudaGetErrorString(cudaGetLastError()));
  return 1;
}

int main(void) {
  float host[4][N], *dev[4], *out, *lr, rate = 0.01f, result[2];
  int64_t *step, zero = 0, count = -1;
  unsigned s = 12345u;
  for (int a = 0; a < 4; ++a)
    for (int i = 0; i < N; ++i) {
      s = s * 1664525u + 1013904223u;
      host[a][i] = (float)(s >> 8) / 16777216.0f - (a == 3 ? 0.0f : 0.5f);
    }
  for (int a = 0; a < 4; ++a) {
    if (cudaMalloc((void**)&dev[a], sizeof(host[a])) != cudaSuccess) return bad(__LINE__);
    if (cudaMemcpy(dev[a], host[a], sizeof(host[a]), cudaMemcpyHostToDevice) != cudaSuccess)
      return bad(__LINE__);
  }
  const int64_t sizes[2] = {N0, N1};
  const double decay[2] = {0.1, 0.0};
  void* params[2] = {dev[0], dev[0] + N0};
  const void* grads[2] = {dev[1], dev[1] + N0};
  float* m[2] = {dev[2], dev[2] + N0};
  float* v[2] = {dev[3], dev[3] + N0};
  size_t ws_size = loom_train_grad_norm_workspace_size(2);
  void* ws = NULL;
  if (loom_train_adamw_workspace_size(2) > ws_size) ws_size = loom_train_adamw_workspace_size(2);
  if (cudaMalloc(&ws, ws_size) != cudaSuccess || cudaMalloc((void**)&out, 8) != cudaSuccess ||
      cudaMalloc((void**)&lr, 4) != cudaSuccess || cudaMalloc((void**)&step, 8) != cudaSuccess)
    return bad(__LINE__);
  cudaMemcpy(lr, &rate, 4, cudaMemcpyHostToDevice);
  cudaMemcpy(step, &zero, 8, cudaMemcpyHostToDevice);
  if (loom_train_grad_norm(2, grads, sizes, LOOM_DTYPE_F32, 1.0f, out, ws, 8) !=
      LOOM_STATUS_WORKSPACE_TOO_SMALL)
    return bad(__LINE__);
  if (loom_train_grad_norm(2, grads, sizes, LOOM_DTYPE_F32, 1.0f, out, ws, ws_size) !=
      LOOM_STATUS_OK)
    return bad(__LINE__);
  if (loom_train_adamw(2, params, grads, m, v, NULL, sizes, decay, LOOM_DTYPE_F32, LOOM_DTYPE_F32,
                       lr, 0.9, 0.95, 1e-8, out + 1, step, ws, ws_size) != LOOM_STATUS_OK)
    return bad(__LINE__);
  float now[N];
  cudaMemcpy(now, dev[0], sizeof(now), cudaMemcpyDeviceToHost);
  cudaMemcpy(result, out, 8, cudaMemcpyDeviceToHost);
  cudaMemcpy(&count, step, 8, cudaMemcpyDeviceToHost);
  double sum = 0.0;
  for (int i = 0; i < N; ++i) sum += (double)host[1][i] * host[1][i];
  const double norm = sqrt(sum), scale = norm > 1.0 ? 1.0 / norm : 1.0;
  if (fabs(result[0] - norm) > 1e-6 * norm || fabs(result[1] - scale) > 1e-6 || count != 1)
    return bad(__LINE__);
  for (int i = 0; i < N; ++i) {
    const double g = scale * host[1][i];
    const double mi = 0.9 * host[2][i] + 0.1 * g, vi = 0.95 * host[3][i] + 0.05 * g * g;
    const double want = host[0][i] * (1.0 - (double)rate * (i < N0 ? 0.1 : 0.0)) -
                        rate * (mi / 0.1) / (sqrt(vi / 0.05) + 1e-8);
    if (fabs(now[i] - want) > 2e-6 * (1.0 + fabs(want - host[0][i]))) return bad(__LINE__);
  }
  printf("train_smoke ok\n");
  return 0;
}
