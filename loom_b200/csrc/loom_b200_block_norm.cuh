// loom_b200_block_norm.cuh -- the norms after and before a block of a network,
// fused with the block's gate and the residual's scale, and their gradients.
//
// With x the residual stream, h a block's output, rows of width D:
//
//   u = h * post_rstd * (post_weight + offset),   post_rstd = 1 / sqrt(mean(h^2) + eps)
//   y = residual_scale * x + branch_scale * gate * u
//   z = y * pre_rstd * (pre_weight + offset),     pre_rstd = 1 / sqrt(mean(y^2) + eps)
//
// Each part may be absent: no h (y is x and only z is made), no post norm
// (u = h), no gate, no weights, no pre norm (only y is made).
//
// HBM-bound: about a dozen operations an element on the 8 to 14 bytes that it
// has to read and write.  So a row is read once and stays in registers between
// its two sums: a row of up to 1024 elements belongs to one warp, a longer one
// to one CTA.
#pragma once

#include "loom_b200_launch.cuh"
#include "loom_b200_types.cuh"

namespace loomb {

constexpr int kRowMaxWidth = 32768;
constexpr int kRowWarps = 4;            // rows (warps) per CTA where a warp holds a row

struct BlockNorm {
  const void* x;                 // [rows, width] at x_stride; y's place in the backward pass
  const void* h;
  const void* gate;              // [rows / rows_per_gate, width] at gate_stride
  const void* post_weight;
  const void* pre_weight;
  int64_t x_stride, h_stride, gate_stride;
  int64_t rows, rows_per_gate;
  int width;
  int post_norm, pre_norm;
  float eps, offset, residual_scale, branch_scale;
};

struct BlockNormOut {
  void* y;
  void* z;
  float* post_rstd;
  float* pre_rstd;
};

// Sum over the threads of a row, the same bits in each of them.  `buf` holds
// two rounds of warp sums; consecutive sums alternate between them, so one
// barrier a sum is enough: a round is written again only after the barrier of
// the next one, which its readers have reached.
template <bool kWarp>
__device__ __forceinline__ float row_sum(float v, float (*buf)[32], int& round) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if constexpr (!kWarp) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
      float* b = buf[round];
      round ^= 1;
      if (lane == 0) b[threadIdx.x >> 5] = v;
      __syncthreads();
      v = lane < warps ? b[lane] : 0.0f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    }
  }
  return v;
}

// The NV groups of V elements of a row that a thread holds: group j starts at
// (j * threads + thread) * V.
template <int V, int NV, Cache kC, class T>
__device__ __forceinline__ void load_row(float (&f)[NV][V], const T* p, int width) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = (j * blockDim.x + threadIdx.x) * V;
    if (d < width) {
      load_vec<V, kC>(f[j], p + d);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[j][i] = 0.0f;
    }
  }
}
template <int V, int NV, class T>
__device__ __forceinline__ void store_row(T* p, const float (&f)[NV][V], int width) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = (j * blockDim.x + threadIdx.x) * V;
    if (d < width) store_vec<V, kKeep>(p + d, f[j]);
  }
}
template <int V, int NV, class T>
__device__ __forceinline__ void load_weight(float (&f)[NV][V], const T* p, float offset,
                                            int width) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) f[j][i] = 1.0f;
    return;
  }
  load_row<V, NV, kKeep>(f, p, width);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) f[j][i] += offset;
}

template <class Tx, class Tb, int V, int NV, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 32 * kRowWarps : 1024)
block_norm_kernel(const BlockNorm a, const BlockNormOut o) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  __shared__ float buf[2][32];
  int round = 0;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;
  const int width = a.width;
  const float mean = 1.0f / (float)width;
  float y[NV][V], u[NV][V], w[NV][V];
  load_row<V, NV, kStream>(y, static_cast<const Tx*>(a.x) + row * a.x_stride, width);
  if (a.h != nullptr) {
    load_row<V, NV, kStream>(u, static_cast<const Tb*>(a.h) + row * a.h_stride, width);
    float gate[NV][V];
    load_weight<V, NV>(gate, a.gate == nullptr
                                 ? nullptr
                                 : static_cast<const Tb*>(a.gate) +
                                       row / a.rows_per_gate * a.gate_stride,
                       0.0f, width);
    load_weight<V, NV>(w, static_cast<const Tb*>(a.post_weight), a.offset, width);
    float rstd = 1.0f;
    if (a.post_norm) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) sum = fmaf(u[j][i], u[j][i], sum);
      sum = row_sum<kWarp>(sum, buf, round);
      rstd = 1.0f / sqrtf(fmaf(sum, mean, a.eps));
      if (threadIdx.x == 0 && o.post_rstd != nullptr) o.post_rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float b = gate[j][i] * (u[j][i] * rstd * w[j][i]);
        y[j][i] = fmaf(a.branch_scale, b, a.residual_scale * y[j][i]);
      }
    store_row<V, NV>(static_cast<Tx*>(o.y) + row * width, y, width);
  }
  if (!a.pre_norm) return;
  load_weight<V, NV>(w, static_cast<const Tb*>(a.pre_weight), a.offset, width);
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fmaf(y[j][i], y[j][i], sum);
  sum = row_sum<kWarp>(sum, buf, round);
  const float rstd = 1.0f / sqrtf(fmaf(sum, mean, a.eps));
  if (threadIdx.x == 0 && o.pre_rstd != nullptr) o.pre_rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) y[j][i] = y[j][i] * rstd * w[j][i];
  store_row<V, NV>(static_cast<Tb*>(o.z) + row * width, y, width);
}

// ---------------------------------------------------------------------------
// gradients
//
//   n = y pre_rstd, t = dz w_pre:        d = dy + pre_rstd (t - n mean(t n)),  dx = residual_scale d
//   k = h post_rstd, e = branch gate d:  dh = post_rstd (e w_post - k mean(e w_post k))
//   dgate = branch d k w_post,  dpost_weight = sum over rows of e k,  dpre_weight = of dz n
//
// The rows are cut into chunks that lie within one gate row's run of rows, and
// a fixed number of row groups (CTAs or warps) walk the chunks.  A group keeps
// its columns' sums of the weights' gradients in fp32 registers over all its
// rows and leaves them as one row of the workspace; a gate row's gradient is
// summed over its run, written where the run is one chunk and left as a
// partial row else.  A second kernel adds the partial rows in a fixed order.

constexpr int kGradCtas = 296;          // two per SM

struct BlockNormGrad {
  const float* post_rstd;
  const float* pre_rstd;
  const void* dy;
  const void* dz;
  int64_t dy_stride, dz_stride;
  void* dx;
  void* dh;
  void* dgate;
  float* pre_rows;               // partial rows: one per row group
  float* post_rows;
  float* gate_rows;              // one per chunk, where a gate row has several
  int64_t chunks;
  int chunks_per_gate;
};

template <class Tx, class Tb, int V, int NV, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 32 * kRowWarps : 1024)
block_norm_grad_kernel(const BlockNorm a, const BlockNormGrad b) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  __shared__ float buf[2][32];
  int round = 0;
  const int width = a.width;
  const float mean = 1.0f / (float)width;
  const int64_t group = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t groups = (int64_t)gridDim.x * blockDim.y;
  float w_pre[NV][V], w_post[NV][V], s_pre[NV][V], s_post[NV][V];
  load_weight<V, NV>(w_pre, static_cast<const Tb*>(a.pre_weight), a.offset, width);
  load_weight<V, NV>(w_post, static_cast<const Tb*>(a.post_weight), a.offset, width);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) s_pre[j][i] = s_post[j][i] = 0.0f;

  for (int64_t chunk = group; chunk < b.chunks; chunk += groups) {
    const int64_t run = chunk / b.chunks_per_gate;
    const int64_t part = chunk - run * b.chunks_per_gate;
    const int64_t row0 = run * a.rows_per_gate + a.rows_per_gate * part / b.chunks_per_gate;
    const int64_t row1 = run * a.rows_per_gate + a.rows_per_gate * (part + 1) / b.chunks_per_gate;
    float gate[NV][V], s_gate[NV][V];
    load_weight<V, NV>(gate, a.gate == nullptr
                                 ? nullptr
                                 : static_cast<const Tb*>(a.gate) + run * a.gate_stride,
                       0.0f, width);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s_gate[j][i] = 0.0f;
    for (int64_t row = row0; row < row1; ++row) {
      float y[NV][V], d[NV][V];
      if (b.dy != nullptr) {
        load_row<V, NV, kStream>(d, static_cast<const Tx*>(b.dy) + row * b.dy_stride, width);
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) d[j][i] = 0.0f;
      }
      float h[NV][V];
      if (a.h != nullptr)
        load_row<V, NV, kStream>(h, static_cast<const Tb*>(a.h) + row * a.h_stride, width);
      if (a.pre_norm) {
        float t[NV][V];
        load_row<V, NV, kStream>(y, static_cast<const Tx*>(a.x) + row * a.x_stride, width);
        load_row<V, NV, kStream>(t, static_cast<const Tb*>(b.dz) + row * b.dz_stride, width);
        const float rstd = b.pre_rstd[row];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            y[j][i] *= rstd;
            s_pre[j][i] = fmaf(t[j][i], y[j][i], s_pre[j][i]);
            t[j][i] *= w_pre[j][i];
            sum = fmaf(t[j][i], y[j][i], sum);
          }
        sum = row_sum<kWarp>(sum, buf, round) * mean;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i)
            d[j][i] = fmaf(rstd, fmaf(-y[j][i], sum, t[j][i]), d[j][i]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) y[j][i] = a.residual_scale * d[j][i];
      store_row<V, NV>(static_cast<Tx*>(b.dx) + row * width, y, width);
      if (a.h == nullptr) continue;
      const float rstd = a.post_norm ? b.post_rstd[row] : 1.0f;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[j][i] *= rstd;
          d[j][i] *= a.branch_scale;
          s_gate[j][i] = fmaf(d[j][i], h[j][i] * w_post[j][i], s_gate[j][i]);
          d[j][i] *= gate[j][i];
          s_post[j][i] = fmaf(d[j][i], h[j][i], s_post[j][i]);
          d[j][i] *= w_post[j][i];
          sum = fmaf(d[j][i], h[j][i], sum);
        }
      if (a.post_norm) {
        sum = row_sum<kWarp>(sum, buf, round) * mean;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) d[j][i] = rstd * fmaf(-h[j][i], sum, d[j][i]);
      }
      store_row<V, NV>(static_cast<Tb*>(b.dh) + row * width, d, width);
    }
    if (b.dgate != nullptr) {
      if (b.chunks_per_gate == 1) {
        store_row<V, NV>(static_cast<Tb*>(b.dgate) + run * width, s_gate, width);
      } else {
        store_row<V, NV>(b.gate_rows + chunk * width, s_gate, width);
      }
    }
  }
  if (b.pre_rows != nullptr) store_row<V, NV>(b.pre_rows + group * width, s_pre, width);
  if (b.post_rows != nullptr) store_row<V, NV>(b.post_rows + group * width, s_post, width);
}

// Sums of partial rows by column: job 0 the pre weight's, job 1 the post
// weight's (each over `groups` rows), from job 2 on a gate row's (over its
// chunks).  32 columns and 8 strides of rows per CTA, the strides folded in
// order.
struct RowSums {
  const float* rows[3];
  void* out[3];
  int64_t groups;
  int chunks_per_gate;
  int width;
};

template <class Tb>
__global__ void __launch_bounds__(256) block_norm_sums_kernel(const RowSums s, int first_job) {
  wait_for_prerequisite_grid();
  allow_dependent_launch();
  __shared__ float part[8][32];
  const int job = first_job + blockIdx.y;
  const int kind = job < 2 ? job : 2;
  if (s.out[kind] == nullptr) return;
  const int64_t count = kind < 2 ? s.groups : s.chunks_per_gate;
  const int64_t line = kind < 2 ? 0 : job - 2;
  const int lane = threadIdx.x & 31, stride = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (d < s.width) {
    const float* p = s.rows[kind] + line * count * s.width + d;
    for (int64_t r = stride; r < count; r += 8) sum += p[r * s.width];
  }
  part[stride][lane] = sum;
  __syncthreads();
  if (stride == 0 && d < s.width) {
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += part[k][lane];
    static_cast<Tb*>(s.out[kind])[line * s.width + d] = narrow<Tb>(sum);
  }
}

// ---------------------------------------------------------------------------
// launchers

// Whether 8 elements at a time can be moved of every row of this array.
inline bool rows_by_8(const void* p, int64_t stride, int width) {
  return p == nullptr || (((uintptr_t)p & 15u) == 0 && stride % 8 == 0 && width % 8 == 0);
}

// How the rows of one launch lie on threads.
struct RowShape {
  int vec, per;        // elements per access, accesses per thread
  bool warp;           // a warp per row
  unsigned threads;    // per row
  dim3 block() const { return dim3(threads, warp ? kRowWarps : 1); }
};

inline RowShape row_shape(int width, bool by8) {
  RowShape s;
  s.vec = by8 ? 8 : 1;
  const int units = by8 ? width / 8 : width;
  const int warp_most = by8 ? 4 : 8;
  s.warp = units <= 32 * warp_most;
  if (s.warp) {
    s.per = by8 ? (units <= 32 ? 1 : units <= 64 ? 2 : 4) : 8;
    s.threads = 32;
    return s;
  }
  s.per = by8 ? (units <= 1024 ? 1 : units <= 2048 ? 2 : 4) : (units <= 8192 ? 8 : 32);
  s.threads = (unsigned)(ceil_div(ceil_div(units, s.per), 32) * 32);
  return s;
}

// Calls f with the shape as constants.
template <class F>
inline int with_shape(const RowShape& s, const F& f) {
  using std::integral_constant;
  if (s.vec == 8) {
    if (s.warp) {
      if (s.per == 1) return f(integral_constant<int, 8>(), integral_constant<int, 1>(), std::true_type());
      if (s.per == 2) return f(integral_constant<int, 8>(), integral_constant<int, 2>(), std::true_type());
      return f(integral_constant<int, 8>(), integral_constant<int, 4>(), std::true_type());
    }
    if (s.per == 1) return f(integral_constant<int, 8>(), integral_constant<int, 1>(), std::false_type());
    if (s.per == 2) return f(integral_constant<int, 8>(), integral_constant<int, 2>(), std::false_type());
    return f(integral_constant<int, 8>(), integral_constant<int, 4>(), std::false_type());
  }
  if (s.warp) return f(integral_constant<int, 1>(), integral_constant<int, 8>(), std::true_type());
  if (s.per == 8) return f(integral_constant<int, 1>(), integral_constant<int, 8>(), std::false_type());
  return f(integral_constant<int, 1>(), integral_constant<int, 32>(), std::false_type());
}

template <class Tx, class Tb>
inline int launch_block_norm(const BlockNorm& a, const BlockNormOut& o, cudaStream_t stream) {
  if (a.rows == 0) return LOOM_STATUS_OK;
  const int w = a.width;
  const bool by8 = rows_by_8(a.x, a.x_stride, w) && rows_by_8(a.h, a.h_stride, w) &&
                   rows_by_8(a.gate, a.gate_stride, w) && rows_by_8(a.post_weight, w, w) &&
                   rows_by_8(a.pre_weight, w, w) && rows_by_8(o.y, w, w) && rows_by_8(o.z, w, w);
  const RowShape s = row_shape(w, by8);
  const int64_t grid = s.warp ? ceil_div(a.rows, kRowWarps) : a.rows;
  if (grid > 0x7fffffff) return LOOM_STATUS_INVALID_ARGUMENT;
  return with_shape(s, [&](auto v, auto nv, auto warp) {
    return launch_dependent(
        block_norm_kernel<Tx, Tb, decltype(v)::value, decltype(nv)::value, decltype(warp)::value>,
        dim3((unsigned)grid), s.block(), stream, a, o);
  });
}

// The chunks of a backward pass: about one per row group, whole gate runs
// where there are more runs than groups.
inline int64_t grad_row_groups() { return (int64_t)kGradCtas * kRowWarps; }

inline int grad_chunks_per_gate(int64_t rows, int64_t gate_rows) {
  if (gate_rows <= 0 || rows <= 0) return 1;
  const int64_t run = rows / gate_rows;
  int64_t c = grad_row_groups() / gate_rows;
  if (c > run) c = run;
  return c < 1 ? 1 : (int)c;
}

inline size_t block_norm_grad_workspace_bytes(int64_t rows, int64_t width, int64_t gate_rows) {
  if (rows < 0 || width <= 0 || gate_rows < 0) return 0;
  const int c = grad_chunks_per_gate(rows, gate_rows);
  const int64_t lines = 2 * grad_row_groups() + (c > 1 ? gate_rows * c : 0);
  return (size_t)lines * (size_t)align_up((size_t)width, 8) * sizeof(float) + 256;
}

template <class Tx, class Tb>
inline int launch_block_norm_grad(const BlockNorm& a0, BlockNormGrad b, int64_t gate_rows,
                                  void* dpost_weight, void* dpre_weight, void* workspace,
                                  cudaStream_t stream) {
  BlockNorm a = a0;
  const int w = a.width;
  const bool by8 = rows_by_8(a.x, a.x_stride, w) && rows_by_8(a.h, a.h_stride, w) &&
                   rows_by_8(a.gate, a.gate_stride, w) && rows_by_8(a.post_weight, w, w) &&
                   rows_by_8(a.pre_weight, w, w) && rows_by_8(b.dy, b.dy_stride, w) &&
                   rows_by_8(b.dz, b.dz_stride, w) && rows_by_8(b.dx, w, w) &&
                   rows_by_8(b.dh, w, w) && rows_by_8(b.dgate, w, w);
  const RowShape s = row_shape(w, by8);
  const int64_t lanes = s.warp ? kRowWarps : 1;
  const int64_t runs = a.gate != nullptr ? gate_rows : 1;
  a.rows_per_gate = a.rows > 0 ? a.rows / runs : 1;
  b.chunks_per_gate = grad_chunks_per_gate(a.rows, runs);
  b.chunks = a.rows > 0 ? runs * b.chunks_per_gate : 0;
  int64_t grid = ceil_div(b.chunks, lanes);
  if (grid > kGradCtas) grid = kGradCtas;
  const int64_t groups = grid * lanes;
  float* rows = reinterpret_cast<float*>(workspace_base(workspace));
  b.pre_rows = dpre_weight != nullptr ? rows : nullptr;
  b.post_rows = dpost_weight != nullptr ? rows + grad_row_groups() * w : nullptr;
  b.gate_rows = rows + 2 * grad_row_groups() * w;
  if (grid > 0) {
    const int st = with_shape(s, [&](auto v, auto nv, auto warp) {
      return launch_dependent(block_norm_grad_kernel<Tx, Tb, decltype(v)::value,
                                                     decltype(nv)::value, decltype(warp)::value>,
                              dim3((unsigned)grid), s.block(), stream, a, b);
    });
    if (st != LOOM_STATUS_OK) return st;
  }
  RowSums sums;
  sums.rows[0] = rows;
  sums.rows[1] = rows + grad_row_groups() * w;
  sums.rows[2] = b.gate_rows;
  sums.out[0] = dpre_weight;
  sums.out[1] = dpost_weight;
  sums.out[2] = b.dgate;
  sums.groups = groups;
  sums.chunks_per_gate = b.chunks_per_gate;
  sums.width = w;
  const bool gate_jobs = b.dgate != nullptr && (b.chunks_per_gate > 1);
  const bool weights = dpre_weight != nullptr || dpost_weight != nullptr;
  const int first = weights ? 0 : 2;
  const int64_t jobs = (weights ? 2 : 0) + (gate_jobs ? runs : 0);
  if (jobs == 0) return LOOM_STATUS_OK;
  return launch_dependent(block_norm_sums_kernel<Tb>,
                          dim3((unsigned)ceil_div(w, 32), (unsigned)jobs), dim3(256), stream, sums,
                          first);
}

}  // namespace loomb
