// loom_b200_block_norm.cuh -- the norms after and before a block of a network,
// fused with the block's gate and the residual's scale, and their gradients.
//
// With x the residual stream, h a block's output, rows of width D:
//
//   u = h * post_rstd * (post_weight + offset),   post_rstd = 1 / sqrt(mean(h^2) + eps)
//   y = residual_scale * x + branch_scale * gate * u
//   z = y * pre_rstd * (pre_weight + offset),     pre_rstd = 1 / sqrt(mean(y^2) + eps)
//
// Each part may be absent: no h (y is x, unscaled, and only z is made), no post
// norm (u = h), no gate, no weights, no pre norm (only y is made).
//
// HBM-bound: about a dozen operations an element on the 8 to 14 bytes that it
// has to read and write.  So a row is read once and stays in registers between
// its two sums: a row of up to 256 elements belongs to one warp, a longer one
// to one CTA (a row group).  Row groups are persistent and walk the rows with a
// stride; their next rows are on the way to shared memory (cp.async) while one
// is computed, since a row's two sums are two barriers with nothing in flight.
// 8192 rows of 4096 bf16 elements with a gate row each: forward 56 us (the 335 MB
// it has to move take 51 at the copy rate), gradients 95 us (537 MB, 82); loading
// each row where it is needed took 115 and 266.
//
// Groups of eight elements move as one access whatever the width: they lie at
// multiples of eight elements from the array's start, not from the row's, so
// a row begins `phase` = row * width mod 8 elements into its first group.  The
// stride over the rows is a multiple of eight where the width is not, so each
// row group has one phase for all its rows and holds the weights, and the
// columns' sums of their gradients, at that phase in registers.
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

// Three sums at once, the same bits in each of the row's threads: the halving
// steps send two of four values away and keep two, then one and one, so that
// three values take six exchanges a level.
struct Sums3 {
  float a, b, c;
};
__device__ __forceinline__ float fold8(float v) {
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
template <bool kWarp>
__device__ __forceinline__ Sums3 row_sums(Sums3 s, float (*buf)[3][32], int& round) {
  const int lane = threadIdx.x & 31;
  const bool high = lane & 16, odd = lane & 8;
  // lanes 0..15 keep a and b, lanes 16..31 keep c (and nothing)
  const float first = (high ? s.c : s.a) + __shfl_xor_sync(0xffffffffu, high ? s.a : s.c, 16);
  const float second = (high ? 0.0f : s.b) + __shfl_xor_sync(0xffffffffu, high ? s.b : 0.0f, 16);
  // of these, lanes 0..7 keep a, 8..15 b, 16..23 c
  float v = (odd ? second : first) + __shfl_xor_sync(0xffffffffu, odd ? first : second, 8);
  v = fold8(v);
  if constexpr (!kWarp) {
    const int warps = blockDim.x >> 5;
    float(*b)[32] = buf[round];
    round ^= 1;
    const int which = lane >> 3, at = lane & 7;
    if (at == 0 && which < 3) b[which][threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    if (which < 3)
      for (int k = at; k < warps; k += 8) v += b[which][k];
    v = fold8(v);
  }
  return {__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 8),
          __shfl_sync(0xffffffffu, v, 16)};
}

// ---------------------------------------------------------------------------
// groups of eight elements, as four pairs

struct Group {
  F2 p[4];
};

__device__ __forceinline__ Group same(float v) {
  Group g;
#pragma unroll
  for (int i = 0; i < 4; ++i) g.p[i] = f2(v, v);
  return g;
}
__device__ __forceinline__ Group operator*(const Group& a, const Group& b) {
  Group r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = mul2(a.p[i], b.p[i]);
  return r;
}
__device__ __forceinline__ Group operator*(const Group& a, float b) {
  Group r;
  const F2 b2 = f2(b, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = mul2(a.p[i], b2);
  return r;
}
__device__ __forceinline__ Group operator+(const Group& a, const Group& b) {
  Group r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = add2(a.p[i], b.p[i]);
  return r;
}
// a * b + c
__device__ __forceinline__ Group fma8(const Group& a, const Group& b, const Group& c) {
  Group r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fma2(a.p[i], b.p[i], c.p[i]);
  return r;
}
__device__ __forceinline__ Group fma8(const Group& a, float b, const Group& c) {
  Group r;
  const F2 b2 = f2(b, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fma2(a.p[i], b2, c.p[i]);
  return r;
}
__device__ __forceinline__ F2 dot8(const Group& a, const Group& b, F2 sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = fma2(a.p[i], b.p[i], sum);
  return sum;
}

// kEdge false: each group lies wholly in the row (and in the staged kernels no
// thread is left over).  True: the first and the last group may be partly outside.
template <bool kEdge>
__device__ __forceinline__ bool inside(int e, int width) {
  return !kEdge || (e >= 0 && e + 8 <= width);
}
template <class T>
__device__ __forceinline__ Group unpack(const Raw8<T>& r) {
  Group g;
#pragma unroll
  for (int i = 0; i < 4; ++i) g.p[i] = pair_of(r, i);
  return g;
}
// Zero outside the row (where a copy leaves a neighbour's values).
template <bool kEdge>
__device__ __forceinline__ Group within(Group g, int e, int width) {
  if (!inside<kEdge>(e, width)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f = halves(g.p[i]);
      if (e + 2 * i < 0 || e + 2 * i >= width) f.x = 0.0f;
      if (e + 2 * i + 1 < 0 || e + 2 * i + 1 >= width) f.y = 0.0f;
      g.p[i] = f2(f.x, f.y);
    }
  }
  return g;
}
// The group of a row that begins `e` elements after the row's start (which may
// be before it), zero outside the row.  kAny: from any place, else each group is
// wholly inside or outside and at a 16-byte boundary.
template <bool kAny = true, class T>
__device__ __forceinline__ Group load_group(const T* row, int e, int width) {
  float f[8];
  if (kAny ? e >= 0 && e + 8 <= width && ((uintptr_t)(row + e) & 15u) == 0 : e < width) {
    load_vec<8, kKeep>(f, row + e);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = kAny && e + i >= 0 && e + i < width ? widen(row[e + i]) : 0.0f;
  }
  Group g;
#pragma unroll
  for (int i = 0; i < 4; ++i) g.p[i] = f2(f[2 * i], f[2 * i + 1]);
  return g;
}
// kPlaced: every whole group is at a 16-byte boundary.
template <bool kPlaced, bool kEdge, class T>
__device__ __forceinline__ void store_group(T* row, const Group& g, int e, int width) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 h = halves(g.p[i]);
    f[2 * i] = h.x;
    f[2 * i + 1] = h.y;
  }
  if (inside<kEdge>(e, width) && (kPlaced || ((uintptr_t)(row + e) & 15u) == 0)) {
    store_vec<8, kKeep>(row + e, f);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (e + i >= 0 && e + i < width) row[e + i] = narrow<T>(f[i]);
}
// A weight with its offset; ones where there is no weight.
template <class T>
__device__ __forceinline__ Group load_weight(const T* w, float offset, int e, int width) {
  if (w == nullptr) return same(1.0f);
  Group g = load_group(w, e, width);
#pragma unroll
  for (int i = 0; i < 4; ++i) g.p[i] = add2(g.p[i], f2(offset, offset));
  return g;
}

// The same as it lies in memory: 16-bit types in half the registers.
template <class T>
__device__ __forceinline__ Raw8<T> load_raw(const T* w, int e, int width) {
  float f[8];
  const Group g = w != nullptr ? load_group(w, e, width) : same(1.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 h = halves(g.p[i]);
    f[2 * i] = h.x;
    f[2 * i + 1] = h.y;
  }
  Raw8<T> r;
  store_vec<8, kKeep>(reinterpret_cast<T*>(r.word), f);
  return r;
}
// 16-byte words of a group of eight.
template <class T>
struct GroupWords {
  static constexpr int value = (int)sizeof(T) / 2;
};

// Starts the copy of a group; `slot` words lie `pitch` apart.  Bytes past the
// row's end are not read.  Bytes before its start (less than one group) are
// read: they belong to the row before it, as the caller's strides are at least
// a width and the phase is that of the row's own place.
template <bool kEdge, class T>
__device__ __forceinline__ void copy_group(uint4* slot, int pitch, const T* row, int e,
                                           int width) {
  const char* from = reinterpret_cast<const char*>(row + e);
  const int bytes = (width - e) * (int)sizeof(T);
#pragma unroll
  for (int k = 0; k < GroupWords<T>::value; ++k) {
    const int some = bytes - 16 * k;
    if (!kEdge || some >= 16) {
      copy16(slot + k * pitch, from + 16 * k);
    } else {
      copy16_some(slot + k * pitch, some > 0 ? from + 16 * k : from, some > 0 ? some : 0);
    }
  }
}
template <class T>
__device__ __forceinline__ Raw8<T> read_raw(const uint4* slot, int pitch) {
  Raw8<T> r;
#pragma unroll
  for (int k = 0; k < GroupWords<T>::value; ++k) r.word[k] = slot[k * pitch];
  return r;
}

template <class T>
__device__ __forceinline__ void store_raw(uint4* slot, int pitch, const Raw8<T>& r) {
#pragma unroll
  for (int k = 0; k < GroupWords<T>::value; ++k) slot[k * pitch] = r.word[k];
}

__device__ __forceinline__ void wait_stage(int stages) {
  if (stages == 4) {
    wait_copies<2>();
  } else if (stages == 3) {
    wait_copies<1>();
  } else {
    wait_copies<0>();
  }
}

__device__ __forceinline__ float total(F2 a) {
  const float2 h = halves(a);
  return h.x + h.y;
}
// Row starts: rows and strides are below 2^31, so one 32-bit product.
template <class T>
__device__ __forceinline__ const T* row_at(const void* p, int64_t row, int64_t stride) {
  return static_cast<const T*>(p) + (uint64_t)(uint32_t)row * (uint32_t)stride;
}
template <class T>
__device__ __forceinline__ T* row_at(void* p, int64_t row, int width) {
  return static_cast<T*>(p) + (uint64_t)(uint32_t)row * (uint32_t)width;
}

// How the rows of one launch lie on threads.
struct RowPlan {
  int per;             // groups of eight per thread
  bool warp;           // a warp per row, else a CTA
  bool edge;           // groups partly outside of a row, or threads left over
  int most;            // threads per CTA that the kernel is compiled for
  unsigned threads;    // per row
  int phased;          // groups lie at multiples of eight from the arrays' starts
  int stages;          // rows on their way at once, 2 to 4; 0: loaded where they are needed
  int64_t groups;      // row groups
  int64_t rows;        // forward: rows of a row group, eight apart; 0: every groups-th row
  size_t shared;       // bytes of the stages
  dim3 block() const { return dim3(threads, warp ? kRowWarps : 1); }
  dim3 grid() const { return dim3((unsigned)(warp ? (groups + kRowWarps - 1) / kRowWarps : groups)); }
};

// ---------------------------------------------------------------------------
// forward

// Stage of one thread: NV groups each of x, h and the gate (where it has a row
// per row).
template <class Tx, class Tb>
struct ForwardStage {
  static constexpr int x = 0, h = GroupWords<Tx>::value, gate = h + GroupWords<Tb>::value;
  static constexpr int words = gate + GroupWords<Tb>::value;
};

template <class Tx, class Tb, bool kStaged, bool kEdge, int NV, bool kWarp, int kMost>
__global__ void __launch_bounds__(kMost, kStaged ? (kMost == 256 ? 2 : 1) : kWarp ? 8 : 1024 / kMost)
block_norm_kernel(const BlockNorm a, const BlockNormOut o, const RowPlan plan) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  using Stage = ForwardStage<Tx, Tb>;
  extern __shared__ uint4 slots[];
  __shared__ float buf[2][32];
  int round = 0;
  const int64_t group = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (group >= plan.groups) return;  // whole warps of a CTA without barriers
  const int width = a.width, threads = blockDim.x, stages = plan.stages;
  const float mean = 1.0f / (float)width;
  const int phase = kEdge && plan.phased ? (int)((group * width) & 7) : 0;
  const int pitch = threads * blockDim.y;
  const bool has_h = a.h != nullptr, row_gate = a.gate != nullptr && a.rows_per_gate == 1;
  const bool run_gate = a.gate != nullptr && !row_gate;

  int e[NV];
  bool any[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    e[j] = (j * threads + (int)threadIdx.x) * 8 - phase;
    any[j] = (kStaged && !kEdge) || e[j] < width;
  }
  uint4* const mine = slots + threadIdx.y * threads + threadIdx.x;
  auto slot = [&](int stage, int j, int part) {
    return mine + ((stage * NV + j) * Stage::words + part) * pitch;
  };
  // All row groups walk the rows side by side (neighbouring rows at one time:
  // 54 against 63 us for 8192 x 4096 bf16 rows), unless that would give each row
  // another gate row; eight rows apart they still have one phase.
  const int64_t step = plan.rows > 0 ? 8 : plan.groups;
  const int64_t row0 = plan.rows > 0 ? (group >> 3) * 8 * plan.rows + (group & 7) : group;
  const int64_t row1 = plan.rows > 0 ? min(a.rows, row0 + 8 * plan.rows) : a.rows;
  auto copy = [&](int64_t row, int stage) {
    if (row < row1) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!any[j]) continue;
        copy_group<kEdge>(slot(stage, j, Stage::x), pitch, row_at<Tx>(a.x, row, a.x_stride), e[j],
                          width);
        if (has_h)
          copy_group<kEdge>(slot(stage, j, Stage::h), pitch, row_at<Tb>(a.h, row, a.h_stride),
                            e[j], width);
        if (row_gate)
          copy_group<kEdge>(slot(stage, j, Stage::gate), pitch,
                            row_at<Tb>(a.gate, row, a.gate_stride), e[j], width);
      }
    }
    copies_done();
  };
  if (kStaged)
    for (int s = 0; s < stages - 1; ++s) copy(row0 + step * s, s);
  Group w_post[NV], w_pre[NV], gate[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    w_post[j] = load_weight(static_cast<const Tb*>(a.post_weight), a.offset, e[j], width);
    w_pre[j] = load_weight(static_cast<const Tb*>(a.pre_weight), a.offset, e[j], width);
    gate[j] = same(1.0f);
  }

  int64_t run_end = 0;  // of the rows that the gate in registers serves
  int stage = 0;
  for (int64_t row = row0; row < row1; row += step) {
    Group y[NV], u[NV];
    if (run_gate && row >= run_end) {
      const uint32_t run = (uint32_t)row / (uint32_t)a.rows_per_gate;
      run_end = (run + 1) * a.rows_per_gate;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        gate[j] = load_group(row_at<Tb>(a.gate, run, a.gate_stride), e[j], width);
    }
    if (kStaged) wait_stage(stages);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!kStaged) {
        y[j] = load_group<kEdge>(row_at<Tx>(a.x, row, a.x_stride), e[j], width);
        if (has_h) u[j] = load_group<kEdge>(row_at<Tb>(a.h, row, a.h_stride), e[j], width);
        if (row_gate)
          gate[j] = load_group<kEdge>(row_at<Tb>(a.gate, row, a.gate_stride), e[j], width);
      } else if (any[j]) {
        y[j] = within<kEdge>(unpack(read_raw<Tx>(slot(stage, j, Stage::x), pitch)), e[j], width);
        if (has_h)
          u[j] = within<kEdge>(unpack(read_raw<Tb>(slot(stage, j, Stage::h), pitch)), e[j], width);
        if (row_gate)
          gate[j] = within<kEdge>(unpack(read_raw<Tb>(slot(stage, j, Stage::gate), pitch)), e[j],
                                  width);
      } else {
        y[j] = u[j] = same(0.0f);
      }
    }
    if (kStaged) {
      // into the stage that the row before this one was read from
      copy(row + step * (stages - 1), stage == 0 ? stages - 1 : stage - 1);
      stage = stage == stages - 1 ? 0 : stage + 1;
    }
    // the statistics by rsqrtf, within 2 ulp: rounded correctly (__frsqrt_rn) they
    // cost short rows most (65536 x 128 bf16: 32.7 against 29.0 us)
    if (has_h) {
      float rstd = 1.0f;
      if (a.post_norm) {
        F2 sum = f2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j) sum = dot8(u[j], u[j], sum);
        rstd = rsqrtf(fmaf(row_sum<kWarp>(total(sum), buf, round), mean, a.eps));
        if (threadIdx.x == 0 && o.post_rstd != nullptr) o.post_rstd[row] = rstd;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        y[j] = fma8(u[j] * rstd * w_post[j] * gate[j], a.branch_scale, y[j] * a.residual_scale);
        if (any[j])
          store_group<kStaged || !kEdge, kEdge>(row_at<Tx>(o.y, row, width), y[j], e[j], width);
      }
    }
    if (!a.pre_norm) continue;
    F2 sum = f2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < NV; ++j) sum = dot8(y[j], y[j], sum);
    const float rstd = rsqrtf(fmaf(row_sum<kWarp>(total(sum), buf, round), mean, a.eps));
    if (threadIdx.x == 0 && o.pre_rstd != nullptr) o.pre_rstd[row] = rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (any[j])
        store_group<kStaged || !kEdge, kEdge>(row_at<Tb>(o.z, row, width),
                                              y[j] * rstd * w_pre[j], e[j], width);
  }
  if (kStaged) wait_copies<0>();
}

// ---------------------------------------------------------------------------
// gradients
//
//   n = y pre_rstd, t = dz w_pre:        d = dy + pre_rstd (t - n mean(t n)),  dx = residual_scale d
//   k = h post_rstd, q = branch gate d:  dh = post_rstd (q w_post - k mean(q w_post k))
//   dgate = branch d k w_post,  dpost_weight = sum over rows of q k,  dpre_weight = of dz n
//
// The second mean would wait for the first.  With f = dy + pre_rstd t and
// c = branch gate w_post, q w_post = c d = c (f - pre_rstd mean(t n) n), so that
//
//   mean(q w_post k) = mean(c f k) - pre_rstd mean(t n) mean(c n k)
//
// and a row takes one round of three sums; the terms are those that d itself
// is made of, so nothing cancels that does not in d.
//
// A row group keeps its columns' sums of the weights' gradients in fp32
// registers over all its rows and leaves them as one row of the workspace.
// Where a gate row serves a run of rows, the run's rows are dealt to
// `chunks_per_gate` chunks, and a row group walks whole chunks: the gate row's
// gradient is written where the run is one chunk, and left as a partial row
// else.  A second kernel adds the partial rows in a fixed order.

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
  int64_t chunks;                // runs * chunks_per_gate; without runs, the row groups
  int64_t run_rows;              // rows of a run
  int chunks_per_gate;
};

// The rows of a row group, chunk after chunk.
struct RowWalk {
  int64_t chunk, row, end;
  __device__ __forceinline__ void enter(const BlockNormGrad& b) {
    if (chunk >= b.chunks) {
      row = -1;
      return;
    }
    const uint32_t run = (uint32_t)chunk / (uint32_t)b.chunks_per_gate;  // below 2^31, all
    row = run * b.run_rows + (chunk - (int64_t)run * b.chunks_per_gate);
    end = (run + 1) * b.run_rows;
  }
  __device__ __forceinline__ void next(const BlockNormGrad& b, int64_t groups) {
    if (row < 0) return;
    row += b.chunks_per_gate;
    if (row >= end) {
      chunk += groups;
      enter(b);
    }
  }
};

template <class Tx, class Tb>
struct GradStage {
  static constexpr int y = 0, dy = GroupWords<Tx>::value, h = dy + GroupWords<Tx>::value;
  static constexpr int dz = h + GroupWords<Tb>::value, gate = dz + GroupWords<Tb>::value;
  static constexpr int words = gate + GroupWords<Tb>::value;
};

// Where the gate's rows are: none, one per row, one per run of rows.
enum Gate : int { kNoGate = 0, kRowGate = 1, kRunGate = 2 };

// kWhole: both norms, h and dy are there (tests of them in the loop are a third
// of the instructions: 103 against 119 us for 8192 x 4096 bf16 rows).
template <class Tx, class Tb, bool kStaged, bool kEdge, int NV, bool kWarp, int kMost, Gate kGate,
          bool kWhole>
__global__ void __launch_bounds__(kMost, kMost == 256 ? 2 : 1)
block_norm_grad_kernel(const BlockNorm a, const BlockNormGrad b, const RowPlan plan) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  using Stage = GradStage<Tx, Tb>;
  extern __shared__ uint4 slots[];
  __shared__ float buf[2][3][32];
  int round = 0;
  const int64_t group = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t groups = plan.groups;
  if (group >= groups) return;  // whole warps of a CTA without barriers
  const int width = a.width, threads = blockDim.x, stages = plan.stages;
  const float mean = 1.0f / (float)width;
  const int phase = kEdge && plan.phased ? (int)((group * width) & 7) : 0;
  const int pitch = threads * blockDim.y;
  const bool has_h = kWhole || a.h != nullptr, has_dy = kWhole || b.dy != nullptr;
  const float post_offset = a.post_weight != nullptr ? a.offset : 0.0f;
  const float pre_offset = a.pre_weight != nullptr ? a.offset : 0.0f;
  const bool pre_norm = kWhole || a.pre_norm, post_norm = kWhole || (a.post_norm && has_h);

  int e[NV];
  bool any[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    e[j] = (j * threads + (int)threadIdx.x) * 8 - phase;
    any[j] = !kEdge || e[j] < width;
  }
  uint4* const mine = slots + threadIdx.y * threads + threadIdx.x;
  auto slot = [&](int stage, int j, int part) {
    return mine + ((stage * NV + j) * Stage::words + part) * pitch;
  };
  auto copy = [&](int64_t row, int stage) {
    if (row >= 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!any[j]) continue;
        if (pre_norm) {
          copy_group<kEdge>(slot(stage, j, Stage::y), pitch, row_at<Tx>(a.x, row, a.x_stride),
                            e[j], width);
          copy_group<kEdge>(slot(stage, j, Stage::dz), pitch, row_at<Tb>(b.dz, row, b.dz_stride),
                            e[j], width);
        }
        if (has_dy)
          copy_group<kEdge>(slot(stage, j, Stage::dy), pitch, row_at<Tx>(b.dy, row, b.dy_stride),
                            e[j], width);
        if (has_h)
          copy_group<kEdge>(slot(stage, j, Stage::h), pitch, row_at<Tb>(a.h, row, a.h_stride),
                            e[j], width);
        if (kGate == kRowGate)
          copy_group<kEdge>(slot(stage, j, Stage::gate), pitch,
                            row_at<Tb>(a.gate, row, a.gate_stride), e[j], width);
      }
    }
    copies_done();
  };
  // a group of this row, from its stage or from memory
  auto fetch = [&](auto type, const void* p, int64_t row, int64_t stride, int stage, int j,
                   int part) {
    using T = decltype(type);
    if (!kStaged) return load_group(row_at<T>(p, row, stride), e[j], width);
    if (!any[j]) return same(0.0f);
    return within<kEdge>(unpack(read_raw<T>(slot(stage, j, part), pitch)), e[j], width);
  };
  RowWalk ahead = {group, 0, 0}, now = {group, 0, 0};
  ahead.enter(b);
  now.enter(b);
  for (int s = 0; kStaged && s < stages - 1; ++s) {
    copy(ahead.row, s);
    ahead.next(b, groups);
  }
  Raw8<Tb> gate[NV];
  Group s_pre[NV], s_post[NV], s_gate[NV];
  // Where registers are short (two groups a thread, or 1024 threads) the weights
  // stay in shared memory, each thread's own beside its stages, or where they are.
  constexpr bool kHold = kStaged && NV == 1 && kMost < 1024;
  Group held[kHold ? 2 : 1];
  auto weight_slot = [&](int j, int part) {
    return mine + ((stages * NV * Stage::words) + (j * 2 + part) * GroupWords<Tb>::value) * pitch;
  };
  auto weight = [&](int j, int part) {
    if (kHold) return held[kHold ? part : 0];
    if (!kStaged)
      return load_weight(static_cast<const Tb*>(part ? a.post_weight : a.pre_weight), a.offset,
                         e[j], width);
    const float offset = part ? post_offset : pre_offset;
    Group w = unpack(read_raw<Tb>(weight_slot(j, part), pitch));
#pragma unroll
    for (int i = 0; i < 4; ++i) w.p[i] = add2(w.p[i], f2(offset, offset));
    return w;
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (kHold) {
      held[0] = load_weight(static_cast<const Tb*>(a.pre_weight), a.offset, e[j], width);
      held[kHold ? 1 : 0] =
          load_weight(static_cast<const Tb*>(a.post_weight), a.offset, e[j], width);
    } else if (kStaged) {
      store_raw(weight_slot(j, 0), pitch,
                load_raw(static_cast<const Tb*>(a.pre_weight), e[j], width));
      store_raw(weight_slot(j, 1), pitch,
                load_raw(static_cast<const Tb*>(a.post_weight), e[j], width));
    }
    gate[j] = load_raw(static_cast<const Tb*>(nullptr), e[j], width);
    s_pre[j] = s_post[j] = s_gate[j] = same(0.0f);
  }

  int64_t chunk = -1;
  int stage = 0;
  while (now.row >= 0) {
    const int64_t row = now.row;
    if (kGate == kRunGate && now.chunk != chunk) {
      chunk = now.chunk;
      const Tb* from = row_at<Tb>(
          a.gate, (uint32_t)chunk / (uint32_t)b.chunks_per_gate, a.gate_stride);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        gate[j] = load_raw(from, e[j], width);
        s_gate[j] = same(0.0f);
      }
    }
    const float pre_rstd = pre_norm ? b.pre_rstd[row] : 1.0f;
    const float post_rstd = post_norm ? b.post_rstd[row] : 1.0f;
    if (kStaged) {
      wait_stage(stages);
      // into the stage that the row before this one was read from
      copy(ahead.row, stage == 0 ? stages - 1 : stage - 1);
      ahead.next(b, groups);
    }
    Group f[NV], n[NV], k[NV];
    F2 tn = f2(0.0f, 0.0f), cfk = tn, cnk = tn;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      f[j] = n[j] = k[j] = same(0.0f);
      if (has_dy) f[j] = fetch(Tx(), b.dy, row, b.dy_stride, stage, j, Stage::dy);
      if (pre_norm) {
        n[j] = fetch(Tx(), a.x, row, a.x_stride, stage, j, Stage::y) * pre_rstd;
        Group t = fetch(Tb(), b.dz, row, b.dz_stride, stage, j, Stage::dz);
        s_pre[j] = fma8(t, n[j], s_pre[j]);
        t = t * weight(j, 0);
        tn = dot8(t, n[j], tn);
        f[j] = fma8(t, pre_rstd, f[j]);
      }
      if (has_h) {
        k[j] = fetch(Tb(), a.h, row, a.h_stride, stage, j, Stage::h) * post_rstd;
        if (kGate == kRowGate) {
          if (!kStaged) gate[j] = load_raw(row_at<Tb>(a.gate, row, a.gate_stride), e[j], width);
          else if (any[j]) gate[j] = read_raw<Tb>(slot(stage, j, Stage::gate), pitch);
        }
        if (post_norm) {
          Group c = weight(j, 1) * k[j];
          if (kGate != kNoGate) c = c * within<kEdge>(unpack(gate[j]), e[j], width);
          cfk = dot8(c, f[j], cfk);
          cnk = dot8(c, n[j], cnk);
        }
      }
    }
    float pull = 0.0f, post_pull = 0.0f;  // the means, with their signs
    if (pre_norm || post_norm) {
      const Sums3 s = row_sums<kWarp>({total(tn), total(cfk), total(cnk)}, buf, round);
      pull = -pre_rstd * (s.a * mean);
      post_pull = -(fmaf(pull, s.c, s.b) * (mean * a.branch_scale));
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Group d = fma8(n[j], pull, f[j]);
      if (any[j])
        store_group<kStaged, kEdge>(row_at<Tx>(b.dx, row, width), d * a.residual_scale, e[j],
                                    width);
      if (has_h) {
        const Group scaled = d * a.branch_scale, own = scaled * k[j];
        const Group w = weight(j, 1);
        Group through = scaled, sum = own;  // with the gate
        if (kGate != kNoGate) {
          const Group g = within<kEdge>(unpack(gate[j]), e[j], width);
          through = scaled * g;
          sum = own * g;
        }
        if (kGate == kRowGate) {
          if (any[j])
            store_group<kStaged, kEdge>(row_at<Tb>(b.dgate, row, width), own * w, e[j], width);
        } else if (kGate == kRunGate) {
          s_gate[j] = fma8(own, w, s_gate[j]);
        }
        s_post[j] = s_post[j] + sum;
        // without the post norm h has no part in it, not even one that is not finite
        Group dh = through * w;
        if (post_norm) dh = fma8(k[j], post_pull, dh) * post_rstd;
        if (any[j])
          store_group<kStaged, kEdge>(row_at<Tb>(b.dh, row, width), dh, e[j], width);
      }
    }
    stage = stage == stages - 1 ? 0 : stage + 1;
    now.next(b, groups);
    if (kGate == kRunGate && now.chunk != chunk) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!any[j]) continue;
        if (b.chunks_per_gate == 1) {
          store_group<false, true>(row_at<Tb>(b.dgate, chunk, width), s_gate[j], e[j], width);
        } else {
          store_group<false, true>(row_at<float>(b.gate_rows, chunk, width), s_gate[j], e[j],
                                   width);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!any[j]) continue;
    if (b.pre_rows != nullptr)
      store_group<false, true>(b.pre_rows + group * width, s_pre[j], e[j], width);
    if (b.post_rows != nullptr)
      store_group<false, true>(b.post_rows + group * width, s_post[j], e[j], width);
  }
  if (kStaged) wait_copies<0>();
}

// Sums of partial rows by column: job 0 the pre weight's, job 1 the post
// weight's (each over `groups` rows), from job 2 on a gate row's (over its
// chunks).  A CTA has 32 columns; each of its warps adds every
// kSumWarps-th row, and the warps' sums of a column are added in a fixed tree.  It reads at most a few
// MB from the second-level cache and is bound by that latency, hence the many
// warps: 32768 x 512 bf16 rows' gradients take 46 us with 32 of them, 49 with 16
// and 56 with 8; from 4096 columns on 16 do it (2048 x 8192: 44 against 47).
struct RowSums {
  const float* rows[3];
  void* out[3];
  int64_t groups;
  int chunks_per_gate;
  int width;
};

constexpr int kSumColumns = 32;

template <class Tb, int kSumWarps>
__global__ void __launch_bounds__(32 * kSumWarps) block_norm_sums_kernel(const RowSums s, int first_job) {
  wait_for_prerequisite_grid();
  allow_dependent_launch();
  __shared__ float part[kSumWarps][kSumColumns + 1];
  const int job = first_job + blockIdx.y;
  const int kind = job < 2 ? job : 2;
  if (s.out[kind] == nullptr) return;
  const int64_t count = kind < 2 ? s.groups : s.chunks_per_gate;
  const int64_t line = kind < 2 ? 0 : job - 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.x * kSumColumns;
  float sum = 0.0f;
  if (first + lane < s.width) {
    const float* p = s.rows[kind] + line * count * s.width + first + lane;
#pragma unroll 4
    for (int64_t r = warp; r < count; r += kSumWarps) sum += p[r * s.width];
  }
  part[warp][lane] = sum;
  __syncthreads();
  const int column = threadIdx.x / kSumWarps, at = threadIdx.x % kSumWarps;
  sum = part[at][column];
#pragma unroll
  for (int off = kSumWarps / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (at == 0 && first + column < s.width)
    static_cast<Tb*>(s.out[kind])[line * s.width + first + column] = narrow<Tb>(sum);
}

// ---------------------------------------------------------------------------
// launchers

constexpr int kSmCount = 148;                  // of a B200
constexpr size_t kStageBytes = 220 * 1024;     // shared memory of an SM that stages may take

// Whether an array's rows have the phase of contiguous ones: copies then find
// every group at a 16-byte boundary, and what lies before a row's first
// element is the row before it.
inline bool in_phase(const void* p, int64_t stride, int64_t rows, int width) {
  return p == nullptr || (((uintptr_t)p & 15u) == 0 &&
                          (rows <= 1 || (stride >= width && (stride - width) % 8 == 0)));
}

// `words`, `fixed`: 16-byte words per thread and group of eight, of a stage and
// beside the stages; `resident`: threads per SM that the kernel's registers
// allow, about; `per`: groups per thread of a staged CTA; `stage`: whether rows
// come through stages at all.
inline RowPlan row_plan(int width, bool phased, bool stage, int words, int fixed, int resident,
                        int per, bool backward) {
  RowPlan s = {};
  s.phased = phased;
  const int units = phased && width % 8 != 0 ? (width + 14) / 8 : (width + 7) / 8;
  for (int staged = phased && stage ? 1 : 0;; --staged) {
    s.warp = units <= 32;
    if (s.warp) {
      s.per = 1;
      s.threads = 32;
      s.most = 32 * kRowWarps;
    } else {
      if (staged) {
        s.per = per;
        s.most = units <= 512 ? 512 / per : units <= 1024 ? 1024 / per : 1024;
      } else {
        s.per = units <= 1024 ? 1 : 4;
        s.most = units <= 512 ? 512 : 1024;
      }
      s.threads = (unsigned)(ceil_div(ceil_div(units, s.per), 32) * 32);
    }
    const int threads = (int)s.threads * (s.warp ? kRowWarps : 1);
    int ctas = resident / threads;
    if (ctas < 1) ctas = 1;
    // weights beside the stages: see kHold
    const bool beside = staged && (s.per > 1 || s.most == 1024);
    const size_t held = beside ? (size_t)s.per * fixed * 16 * threads : 0;
    s.edge = width % 8 != 0 || (staged ? units != (int)s.threads * s.per : !phased || backward);
    if (staged) {
      const size_t bytes = (size_t)s.per * words * 16 * threads;
      // wider than the staged kernels go, or than shared memory holds two rows of
      if (threads > s.most || (per == 2 && backward && s.most == 1024) ||
          2 * bytes + held > kStageBytes)
        continue;
      if ((2 * bytes + held) * ctas > kStageBytes) ctas = (int)(kStageBytes / (2 * bytes + held));
      const size_t fit = (kStageBytes / ctas - held) / bytes;
      s.stages = fit < 4 ? (int)fit : 4;
      s.shared = (size_t)s.stages * bytes;
    } else if (units > 4096) {
      // an odd width whose shifted groups pass the widest CTA: unshifted
      return row_plan(width, false, false, words, fixed, resident, per, backward);
    }
    s.shared += held;
    s.groups = (int64_t)kSmCount * ctas * (s.warp ? kRowWarps : 1);
    return s;
  }
}

// A row group that takes several rows of one phase steps by a multiple of
// eight rows, unless every row has it.
inline int64_t step_groups(int64_t groups, int64_t rows, int width, bool phased) {
  if (groups >= rows) return rows;
  return phased && width % 8 != 0 && groups >= 8 ? groups / 8 * 8 : groups;
}

template <class Kern, class... Args>
inline int launch_rows(Kern kernel, const RowPlan& s, cudaStream_t stream, const Args&... args) {
  // Without the attribute 48 KiB, the kernel's own (under 1 KiB) among them.  It
  // belongs to the function, which serves many widths and host threads: every
  // call asks for the most that any plan takes, so none lowers another's.
  if (s.shared > 47 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)kStageBytes) != cudaSuccess) {
    cudaGetLastError();
    return LOOM_STATUS_CUDA_ERROR;
  }
  return launch_dependent(kernel, s.grid(), s.block(), stream, s.shared, args..., s);
}

// Calls f with the plan as constants.
template <bool kBackward, class F>
inline int with_plan(const RowPlan& s, const F& f) {
  using std::integral_constant;
  const std::true_type yes;
  const std::false_type no;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  const integral_constant<int, 4> four;
  const integral_constant<int, 32 * kRowWarps> warps;
  const integral_constant<int, 256> quarter;
  const integral_constant<int, 512> half;
  const integral_constant<int, 1024> full;
  if (s.stages == 0) {
    if (s.per == 4) return f(no, yes, four, no, full);
    auto direct = [&](auto edge) {
      return s.warp          ? f(no, edge, one, yes, warps)
             : s.most == 512 ? f(no, edge, one, no, half)
                             : f(no, edge, one, no, full);
    };
    if constexpr (!kBackward)
      if (!s.edge) return direct(no);
    return direct(yes);
  }
  auto staged = [&](auto edge) {
    if (s.warp) return f(yes, edge, one, yes, warps);
    if (s.per == 2 && s.most == 256) return f(yes, edge, two, no, quarter);
    if (s.per == 2 && s.most == 512) return f(yes, edge, two, no, half);
    if constexpr (kBackward) {
      return s.most == 512 ? f(yes, edge, one, no, half) : f(yes, edge, one, no, full);
    } else {
      return f(yes, edge, two, no, full);
    }
  };
  return s.edge ? staged(yes) : staged(no);
}

template <class Tx, class Tb>
int launch_block_norm(const BlockNorm& a, const BlockNormOut& o, cudaStream_t stream) {
  const int w = a.width;
  const bool row_gate = a.gate != nullptr && a.rows_per_gate == 1;
  const bool phased = in_phase(a.x, a.x_stride, a.rows, w) &&
                      in_phase(a.h, a.h_stride, a.rows, w) &&
                      (!row_gate || in_phase(a.gate, a.gate_stride, a.rows, w)) &&
                      in_phase(o.y, w, a.rows, w) && in_phase(o.z, w, a.rows, w);
  // two groups a thread and 512 threads an SM: with one group and twice the
  // threads the registers spill (62 against 54 us for 8192 x 4096 bf16 rows).
  // Where there are hardly more rows than row groups, nothing is gained by
  // staging: every row has a CTA or a warp of its own.
  RowPlan s = row_plan(w, phased, true, ForwardStage<Tx, Tb>::words, 0, 512, 2, false);
  // Unstaged against staged, us in a graph, a gate row per row.  Up to here: 1533
  // rows of 1024, fp32 beside bf16, 6.1 against 7.3; of 1040, which leave threads
  // over, 6.7 against 9.2; of 1000, 6.5 against 9.0; of 511, 8.4 against 8.6.  Past
  // it: 3000 bf16 rows of 1024 10.4 against 8.2; of 1023, fp32 beside bf16, 23.3
  // against 16.6.  The rule is one for all types: it loses up to a quarter with odd
  // bf16 rows below it (1533 of 1023: 10.4 against 9.3; of 255: 6.5 against 5.3) and
  // more with fp32 rows beside fp32 past it (3000 of 1024: 12.6 against 20.5).
  if (s.stages == 0 || a.rows <= (w > 1088 ? 1 : s.edge ? 3 : 2) * s.groups) {
    s = row_plan(w, phased, false, 0, 0, 1024, 1, false);
    s.groups = a.rows;
  }
  s.groups = step_groups(s.groups, a.rows, w, s.phased);
  if (a.gate != nullptr && !row_gate && s.groups < a.rows && a.rows_per_gate < s.groups) {
    s.rows = ceil_div(a.rows, s.groups / 8 * 8);
    s.groups = ceil_div(a.rows, 8 * s.rows) * 8;
  }
  return with_plan<false>(s, [&](auto staged, auto edge, auto per, auto warp, auto most) {
    return launch_rows(block_norm_kernel<Tx, Tb, decltype(staged)::value, decltype(edge)::value,
                                         decltype(per)::value, decltype(warp)::value,
                                         decltype(most)::value>,
                       s, stream, a, o);
  });
}

// Rows that a row group of the backward pass takes at least, where the SMs have
// one group each: it leaves a partial row for them (777 x 1535 fp16 rows: 16.4 us
// with 2, 17.6 with 4, 21 with 8).
constexpr int kGroupRows = 2;

// Row groups of the backward pass at most (partial rows of the workspace).
inline int64_t grad_groups_most(int64_t rows, int64_t width) {
  const int64_t most = width <= 1024 ? (int64_t)kSmCount * 8 : (int64_t)kSmCount * 2;
  return rows < most ? rows : most;
}

inline size_t block_norm_grad_workspace_bytes(int64_t rows, int64_t width, int64_t gate_rows) {
  if (rows < 0 || width <= 0 || gate_rows < 0) return 0;
  const int64_t lines = grad_groups_most(rows, width) * (gate_rows > 0 ? 3 : 2);
  return (size_t)lines * (size_t)width * sizeof(float) + 512;
}

template <class Tx, class Tb>
int launch_block_norm_grad(const BlockNorm& a0, BlockNormGrad b, int64_t gate_rows,
                                  void* dpost_weight, void* dpre_weight, void* workspace,
                                  cudaStream_t stream) {
  BlockNorm a = a0;
  if (a.h == nullptr) a.residual_scale = 1.0f;  // y is x: nothing scaled it
  const int w = a.width;
  const int64_t rows = a.rows, most = grad_groups_most(rows, w);
  a.rows_per_gate = a.gate != nullptr && rows > 0 ? rows / gate_rows : rows;
  const bool row_gate = a.gate != nullptr && a.rows_per_gate == 1;
  const int64_t runs = a.gate != nullptr && !row_gate ? gate_rows : 1;
  b.run_rows = runs > 0 ? rows / runs : rows;
  bool phased = in_phase(a.x, a.x_stride, rows, w) && in_phase(a.h, a.h_stride, rows, w) &&
                (!row_gate || in_phase(a.gate, a.gate_stride, rows, w)) &&
                in_phase(b.dy, b.dy_stride, rows, w) && in_phase(b.dz, b.dz_stride, rows, w) &&
                in_phase(b.dx, w, rows, w) && in_phase(b.dh, w, rows, w) &&
                (!row_gate || in_phase(b.dgate, w, rows, w));
  // chunks of several runs have one phase where runs and chunks keep it
  if (w % 8 != 0 && runs > 1 && (b.run_rows % 8 != 0 || 8 * runs > most)) phased = false;
  // Two groups a thread and 256 threads: two CTAs share an SM and cover each
  // other's barriers (8192 x 4096 bf16 rows: 95 against 105 us); with edges or a
  // gate row's sums beside, the registers spill (25 against 16 us for 777 x 1535
  // fp16 rows), and few or narrow rows gain nothing (2048 wide: 53 against 47).
  const bool run_gate = a.gate != nullptr && !row_gate;
  const bool two = w % 8 == 0 && !run_gate && (w > 4096 || (w > 2048 && rows >= 2048));
  RowPlan s = row_plan(w, phased, true, GradStage<Tx, Tb>::words, 2 * GroupWords<Tb>::value, 512,
                       two ? 2 : 1, true);
  if (!(a.h != nullptr && b.dy != nullptr && a.pre_norm && a.post_norm)) s.edge = true;
  int64_t groups = ceil_div(rows, (int64_t)kGroupRows);
  if (groups < kSmCount) groups = kSmCount;
  if (groups > s.groups) groups = s.groups;
  if (groups > most) groups = most;
  if (runs == 1) {
    groups = step_groups(groups, rows, w, s.phased);
    b.chunks_per_gate = (int)groups;
    b.chunks = groups;
  } else {
    int64_t c = groups / runs;
    if (s.phased && w % 8 != 0) c = c < 8 ? 8 : c / 8 * 8;
    if (c > b.run_rows) c = b.run_rows;
    b.chunks_per_gate = (int)(c < 1 ? 1 : c);
    b.chunks = runs * b.chunks_per_gate;
    groups = step_groups(groups, b.chunks, w, s.phased);
  }
  s.groups = groups;
  float* partial = reinterpret_cast<float*>(workspace_base(workspace));
  b.pre_rows = dpre_weight != nullptr ? partial : nullptr;
  b.post_rows = dpost_weight != nullptr ? partial + most * w : nullptr;
  b.gate_rows = partial + 2 * most * w;
  if (rows > 0) {
    const bool whole = a.h != nullptr && b.dy != nullptr && a.pre_norm && a.post_norm;
    const int st = with_plan<true>(s, [&](auto staged, auto edge, auto per, auto warp, auto most) {
      auto launch = [&](auto gate, auto all) {
        return launch_rows(
            block_norm_grad_kernel<Tx, Tb, decltype(staged)::value, decltype(edge)::value,
                                   decltype(per)::value, decltype(warp)::value,
                                   decltype(most)::value, (Gate)decltype(gate)::value,
                                   decltype(all)::value>,
            s, stream, a, b);
      };
      auto by_gate = [&](auto all) {
        if constexpr (decltype(per)::value != 2)  // `two` above leaves run gates out
          if (run_gate) return launch(std::integral_constant<int, kRunGate>(), all);
        return row_gate ? launch(std::integral_constant<int, kRowGate>(), all)
                        : launch(std::integral_constant<int, kNoGate>(), all);
      };
      if constexpr (decltype(staged)::value)
        if (whole) return by_gate(std::true_type());
      if constexpr (decltype(edge)::value) return by_gate(std::false_type());
      return (int)LOOM_STATUS_CUDA_ERROR;
    });
    if (st != LOOM_STATUS_OK) return st;
  }
  RowSums sums;
  sums.rows[0] = partial;
  sums.rows[1] = partial + most * w;
  sums.rows[2] = b.gate_rows;
  sums.out[0] = dpre_weight;
  sums.out[1] = dpost_weight;
  sums.out[2] = b.dgate;
  sums.groups = rows > 0 ? groups : 0;
  sums.chunks_per_gate = b.chunks_per_gate;
  sums.width = w;
  const bool gate_jobs = b.dgate != nullptr && !row_gate && b.chunks_per_gate > 1;
  const bool weights = dpre_weight != nullptr || dpost_weight != nullptr;
  const int first = weights ? 0 : 2;
  const int64_t jobs = (weights ? 2 : 0) + (gate_jobs ? runs : 0);
  if (jobs == 0) return LOOM_STATUS_OK;
  const dim3 grid((unsigned)ceil_div(w, kSumColumns), (unsigned)jobs);
  return w >= 4096 ? launch_dependent(block_norm_sums_kernel<Tb, 16>, grid, dim3(512), stream,
                                      (size_t)0, sums, first)
                   : launch_dependent(block_norm_sums_kernel<Tb, 32>, grid, dim3(1024), stream,
                                      (size_t)0, sums, first);
}

// The pairs of a residual stream's and a branch's element types.  Each pair and
// direction is compiled on its own (b200_train_rows.cu).
#define LOOM_ROW_TYPES(X)          \
  X(float, float)                  \
  X(float, __nv_bfloat16)          \
  X(float, __half)                 \
  X(__nv_bfloat16, __nv_bfloat16)  \
  X(__half, __half)

}  // namespace loomb
