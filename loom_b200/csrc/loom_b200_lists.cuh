// loom_b200_lists.cuh -- operators over lists of tensors: the norm of a
// gradient list with its clipping factor, and the AdamW step with its states
// in 32 bits or in 8.
//
// A list travels in the kernel's parameters (sm_100a takes 32 KiB of them):
// no device table has to be uploaded, kept alive or guarded, and a captured
// launch holds its own copy.  The grid has one CTA per tile of the whole list;
// a CTA finds its tensor by a binary search over the first tile of each
// (10 steps at most, uniform over the CTA, in the constant bank).
//
// Every kernel is a programmatic dependent launch of the one before it, as in
// loom_b200_device.cuh.
#pragma once

#include "loom_b200_launch.cuh"
#include "loom_b200_types.cuh"

namespace loomb {

// Largest number of tensors per launch: a table fits the 32764 bytes of a
// kernel's parameters.  Longer lists take several launches.
constexpr int kNormCap = 1024;
constexpr int kAdamCap = 480;
constexpr int kAdam8Cap = 360;

// What a kernel's parameters may take beside its table.
constexpr size_t kParamBytes = 32764, kOtherParams = 256;

// Index of the last entry of first[0..count) that is at most `tile`.
__device__ __forceinline__ int find_tensor(const uint32_t* first, int count, uint32_t tile) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= tile) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// ---------------------------------------------------------------------------
// norm of a list

constexpr int kNormUnroll = 4;          // 16-byte loads per thread per tile
constexpr int kNormMaxCtas = 4096;      // CTAs (fp64 partial slots) per launch

template <class T>
struct NormTile {
  static constexpr int value = kThreads * kNormUnroll * (16 / (int)sizeof(T));
};

struct NormTable {
  const void* g[kNormCap];
  int64_t n[kNormCap];
  uint32_t first[kNormCap];
  int count;
  uint32_t tiles;
};

// Sum of squares of the list, one fp64 partial per CTA.  HBM-bound: one read
// of each element and two operations on it.  A thread adds its up to 32
// squares of a tile in fp32 (a fixed tree: no cancellation, at most 5
// roundings, 3e-7 of the tile's sum) and everything past that in fp64.  A
// square beyond the fp32 range makes the sum infinite.
template <class T>
__global__ void __launch_bounds__(kThreads)
list_norm_kernel(const __grid_constant__ NormTable t, double* __restrict__ partials) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  constexpr int V = 16 / (int)sizeof(T);
  double acc = 0.0;
  for (uint32_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const int i = find_tensor(t.first, t.count, tile);
    const T* __restrict__ g = static_cast<const T*>(t.g[i]);
    const int64_t n = t.n[i];
    // elements before the first 16-byte boundary, and whole vectors after it
    const int64_t lead = (int64_t)((16u - ((uintptr_t)g & 15u)) & 15u) / (int)sizeof(T);
    const int64_t head = lead < n ? lead : n;
    const int64_t nvec = (n - head) / V;
    const int64_t v0 = (int64_t)(tile - t.first[i]) * (kThreads * kNormUnroll);
    const T* __restrict__ body = g + head;
    float s[kNormUnroll];
#pragma unroll
    for (int u = 0; u < kNormUnroll; ++u) s[u] = 0.0f;
    if (v0 + kThreads * kNormUnroll <= nvec) {
      float f[kNormUnroll][V];
#pragma unroll
      for (int u = 0; u < kNormUnroll; ++u)
        load_vec<V, kStream>(f[u], body + (v0 + u * kThreads + threadIdx.x) * V);
#pragma unroll
      for (int u = 0; u < kNormUnroll; ++u) {
#pragma unroll
        for (int w = V / 2; w > 0; w >>= 1)
#pragma unroll
          for (int j = 0; j < w; ++j)
            f[u][j] = w == V / 2 ? fmaf(f[u][j], f[u][j], f[u][j + w] * f[u][j + w])
                                 : f[u][j] + f[u][j + w];
        s[u] = f[u][0];
      }
    } else {
#pragma unroll
      for (int u = 0; u < kNormUnroll; ++u) {
        const int64_t v = v0 + u * kThreads + threadIdx.x;
        if (v < nvec) {
          float f[V];
          load_vec<V, kStream>(f, body + v * V);
#pragma unroll
          for (int j = 0; j < V; ++j) s[u] = fmaf(f[j], f[j], s[u]);
        }
      }
    }
    acc += (double)((s[0] + s[1]) + (s[2] + s[3]));
    if (v0 == 0) {  // the tensor's first tile takes its ragged ends
      const int64_t tail0 = head + nvec * V;
      const int r = threadIdx.x;
      int64_t e = -1;
      if (r < head) e = r;
      else if (r >= V && (int64_t)(r - V) < n - tail0) e = tail0 + (r - V);
      if (e >= 0) {
        const float f = widen(g[e]);
        acc += (double)(f * f);
      }
    }
  }
  acc = block_reduce<SumOp>(acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

static_assert(sizeof(NormTable) + kOtherParams <= kParamBytes, "the list fits the parameters");

// out[0] = the norm, out[1] = the factor that brings it down to max_norm: 1
// where it is no larger, NaN where the sum is not finite (a step given that
// factor changes nothing).
__global__ void __launch_bounds__(kFinalizeThreads)
list_norm_finalize_kernel(const double* __restrict__ partials, const int count,
                          const float max_norm, float* __restrict__ out) {
  wait_for_prerequisite_grid();
  allow_dependent_launch();
  const double sum = fold_partials<SumOp>(partials, count);
  if (threadIdx.x == 0) {
    const double norm = sqrt(sum);
    out[0] = (float)norm;
    out[1] = !(sum < (double)INFINITY) ? __int_as_float(0x7fc00000)
             : norm > (double)max_norm ? (float)((double)max_norm / norm)
                                       : 1.0f;
  }
}

inline int64_t list_launches(int64_t count, int cap) {
  return count <= 0 ? 1 : ceil_div(count, (int64_t)cap);
}

inline size_t list_norm_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  return (size_t)list_launches(count, kNormCap) * kNormMaxCtas * sizeof(double) + 256;
}

template <class T>
inline int launch_list_norm(int64_t count, const void* const* grads, const int64_t* sizes,
                            float max_norm, float* out, void* workspace, cudaStream_t stream) {
  double* partials = reinterpret_cast<double*>(workspace_base(workspace));
  int filled = 0;
  NormTable t;
  int64_t i = 0;
  while (i < count) {
    t.count = 0;
    int64_t tiles = 0;
    for (; i < count && t.count < kNormCap; ++i) {
      if (sizes[i] == 0) continue;
      const int64_t more = ceil_div(sizes[i], (int64_t)NormTile<T>::value);
      if (tiles + more > 0x7fffffff) return LOOM_STATUS_INVALID_ARGUMENT;
      t.g[t.count] = grads[i];
      t.n[t.count] = sizes[i];
      t.first[t.count] = (uint32_t)tiles;
      ++t.count;
      tiles += more;
    }
    if (t.count == 0) break;
    t.tiles = (uint32_t)tiles;
    const unsigned grid = clamp_grid(tiles, kNormMaxCtas);
    const int st = launch_dependent(list_norm_kernel<T>, dim3(grid), dim3(kThreads),
                                    stream, t, partials + filled);
    if (st != LOOM_STATUS_OK) return st;
    filled += (int)grid;
  }
  return launch_dependent(list_norm_finalize_kernel, dim3(1), dim3(kFinalizeThreads), stream,
                          (const double*)partials, filled, max_norm, out);
}

// ---------------------------------------------------------------------------
// AdamW

// What a step computes once: left in the workspace by adamw_begin_kernel.
struct StepValues {
  float scale;    // gradient factor
  float rate;     // lr / (1 - beta1^t)
  float root;     // 1 / sqrt(1 - beta2^t)
  float lr;
  uint32_t key;   // of this step's random numbers
  uint32_t skip;  // the factor is not finite: nothing is changed
};

// The constants of a step, rounded once on the host from fp64.
struct StepConst {
  float beta1, rest1;  // beta, 1 - beta
  float beta2, rest2;
  float eps;
};

// A bijection of 32-bit words in which each input bit moves about half of the
// output bits: two odd multipliers (the fractions of sqrt 2 and sqrt 3) and
// three folds.
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

constexpr uint32_t kGolden = 0x9E3779B9u;

__global__ void adamw_begin_kernel(StepValues* __restrict__ out, const float* __restrict__ lr,
                                   const float* __restrict__ grad_scale,
                                   int64_t* __restrict__ step, const double beta1,
                                   const double beta2, const uint64_t seed) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  if (threadIdx.x != 0) return;
  StepValues s;
  s.scale = grad_scale != nullptr ? *grad_scale : 1.0f;
  s.skip = !(fabsf(s.scale) < INFINITY);
  const int64_t t = *step + (s.skip ? 0 : 1);
  s.lr = *lr;
  s.rate = (float)((double)s.lr / (1.0 - pow(beta1, (double)t)));
  s.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
  uint32_t k = mix32((uint32_t)seed ^ kGolden);
  k = mix32(k ^ (uint32_t)(seed >> 32));
  k = mix32(k ^ (uint32_t)t);
  s.key = mix32(k ^ (uint32_t)((uint64_t)t >> 32));
  *step = t;
  *out = s;
}

inline size_t adamw_workspace_bytes() { return 256 + 256; }

__device__ __forceinline__ StepValues step_values(const StepValues* p) {
  StepValues s;
  s.scale = __ldcg(&p->scale);
  s.rate = __ldcg(&p->rate);
  s.root = __ldcg(&p->root);
  s.lr = __ldcg(&p->lr);
  s.key = __ldcg(&p->key);
  s.skip = __ldcg(&p->skip);
  return s;
}

// The step of one element.  Each operation of the moments is rounded on its
// own (this file is compiled with -fmad=false): a stored 8-bit moment hangs on
// which side of a code's border the fp32 value falls, so the order is part of
// the definition.
__device__ __forceinline__ void moments(float& m, float& v, float g, const StepConst& c,
                                        float scale) {
  g = __fmul_rn(g, scale);
  m = __fadd_rn(__fmul_rn(m, c.beta1), __fmul_rn(g, c.rest1));
  v = __fadd_rn(__fmul_rn(v, c.beta2), __fmul_rn(__fmul_rn(g, g), c.rest2));
}
__device__ __forceinline__ float stepped(float p, float m, float v, const StepConst& c,
                                         const StepValues& s, float keep) {
  const float move = m / (sqrtf(v) * s.root + c.eps);
  return p * keep - s.rate * move;
}

constexpr int kAdamUnroll = 2;                           // groups of four elements per thread
constexpr int kAdamTile = kThreads * 4 * kAdamUnroll;    // elements per CTA

struct AdamTable {
  void* p[kAdamCap];
  const void* g[kAdamCap];
  float* m[kAdamCap];
  float* v[kAdamCap];
  float* w[kAdamCap];         // fp32 master copies (unused without them)
  int64_t n[kAdamCap];
  double decay[kAdamCap];
  uint32_t first[kAdamCap];
  int count;
};

template <class T>
__device__ __forceinline__ unsigned phase4(const T* p) {
  return (unsigned)((uintptr_t)p / sizeof(T)) & 3u;
}

// HBM-bound: 28 bytes and about 14 operations an element with fp32 parameters
// or with fp32 masters.  Four consecutive elements per access (16 bytes of
// every fp32 array); where the arrays of a tensor stand at different places
// mod 4 elements, single elements are moved instead.
template <class Tp, class Tg, bool kMaster>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ AdamTable t, const StepValues* __restrict__ values,
             const StepConst c) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  const int i = find_tensor(t.first, t.count, blockIdx.x);
  const StepValues s = step_values(values);
  if (s.skip) return;
  Tp* const p = static_cast<Tp*>(t.p[i]);
  const Tg* const g = static_cast<const Tg*>(t.g[i]);
  float* const m = t.m[i];
  float* const v = t.v[i];
  float* const w = kMaster ? t.w[i] : nullptr;
  const int64_t n = t.n[i];
  const float keep = (float)(1.0 - (double)s.lr * t.decay[i]);
  const int64_t tile = blockIdx.x - t.first[i];

  auto one = [&](int64_t e) {
    float me = m[e], ve = v[e];
    float pe = kMaster ? w[e] : widen(p[e]);
    moments(me, ve, widen(g[e]), c, s.scale);
    pe = stepped(pe, me, ve, c, s, keep);
    m[e] = me;
    v[e] = ve;
    if (kMaster) w[e] = pe;
    p[e] = narrow<Tp>(pe);
  };

  const unsigned ph = phase4(m);
  const bool together = phase4(v) == ph && phase4(p) == ph && phase4(g) == ph &&
                        (!kMaster || phase4(w) == ph);
  if (!together) {
#pragma unroll 1
    for (int u = 0; u < 4 * kAdamUnroll; ++u) {
      const int64_t e = tile * kAdamTile + u * kThreads + threadIdx.x;
      if (e < n) one(e);
    }
    return;
  }
  const int64_t lead = (4u - ph) & 3u;
  const int64_t head = lead < n ? lead : n;
  const int64_t nvec = (n - head) >> 2;
  const int64_t v0 = tile * (kThreads * kAdamUnroll) + threadIdx.x;
  float fp[kAdamUnroll][4], fg[kAdamUnroll][4], fm[kAdamUnroll][4], fv[kAdamUnroll][4];
#pragma unroll
  for (int u = 0; u < kAdamUnroll; ++u) {
    const int64_t at = v0 + u * kThreads;
    if (at < nvec) {
      const int64_t e = head + at * 4;
      if (kMaster) {
        load_vec<4, kStream>(fp[u], (const float*)w + e);
      } else {
        load_vec<4, kStream>(fp[u], (const Tp*)p + e);
      }
      load_vec<4, kStream>(fg[u], g + e);
      load_vec<4, kStream>(fm[u], (const float*)m + e);
      load_vec<4, kStream>(fv[u], (const float*)v + e);
    }
  }
#pragma unroll
  for (int u = 0; u < kAdamUnroll; ++u) {
    const int64_t at = v0 + u * kThreads;
    if (at < nvec) {
      const int64_t e = head + at * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        moments(fm[u][j], fv[u][j], fg[u][j], c, s.scale);
        fp[u][j] = stepped(fp[u][j], fm[u][j], fv[u][j], c, s, keep);
      }
      store_vec<4, kStream>(m + e, fm[u]);
      store_vec<4, kStream>(v + e, fv[u]);
      if (kMaster) store_vec<4, kStream>(w + e, fp[u]);
      store_vec<4, kStream>(p + e, fp[u]);
    }
  }
  if (tile == 0) {  // the tensor's first tile takes its ragged ends
    const int64_t tail0 = head + (nvec << 2);
    const int r = threadIdx.x;
    if (r < head) one(r);
    else if (r >= 4 && (int64_t)(r - 4) < n - tail0) one(tail0 + (r - 4));
  }
}

// ---------------------------------------------------------------------------
// AdamW with 8-bit states

constexpr int kBlock = 256;                              // values that share one top
constexpr int kTileBlocks = kThreads / 32;               // one block per warp
constexpr float kTop = 256.0f;                           // code value of a block's largest
constexpr float kTinyTop = 7.8886090522101181e-31f;      // 2^-100: smaller blocks hold zeros

struct Adam8Table {
  void* p[kAdam8Cap];
  const void* g[kAdam8Cap];
  uint8_t* m[kAdam8Cap];
  uint8_t* v[kAdam8Cap];
  float* mtop[kAdam8Cap];
  float* vtop[kAdam8Cap];
  float* w[kAdam8Cap];
  int64_t n[kAdam8Cap];
  double decay[kAdam8Cap];
  uint32_t first[kAdam8Cap];   // first tile
  uint32_t block[kAdam8Cap];   // first block, counted through the whole list
  int count;
};

// Eight consecutive elements of which the first `left` exist; the others are
// zero.  `whole`: p is aligned for one vector access.
template <class T>
__device__ __forceinline__ void load8(float (&f)[8], const T* p, int left, bool whole) {
  if (whole && left >= 8) {
    load_vec<8, kStream>(f, p);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = j < left ? widen(p[j]) : 0.0f;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8], int left, bool whole) {
  if (whole && left >= 8) {
    store_vec<8, kStream>(p, f);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) p[j] = narrow<T>(f[j]);
}
__device__ __forceinline__ uint2 load8_codes(const uint8_t* p, int left, bool whole) {
  if (whole && left >= 8) return __ldcs(reinterpret_cast<const uint2*>(p));
  uint2 w = make_uint2(0, 0);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) (j < 4 ? w.x : w.y) |= (unsigned)p[j] << (8 * (j & 3));
  return w;
}
__device__ __forceinline__ void store8_codes(uint8_t* p, uint2 w, int left, bool whole) {
  if (whole && left >= 8) {
    __stcs(reinterpret_cast<uint2*>(p), w);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) p[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
}

// Two e4m3 codes (the low 16 bits of `pair`) as fp32.
__device__ __forceinline__ float2 open2(unsigned pair) {
  unsigned h;
  asm("{.reg .b16 c; cvt.u16.u32 c, %1; cvt.rn.f16x2.e4m3x2 %0, c;}" : "=r"(h) : "r"(pair));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void open8(float (&f)[8], uint2 w, float unit) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned word = j < 2 ? w.x : w.y;
    const float2 a = open2((j & 1) ? word >> 16 : word);
    f[2 * j] = __fmul_rn(a.x, unit);
    f[2 * j + 1] = __fmul_rn(a.y, unit);
  }
}

// The e4m3 code of a >= 0 (a <= 256 and a little), rounded up with the
// probability of its distance from the code below, by the 20-bit number r.
// A code keeps 3 bits after the leading one: the upper 12 bits of the fp32
// word, after adding r to the 20 that are cut off.  Below 2^-6 codes are
// evenly spaced; adding 2^-6 moves that range onto the spacing above it.
__device__ __forceinline__ unsigned close1(float a, unsigned r) {
  const bool low = a < 0.015625f;
  const unsigned bits = __float_as_uint(__fadd_rn(a, low ? 0.015625f : 0.0f)) + r;
  return (bits >> 20) - (low ? (120u << 3) + 8u : (120u << 3));
}

// HBM-bound by its bytes (10 and a sixteenth an element with bf16 parameters
// and gradients), and close to bound by issue: about 75 instructions an
// element for opening and closing two codes, the random bits and the step.
// A warp holds one block, eight consecutive values a lane, so a block's
// largest is one warp-wide maximum of the values' bit patterns; as unsigned
// words these order NaN above infinity above every number, so a block that
// holds one that is not finite gets it as its top and reads back as such.
template <class Tp, class Tg, bool kMaster>
__global__ void __launch_bounds__(kThreads)
adamw8_kernel(const __grid_constant__ Adam8Table t, const StepValues* __restrict__ values,
              const StepConst c) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  const int i = find_tensor(t.first, t.count, blockIdx.x);
  const StepValues s = step_values(values);
  if (s.skip) return;
  const int lane = threadIdx.x & 31;
  const int64_t block = (int64_t)(blockIdx.x - t.first[i]) * kTileBlocks + (threadIdx.x >> 5);
  const int64_t n = t.n[i];
  if (block * kBlock >= n) return;
  const int64_t e = block * kBlock + lane * 8;
  const int left = (int)(n - e < 0 ? 0 : n - e > 8 ? 8 : n - e);
  Tp* const p = static_cast<Tp*>(t.p[i]);
  const Tg* const g = static_cast<const Tg*>(t.g[i]);
  uint8_t* const m = t.m[i];
  uint8_t* const v = t.v[i];
  float* const w = kMaster ? t.w[i] : nullptr;
  const bool p_whole = ((uintptr_t)p & 15u) == 0, g_whole = ((uintptr_t)g & 15u) == 0;
  const bool m_whole = ((uintptr_t)m & 7u) == 0, v_whole = ((uintptr_t)v & 7u) == 0;
  const bool w_whole = ((uintptr_t)w & 15u) == 0;

  float fp[8], fg[8], fm[8], fv[8];
  if (kMaster) {
    load8(fp, (const float*)w + e, left, w_whole);
  } else {
    load8(fp, (const Tp*)p + e, left, p_whole);
  }
  load8(fg, g + e, left, g_whole);
  const uint2 mc = load8_codes(m + e, left, m_whole);
  const uint2 vc = load8_codes(v + e, left, v_whole);
  const float mt = t.mtop[i][block], vt = t.vtop[i][block];
  const float keep = (float)(1.0 - (double)s.lr * t.decay[i]);
  open8(fm, mc, __fmul_rn(mt, 1.0f / kTop));
  open8(fv, vc, __fmul_rn(vt, 1.0f / kTop));
  unsigned mbig = 0, vbig = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    moments(fm[j], fv[j], fg[j], c, s.scale);
    fp[j] = stepped(fp[j], fm[j], fv[j], c, s, keep);
    mbig = max(mbig, __float_as_uint(fm[j]) & 0x7fffffffu);
    vbig = max(vbig, __float_as_uint(fv[j]) & 0x7fffffffu);
  }
  if (kMaster) store8(w + e, fp, left, w_whole);
  store8(p + e, fp, left, p_whole);

  mbig = __reduce_max_sync(0xffffffffu, mbig);
  vbig = __reduce_max_sync(0xffffffffu, vbig);
  float mtop = __uint_as_float(mbig), vtop = __uint_as_float(vbig);
  const bool mgood = mbig < 0x7f800000u, vgood = vbig < 0x7f800000u;
  if (mtop < kTinyTop) mtop = 0.0f;
  if (vtop < kTinyTop) vtop = 0.0f;
  const float minv = mgood && mtop > 0.0f ? __fmul_rn(__fdiv_rn(1.0f, mtop), kTop) : 0.0f;
  const float vinv = vgood && vtop > 0.0f ? __fmul_rn(__fdiv_rn(1.0f, vtop), kTop) : 0.0f;

  // 32 random bits a value: a full mix for the lane's eight, half a mix each
  const uint32_t count = (uint32_t)(t.block[i] + block) * 32u + lane;
  const uint32_t h = mix32(mix32(count) + s.key);
  uint2 mo = make_uint2(0, 0), vo = make_uint2(0, 0);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t x = h + (uint32_t)j * kGolden;
    x ^= x >> 17;
    x *= 0xBB67AE85u;
    x ^= x >> 15;
    unsigned cm = close1(__fmul_rn(fabsf(fm[j]), minv), ((x & 0xffffu) << 4) + 8u);
    unsigned cv = close1(__fmul_rn(fabsf(fv[j]), vinv), ((x >> 12) & 0xffff0u) + 8u);
    if (fv[j] > 0.0f) cv = max(cv, 1u);  // a second moment above zero stays above it
    if (fm[j] < 0.0f) cm |= 0x80u;
    (j < 4 ? mo.x : mo.y) |= cm << (8 * (j & 3));
    (j < 4 ? vo.x : vo.y) |= cv << (8 * (j & 3));
  }
  if (!mgood) mo = make_uint2(0, 0);
  if (!vgood) vo = make_uint2(0, 0);
  store8_codes(m + e, mo, left, m_whole);
  store8_codes(v + e, vo, left, v_whole);
  if (lane == 0) {
    t.mtop[i][block] = mtop;
    t.vtop[i][block] = vtop;
  }
}

static_assert(sizeof(AdamTable) + kOtherParams <= kParamBytes, "the list fits the parameters");
static_assert(sizeof(Adam8Table) + kOtherParams <= kParamBytes, "the list fits the parameters");

// ---------------------------------------------------------------------------
// launchers

struct AdamLists {
  int64_t count;
  void* const* params;
  const void* const* grads;
  void* const* exp_avg;
  void* const* exp_avg_sq;
  float* const* exp_avg_top;      // 8-bit states only
  float* const* exp_avg_sq_top;
  float* const* master;           // or null
  const int64_t* sizes;
  const double* weight_decay;
};

template <class Tp, class Tg, bool kMaster>
inline int launch_adamw_lists(const AdamLists& l, const StepConst& c, const StepValues* values,
                              cudaStream_t stream) {
  AdamTable t;
  int64_t i = 0;
  while (i < l.count) {
    t.count = 0;
    int64_t tiles = 0;
    for (; i < l.count && t.count < kAdamCap; ++i) {
      if (l.sizes[i] == 0) continue;
      const int64_t more = ceil_div(l.sizes[i], (int64_t)kAdamTile);
      if (tiles + more > 0x7fffffff) return LOOM_STATUS_INVALID_ARGUMENT;
      const int k = t.count++;
      t.p[k] = l.params[i];
      t.g[k] = l.grads[i];
      t.m[k] = static_cast<float*>(l.exp_avg[i]);
      t.v[k] = static_cast<float*>(l.exp_avg_sq[i]);
      t.w[k] = kMaster ? l.master[i] : nullptr;
      t.n[k] = l.sizes[i];
      t.decay[k] = l.weight_decay[i];
      t.first[k] = (uint32_t)tiles;
      tiles += more;
    }
    if (t.count == 0) break;
    const int st = launch_dependent(adamw_kernel<Tp, Tg, kMaster>, dim3((unsigned)tiles),
                                    dim3(kThreads), stream, t, values, c);
    if (st != LOOM_STATUS_OK) return st;
  }
  return LOOM_STATUS_OK;
}

template <class Tp, class Tg, bool kMaster>
inline int launch_adamw8_lists(const AdamLists& l, const StepConst& c, const StepValues* values,
                               cudaStream_t stream) {
  Adam8Table t;
  int64_t i = 0, block = 0;
  while (i < l.count) {
    t.count = 0;
    int64_t tiles = 0;
    for (; i < l.count && t.count < kAdam8Cap; ++i) {
      if (l.sizes[i] == 0) continue;
      const int64_t blocks = ceil_div(l.sizes[i], (int64_t)kBlock);
      const int64_t more = ceil_div(blocks, (int64_t)kTileBlocks);
      if (tiles + more > 0x7fffffff) return LOOM_STATUS_INVALID_ARGUMENT;
      const int k = t.count++;
      t.p[k] = l.params[i];
      t.g[k] = l.grads[i];
      t.m[k] = static_cast<uint8_t*>(l.exp_avg[i]);
      t.v[k] = static_cast<uint8_t*>(l.exp_avg_sq[i]);
      t.mtop[k] = l.exp_avg_top[i];
      t.vtop[k] = l.exp_avg_sq_top[i];
      t.w[k] = kMaster ? l.master[i] : nullptr;
      t.n[k] = l.sizes[i];
      t.decay[k] = l.weight_decay[i];
      t.first[k] = (uint32_t)tiles;
      t.block[k] = (uint32_t)block;
      tiles += more;
      block += blocks;
    }
    if (t.count == 0) break;
    const int st = launch_dependent(adamw8_kernel<Tp, Tg, kMaster>, dim3((unsigned)tiles),
                                    dim3(kThreads), stream, t, values, c);
    if (st != LOOM_STATUS_OK) return st;
  }
  return LOOM_STATUS_OK;
}

}  // namespace loomb
