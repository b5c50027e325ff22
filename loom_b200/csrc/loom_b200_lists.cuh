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
// loom_b200_device.cuh.  What it reads may be written while it is already
// resident, before its wait: no pointer to that promises read-only data.
#pragma once

#include "loom_b200_launch.cuh"
#include "loom_b200_types.cuh"

namespace loomb {

// Largest number of tensors per launch: a table fits the 32764 bytes of a
// kernel's parameters.  Longer lists take several launches; lists of at most
// kShortCap tensors take a table of that size, since a launch costs the more the
// more parameters it has (a step of six tensors: 5.8 against 7.5 us).
constexpr int kShortCap = 32;
constexpr int kNormCap = 1024;
constexpr int kAdamCap = 480;
constexpr int kAdam8Cap = 360;
constexpr int kSms = 148;                // of a B200

// Values of a list at most (2^30 tiles of 1024 and one more a tensor).
constexpr int64_t kListMost = (int64_t)1 << 40;

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

struct NormItem {
  const void* g;
  int64_t n;
};

template <int kCap>
struct NormTable {
  NormItem item[kCap];
  uint32_t first[kCap];
  int count;
  uint32_t tiles;
};

// A square in fp64; one beyond the fp32 range counts as infinite.
__device__ __forceinline__ double wide_square(float f) {
  const float q = f * f;
  return q < INFINITY ? (double)f * (double)f : (double)q;
}

// Below this a sum of 32 fp32 squares may have lost more than it keeps bits for:
// squares below 2^-126 are rounded to multiples of 2^-149, so 32 of them are off
// by 2^-145 at most, 2^-45 of the bound.
constexpr float kLeastSum = 7.8886090522101181e-31f;      // 2^-100

// Sum of squares of the list, one fp64 partial per CTA.  HBM-bound: one read of
// each element and two operations on it (411M bf16 values: 120 to 127 us by the
// box, 105 to 99% of the copy rate).  A thread adds its up to 32 squares of a tile
// in fp32 (a fixed tree: no cancellation, at most 6 roundings, 3.6e-7 of the
// tile's sum) and everything past that in fp64.  Where that sum leaves the range in
// which this holds, on either side, the thread adds the same squares in fp64 (134M
// fp32 values of 1e-24: 106 us, else 77).
template <class T, int kCap>
__global__ void __launch_bounds__(kThreads)
list_norm_kernel(const __grid_constant__ NormTable<kCap> t, double* __restrict__ partials) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  constexpr int V = 16 / (int)sizeof(T);
  double acc = 0.0;
  for (uint32_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const int i = find_tensor(t.first, t.count, tile);
    const T* const g = static_cast<const T*>(t.item[i].g);
    const int64_t n = t.item[i].n;
    // elements before the first 16-byte boundary, and whole vectors after it
    const int64_t lead = (int64_t)((16u - ((uintptr_t)g & 15u)) & 15u) / (int)sizeof(T);
    const int64_t head = lead < n ? lead : n;
    const int64_t nvec = (n - head) / V;
    const int64_t v0 = (int64_t)(tile - t.first[i]) * (kThreads * kNormUnroll);
    const T* const body = g + head;
    if (v0 + (int)threadIdx.x < nvec) {
      const uint4* const vecs = reinterpret_cast<const uint4*>(body);
      uint4 raw[kNormUnroll];
      if (v0 + kThreads * kNormUnroll <= nvec) {
#pragma unroll
        for (int u = 0; u < kNormUnroll; ++u)
          raw[u] = load_word<kStream>(vecs + v0 + u * kThreads + threadIdx.x);
      } else {
#pragma unroll
        for (int u = 0; u < kNormUnroll; ++u) {
          const int64_t v = v0 + u * kThreads + threadIdx.x;
          raw[u] = v < nvec ? load_word<kStream>(vecs + v) : make_uint4(0, 0, 0, 0);
        }
      }
      float s[kNormUnroll];
#pragma unroll
      for (int u = 0; u < kNormUnroll; ++u) {
        float f[V];
        widen_word(f, raw[u], T());
#pragma unroll
        for (int w = V / 2; w > 0; w >>= 1)
#pragma unroll
          for (int j = 0; j < w; ++j)
            f[j] = w == V / 2 ? fmaf(f[j], f[j], f[j + w] * f[j + w]) : f[j] + f[j + w];
        s[u] = f[0];
      }
      const float sum = (s[0] + s[1]) + (s[2] + s[3]);
      if (sum >= kLeastSum && sum < INFINITY) {
        acc += (double)sum;
      } else {
        unsigned any = 0;
#pragma unroll
        for (int u = 0; u < kNormUnroll; ++u) any |= raw[u].x | raw[u].y | raw[u].z | raw[u].w;
        if (any & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) {  // not zeros alone
#pragma unroll 1
          for (int u = 0; u < kNormUnroll; ++u) {
            float f[V];
            widen_word(f, raw[0], T());
#pragma unroll
            for (int j = 0; j < V; ++j) acc += wide_square(f[j]);
#pragma unroll
            for (int k = 1; k < kNormUnroll; ++k) raw[k - 1] = raw[k];
          }
        }
      }
    }
    if (v0 == 0) {  // the tensor's first tile takes its ragged ends
      const int64_t tail0 = head + nvec * V;
      const int r = threadIdx.x;
      int64_t e = -1;
      if (r < head) e = r;
      else if (r >= V && (int64_t)(r - V) < n - tail0) e = tail0 + (r - V);
      if (e >= 0) acc += wide_square(widen(g[e]));
    }
  }
  acc = block_reduce<SumOp>(acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

static_assert(sizeof(NormTable<kNormCap>) + kOtherParams <= kParamBytes, "the list fits the parameters");

// out[0] = the norm, out[1] = the factor that brings it down to max_norm: 1
// where it is no larger, NaN where the sum is not finite (a step given that
// factor changes nothing).
__global__ void __launch_bounds__(kFinalizeThreads)
list_norm_finalize_kernel(const double* partials, const int count, const float max_norm,
                          float* out) {
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

template <class T, int kCap>
inline int launch_list_norm_parts(int64_t count, const void* const* grads, const int64_t* sizes,
                            float max_norm, float* out, void* workspace, cudaStream_t stream) {
  double* partials = reinterpret_cast<double*>(workspace_base(workspace));
  int filled = 0;
  NormTable<kCap> t;
  int64_t i = 0;
  while (i < count) {
    t.count = 0;
    int64_t tiles = 0;
    for (; i < count && t.count < kCap; ++i) {
      if (sizes[i] == 0) continue;
      const int64_t more = ceil_div(sizes[i], (int64_t)NormTile<T>::value);
      t.item[t.count] = {grads[i], sizes[i]};
      t.first[t.count] = (uint32_t)tiles;
      ++t.count;
      tiles += more;
    }
    if (t.count == 0) break;
    t.tiles = (uint32_t)tiles;
    const unsigned grid = clamp_grid(tiles, kNormMaxCtas);
    const int st = launch_dependent(list_norm_kernel<T, kCap>, dim3(grid), dim3(kThreads),
                                    stream, (size_t)0, t, partials + filled);
    if (st != LOOM_STATUS_OK) return st;
    filled += (int)grid;
  }
  return launch_dependent(list_norm_finalize_kernel, dim3(1), dim3(kFinalizeThreads), stream,
                          (size_t)0, (const double*)partials, filled, max_norm, out);
}

// ---------------------------------------------------------------------------
// AdamW

// What a step computes once: left in the workspace by adamw_begin_kernel.
struct alignas(16) StepValues {
  float scale;    // gradient factor
  float rate;     // lr / (1 - beta1^t)
  float root;     // 1 / sqrt(1 - beta2^t)
  float lr;
  uint32_t key;   // of this step's random numbers
  uint32_t skip;  // the factor is not finite: nothing is changed
  uint32_t unused[2];
};

// The constants of a step, rounded once on the host from fp64.
struct StepConst {
  float beta1, rest1;  // beta, 1 - beta
  float beta2, rest2;
  float eps;
  float zero;           // -0, added to a product that must be rounded on its own
  uint32_t sixteen;     // 16, for a shift on the multiplier
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

__global__ void adamw_begin_kernel(StepValues* out, const float* lr, const float* grad_scale,
                                   int64_t* step, const double beta1, const double beta2,
                                   const uint64_t seed) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  StepValues s = {};
  s.scale = grad_scale != nullptr ? *grad_scale : 1.0f;
  s.skip = !(fabsf(s.scale) < INFINITY);
  const int64_t t = *step + (s.skip ? 0 : 1);
  s.lr = *lr;
  // even lanes raise the one beta, odd lanes the other: the two powers one after
  // the other were a fifth of a short list's step (8-bit: 4.9 against 6.0 us)
  const bool second = threadIdx.x & 1;
  const double rest = 1.0 - pow(second ? beta2 : beta1, (double)t);
  const float mine = second ? (float)(1.0 / sqrt(rest)) : (float)((double)s.lr / rest);
  s.rate = __shfl_sync(0xffffffffu, mine, 0);
  s.root = __shfl_sync(0xffffffffu, mine, 1);
  if (threadIdx.x != 0) return;
  uint32_t k = mix32((uint32_t)seed ^ kGolden);
  k = mix32(k ^ (uint32_t)(seed >> 32));
  k = mix32(k ^ (uint32_t)t);
  s.key = mix32(k ^ (uint32_t)((uint64_t)t >> 32));
  *step = t;
  *out = s;
}

inline size_t adamw_workspace_bytes() { return 256 + 256; }

// Plain loads, which stay in an SM's first-level cache: every warp of the grid
// reads these 32 bytes, and asking the second level for them each time made
// its one line the whole step's limit (1026 us for 109M fp32 parameters in
// tiles of 1024, against 466 for their bytes).  The wait at the kernel's start
// makes what the kernel before it wrote visible to them, as ordinary loads: the
// pointer carries no __restrict__, which would allow the read-only path.
__device__ __forceinline__ StepValues step_values(const StepValues* p) {
  const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
  StepValues s;
  s.scale = __uint_as_float(a.x);
  s.rate = __uint_as_float(a.y);
  s.root = __uint_as_float(a.z);
  s.lr = __uint_as_float(a.w);
  s.key = b.x;
  s.skip = b.y;
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

constexpr int kAdamTile = kThreads * 4;                  // elements per CTA

struct AdamItem {
  void* p;
  const void* g;
  float* m;
  float* v;
  float* w;                   // fp32 master copy (unused without them)
  int64_t n;
  double decay;
};

template <int kCap>
struct AdamTable {
  AdamItem item[kCap];
  uint32_t first[kCap];
  int count;
};

template <class T>
__device__ __forceinline__ unsigned phase4(const T* p) {
  return (unsigned)((uintptr_t)p / sizeof(T)) & 3u;
}

// HBM-bound: 28 bytes and about 14 operations an element with fp32 parameters
// or with fp32 masters; 109M fp32 parameters take 442 to 447 us by the box, 105 to
// 104% of the copy rate.  Four consecutive elements per thread (16 bytes of every fp32 array)
// and six CTAs per SM: eight or sixteen elements a thread leave fewer warps to
// cover the loads' latency (455 and 453 us).  Where the arrays of a tensor stand
// at different places mod 4 elements, single elements are moved instead.
template <class Tp, class Tg, bool kMaster, int kCap>
__global__ void __launch_bounds__(kThreads, 6)
adamw_kernel(const __grid_constant__ AdamTable<kCap> t, const StepValues* values,
             const StepConst c) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  const int i = find_tensor(t.first, t.count, blockIdx.x);
  const StepValues s = step_values(values);
  const AdamItem& item = t.item[i];
  Tp* const p = static_cast<Tp*>(item.p);
  const Tg* const g = static_cast<const Tg*>(item.g);
  float* const m = item.m;
  float* const v = item.v;
  float* const w = kMaster ? item.w : nullptr;
  const int64_t n = item.n;
  const float keep = (float)(1.0 - (double)s.lr * item.decay);
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
    if (s.skip) return;
#pragma unroll 1
    for (int u = 0; u < 4; ++u) {
      const int64_t e = tile * kAdamTile + u * kThreads + threadIdx.x;
      if (e < n) one(e);
    }
    return;
  }
  const int64_t lead = (4u - ph) & 3u;
  const int64_t head = lead < n ? lead : n;
  const int64_t nvec = (n - head) >> 2;
  const int64_t at = tile * kThreads + threadIdx.x;
  const int64_t e = head + at * 4;
  float fp[4], fg[4], fm[4], fv[4];
  if (at < nvec) {
    if (kMaster) {
      load_vec<4, kStream>(fp, (const float*)w + e);
    } else {
      load_vec<4, kStream>(fp, (const Tp*)p + e);
    }
    load_vec<4, kStream>(fg, g + e);
    load_vec<4, kStream>(fm, (const float*)m + e);
    load_vec<4, kStream>(fv, (const float*)v + e);
  }
  if (s.skip) return;  // looked at when the data is on its way
  if (at < nvec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      moments(fm[j], fv[j], fg[j], c, s.scale);
      fp[j] = stepped(fp[j], fm[j], fv[j], c, s, keep);
    }
    store_vec<4, kStream>(m + e, fm);
    store_vec<4, kStream>(v + e, fv);
    if (kMaster) store_vec<4, kStream>(w + e, fp);
    store_vec<4, kStream>(p + e, fp);
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
constexpr int kMaxWarpBlocks = 16;                       // consecutive blocks per warp
constexpr float kTop = 256.0f;                           // code value of a block's largest
constexpr float kTinyTop = 7.8886090522101181e-31f;      // 2^-100: smaller blocks hold zeros

struct Adam8Item {
  void* p;
  const void* g;
  uint8_t* m;
  uint8_t* v;
  float* mtop;
  float* vtop;
  float* w;
  int64_t n;
  double decay;
  uint64_t block;              // first block, counted through the whole list
};

template <int kCap>
struct Adam8Table {
  Adam8Item item[kCap];
  uint32_t first[kCap];   // first tile
  int count;
  int warp_blocks;             // consecutive blocks that each warp takes
};

// Eight consecutive elements of which the first `left` exist; the others are
// zero.
template <class T>
__device__ __forceinline__ void load8_some(Raw8<T>& r, const T* p, int left) {
  using Bits = typename Word<sizeof(T)>::T;
  const Bits* q = reinterpret_cast<const Bits*>(p);
  unsigned u[2 * sizeof(T)];
#pragma unroll
  for (int k = 0; k < 2 * (int)sizeof(T); ++k) {
    if constexpr (sizeof(T) == 4) {
      u[k] = k < left ? q[k] : 0u;
    } else {
      u[k] = (2 * k < left ? q[2 * k] : 0u) | (2 * k + 1 < left ? q[2 * k + 1] : 0u) << 16;
    }
  }
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k)
    r.word[k] = make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
}
template <class T>
__device__ __forceinline__ void store8_some(T* p, const float (&f)[8], int left) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) p[j] = narrow<T>(f[j]);
}
__device__ __forceinline__ uint2 load8_codes_some(const uint8_t* p, int left) {
  uint2 w = make_uint2(0, 0);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) (j < 4 ? w.x : w.y) |= (unsigned)p[j] << (8 * (j & 3));
  return w;
}
__device__ __forceinline__ void store8_codes_some(uint8_t* p, uint2 w, int left) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) p[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
}

// Four e4m3 codes as fp32.
__device__ __forceinline__ void open4(F2& lo, F2& hi, unsigned codes) {
  unsigned a, b;
  asm("{.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;}"
      : "=r"(a), "=r"(b)
      : "r"(codes));
  const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
  lo = f2(fa.x, fa.y);
  hi = f2(fb.x, fb.y);
}

// Rounds a >= 0 (a <= 256 and a little) to an e4m3 code, up with the
// probability of its distance from the code below, by the 16 random bits r.
// A code keeps 3 bits after the leading one, so it is the upper 12 bits of
// the fp32 word, less the difference of the exponents' offsets (120 << 3),
// after adding the 20 random bits (r << 4 | 8) to those that are cut off.
// Below 2^-6 codes are evenly spaced: adding 2^-6 to the value (`lifted`)
// moves that range onto the binade above it, whose spacing it has, and
// subtracting a binade from the word moves it back.  The fp32 word as a
// function of the value is concave, so the lifted word is the larger of the
// two below 2^-6 and the smaller above, and no comparison of a is needed.
__device__ __forceinline__ int rounding_word(float a, float lifted) {
  return __viaddmax_s32(__float_as_int(lifted), -(1 << 23), __float_as_int(a));
}
constexpr int kCodeOffset = 960 << 20;
// The code in the upper byte: word + 8 - offset, moved up by 4.  Written as a
// product with a kernel argument, the shift goes to the multiplier: the integer
// pipe is the busiest one here (226 against 229 us for 109M bf16 parameters;
// moving the random bits' shifts as well made it 233).
__device__ __forceinline__ unsigned upper_code(int word, unsigned sixteen) {
  return (unsigned)word * sixteen + ((unsigned)(8 - kCodeOffset) << 4);
}

// Rates of two and one instructions for the parameter's move, which hangs on
// no border: about 2 ulp each.
__device__ __forceinline__ float root_approx(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float inverse_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float largest(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One lane's part of a block on its way through shared memory.
template <class Tw, class Tg>
struct BlockStage {
  uint4 w[sizeof(Tw) / 2][kThreads];
  uint4 g[sizeof(Tg) / 2][kThreads];
  uint2 m[kThreads];
  uint2 v[kThreads];
};

// 10 and a sixteenth bytes an element with bf16 parameters and gradients, but
// bound by issue before HBM: about 60 instructions an element for opening and
// closing two codes, the random bits and the step.  109M bf16 parameters take
// 226 to 246 us by the box, 74 to 68% of the copy rate (one block per warp, 115
// instructions an element and loads that nothing overlapped: 587 us); 114M with
// fp32 masters 359, with fp32 parameters and gradients 396, 78 and 71%.  A tensor
// with an array that is not aligned takes single elements (101M bf16: 351 against
// 204).  What it rests on:
//  * a warp holds a block, eight consecutive values a lane, so a block's
//    largest is one warp-wide maximum of the values' bit patterns; as unsigned
//    words these order NaN above infinity above every number, so a block that
//    holds one that is not finite gets it as its top and reads back as such;
//  * a warp walks up to 16 consecutive blocks; whole blocks come through shared
//    memory, three ahead with 16-bit types, two where what the step reads or the
//    gradients are fp32, one where both are, at no registers' cost;
//  * packed fp32 instructions for two values at a time;
//  * three CTAs per SM: bounding the registers for four spills them and is 8%
//    slower.
template <class Tp, class Tg, bool kMaster, int kCap>
__global__ void __launch_bounds__(kThreads, 3)
adamw8_kernel(const __grid_constant__ Adam8Table<kCap> t, const StepValues* values,
              const StepConst c) {
  allow_dependent_launch();
  wait_for_prerequisite_grid();
  using Tw = typename std::conditional<kMaster, float, Tp>::type;  // what the step reads
  const int i = find_tensor(t.first, t.count, blockIdx.x);
  const Adam8Item& item = t.item[i];
  const int lane = threadIdx.x & 31;
  const int blocks = t.warp_blocks;
  const int64_t block =
      ((int64_t)(blockIdx.x - t.first[i]) * (kThreads / 32) + (threadIdx.x >> 5)) * blocks;
  const int64_t rest = item.n - block * kBlock;  // elements from the warp's first on
  const int64_t at = block * kBlock + lane * 8;
  Tp* p = static_cast<Tp*>(item.p) + at;
  Tw* w = (kMaster ? (Tw*)item.w : (Tw*)item.p) + at;
  const Tg* g = static_cast<const Tg*>(item.g) + at;
  uint8_t* m = item.m + at;
  uint8_t* v = item.v + at;
  const bool aligned = (((uintptr_t)p | (uintptr_t)w | (uintptr_t)g) & 15u) == 0 &&
                       (((uintptr_t)m | (uintptr_t)v) & 7u) == 0;
  // the warp's blocks, and those of them that lie wholly in the tensor (none
  // where an array is not aligned for vector access)
  const int here = rest <= 0 ? 0 : (int)min((rest + kBlock - 1) / kBlock, (int64_t)blocks);
  const int whole = aligned && rest > 0 ? (int)min(rest / kBlock, (int64_t)blocks) : 0;
  uint32_t count = (uint32_t)(item.block + block) * 32u + lane;

  // Whole blocks come through shared memory, kStages - 1 of them ahead of the
  // one that is computed; the others are loaded where they are needed.
  constexpr int kStages = 49152 / (int)sizeof(BlockStage<Tw, Tg>) > 4
                              ? 4
                              : 49152 / (int)sizeof(BlockStage<Tw, Tg>);
  static_assert(kStages >= 2, "two blocks fit the shared memory");
  __shared__ BlockStage<Tw, Tg> stages[kStages];
  const int tid = threadIdx.x;
  // starts the copies of the warp's block k, `ahead` of the pointers' one
  auto copy = [&](int k, int ahead, int stage) {
    const int o = ahead * kBlock;
    if (k < whole) {
      BlockStage<Tw, Tg>& b = stages[stage];
#pragma unroll
      for (int k = 0; k < (int)sizeof(Tw) / 2; ++k)
        copy16(&b.w[k][tid], reinterpret_cast<const uint4*>(w + o) + k);
#pragma unroll
      for (int k = 0; k < (int)sizeof(Tg) / 2; ++k)
        copy16(&b.g[k][tid], reinterpret_cast<const uint4*>(g + o) + k);
      copy8(&b.m[tid], m + o);
      copy8(&b.v[tid], v + o);
    }
    copies_done();
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) copy(k, k, k);
  // the lane's elements of a block that is not whole
  auto some_of = [&](int k) {
    const int64_t left = rest - k * kBlock - lane * 8;
    return (int)(left < 0 ? 0 : left > 8 ? 8 : left);
  };
  // lane k holds the tops of the warp's block k, the old ones and then the new:
  // one coalesced access for all of them (a load and a store of 4 bytes in the
  // loop cost 20% of the whole step)
  float mtops = 0.0f, vtops = 0.0f;
  const bool has_tops = lane < here;
  if (has_tops) {
    mtops = item.mtop[block + lane];
    vtops = item.vtop[block + lane];
  }
  const StepValues s = step_values(values);
  if (s.skip) {
    wait_copies<0>();
    return;
  }
  const float keep = (float)(1.0 - (double)s.lr * item.decay);
  const F2 scale = f2(s.scale, s.scale), beta1 = f2(c.beta1, c.beta1), rest1 = f2(c.rest1, c.rest1),
           beta2 = f2(c.beta2, c.beta2), rest2 = f2(c.rest2, c.rest2), eps = f2(c.eps, c.eps),
           root = f2(s.root, s.root), rate = f2(-s.rate, -s.rate), keep2 = f2(keep, keep),
           zero = f2(c.zero, c.zero), lift = f2(0.015625f, 0.015625f);
  int stage = 0;
#pragma unroll 1
  for (int k = 0; k < here; ++k) {
    struct {
      Raw8<Tw> p;
      Raw8<Tg> g;
      uint2 m, v;
    } x;
    wait_copies<kStages - 2>();
    if (k < whole) {
      const BlockStage<Tw, Tg>& b = stages[stage];
#pragma unroll
      for (int q = 0; q < (int)sizeof(Tw) / 2; ++q) x.p.word[q] = b.w[q][tid];
#pragma unroll
      for (int q = 0; q < (int)sizeof(Tg) / 2; ++q) x.g.word[q] = b.g[q][tid];
      x.m = b.m[tid];
      x.v = b.v[tid];
    } else {
      const int some = some_of(k);
      load8_some(x.p, (const Tw*)w, some);
      load8_some(x.g, g, some);
      x.m = load8_codes_some(m, some);
      x.v = load8_codes_some(v, some);
    }
    // into the stage that the block before this one was read from
    const int freed = stage == 0 ? kStages - 1 : stage - 1;
    copy(k + kStages - 1, kStages - 1, freed);
    stage = stage == kStages - 1 ? 0 : stage + 1;
    const float munit = __fmul_rn(__shfl_sync(0xffffffffu, mtops, k), 1.0f / kTop);
    const float vunit = __fmul_rn(__shfl_sync(0xffffffffu, vtops, k), 1.0f / kTop);
    const F2 munit2 = f2(munit, munit), vunit2 = f2(vunit, vunit);
    F2 fm[4], fv[4];
    float fp[8];
    float mbig = 0.0f, vbig = 0.0f;
    open4(fm[0], fm[1], x.m.x);
    open4(fm[2], fm[3], x.m.y);
    open4(fv[0], fv[1], x.v.x);
    open4(fv[2], fv[3], x.v.y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      fm[j] = mul2(fm[j], munit2);
      fv[j] = mul2(fv[j], vunit2);
      const F2 fg = mul2(pair_of(x.g, j), scale);
      // the assembler joins a packed product with the sum that takes it into one
      // rounding; a product written as a sum with -0 is left alone
      fm[j] = add2(fma2(fm[j], beta1, zero), fma2(fg, rest1, zero));
      fv[j] = add2(fma2(fv[j], beta2, zero), fma2(mul2(fg, fg), rest2, zero));
      const float2 a = halves(fm[j]), b = halves(fv[j]);
      mbig = largest(mbig, a.x, a.y);
      vbig = largest(vbig, b.x, b.y);
      const float2 d = halves(fma2(f2(root_approx(b.x), root_approx(b.y)), root, eps));
      const F2 move = mul2(fm[j], f2(inverse_approx(d.x), inverse_approx(d.y)));
      const float2 q = halves(fma2(move, rate, mul2(pair_of(x.p, j), keep2)));
      fp[2 * j] = q.x;
      fp[2 * j + 1] = q.y;
    }

    const unsigned mmax = __reduce_max_sync(0xffffffffu, __float_as_uint(mbig) & 0x7fffffffu);
    const unsigned vmax = __reduce_max_sync(0xffffffffu, __float_as_uint(vbig) & 0x7fffffffu);
    // a top that is not finite or too small makes the block's codes zero; even
    // lanes invert the one top, odd lanes the other
    float mtop = __uint_as_float(mmax), vtop = __uint_as_float(vmax);
    if (mtop < kTinyTop) mtop = 0.0f;
    if (vtop < kTinyTop) vtop = 0.0f;
    const float own = (lane & 1) ? vtop : mtop;
    const float inverse = own > 0.0f && own < INFINITY ? __fmul_rn(__frcp_rn(own), kTop) : 0.0f;
    const float minv = __shfl_sync(0xffffffffu, inverse, 0);
    const float vinv = __shfl_sync(0xffffffffu, inverse, 1);
    const F2 vinv2 = f2(vinv, vinv);

    // 32 random bits a value: a full mix for the lane's eight, half a mix each
    const uint32_t h = mix32(mix32(count) + s.key);
    unsigned mw[8], vw[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t rm[2], rv[2];  // 16 bits each, at the bottom and at the top
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t y = h + (uint32_t)(2 * j + q) * kGolden;
        y ^= y >> 17;
        y *= 0xBB67AE85u;
        const uint32_t z = y >> 15;
        rm[q] = (y ^ z) & 0xffffu;
        rv[q] = (y ^ z) & 0xffff0000u;
      }
      const float2 a = halves(fm[j]), b = halves(fv[j]);
      const float2 ma = make_float2(__fmul_rn(fabsf(a.x), minv), __fmul_rn(fabsf(a.y), minv));
      const float2 ml = halves(add2(f2(ma.x, ma.y), lift));
      const F2 tb = fma2(fv[j], vinv2, zero);
      const float2 va = halves(tb), vl = halves(add2(tb, lift));
      const int m0 = rounding_word(ma.x, ml.x) + (int)(rm[0] << 4);
      const int m1 = rounding_word(ma.y, ml.y) + (int)(rm[1] << 4);
      int v0 = rounding_word(va.x, vl.x) + (int)(rv[0] >> 12);
      int v1 = rounding_word(va.y, vl.y) + (int)(rv[1] >> 12);
      // a second moment above zero stays above it
      if (b.x > 0.0f) v0 = max(v0, kCodeOffset + (1 << 20));
      if (b.y > 0.0f) v1 = max(v1, kCodeOffset + (1 << 20));
      mw[2 * j] = upper_code(m0, c.sixteen) | (__float_as_uint(a.x) & 0x80000000u);
      mw[2 * j + 1] = upper_code(m1, c.sixteen) | (__float_as_uint(a.y) & 0x80000000u);
      vw[2 * j] = upper_code(v0, c.sixteen);
      vw[2 * j + 1] = upper_code(v1, c.sixteen);
    }
    auto upper4 = [](const unsigned* u) {
      return __byte_perm(__byte_perm(u[0], u[1], 0x0073), __byte_perm(u[2], u[3], 0x0073), 0x5410);
    };
    uint2 mo = make_uint2(upper4(mw), upper4(mw + 4)), vo = make_uint2(upper4(vw), upper4(vw + 4));
    if (mmax >= 0x7f800000u) mo = make_uint2(0, 0);
    if (vmax >= 0x7f800000u) vo = make_uint2(0, 0);
    if (k < whole) {
      if (kMaster) store_vec<8, kStream>((float*)w, fp);
      store_vec<8, kStream>(p, fp);
      __stcs(reinterpret_cast<uint2*>(m), mo);
      __stcs(reinterpret_cast<uint2*>(v), vo);
    } else {
      const int some = some_of(k);
      if (kMaster) store8_some((float*)w, fp, some);
      store8_some(p, fp, some);
      store8_codes_some(m, mo, some);
      store8_codes_some(v, vo, some);
    }
    if (lane == k) {
      mtops = mtop;
      vtops = vtop;
    }
    p += kBlock;
    w += kBlock;
    g += kBlock;
    m += kBlock;
    v += kBlock;
    count += 32;
  }
  if (has_tops) {
    item.mtop[block + lane] = mtops;
    item.vtop[block + lane] = vtops;
  }
  wait_copies<0>();
}

static_assert(sizeof(AdamTable<kAdamCap>) + kOtherParams <= kParamBytes, "the list fits the parameters");
static_assert(sizeof(Adam8Table<kAdam8Cap>) + kOtherParams <= kParamBytes, "the list fits the parameters");

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

template <class Tp, class Tg, bool kMaster, int kCap>
inline int launch_adamw_parts(const AdamLists& l, const StepConst& c, const StepValues* values,
                              cudaStream_t stream) {
  AdamTable<kCap> t;
  int64_t i = 0;
  while (i < l.count) {
    t.count = 0;
    int64_t tiles = 0;
    for (; i < l.count && t.count < kCap; ++i) {
      if (l.sizes[i] == 0) continue;
      const int64_t more = ceil_div(l.sizes[i], (int64_t)kAdamTile);
      const int k = t.count++;
      t.item[k] = {l.params[i],
                   l.grads[i],
                   static_cast<float*>(l.exp_avg[i]),
                   static_cast<float*>(l.exp_avg_sq[i]),
                   kMaster ? l.master[i] : nullptr,
                   l.sizes[i],
                   l.weight_decay[i]};
      t.first[k] = (uint32_t)tiles;
      tiles += more;
    }
    if (t.count == 0) break;
    const int st = launch_dependent(adamw_kernel<Tp, Tg, kMaster, kCap>, dim3((unsigned)tiles),
                                    dim3(kThreads), stream, (size_t)0, t, values, c);
    if (st != LOOM_STATUS_OK) return st;
  }
  return LOOM_STATUS_OK;
}

template <class Tp, class Tg, bool kMaster, int kCap>
inline int launch_adamw8_parts(const AdamLists& l, const StepConst& c, const StepValues* values,
                               cudaStream_t stream) {
  Adam8Table<kCap> t;
  int64_t i = 0, block = 0, all = 0;
  for (int64_t k = 0; k < l.count; ++k) all += ceil_div(l.sizes[k], (int64_t)kBlock);
  // one block per warp while these are fewer than the warps that the GPU holds
  // at once, then as many as keep them all busy, up to kMaxWarpBlocks
  int64_t per = all / (kSms * 4 * (kThreads / 32));
  per = per < 1 ? 1 : per > kMaxWarpBlocks ? kMaxWarpBlocks : per;
  t.warp_blocks = (int)per;
  while (i < l.count) {
    t.count = 0;
    int64_t tiles = 0;
    for (; i < l.count && t.count < kCap; ++i) {
      if (l.sizes[i] == 0) continue;
      const int64_t blocks = ceil_div(l.sizes[i], (int64_t)kBlock);
      const int64_t more = ceil_div(blocks, per * (kThreads / 32));
      const int k = t.count++;
      t.item[k] = {l.params[i],
                   l.grads[i],
                   static_cast<uint8_t*>(l.exp_avg[i]),
                   static_cast<uint8_t*>(l.exp_avg_sq[i]),
                   l.exp_avg_top[i],
                   l.exp_avg_sq_top[i],
                   kMaster ? l.master[i] : nullptr,
                   l.sizes[i],
                   l.weight_decay[i],
                   (uint64_t)block};
      t.first[k] = (uint32_t)tiles;
      tiles += more;
      block += blocks;
    }
    if (t.count == 0) break;
    const int st = launch_dependent(adamw8_kernel<Tp, Tg, kMaster, kCap>, dim3((unsigned)tiles),
                                    dim3(kThreads), stream, (size_t)0, t, values, c);
    if (st != LOOM_STATUS_OK) return st;
  }
  return LOOM_STATUS_OK;
}

template <class T>
inline int launch_list_norm(int64_t count, const void* const* grads, const int64_t* sizes,
                            float max_norm, float* out, void* workspace, cudaStream_t stream) {
  return count <= kShortCap ? launch_list_norm_parts<T, kShortCap>(count, grads, sizes, max_norm,
                                                                   out, workspace, stream)
                            : launch_list_norm_parts<T, kNormCap>(count, grads, sizes, max_norm,
                                                                  out, workspace, stream);
}

template <class Tp, class Tg, bool kMaster>
inline int launch_adamw_lists(const AdamLists& l, const StepConst& c, const StepValues* values,
                              cudaStream_t stream) {
  return l.count <= kShortCap
             ? launch_adamw_parts<Tp, Tg, kMaster, kShortCap>(l, c, values, stream)
             : launch_adamw_parts<Tp, Tg, kMaster, kAdamCap>(l, c, values, stream);
}

template <class Tp, class Tg, bool kMaster>
inline int launch_adamw8_lists(const AdamLists& l, const StepConst& c, const StepValues* values,
                               cudaStream_t stream) {
  return l.count <= kShortCap
             ? launch_adamw8_parts<Tp, Tg, kMaster, kShortCap>(l, c, values, stream)
             : launch_adamw8_parts<Tp, Tg, kMaster, kAdam8Cap>(l, c, values, stream);
}

}  // namespace loomb
