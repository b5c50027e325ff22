// loom_b200_types.cuh -- the element types of the training-step operators and
// their loads and stores.
//
// Every operator computes in fp32 whatever its tensors hold; a 16-bit value is
// widened exactly on the way in and rounded once, to nearest even, on the way
// out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace loomb {

// Type codes of the C entries.
enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

inline bool valid_dtype(int t) { return t >= kF32 && t <= kF16; }
inline int dtype_bytes(int t) { return t == kF32 ? 4 : 2; }

// 4, 8 or 16 bytes moved by one instruction.
template <int kBytes>
struct Word;
template <>
struct Word<2> {
  using T = unsigned short;
};
template <>
struct Word<4> {
  using T = unsigned;
};
template <>
struct Word<8> {
  using T = uint2;
};
template <>
struct Word<16> {
  using T = uint4;
};

__device__ __forceinline__ void widen2(float& a, float& b, unsigned w, __nv_bfloat16) {
  // a bf16 is the upper half of the fp32 of the same value
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void widen2(float& a, float& b, unsigned w, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ unsigned narrow2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&p);
}
__device__ __forceinline__ unsigned narrow2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&p);
}

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}

// How a load or a store treats the caches: kStream marks data that is touched
// once (evict first); kKeep leaves the default.
enum Cache : int { kKeep = 0, kStream = 1 };

template <Cache kC, class W>
__device__ __forceinline__ W load_word(const W* p) {
  if constexpr (kC == kStream) return __ldcs(p);
  return *p;
}
template <Cache kC, class W>
__device__ __forceinline__ void store_word(W* p, const W& w) {
  if constexpr (kC == kStream) {
    __stcs(p, w);
  } else {
    *p = w;
  }
}

// V consecutive elements of T from `p`, which is aligned to min(16, V *
// sizeof(T)) bytes, as fp32.
template <int V, Cache kC, class T>
__device__ __forceinline__ void load_vec(float (&f)[V], const T* p) {
  constexpr int kBytes = V * (int)sizeof(T);
  if constexpr (sizeof(T) == 4) {
    constexpr int kW = kBytes >= 16 ? 16 : kBytes;
    using W = typename Word<kW>::T;
    constexpr int kPer = kW / 4;
#pragma unroll
    for (int i = 0; i < V / kPer; ++i) {
      const W w = load_word<kC>(reinterpret_cast<const W*>(p) + i);
      if constexpr (kPer == 4) {
        f[4 * i + 0] = __uint_as_float(w.x);
        f[4 * i + 1] = __uint_as_float(w.y);
        f[4 * i + 2] = __uint_as_float(w.z);
        f[4 * i + 3] = __uint_as_float(w.w);
      } else if constexpr (kPer == 2) {
        f[2 * i + 0] = __uint_as_float(w.x);
        f[2 * i + 1] = __uint_as_float(w.y);
      } else {
        f[i] = __uint_as_float(w);
      }
    }
  } else if constexpr (V == 1) {
    const unsigned short w = load_word<kC>(reinterpret_cast<const unsigned short*>(p));
    f[0] = widen(*reinterpret_cast<const T*>(&w));
  } else {
    using W = typename Word<kBytes>::T;
    static_assert(kBytes <= 16, "at most one 16-byte word of 16-bit elements");
    const W w = load_word<kC>(reinterpret_cast<const W*>(p));
    const unsigned* u = reinterpret_cast<const unsigned*>(&w);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) widen2(f[2 * i], f[2 * i + 1], u[i], T());
  }
}

// The elements of a 16-byte word as fp32.
template <class T>
__device__ __forceinline__ void widen_word(float (&f)[8], const uint4& w, T) {
  const unsigned* u = reinterpret_cast<const unsigned*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) widen2(f[2 * i], f[2 * i + 1], u[i], T());
}
__device__ __forceinline__ void widen_word(float (&f)[4], const uint4& w, float) {
  f[0] = __uint_as_float(w.x);
  f[1] = __uint_as_float(w.y);
  f[2] = __uint_as_float(w.z);
  f[3] = __uint_as_float(w.w);
}

template <int V, Cache kC, class T>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  constexpr int kBytes = V * (int)sizeof(T);
  if constexpr (sizeof(T) == 4) {
    constexpr int kW = kBytes >= 16 ? 16 : kBytes;
    using W = typename Word<kW>::T;
    constexpr int kPer = kW / 4;
#pragma unroll
    for (int i = 0; i < V / kPer; ++i) {
      W w;
      if constexpr (kPer == 4) {
        w.x = __float_as_uint(f[4 * i + 0]);
        w.y = __float_as_uint(f[4 * i + 1]);
        w.z = __float_as_uint(f[4 * i + 2]);
        w.w = __float_as_uint(f[4 * i + 3]);
      } else if constexpr (kPer == 2) {
        w.x = __float_as_uint(f[2 * i + 0]);
        w.y = __float_as_uint(f[2 * i + 1]);
      } else {
        w = __float_as_uint(f[i]);
      }
      store_word<kC>(reinterpret_cast<W*>(p) + i, w);
    }
  } else if constexpr (V == 1) {
    const T t = narrow<T>(f[0]);
    store_word<kC>(reinterpret_cast<unsigned short*>(p),
                   *reinterpret_cast<const unsigned short*>(&t));
  } else {
    using W = typename Word<kBytes>::T;
    static_assert(kBytes <= 16, "at most one 16-byte word of 16-bit elements");
    W w;
    unsigned* u = reinterpret_cast<unsigned*>(&w);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) u[i] = narrow2(f[2 * i], f[2 * i + 1], T());
    store_word<kC>(reinterpret_cast<W*>(p), w);
  }
}

// Two fp32 values in one register pair.  The packed instructions round each
// half on its own, as the single ones do, and take one issue slot for both.
struct F2 {
  unsigned long long bits;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.bits));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}

// Eight consecutive elements as they lie in memory.
template <class T>
struct Raw8 {
  uint4 word[sizeof(T) / 2];
};

template <class T>
__device__ __forceinline__ F2 pair_of(const Raw8<T>& r, int j) {
  const unsigned* u = reinterpret_cast<const unsigned*>(r.word);
  if constexpr (sizeof(T) == 4) {
    return f2(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1]));
  } else {
    float a, b;
    widen2(a, b, u[j], T());
    return f2(a, b);
  }
}
// Asynchronous copies to shared memory.  Every user here lets a thread copy
// what the same thread reads, so that its own wait is all that is needed
// between the two.
__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   (unsigned)__cvta_generic_to_shared(to)),
               "l"(from)
               : "memory");
}
// The first `bytes` of 16; the rest become zeros and are not read.
__device__ __forceinline__ void copy16_some(void* to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   (unsigned)__cvta_generic_to_shared(to)),
               "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copy8(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(
                   (unsigned)__cvta_generic_to_shared(to)),
               "l"(from)
               : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLater>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLater) : "memory");
}

}  // namespace loomb
