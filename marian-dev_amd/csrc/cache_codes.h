// Rows of activations and of 8-bit codes as the kernels over a quantized cache take them (device code).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace marian_hip {

enum class CacheFormat { int8 = 0, e4m3 = 1 };

typedef float cache_f4 __attribute__((ext_vector_type(4)));
typedef unsigned cache_u2 __attribute__((ext_vector_type(2)));
typedef unsigned cache_u4 __attribute__((ext_vector_type(4)));
typedef _Float16 cache_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 cache_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 cache_b2 __attribute__((ext_vector_type(2)));
typedef short cache_s2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

struct bf16_t {   // sixteen bits of a bfloat16
  uint16_t bits;
};

// ---- activations ----------------------------------------------------------------------------------
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(bf16_t x) { return __builtin_bit_cast(float, (unsigned)x.bits << 16); }

// COUNT (4 or 8) values from an address of whole vectors.
template <int COUNT, typename T>
__device__ __forceinline__ void load_row(const T* p, float (&x)[COUNT]) {
  if constexpr(sizeof(T) == 4) {
#pragma unroll
    for(int i = 0; i < COUNT / 4; ++i) {
      const cache_f4 v = reinterpret_cast<const cache_f4*>(p)[i];
#pragma unroll
      for(int e = 0; e < 4; ++e) x[4 * i + e] = v[e];
    }
  } else {
    unsigned w[COUNT / 2];
    if constexpr(COUNT == 8) {
      const cache_u4 v = *reinterpret_cast<const cache_u4*>(p);
#pragma unroll
      for(int e = 0; e < 4; ++e) w[e] = v[e];
    } else {
      const cache_u2 v = *reinterpret_cast<const cache_u2*>(p);
      w[0] = v[0];
      w[1] = v[1];
    }
#pragma unroll
    for(int e = 0; e < COUNT; ++e) {
      const uint16_t b = (uint16_t)(w[e / 2] >> (e % 2 * 16));
      x[e] = to_float(__builtin_bit_cast(T, b));
    }
  }
}

// Two values rounded to T (nearest, ties to even), in the order of memory.
template <typename T>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr(sizeof(T) == 2 && !__is_same(T, bf16_t)) {
    const cache_h2 h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(unsigned, h);
  } else {
    const cache_b2 h = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, h);
  }
}

template <int COUNT, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&x)[COUNT]) {
  if constexpr(sizeof(T) == 4) {
#pragma unroll
    for(int i = 0; i < COUNT / 4; ++i)
      reinterpret_cast<cache_f4*>(p)[i] = cache_f4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
  } else if constexpr(COUNT % 8 == 0) {
#pragma unroll
    for(int i = 0; i < COUNT / 8; ++i)
      reinterpret_cast<cache_u4*>(p)[i] = cache_u4{pack2<T>(x[8 * i], x[8 * i + 1]), pack2<T>(x[8 * i + 2], x[8 * i + 3]),
                                                   pack2<T>(x[8 * i + 4], x[8 * i + 5]), pack2<T>(x[8 * i + 6], x[8 * i + 7])};
  } else {
    *reinterpret_cast<cache_u2*>(p) = cache_u2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
  }
}

// ---- codes as float16 -------------------------------------------------------------------------------
// Both kinds of code become float16 exactly, times a power of two, in two or three instructions for two of them:
//   int8: the byte plus 128, as the bits of a float16, is (code + 128) 2^-24; times 2^15 minus 2^-2 that is code * 2^-9.
//   e4m3: sign, four exponent bits and mantissa in the upper byte, everything but the sign moved down by one: the
//   exponent then counts from 15 in place of 7, code * 2^-8 (small values without an exponent included).
// (0x7f, which e4m3 reads as NaN and nothing here writes, is 480.)
template <CacheFormat F>
constexpr float kCodeUnit = F == CacheFormat::int8 ? 1.0f / 512 : 1.0f / 256;

// Four codes as they are held ahead of half2_of.
template <CacheFormat F>
__device__ __forceinline__ unsigned held(unsigned x) { return F == CacheFormat::int8 ? x ^ 0x80808080u : x; }

// Byte I of a and byte J of b as two float16.
template <CacheFormat F, int I, int J>
__device__ __forceinline__ cache_h2 half2_of(unsigned a, unsigned b) {
  constexpr unsigned none = 0x0c;
  if constexpr(F == CacheFormat::int8) {
    const unsigned w = __builtin_amdgcn_perm(b, a, I | none << 8 | (4u + J) << 16 | none << 24);
    const cache_h2 up = {(_Float16)32768.0f, (_Float16)32768.0f}, down = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_elementwise_fma(__builtin_bit_cast(cache_h2, w), up, down);
  } else {
    const unsigned w = __builtin_amdgcn_perm(b, a, none | (unsigned)I << 8 | none << 16 | (4u + J) << 24);
    const cache_s2 s = __builtin_bit_cast(cache_s2, w) >> 1;
    return __builtin_bit_cast(cache_h2, __builtin_bit_cast(unsigned, s) & 0xbfffbfffu);
  }
}

// Eight codes in a row.
template <CacheFormat F>
__device__ __forceinline__ cache_h8 half8_of(unsigned lo, unsigned hi) {
  const unsigned a = held<F>(lo), b = held<F>(hi);
  const cache_h2 h[4] = {half2_of<F, 0, 1>(a, a), half2_of<F, 2, 3>(a, a), half2_of<F, 0, 1>(b, b), half2_of<F, 2, 3>(b, b)};
  return cache_h8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// ---- quantizing -------------------------------------------------------------------------------------
template <CacheFormat F>
constexpr float kCodeMost = F == CacheFormat::int8 ? 127.0f : 448.0f;

// The code of x in a row whose largest magnitude is `most` (finite, above zero): the exact quotient x * 127 / most (448),
// rounded to the nearest step, ties to even.  float32 finds the step but for quotients within a thousandth of a
// border, which 64 bits decide: there the product is exact and the quotient, if no tie, stays on its side (it is off a border by
// 2^-32 at least).  fast = 127 / most, or 0 where that is not a normal number: then all go by 64 bits.
template <CacheFormat F>
__device__ __forceinline__ unsigned code_of(float x, float fast, float most) {
  float t = x * fast;
  int e = 0;   // e4m3: steps of 2^(e - 9), 2^-9 the smallest
  if(fast == 0.0f) t = (float)((double)x * (double)kCodeMost<F> / (double)most);
  if constexpr(F == CacheFormat::e4m3) {
    e = max((int)(__builtin_bit_cast(unsigned, t) >> 23 & 0xff) - (127 - 6), 0);
    t *= __builtin_bit_cast(float, (unsigned)(127 + 9 - e) << 23);
  }
  float r = __builtin_rintf(t);
  if(fast == 0.0f || __builtin_fabsf(t - r) > 0.499f) {
    double q = (double)x * (double)kCodeMost<F> / (double)most;
    if constexpr(F == CacheFormat::e4m3) q *= (double)__builtin_bit_cast(float, (unsigned)(127 + 9 - e) << 23);
    r = (float)__builtin_rint(q);
  }
  if constexpr(F == CacheFormat::int8) return (unsigned)(int)r & 0xffu;
  // (a step up to the next power of two runs over into the exponent)
  return (unsigned)((e << 3) + (int)__builtin_fabsf(r)) | (__builtin_bit_cast(unsigned, x) >> 31 << 7);
}

template <CacheFormat F>
__device__ __forceinline__ float code_factor(float most) {
  const float fast = kCodeMost<F> / most;
  return fast < 1e30f && most < 1e30f ? fast : 0.0f;
}

// Four codes as float32 values.
template <CacheFormat F>
__device__ __forceinline__ void values_of(unsigned w, float (&x)[4]) {
  if constexpr(F == CacheFormat::int8) {
#pragma unroll
    for(int i = 0; i < 4; ++i) x[i] = (float)(int)(int8_t)(w >> (8 * i));
  } else {
    const cache_h2 lo = half2_of<F, 0, 1>(w, w), hi = half2_of<F, 2, 3>(w, w);
    x[0] = (float)lo[0] * 256.0f;
    x[1] = (float)lo[1] * 256.0f;
    x[2] = (float)hi[0] * 256.0f;
    x[3] = (float)hi[1] * 256.0f;
  }
}

// ---- trees of drafted tokens ---------------------------------------------------------------------------
// Lane i: the drafted tokens that token i (of n <= 64) descends from and itself, one bit each.  A wave's work.
__device__ __forceinline__ unsigned long long lineage(const int* __restrict__ parents, int n, int lane) {
  int p = lane < n ? parents[lane] : -1;
  if(p >= lane) p = -1;
  unsigned long long seen = 1ull << lane;
  while(__any(p >= 0)) {   // (a parent is before its child: six rounds at the most, each twice as far up)
    const unsigned lo = __shfl((unsigned)seen, p & 63, 64), hi = __shfl((unsigned)(seen >> 32), p & 63, 64);
    const int up = __shfl(p, p & 63, 64);
    if(p >= 0) {
      seen |= (unsigned long long)hi << 32 | lo;
      p = up;
    }
  }
  return seen;
}

}  // namespace marian_hip
