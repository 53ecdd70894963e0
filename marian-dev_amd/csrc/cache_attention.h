// What the launchers of the attention over a quantized cache are handed; one source file for each type of activations.
#pragma once

#include <hip/hip_runtime.h>

#include "cache_plan.h"

namespace marian_hip {

// Division of numbers below 2^32 by a number that the host knows: the high half of the product with 2^32 / d falls short by one at the most.
struct CacheDivisor {
  unsigned d, m;
  CacheDivisor() = default;
  explicit CacheDivisor(unsigned by) : d(by), m(by == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / by)) {}
  __device__ __forceinline__ unsigned of(unsigned n, unsigned& rest) const {
    unsigned q = __umulhi(n, m);
    rest = n - q * d;
    if(rest >= d) {
      ++q;
      rest -= d;
    }
    return q;
  }
  __device__ __forceinline__ unsigned of(unsigned n) const {
    unsigned rest;
    return of(n, rest);
  }
};

struct CacheAttentionArgs {
  const void* q;
  long long q_s, q_h, q_n;   // in values
  void* out;
  long long o_s, o_h, o_n;
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int *lens, *counts, *parents;
  float* part;          // partial results, row_floats to a row: the rows' values, then their logarithms
  unsigned* counters;   // parts that have arrived, zero between calls
  int S, Hk, G, n, cap, dk, row_tiles, target, least, items;
  CacheDivisor by_tiles, by_heads, by_group;
  float scale_log2;     // scale / ln 2
};

int launch_cache_attention_float32(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st);
int launch_cache_attention_float16(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st);
int launch_cache_attention_bfloat16(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st);

}  // namespace marian_hip
