// What the launchers of the attention over a quantized cache are handed; one source file for each type of activations.
#pragma once

#include <hip/hip_runtime.h>

#include "cache_plan.h"

namespace marian_hip {

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
  int S, Hk, G, n, cap, dk, row_tiles, target, items;
  float scale_log2;     // scale / ln 2
};

int launch_cache_attention_float32(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st);
int launch_cache_attention_float16(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st);
int launch_cache_attention_bfloat16(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st);

}  // namespace marian_hip
