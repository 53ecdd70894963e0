// The form of the attention that a plan says, for one type of activations.
#pragma once

#include <type_traits>

#include "../../include/marian_hip_ops.h"
#include "abi_common.h"
#include "cache_attention_kernel.h"

namespace marian_hip {

template <typename T, CacheFormat F, int W>
int launch_cache_attention(const CacheAttentionArgs& a, const CacheAttentionPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.grid), block(64 * W);
  auto few = [&](auto rows) -> int {
    constexpr int R = decltype(rows)::value;
    if(p.dp == 64) MH_LAUNCH((cache_attention_few_kernel<T, F, 64, R, W>), grid, block, 0, st, a);
    else MH_LAUNCH((cache_attention_few_kernel<T, F, 128, R, W>), grid, block, 0, st, a);
    return MARIAN_HIP_OK;
  };
  if(p.few == 1) return few(std::integral_constant<int, 1>());
  if(p.few == 2) return few(std::integral_constant<int, 2>());
  if(p.few == 4) return few(std::integral_constant<int, 4>());
  if(p.few == 8) return few(std::integral_constant<int, 8>());
  if(p.dp == 64 && p.qt == 1) MH_LAUNCH((cache_attention_kernel<T, F, 64, 1, W>), grid, block, 0, st, a);
  else if(p.dp == 64) MH_LAUNCH((cache_attention_kernel<T, F, 64, 2, W>), grid, block, 0, st, a);
  else if(p.dp == 128 && p.qt == 1) MH_LAUNCH((cache_attention_kernel<T, F, 128, 1, W>), grid, block, 0, st, a);
  else if(p.dp == 128) MH_LAUNCH((cache_attention_kernel<T, F, 128, 2, W>), grid, block, 0, st, a);
  else MH_LAUNCH((cache_attention_kernel<T, F, 256, 1, W>), grid, block, 0, st, a);
  return MARIAN_HIP_OK;
}

template <typename T, CacheFormat F>
int launch_cache_attention_many(const CacheAttentionArgs& a, const CacheAttentionPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.grid), block(256);
  if(p.dp == 64 && p.qt == 1) MH_LAUNCH((cache_attention_many_kernel<T, F, 64, 1>), grid, block, 0, st, a);
  else if(p.dp == 64) MH_LAUNCH((cache_attention_many_kernel<T, F, 64, 2>), grid, block, 0, st, a);
  else if(p.dp == 128 && p.qt == 1) MH_LAUNCH((cache_attention_many_kernel<T, F, 128, 1>), grid, block, 0, st, a);
  else if(p.dp == 128) MH_LAUNCH((cache_attention_many_kernel<T, F, 128, 2>), grid, block, 0, st, a);
  else MH_LAUNCH((cache_attention_many_kernel<T, F, 256, 1>), grid, block, 0, st, a);
  return MARIAN_HIP_OK;
}

template <typename T, CacheFormat F>
int launch_cache_attention(const CacheAttentionArgs& a, const CacheAttentionPlan& p, hipStream_t st) {
  if(p.many) return launch_cache_attention_many<T, F>(a, p, st);
  if(p.waves == 4) return launch_cache_attention<T, F, 4>(a, p, st);
  if(p.waves == 2) return launch_cache_attention<T, F, 2>(a, p, st);
  return launch_cache_attention<T, F, 1>(a, p, st);
}

template <typename T>
int launch_cache_attention(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st) {
  if(format == MARIAN_HIP_CACHE_INT8) return launch_cache_attention<T, CacheFormat::int8>(a, p, st);
  return launch_cache_attention<T, CacheFormat::e4m3>(a, p, st);
}

}  // namespace marian_hip
