// The form of the attention over pages that a plan says, for one type.
#pragma once

#include "../../include/marian_hip_ops.h"
#include "abi_common.h"
#include "pages_attention_kernel.h"

namespace marian_hip {

template <typename T, int DP, bool WHOLE, int W>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  constexpr int kMost = pages_most_qt(sizeof(T), DP);
  const dim3 grid((unsigned)p.grid), block(64 * W);
  if constexpr(kMost >= 2) {
    if(p.qt == 2) {
      MH_LAUNCH((pages_attention_kernel<T, DP, WHOLE, 2, W>), grid, block, 0, st, a);
      return MARIAN_HIP_OK;
    }
  }
  MH_LAUNCH((pages_attention_kernel<T, DP, WHOLE, 1, W>), grid, block, 0, st, a);
  return MARIAN_HIP_OK;
}

template <typename T, int DP, bool WHOLE>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  if constexpr(pages_has_many(sizeof(T), DP)) {
    if(p.many) {
      const dim3 grid((unsigned)p.grid), block(64 * p.waves);
      if(p.tile_rows == 64) MH_LAUNCH((pages_attention_many_kernel<T, DP, WHOLE, 64>), grid, block, 0, st, a);
      else MH_LAUNCH((pages_attention_many_kernel<T, DP, WHOLE, 128>), grid, block, 0, st, a);
      return MARIAN_HIP_OK;
    }
  }
  return p.waves == 1 ? launch_pages_attention<T, DP, WHOLE, 1>(a, p, st) : launch_pages_attention<T, DP, WHOLE, 4>(a, p, st);
}

// WHOLE: rows of dp values; their places are constants then.
template <typename T, int DP>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  return a.dk == DP ? launch_pages_attention<T, DP, true>(a, p, st) : launch_pages_attention<T, DP, false>(a, p, st);
}

template <typename T>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  if(p.dp == 64) return launch_pages_attention<T, 64>(a, p, st);
  if(p.dp == 128) return launch_pages_attention<T, 128>(a, p, st);
  return launch_pages_attention<T, 256>(a, p, st);
}

}  // namespace marian_hip
