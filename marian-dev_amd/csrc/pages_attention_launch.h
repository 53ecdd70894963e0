// The form of the attention over pages that a plan says, for one type.
#pragma once

#include "../../include/marian_hip_ops.h"
#include "abi_common.h"
#include "pages_attention_kernel.h"

namespace marian_hip {

template <typename T, int DP, int W>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  constexpr int kMost = pages_most_qt(sizeof(T), DP);
  const dim3 grid((unsigned)p.grid), block(64 * W);
  if(p.qt == 1) {
    MH_LAUNCH((pages_attention_kernel<T, DP, 1, W>), grid, block, 0, st, a);
    return MARIAN_HIP_OK;
  }
  if constexpr(kMost >= 2) {
    if(p.qt == 2) {
      MH_LAUNCH((pages_attention_kernel<T, DP, 2, W>), grid, block, 0, st, a);
      return MARIAN_HIP_OK;
    }
  }
  if constexpr(kMost >= 4) {
    if(p.qt == 4) {
      MH_LAUNCH((pages_attention_kernel<T, DP, 4, W>), grid, block, 0, st, a);
      return MARIAN_HIP_OK;
    }
  }
  return MARIAN_HIP_ERR_SHAPE;
}

template <typename T, int W>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  if(p.dp == 64) return launch_pages_attention<T, 64, W>(a, p, st);
  if(p.dp == 128) return launch_pages_attention<T, 128, W>(a, p, st);
  return launch_pages_attention<T, 256, W>(a, p, st);
}

template <typename T>
int launch_pages_attention(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  return p.waves == 1 ? launch_pages_attention<T, 1>(a, p, st) : launch_pages_attention<T, 4>(a, p, st);
}

}  // namespace marian_hip
