// Attention over a quantized cache, bfloat16 activations.
#include "cache_attention_launch.h"

namespace marian_hip {

int launch_cache_attention_bfloat16(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st) {
  return launch_cache_attention<bf16_t>(a, p, format, st);
}

}  // namespace marian_hip
