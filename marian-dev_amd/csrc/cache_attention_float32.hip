// Attention over a quantized cache, float32 activations.
#include "cache_attention_launch.h"

namespace marian_hip {

int launch_cache_attention_float32(const CacheAttentionArgs& a, const CacheAttentionPlan& p, int format, hipStream_t st) {
  return launch_cache_attention<float>(a, p, format, st);
}

}  // namespace marian_hip
