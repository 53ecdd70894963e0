// Attention over pages of float32 keys and values.
#include "pages_attention_launch.h"

namespace marian_hip {

int launch_pages_attention_float32(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  return launch_pages_attention<float>(a, p, st);
}

}  // namespace marian_hip
