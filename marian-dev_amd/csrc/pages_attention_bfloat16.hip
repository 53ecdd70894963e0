// Attention over pages of bfloat16 keys and values.
#include "pages_attention_launch.h"

namespace marian_hip {

int launch_pages_attention_bfloat16(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  return launch_pages_attention<bf16_t>(a, p, st);
}

}  // namespace marian_hip
