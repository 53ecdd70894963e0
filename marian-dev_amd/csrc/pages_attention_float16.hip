// Attention over pages of float16 keys and values.
#include "pages_attention_launch.h"

namespace marian_hip {

int launch_pages_attention_float16(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st) {
  return launch_pages_attention<_Float16>(a, p, st);
}

}  // namespace marian_hip
