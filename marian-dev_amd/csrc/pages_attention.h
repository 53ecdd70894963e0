// What the launchers of the attention over pages are handed; one source file for each type.
#pragma once

#include <hip/hip_runtime.h>

#include "cache_attention.h"
#include "pages_plan.h"

namespace marian_hip {

// cap: positions that a row of the table has room for; k, v, their scales and parents are not used
struct PagesAttentionArgs : CacheAttentionArgs {
  const unsigned char *k_pages, *v_pages;
  const int* table;
  int row, pages, page;             // of the table; there are; positions of a page
  long long page_bytes, head_bytes; // from a page to the next, from a head of it to the next
  CacheDivisor by_eights;           // eights of positions of a page
};

int launch_pages_attention_float32(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st);
int launch_pages_attention_float16(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st);
int launch_pages_attention_bfloat16(const PagesAttentionArgs& a, const PagesAttentionPlan& p, hipStream_t st);

}  // namespace marian_hip
