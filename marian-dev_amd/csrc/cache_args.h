// What the host side of the operators over caches looks at in their arguments (host code).
#pragma once

#include <algorithm>
#include <array>
#include <cstdint>
#include <utility>

#include "../../include/marian_hip_ops.h"
#include "abi_common.h"
#include "cache_codes.h"

namespace marian_hip {

struct Strides {   // in values
  long long s, h, n;
};

template <typename F>
int for_type(int type, F f) {
  if(type == MARIAN_HIP_FLOAT32) return f(float());
  if(type == MARIAN_HIP_FLOAT16) return f(_Float16());
  return f(bf16_t());
}

inline int width_of(int type) { return type == MARIAN_HIP_FLOAT32 ? 4 : 2; }
inline bool aligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool row_size(int64_t dk) { return dk >= 16 && dk <= 256 && dk % 16 == 0; }
constexpr int64_t kMostThreads = 0xffffffff;   // of a launch, in one dimension
constexpr int64_t kMaxTokens = 1 << 20, kMaxHeads = 4096, kMaxSequences = 65535;

#define MH_CHECK(expr)                             \
  do {                                             \
    const int check_status_ = (expr);              \
    if(check_status_ != MARIAN_HIP_OK) return check_status_; \
  } while(0)

inline int check_type(int type) { return type >= MARIAN_HIP_FLOAT32 && type <= MARIAN_HIP_BFLOAT16 ? MARIAN_HIP_OK : MARIAN_HIP_ERR_SHAPE; }

// A tensor [sequences, heads, n, dk]: from its first to its last byte in `span`.
inline int check_rows(const void* p, const int64_t* st, int type, int64_t sequences, int64_t heads, int64_t n, int64_t dk, Span* span) {
  if(!p || !st) return MARIAN_HIP_ERR_NULL;
  const int64_t whole = 16 / width_of(type);
  if(!aligned(p, 16)) return MARIAN_HIP_ERR_ALIGN;
  int64_t last = dk;
  const int64_t size[3] = {sequences, heads, n};
  for(int i = 0; i < 3; ++i) {
    if(size[i] <= 1) continue;
    if(st[i] < 0 || st[i] > (int64_t)1 << 44) return MARIAN_HIP_ERR_SHAPE;
    if(st[i] % whole != 0) return MARIAN_HIP_ERR_ALIGN;
    last += (size[i] - 1) * st[i];
  }
  *span = Span{p, last * width_of(type)};
  return MARIAN_HIP_OK;
}
// ... that is written: its rows share no memory, each dimension's step reaching over all that lies within one of its steps.
inline int check_written(const void* p, const int64_t* st, int type, int64_t sequences, int64_t heads, int64_t n, int64_t dk, Span* span) {
  MH_CHECK(check_rows(p, st, type, sequences, heads, n, dk, span));
  std::array<std::pair<int64_t, int64_t>, 3> dim{{{sequences > 1 ? st[0] : 0, sequences}, {heads > 1 ? st[1] : 0, heads}, {n > 1 ? st[2] : 0, n}}};
  std::sort(dim.begin(), dim.end());
  int64_t within = dk;
  for(const auto& [step, size] : dim) {
    if(size <= 1) continue;
    if(step < within) return MARIAN_HIP_ERR_ALIAS;
    within += (size - 1) * step;
  }
  return MARIAN_HIP_OK;
}
inline Strides strides(const int64_t* st) { return Strides{st[0], st[1], st[2]}; }
inline bool same_rows(const void* a, const int64_t* x, const void* b, const int64_t* y, int64_t sequences, int64_t heads, int64_t n) {
  return a == b && (sequences <= 1 || x[0] == y[0]) && (heads <= 1 || x[1] == y[1]) && (n <= 1 || x[2] == y[2]);
}

}  // namespace marian_hip
