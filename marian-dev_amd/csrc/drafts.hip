// Verification of drafted tokens.  Declarations: include/marian_hip_ops.h
#include "../../include/marian_hip_ops.h"

#include <hip/hip_runtime.h>

#include <algorithm>

#include "abi_common.h"
#include "cache_args.h"
#include "cache_attention_kernel.h"

using namespace marian_hip;

namespace {

struct VerifyArgs {
  const int *tokens, *counts, *parents;
  const void *target, *draft;
  const float* random;
  long long t_s, t_n, d_s, d_n;   // values from a sequence and a row of the target's and the draft's to the next
  int *path, *accepted, *next;
  unsigned* counters;
  double* sums;   // of what is drawn from, and of the target's row, of every part
  int n, vocab, parts;
};

constexpr int kVerifyThreads = 256, kEach = 16;            // words of a thread
constexpr int kVerifyPart = kVerifyThreads * kEach;        // ... and of a workgroup
constexpr int64_t kVerifySequences = kCacheMost;           // of a launch: a counter each

__device__ __forceinline__ double lane_double(double x, int lane) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_readlane((unsigned)b, lane), hi = __builtin_amdgcn_readlane((unsigned)(b >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// A probability as it counts: nothing where it is below zero or NaN.
__device__ __forceinline__ double counted(double x) { return x > 0.0 ? x : 0.0; }

// What became of a sequence's tokens: a bit for each kept one, the last of these, and the ones refused as its children.
struct Verdict {
  unsigned long long kept, refused;
  int last, token;   // token: the lane's
};

// All waves do the same, lanes being tokens.  A token is judged as if its parent were kept - the row that it is held against is known -,
// and is kept if all that it descends from are.
template <typename T>
__device__ __forceinline__ Verdict judge(const VerifyArgs& a, int s, int lane, int count) {
  const long long at = (long long)s * a.n + lane;
  const bool there = lane < count;
  Verdict y;
  y.token = there ? a.tokens[at] : -1;
  int parent = !there || !a.parents ? lane - 1 : a.parents[at];
  if(parent >= lane || parent < 0) parent = -1;
  const bool judged = there && parent >= 0 && (unsigned)y.token < (unsigned)a.vocab;
  double p = 0.0, q = 1.0;
  if(judged) p = counted(to_float(static_cast<const T*>(a.target)[s * a.t_s + parent * a.t_n + y.token]));
  if(judged && a.draft) q = to_float(static_cast<const T*>(a.draft)[s * a.d_s + parent * a.d_n + y.token]);
  const double u = there ? a.random[at] : 0.0;
  unsigned long long siblings = 0;   // that come before
  double gone = 0.0;                 // their probabilities
  if(a.parents) {
    for(int j = 1; j < count; ++j) {
      const double pj = lane_double(p, j);   // (by now without what a sibling had already)
      const int parent_j = __builtin_amdgcn_readlane(parent, j), token_j = __builtin_amdgcn_readlane(y.token, j);
      if(lane > j && parent == parent_j) {
        siblings |= 1ull << j;
        if(y.token == token_j) p = 0.0;
        gone += pj;
      }
    }
  }
  const bool likes = judged && u * (a.draft ? q : 1.0 - gone) < p;
  const unsigned long long liked = __ballot(likes), chosen = __ballot(likes && !(liked & siblings));
  if(a.parents) {
    int up = parent;
    unsigned long long line = 1ull << lane;   // itself and what it descends from
    while(__any(up >= 0)) {   // (a parent is before its child: six rounds at the most, each twice as far up)
      const unsigned lo = __shfl((unsigned)line, up & 63, 64), hi = __shfl((unsigned)(line >> 32), up & 63, 64);
      const int next = __shfl(up, up & 63, 64);
      if(up >= 0) {
        line |= (unsigned long long)hi << 32 | lo;
        up = next;
      }
    }
    y.kept = __ballot(there && (line & 1) && !(line & ~1ull & ~chosen));
  } else {
    const int row = __builtin_ctzll(~(chosen >> 1));   // (the shift leaves a zero on top)
    y.kept = count > 0 ? (2ull << row) - 1 : 0;
  }
  y.last = y.kept ? 63 - __builtin_clzll(y.kept) : 0;
  y.refused = __ballot(there && lane > 0 && parent == y.last) & ~y.kept;
  return y;
}

// What the next token is drawn from: words of the target's row, less the draft's or the refused words.
template <typename T>
struct Weights {
  static constexpr int kTogether = 16 / sizeof(T), kVectors = kEach / kTogether;
  const T *p, *q;   // q null: not taken away
  const Verdict& y;
  int vocab;
  // A vector of words from `at` on: what is left, and the target's own.
  __device__ __forceinline__ void load(int at, double (&left)[kTogether], double (&own)[kTogether]) const {
    T x[kTogether], z[kTogether];
    const bool whole = at + kTogether <= vocab;
    if(whole) {
      __builtin_memcpy(x, p + at, 16);
      if(q) __builtin_memcpy(z, q + at, 16);
    }
#pragma unroll
    for(int e = 0; e < kTogether; ++e) {
      const bool is = at + e < vocab;
      if(!whole && is) {
        x[e] = p[at + e];
        if(q) z[e] = q[at + e];
      }
      own[e] = is ? counted(to_float(x[e])) : 0.0;
      left[e] = is && q ? counted((double)to_float(x[e]) - (double)to_float(z[e])) : own[e];
    }
  }
  // ... without the refused words among `size` from `from` on.
  template <int COUNT>
  __device__ __forceinline__ void refuse(double (&left)[COUNT], int at) const {
#pragma unroll 1
    for(unsigned long long bits = q ? 0 : y.refused; bits; bits &= bits - 1) {
      const int word = __builtin_amdgcn_readlane(y.token, __builtin_ctzll(bits)) - at;
#pragma unroll
      for(int e = 0; e < COUNT; ++e) left[e] = word == e ? 0.0 : left[e];
    }
  }
};

__device__ __forceinline__ double wave_sum_before(double x, int lane, double& all) {   // exclusive, in the lanes' order
  double sum = x;
#pragma unroll
  for(int o = 1; o < 64; o <<= 1) {
    const double other = __shfl_up(sum, o, 64);
    if(lane >= o) sum += other;
  }
  all = lane_double(sum, 63);
  const double before = __shfl_up(sum, 1, 64);
  return lane == 0 ? 0.0 : before;
}

struct VerifyShared {
  double wave[2][kVerifyThreads / 64];
  double before;
  int found, last, is_last;
};

// The exclusive sum over a workgroup's threads, and the sum of all; `which`: a place in LDS that nobody reads any more.
__device__ __forceinline__ double group_sum_before(VerifyShared& sh, int which, double x, double& all) {
  const int tid = threadIdx.x, wave = tid >> 6;
  double mine, before = wave_sum_before(x, tid & 63, mine);
  if((tid & 63) == 0) sh.wave[which][wave] = mine;
  __syncthreads();
  double ahead = 0.0;
  all = 0.0;
#pragma unroll
  for(int i = 0; i < kVerifyThreads / 64; ++i) {
    if(i == wave) ahead = all;
    all += sh.wave[which][i];
  }
  return ahead + before;
}

// Every workgroup judges the tokens of a sequence anew - a chain of three loads - and sums its part of the words that the next token is drawn from; the
// last one to arrive finds the part in which the drawn number lies, and the word in it.  All sums are in 64 bits and in the words' order.
// The kept tokens cost nothing but their own probabilities, so what moves is one row of the target's, and one of the draft's where a
// token was refused.
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyArgs a, int first) {
  using W = Weights<T>;
  constexpr int kTogether = W::kTogether, kVectors = W::kVectors;
  __shared__ VerifyShared sh;
  const int tid = threadIdx.x, lane = tid & 63, s = first + blockIdx.y, part = blockIdx.x;
  const int count = a.counts ? clamp_int(a.counts[s], 0, a.n) : a.n;
  const Verdict y = judge<T>(a, s, lane, count);
  const double u = a.random[(long long)s * a.n];
  if(part == 0 && tid < 64) {
    const int accepted = __builtin_popcountll(y.kept);
    const long long row = (long long)s * a.n;
    if(lane < a.n && lane >= accepted) a.path[row + lane] = -1;
    if(y.kept >> lane & 1) a.path[row + __builtin_popcountll(y.kept & ((1ull << lane) - 1))] = lane;
    if(lane == 0) a.accepted[s] = accepted;
    if(lane == 0 && count == 0) a.next[s] = -1;
  }
  if(count == 0) return;
  const W w{static_cast<const T*>(a.target) + s * a.t_s + y.last * a.t_n,
            a.draft && y.refused ? static_cast<const T*>(a.draft) + s * a.d_s + y.last * a.d_n : nullptr, y, a.vocab};
  if(tid == 0) {
    sh.found = 0x7fffffff;
    sh.last = -1;
  }
  const int from = part * kVerifyPart;
  double left_sum = 0.0, own_sum = 0.0;
  {
    double left[kVectors][kTogether], own[kVectors][kTogether];
#pragma unroll
    for(int v = 0; v < kVectors; ++v) w.load(from + (v * kVerifyThreads + tid) * kTogether, left[v], own[v]);
#pragma unroll
    for(int v = 0; v < kVectors; ++v) {
      w.refuse(left[v], from + (v * kVerifyThreads + tid) * kTogether);
#pragma unroll
      for(int e = 0; e < kTogether; ++e) {
        left_sum += left[v][e];
        own_sum += own[v][e];
      }
    }
  }
  double left_all, own_all;
  group_sum_before(sh, 0, left_sum, left_all);
  group_sum_before(sh, 1, own_sum, own_all);
  int found_part = 0;
  double ahead = 0.0;   // of the part that the word is in
  if(a.parts > 1) {
    unsigned long long* const sums = reinterpret_cast<unsigned long long*>(a.sums) + 2 * (long long)blockIdx.y * a.parts;
    if(tid == 0) {
      __hip_atomic_store(sums + 2 * part, __builtin_bit_cast(unsigned long long, left_all), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(sums + 2 * part + 1, __builtin_bit_cast(unsigned long long, own_all), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if(!cache_arrived_last(a.counters + blockIdx.y, a.parts, sh.is_last)) return;
    const int each = (a.parts + kVerifyThreads - 1) / kVerifyThreads, i0 = tid * each, i1 = min(i0 + each, a.parts);
    auto sum_of = [&](int i, int which) {
      return __builtin_bit_cast(double, __hip_atomic_load(sums + 2 * i + which, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    };
    double mine[2] = {0.0, 0.0};
    for(int i = i0; i < i1; ++i) {
      mine[0] += sum_of(i, 0);
      mine[1] += sum_of(i, 1);
    }
    double before = group_sum_before(sh, 0, mine[0], left_all);
    const double before_own = group_sum_before(sh, 1, mine[1], own_all);
    const int which = left_all > 0.0 ? 0 : 1;
    if(which) before = before_own;
    const double bar = u * (which ? own_all : left_all);
    double sum = before;
    for(int i = i0; i < i1; ++i) {
      const double x = sum_of(i, which);
      sum += x;
      if(x > 0.0) atomicMax(&sh.last, i);
      if(x > 0.0 && sum > bar) {
        atomicMin(&sh.found, i);
        break;
      }
    }
    __syncthreads();
    // (rounding may leave none where the drawn number is next to one: the last that has anything)
    found_part = sh.found != 0x7fffffff ? sh.found : max(sh.last, 0);
    if(found_part >= i0 && found_part < i1) {
      for(int i = i0; i < found_part; ++i) before += sum_of(i, which);
      sh.before = before;
    }
    __syncthreads();
    ahead = sh.before;
    if(tid == 0) {
      sh.found = 0x7fffffff;
      sh.last = -1;
    }
    __syncthreads();
  }
  const bool of_left = left_all > 0.0;
  const double bar = u * (of_left ? left_all : own_all);
  // sixteen words that follow each other to a thread
  const int at = found_part * kVerifyPart + tid * kEach;
  double x[kEach], sum = 0.0;
#pragma unroll
  for(int v = 0; v < kVectors; ++v) {
    double left[kTogether], own[kTogether];
    w.load(at + v * kTogether, left, own);
    w.refuse(left, at + v * kTogether);
#pragma unroll
    for(int e = 0; e < kTogether; ++e) {
      x[v * kTogether + e] = of_left ? left[e] : own[e];
      sum += x[v * kTogether + e];
    }
  }
  double all;
  double running = ahead + group_sum_before(sh, 0, sum, all);
  int found = 0x7fffffff, last = -1;
#pragma unroll
  for(int e = 0; e < kEach; ++e) {
    running += x[e];
    if(x[e] > 0.0) last = at + e;
    if(x[e] > 0.0 && running > bar && found == 0x7fffffff) found = at + e;
  }
  if(found != 0x7fffffff) atomicMin(&sh.found, found);
  if(last >= 0) atomicMax(&sh.last, last);
  __syncthreads();
  if(tid == 0) a.next[s] = sh.found != 0x7fffffff ? sh.found : sh.last;
}

}  // namespace

extern "C" {

size_t marian_hip_verify_drafts_workspace_bytes(int64_t sequences, int64_t vocab) {
  if(sequences < 1 || vocab < 1 || sequences > kMaxSequences || vocab >= 1 << 24 || vocab <= kVerifyPart) return 0;
  return (size_t)(kCacheCounterBytes + std::min(sequences, kVerifySequences) * ((vocab + kVerifyPart - 1) / kVerifyPart) * 16);
}

int marian_hip_verify_drafts(const marian_hip_drafted* d, int32_t* path, int32_t* accepted, int32_t* next, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if(!d) return MARIAN_HIP_ERR_NULL;
  MH_CHECK(check_type(d->type));
  const int64_t S = d->sequences, n = d->n, vocab = d->vocab;
  if(S < 0 || n < 1 || n > MARIAN_HIP_TREE_MAX || vocab < 1 || (d->draft && d->parents)) return MARIAN_HIP_ERR_SHAPE;
  if(S > kMaxSequences || vocab >= 1 << 24) return MARIAN_HIP_ERR_RANGE;
  if(S == 0) return MARIAN_HIP_OK;
  if(!d->tokens || !d->target || !d->random || !path || !accepted || !next) return MARIAN_HIP_ERR_NULL;
  const void* words[] = {d->tokens, d->counts, d->parents, d->random, path, accepted, next};
  for(const void* p : words)
    if(!aligned(p, 4)) return MARIAN_HIP_ERR_ALIGN;
  const int width = width_of(d->type);
  if(!aligned(d->target, width) || !aligned(d->draft, width)) return MARIAN_HIP_ERR_ALIGN;
  auto rows = [&](const void* p, const int64_t* st, int64_t count, Span* span) -> int {
    *span = Span{nullptr, 0};
    if(!p || count == 0) return MARIAN_HIP_OK;
    int64_t last = vocab;
    const int64_t size[2] = {S, count};
    for(int i = 0; i < 2; ++i) {
      if(size[i] <= 1) continue;
      if(st[i] < 0 || st[i] > (int64_t)1 << 44) return MARIAN_HIP_ERR_SHAPE;
      last += (size[i] - 1) * st[i];
    }
    *span = Span{p, last * width};
    return MARIAN_HIP_OK;
  };
  Span target, draft;
  MH_CHECK(rows(d->target, d->target_strides, n, &target));
  MH_CHECK(rows(d->draft, d->draft_strides, n - 1, &draft));
  const int64_t need = (int64_t)marian_hip_verify_drafts_workspace_bytes(S, vocab);
  if(need > 0 && !workspace) return MARIAN_HIP_ERR_NULL;
  if((int64_t)workspace_bytes < need) return MARIAN_HIP_ERR_WORKSPACE;
  if(!aligned(workspace, 256)) return MARIAN_HIP_ERR_ALIGN;
  const int64_t each = 4 * S, all = 4 * S * n;
  const Span work{need > 0 ? workspace : nullptr, need};
  MH_CHECK(apart({{path, all}, {accepted, each}, {next, each}, work}, {{d->tokens, all}, {d->counts, each}, {d->parents, all}, {d->random, all}, target, draft}));
  MH_CHECK(apart({{path, all}}, {{accepted, each}, {next, each}, work}));
  MH_CHECK(apart({{accepted, each}}, {{next, each}, work}));
  MH_CHECK(apart({{next, each}}, {work}));
  VerifyArgs a{};
  a.tokens = d->tokens;
  a.counts = d->counts;
  a.parents = d->parents;
  a.target = d->target;
  a.draft = n > 1 ? d->draft : nullptr;
  a.random = d->random;
  a.t_s = S > 1 ? d->target_strides[0] : 0;
  a.t_n = d->target_strides[1];
  a.d_s = S > 1 ? d->draft_strides[0] : 0;
  a.d_n = d->draft_strides[1];
  a.path = path;
  a.accepted = accepted;
  a.next = next;
  a.counters = static_cast<unsigned*>(workspace);
  a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + kCacheCounterBytes);
  a.n = (int)n;
  a.vocab = (int)vocab;
  a.parts = (int)((vocab + kVerifyPart - 1) / kVerifyPart);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for(int64_t first = 0; first < S; first += kVerifySequences) {
    const dim3 grid((unsigned)a.parts, (unsigned)std::min(S - first, kVerifySequences));
    MH_CHECK(for_type(d->type, [&](auto t) -> int {
      MH_LAUNCH(verify_kernel<decltype(t)>, grid, dim3(kVerifyThreads), 0, st, a, (int)first);
      return MARIAN_HIP_OK;
    }));
  }
  return MARIAN_HIP_OK;
}

}  // extern "C"
