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
  double* sums;   // of what is drawn from, of every share
  int n, vocab, parts;
};

// Eight waves: a sequence's workgroups judge its tokens each, ahead of all else, and a workgroup's words are summed in 64 bits, five operations a
// word. With 4, 8 and 16 of them 32000 words of one sequence took 5.7, 6.3 and 9.1 us, 131071 words of 64 sequences 44.0, 20.2 and 22.0.
constexpr int kVerifyWaves = 8, kVerifyThreads = 64 * kVerifyWaves;
constexpr int kShare = 2 * kVerifyThreads;                 // words of a wave ...
constexpr int kVerifyPart = kVerifyWaves * kShare;         // ... and of a workgroup
constexpr int64_t kVerifySequences = kCacheMost;           // of a launch: a counter each

// x of the lane that a control of lane movement says, zero where there is none.
template <int CONTROL, int ROWS, bool ZERO>
__device__ __forceinline__ double moved(double x) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CONTROL, ROWS, 0xf, ZERO);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CONTROL, ROWS, 0xf, ZERO);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// Inclusive sum over the lanes of a wave: within rows of sixteen lanes, then over the rows, without LDS.
__device__ __forceinline__ double lanes_sum(double x) {
  x += moved<0x111, 0xf, true>(x);    // row_shr:1
  x += moved<0x112, 0xf, true>(x);    // row_shr:2
  x += moved<0x114, 0xf, true>(x);    // row_shr:4
  x += moved<0x118, 0xf, true>(x);    // row_shr:8
  x += moved<0x142, 0xa, false>(x);   // row_bcast:15
  x += moved<0x143, 0xc, false>(x);   // row_bcast:31
  return x;
}

// What became of a sequence's tokens: a bit for each kept one, the last of these, and the ones refused as its children.
struct Verdict {
  unsigned long long kept, refused;
  int last;
  int token[64];
};

__device__ __forceinline__ double lane_double(double x, int lane) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_readlane((unsigned)b, lane), hi = __builtin_amdgcn_readlane((unsigned)(b >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// A wave's work, lanes being tokens.  The row that a token is held against is its parent's, so all probabilities are asked for at once; then the
// kept tokens are followed from the first on.
template <typename T>
__device__ __forceinline__ void judge(const VerifyArgs& a, int s, int lane, int count, Verdict& y) {
  const long long at = (long long)s * a.n + lane;
  const bool inside = lane < a.n, there = lane < count;
  const int token = inside ? a.tokens[at] : -1;   // (asked for beside the count)
  int parent = !inside || !a.parents ? lane - 1 : a.parents[at];
  const double u = inside ? a.random[at] : 0.0;
  if(parent >= lane || parent < 0) parent = -1;
  const bool judged = inside && parent >= 0 && (unsigned)token < (unsigned)a.vocab;
  double p = 0.0, q = 1.0;
  if(judged) {
    p = fmaxf(to_float(static_cast<const T*>(a.target)[s * a.t_s + parent * a.t_n + token]), 0.0f);
    if(a.draft) q = fmaxf(to_float(static_cast<const T*>(a.draft)[s * a.d_s + parent * a.d_n + token]), 0.0f);
  }
  unsigned long long kept = count > 0, refused = 0;
  int last = 0;
  if(a.parents) {
    for(;;) {
      unsigned long long children = __ballot(there && parent == last);
      double gone = 0.0;
      int next = 0;
      for(refused = 0; children && !next; children &= children - 1) {
        const int i = __builtin_ctzll(children);
        const unsigned long long alike = __ballot(token == __builtin_amdgcn_readlane(token, i));
        const double its = alike & refused ? 0.0 : lane_double(p, i);   // (a token that a sibling had already has nothing left)
        if(lane_double(u, i) * (1.0 - gone) < its) {
          next = i;
        } else {
          refused |= 1ull << i;
          gone += its;
        }
      }
      if(!next) break;
      kept |= 1ull << next;
      last = next;
    }
  } else {
    const unsigned long long likes = __ballot(there && u * q < p);
    last = __builtin_ctzll(~(likes >> 1));   // (the shift leaves a zero on top)
    kept = count > 0 ? (2ull << last) - 1 : 0;
    refused = last + 1 < count ? 2ull << last : 0;
  }
  y.token[lane] = token;
  if(lane == 0) {
    y.kept = kept;
    y.refused = refused;
    y.last = last;
  }
}

// What the next token is drawn from: words of the target's row, less the draft's or the refused words.  Negative numbers and NaN count as nothing.
template <typename T>
struct Weights {
  static constexpr int kTogether = 16 / sizeof(T);
  const T *p, *q;   // q null: not taken away
  const int* token;
  int vocab;
  struct Raw {
    T x[kTogether], z[kTogether];
  };
  // Sixteen bytes of words from `at` on; WHOLE: all of them are there.
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(Raw& r, int at) const {
    if constexpr(WHOLE) {
      __builtin_memcpy(r.x, p + at, 16);
      if(q) __builtin_memcpy(r.z, q + at, 16);
    } else {
#pragma unroll
      for(int e = 0; e < kTogether; ++e) {
        r.x[e] = at + e < vocab ? p[at + e] : T{};
        if(q) r.z[e] = at + e < vocab ? q[at + e] : T{};
      }
    }
  }
  // (Differences of two numbers of up to 24 bits and their sums are taken in 64 bits.  A maximum with zero leaves NaN out.)
  template <int COUNT>
  __device__ __forceinline__ void weigh(const T (&x)[COUNT], const T (&z)[COUNT], int at, unsigned long long refused, double (&left)[COUNT]) const {
#pragma unroll
    for(int e = 0; e < COUNT; ++e) {
      const float own = fmaxf(to_float(x[e]), 0.0f);
      left[e] = q ? fmax((double)own - (double)fmaxf(to_float(z[e]), 0.0f), 0.0) : (double)own;
    }
#pragma unroll 1
    for(; refused; refused &= refused - 1) {
      const int word = token[__builtin_ctzll(refused)] - at;
#pragma unroll
      for(int e = 0; e < COUNT; ++e) left[e] = word == e ? 0.0 : left[e];
    }
  }
  // Words at and at + 1.
  __device__ __forceinline__ void two(int at, unsigned long long refused, double (&left)[2]) const {
    T x[2], z[2];
#pragma unroll
    for(int e = 0; e < 2; ++e) {
      x[e] = at + e < vocab ? p[at + e] : T{};
      z[e] = q && at + e < vocab ? q[at + e] : T{};
    }
    weigh(x, z, at, refused, left);
  }
};

struct VerifyShared {
  Verdict verdict;
  double wave[kVerifyWaves], share[kVerifyWaves];
  double before, bar;
  int found, is_last;
};

// The sum of a share that a workgroup's threads have two words each of; in the end all have read it.
__device__ __forceinline__ double share_sum(VerifyShared& sh, double x) {
  const double sum = lanes_sum(x);
  if((threadIdx.x & 63) == 63) sh.wave[threadIdx.x >> 6] = sum;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for(int i = 0; i < kVerifyWaves; ++i) all += sh.wave[i];
  __syncthreads();
  return all;
}

// A workgroup judges the tokens of a sequence - a chain of three loads - and sums a part of the words that the next token is drawn from, a share
// to each wave.  The last workgroup of a sequence finds the share in which the drawn number lies, and the word in it.  All sums are in 64
// bits and in an order of their own, whoever comes last.
// The kept tokens cost nothing but their own probabilities, so what moves is one row of the target's, and one of the draft's where a
// token was refused.  64 sequences, 131071 words, float32: 18.5 us, 3.6 TB/s; their bytes take 13 us, the judgement ahead of them and the join
// behind them the rest.  32000 words of one sequence: 6.3 us, a chain of some nine steps through memory.
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyArgs a, int first) {
  using W = Weights<T>;
  constexpr int kTogether = W::kTogether, kTurns = kShare / (64 * kTogether);
  __shared__ VerifyShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), s = first + blockIdx.y, part = blockIdx.x;
  const int count = a.counts ? clamp_int(a.counts[s], 0, a.n) : a.n;
  const double u = a.random[(long long)s * a.n];
  if(wave == 0) judge<T>(a, s, lane, count, sh.verdict);
  __syncthreads();
  const unsigned long long kept = sh.verdict.kept, refused = sh.verdict.refused;
  const int row = sh.verdict.last;
  if(part == 0 && wave == 0) {
    const int accepted = __builtin_popcountll(kept);
    const long long to = (long long)s * a.n;
    if(lane < a.n && lane >= accepted) a.path[to + lane] = -1;
    if(kept >> lane & 1) a.path[to + __builtin_popcountll(kept & ((1ull << lane) - 1))] = lane;
    if(lane == 0) a.accepted[s] = accepted;
    if(lane == 0 && count == 0) a.next[s] = -1;
  }
  if(count == 0) return;
  W w{static_cast<const T*>(a.target) + s * a.t_s + row * a.t_n,
      a.draft && refused ? static_cast<const T*>(a.draft) + s * a.d_s + row * a.d_n : nullptr, sh.verdict.token, a.vocab};
  // The refused words among a share's.
  auto refused_in = [&](int share) {
    return a.draft ? 0 : refused & __ballot((unsigned)(sh.verdict.token[lane] - share * kShare) < (unsigned)kShare);
  };
  const int mine = part * kVerifyWaves + wave, from = mine * kShare, shares = (a.vocab + kShare - 1) / kShare;
  double sum = 0.0;
  if(from < a.vocab) {
    const unsigned long long out = refused_in(mine);
    auto add = [&](const typename W::Raw& raw, int at) __attribute__((always_inline)) {
      double left[kTogether];
      w.weigh(raw.x, raw.z, at, out, left);
#pragma unroll
      for(int e = 0; e < kTogether; ++e) sum += left[e];
    };
    if(from + kShare <= a.vocab) {   // (all are asked for at once)
      typename W::Raw raw[kTurns];
#pragma unroll
      for(int i = 0; i < kTurns; ++i) w.template fetch<true>(raw[i], from + (i * 64 + lane) * kTogether);
#pragma unroll
      for(int i = 0; i < kTurns; ++i) add(raw[i], from + (i * 64 + lane) * kTogether);
    } else {
#pragma unroll 1
      for(int at = from + lane * kTogether; at < a.vocab; at += 64 * kTogether) {
        typename W::Raw raw;
        w.template fetch<false>(raw, at);
        add(raw, at);
      }
    }
    sum = lanes_sum(sum);
  }
  unsigned long long* const sums = reinterpret_cast<unsigned long long*>(a.sums) + (long long)blockIdx.y * shares;
  if(a.parts == 1) {
    if(lane == 63) sh.share[wave] = sum;
    __syncthreads();
  } else {
    if(lane == 63 && from < a.vocab)
      __hip_atomic_store(sums + mine, __builtin_bit_cast(unsigned long long, sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if(!cache_arrived_last(a.counters + blockIdx.y, a.parts, sh.is_last)) return;
  }
  // The share: the first one up to which the sum is above u of all (rounding may leave none where u is next to one: the last that has anything).
  if(wave == 0) {
    auto sum_of = [&](int i) {
      return a.parts == 1 ? sh.share[i] : __builtin_bit_cast(double, __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    };
    const int each = (shares + 63) / 64, i0 = min(lane * each, shares), i1 = min(i0 + each, shares);
    double some = 0.0;
    for(int i = i0; i < i1; ++i) some += sum_of(i);
    const double upto = lanes_sum(some), bar = u * lane_double(upto, 63), shifted = __shfl_up(upto, 1, 64);
    const unsigned long long above = __ballot(some > 0.0 && upto > bar), any = __ballot(some > 0.0);
    const int l = above ? __builtin_ctzll(above) : any ? 63 - __builtin_clzll(any) : -1;
    if(l < 0 ? lane == 0 : lane == l) {
      double running = lane == 0 ? 0.0 : shifted, before = running;
      int found = l < 0 ? -1 : i0;
      for(int i = i0; i < i1 && l >= 0; ++i) {
        const double x = sum_of(i);
        if(x > 0.0) {
          found = i;
          before = running;
          if(running + x > bar) break;
        }
        running += x;
      }
      sh.found = found;
      sh.before = before;
      sh.bar = bar;
    }
  }
  __syncthreads();
  int share = sh.found;
  double before = sh.before, bar = sh.bar;
  if(share < 0) {
    // Nothing is left: the target's own probabilities, summed anew by this workgroup, twice (to be seen only where the draft was not drawn from
    // its distribution, or probabilities are none).
    w.q = nullptr;
    double all = 0.0, left[2];
    for(int i = 0; i < shares; ++i) {
      w.two(i * kShare + 2 * tid, 0, left);
      all += share_sum(sh, left[0] + left[1]);
    }
    bar = u * all;
    double running = 0.0;
    for(int i = 0; i < shares; ++i) {
      w.two(i * kShare + 2 * tid, 0, left);
      const double x = share_sum(sh, left[0] + left[1]);
      if(x > 0.0) {
        share = i;
        before = running;
        if(running + x > bar) break;
      }
      running += x;
    }
    if(share < 0) {
      if(tid == 0) a.next[s] = -1;
      return;
    }
  }
  // The word, likewise: two that follow each other to a thread.
  const int at = share * kShare + 2 * tid;
  double left[2];
  w.two(at, sh.found < 0 ? 0 : refused_in(share), left);
  const double upto = lanes_sum(left[0] + left[1]), shifted = __shfl_up(upto, 1, 64);
  if(lane == 63) sh.wave[wave] = upto;
  __syncthreads();
  double ahead = before, running = before;
  int here = -1;
#pragma unroll
  for(int i = 0; i < kVerifyWaves; ++i) {
    const double x = sh.wave[i];
    const bool passed = here >= 0 && running > bar;
    if(x > 0.0 && !passed) {
      here = i;
      ahead = running;
    }
    if(!passed) running += x;
  }
  if(wave != here) return;
  const double start = lane == 0 ? ahead : ahead + shifted;
  const bool zero = left[0] > 0.0 && start + left[0] > bar, one = left[1] > 0.0 && start + left[0] + left[1] > bar;
  const unsigned long long hits = __ballot(zero || one), any = __ballot(left[0] > 0.0 || left[1] > 0.0);
  const int l = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(any);
  if(lane == l) a.next[s] = hits ? (zero ? at : at + 1) : left[1] > 0.0 ? at + 1 : at;
}

}  // namespace

extern "C" {

size_t marian_hip_verify_drafts_workspace_bytes(int64_t sequences, int64_t vocab) {
  if(sequences < 1 || vocab < 1 || sequences > kMaxSequences || vocab >= 1 << 24 || vocab <= kVerifyPart) return 0;
  return (size_t)(kCacheCounterBytes + std::min(sequences, kVerifySequences) * ((vocab + kShare - 1) / kShare) * 8);
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
