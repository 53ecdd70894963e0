// Attention of new tokens over a quantized cache (marian_hip_cache_attention; device code).
//
// For the rows r of an entry (token i of the n new ones, query head g of the group that shares the entry's keys) and
// its positions j:
//   s_rj = scale * q_r . k_j,  p_rj = exp(s_rj - m_r),  out_r = sum_j p_rj v_j / sum_j p_rj
// over the j that token i sees.  One pass: maximum, sum and weighted values are carried along and scaled down when
// the maximum grows.
//
// What has to move is dk bytes and a scale of each position's key and value, 2 * (dk + 4) bytes; the products are
// 4 * dk operations a row and position.  Up to some sixty rows an entry the bytes are the bound, beyond it the matrix
// instructions.
//
// Layout: a wave takes 32 positions at a time and 16 * QT rows, all in registers.
//   S^T = K Q^T (16x16x32): lane (c = lane % 16, g = lane / 16) loads sixteen codes at a time of key c - whole 64-byte
//   pieces of a row between four lanes - and uses them as two operands; which codes a step of the product takes is the same
//   for Q, so no code moves between lanes.  The result has row c's scores of keys 4 g .. 4 g + 3, for two blocks of 16 keys.
//   O^T = V^T P^T: those eight weights of a lane are its operand as they are, if V's operand has the keys in that
//   order: lane (c, g) loads DP / 16 codes at c * DP / 16 of each of these eight keys - a row of keys between
//   sixteen lanes - and picks a dimension's eight codes out of its registers, two at a time, while they become float16.
//   So neither keys, values nor weights go through LDS.
// Codes are exact in float16.  Q is scaled row by row by a power of two up to 2^14 .. 2^15 and enters in one float16
// (float16 and bfloat16: exact but for values 2^-29 below the row's largest) or two (float32: 22 bits).  A weight is
// p_rj times the value's scale over a running scale S_r (as the maximum runs), times 2^9: in one float16 or two, rounded
// to nearest, of what is at most 2^15 and, with normal numbers, down to 2^-14: 11 (22) bits of weights up to 2^-24 below the
// largest.  Their sum is of the weights in float32.
// Positions that a row does not see, and rows past the end that pad a block, weigh a selected zero; loads past the end go to the
// last position in reach, whose codes are finite whatever they hold.
#pragma once

#include "cache_codes.h"
#include "cache_plan.h"

namespace marian_hip {

struct CacheAttentionArgs {
  const void* q;
  long long q_s, q_h, q_n;   // in values
  void* out;
  long long o_s, o_h, o_n;
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int *lens, *counts, *parents;
  float* part;          // partial results, row_floats to a row: the rows' values, then their logarithms
  unsigned* counters;   // parts that have arrived, zero between calls
  int S, Hk, G, n, cap, dk, row_tiles, target, items;
  float scale_log2;     // scale / ln 2
};

constexpr float kWeightUnit = 512.0f;     // 2^9, see above
constexpr float kMaximumSlack = 4.0f;     // weights may be 2^4 above the carried maximum's ...
constexpr float kScaleSlack = 4.0f;       // ... and scales four times the carried one before the sums are scaled down

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// The part of a workgroup: sequence, positions from..to (of the `used` in reach), and its place among the parts.
struct CachePart {
  int s, len, count, used, from, to, parts, part, slot;
};

// Inclusive sum over the lanes of a wave: within rows of sixteen lanes, then over the rows, without LDS.
__device__ __forceinline__ unsigned lanes_sum(unsigned x) {
  int v = (int)x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return (unsigned)v;
}

// Finds part `item`; false where there are fewer.  All waves do the same, lanes being sequences.
__device__ __forceinline__ bool cache_part(const CacheAttentionArgs& a, int item, int lane, CachePart& w) {
  auto blocks_of = [&](int s) -> unsigned {   // of positions that sequence s has in reach
    if(s >= a.S) return 0;
    const int len = clamp_int(a.lens[s], 0, a.cap), count = a.counts ? clamp_int(a.counts[s], 0, a.n) : a.n;
    return count > 0 ? (unsigned)(min(len + count, a.cap) + kCacheBlock - 1) / kCacheBlock : 0;
  };
  w.parts = 1;
  w.part = 0;
  w.slot = 0;
  unsigned each = 1u << 20;   // blocks of a part
  w.s = item;
  if(a.target > 1) {
    constexpr int kHeld = 4;   // up to 256 sequences are asked for once, all at a time
    unsigned held[kHeld], total = 0;
#pragma unroll
    for(int i = 0; i < kHeld; ++i) held[i] = blocks_of(64 * i + lane);
#pragma unroll
    for(int i = 0; i < kHeld; ++i) total += held[i];
    for(int base = 64 * kHeld; base < a.S; base += 64) total += blocks_of(base + lane);
    total = (unsigned)__builtin_amdgcn_readlane((int)lanes_sum(total), 63);
    each = max(1u, (total + a.target - 1) / a.target);
    // parts in the lower bits, those of sequences with several in the upper twelve (less than 2 * target)
    unsigned before = 0;
    bool found = false;
    auto look = [&](int base, unsigned mine) __attribute__((always_inline)) {
      const unsigned parts = base + lane < a.S ? max(1u, (mine + each - 1) / each) : 0;
      const unsigned sum = before + lanes_sum(parts > 1 ? parts | parts << 20 : parts);
      const unsigned long long at = __ballot((int)(sum & 0xfffff) > item);
      if(at) {
        const int l = __ffsll((long long)at) - 1;
        const unsigned upto = (unsigned)__builtin_amdgcn_readlane((int)sum, l);
        w.s = base + l;
        w.parts = __builtin_amdgcn_readlane((int)parts, l);
        w.part = item - ((int)(upto & 0xfffff) - w.parts);
        w.slot = w.parts > 1 ? (int)(upto >> 20) - w.parts : 0;
        found = true;
      }
      before = (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
    };
#pragma unroll
    for(int i = 0; i < kHeld; ++i)
      if(!found && 64 * i < a.S) look(64 * i, held[i]);
    for(int base = 64 * kHeld; base < a.S && !found; base += 64) look(base, blocks_of(base + lane));
    if(!found) return false;
  }
  w.len = clamp_int(a.lens[w.s], 0, a.cap);
  w.count = a.counts ? clamp_int(a.counts[w.s], 0, a.n) : a.n;
  w.used = w.count > 0 ? min(w.len + w.count, a.cap) : 0;
  w.from = a.target > 1 ? w.part * (int)each * kCacheBlock : 0;
  w.to = a.target > 1 ? min(w.from + (int)each * kCacheBlock, w.used) : w.used;
  return true;
}

template <typename T, CacheFormat F, int DP, int QT>
struct CacheAttention {
  static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;   // float16 to a query value or weight
  static constexpr int kSteps = DP / 32;                  // of a product over a row
  static constexpr int kPieces = DP / 64;                 // sixteen codes of a key to a lane
  static constexpr int kDims = DP / 16;                   // of a value's row to a lane
  static constexpr int kWords = kDims / 4;

  // 32 positions as they are loaded: what is needed for the scores, and what is needed behind them.
  struct Keys {
    cache_u4 code[2][kPieces];
    cache_f4 scale[2];
  };
  struct Values {
    unsigned code[8][kWords];
    cache_f4 scale[2];
  };

  // Positions at .. at + 31 of an entry; ENDS: those behind `last` are `last`.  Lanes past a row's end (dk < DP) take its start: the
  // queries are zero there, and the values are not stored.
  template <bool ENDS>
  static __device__ __forceinline__ void load(Keys& t, const unsigned char* k, const float* scale, int at, int last, int dk, int lane) {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for(int b = 0; b < 2; ++b) {
      const unsigned row = ENDS ? (unsigned)min(at + 16 * b + c, last) * dk : (unsigned)(at + c) * dk;
      const unsigned char* p = ENDS ? k : k + (size_t)(16 * b * dk);
#pragma unroll
      for(int i = 0; i < kPieces; ++i) {
        const unsigned d = 64 * i + 16 * g;
        t.code[b][i] = *reinterpret_cast<const cache_u4*>(p + (row + (d < (unsigned)dk ? d : 0)));
      }
    }
    load_scales<ENDS>(t.scale, scale, at, last, g);
  }
  template <bool ENDS>
  static __device__ __forceinline__ void load(Values& t, const unsigned char* v, const float* scale, int at, int last, int dk, int lane) {
    const int c = lane & 15, g = lane >> 4;
    const unsigned d = (unsigned)(kDims * c) < (unsigned)dk ? kDims * c : 0;
#pragma unroll
    for(int e = 0; e < 8; ++e) {
      const int key = 16 * (e / 4) + e % 4;
      const unsigned row = ENDS ? (unsigned)min(at + 4 * g + key, last) * dk : (unsigned)(at + 4 * g) * dk;
      const unsigned char* p = (ENDS ? v : v + (size_t)(key * dk)) + (row + d);
      if constexpr(kWords == 1) {
        t.code[e][0] = *reinterpret_cast<const unsigned*>(p);
      } else if constexpr(kWords == 2) {
        const cache_u2 x = *reinterpret_cast<const cache_u2*>(p);
        t.code[e][0] = x[0];
        t.code[e][1] = x[1];
      } else {
        const cache_u4 x = *reinterpret_cast<const cache_u4*>(p);
#pragma unroll
        for(int w = 0; w < 4; ++w) t.code[e][w] = x[w];
      }
    }
    load_scales<ENDS>(t.scale, scale, at, last, g);
  }
  template <bool ENDS>
  static __device__ __forceinline__ void load_scales(cache_f4 (&to)[2], const float* scale, int at, int last, int g) {
#pragma unroll
    for(int b = 0; b < 2; ++b) {
      if(ENDS) {
#pragma unroll
        for(int e = 0; e < 4; ++e) to[b][e] = scale[(unsigned)min(at + 16 * b + 4 * g + e, last)];
      } else {
        to[b] = *reinterpret_cast<const cache_f4_any*>(scale + 16 * b + (unsigned)(at + 4 * g));
      }
    }
  }

  // Dimension B of word W of the lane's values, eight keys.
  template <int B>
  static __device__ __forceinline__ cache_h8 value_operand(const unsigned (&v)[8][kWords], int w) {
    const cache_h2 h[4] = {half2_of<F, B, B>(v[0][w], v[1][w]), half2_of<F, B, B>(v[2][w], v[3][w]),
                           half2_of<F, B, B>(v[4][w], v[5][w]), half2_of<F, B, B>(v[6][w], v[7][w])};
    return cache_h8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
  }
};

// The maximum over the four lanes of a query row.
__device__ __forceinline__ float over_lanes_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float over_lanes_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

constexpr float kNone = -__builtin_huge_valf();

template <typename T, CacheFormat F, int DP, int QT>
__global__ __launch_bounds__(256, (DP == 64 ? 5 - QT : DP == 128 ? 4 - QT : 2)) void cache_attention_kernel(CacheAttentionArgs a) {
  using A = CacheAttention<T, F, DP, QT>;
  constexpr int kTerms = A::kTerms, kSteps = A::kSteps, kDims = A::kDims;
  constexpr int kHalf = DP < 128 ? DP : 128;   // dimensions that are joined at a time
  __shared__ float joined[4][16][kHalf + 4];
  __shared__ float row_max[4][16 * QT], row_sum[4][16 * QT];
  __shared__ int is_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  // Workgroups with the same positions follow each other on one XCD (a workgroup to each of the eight in turn).
  const int place = blockIdx.x >> 3, tile = place % a.row_tiles, entry = place / a.row_tiles * 8 + (blockIdx.x & 7);
  if(entry >= a.items * a.Hk) return;
  const int head = entry % a.Hk;
  CachePart w;
  if(!cache_part(a, entry / a.Hk, lane, w)) return;
  const int rows = w.count * a.G, row0 = tile * 16 * QT;   // rows of the sequence that are there
  T* const out = static_cast<T*>(a.out) + w.s * a.o_s;
  auto row_out = [&](int r) { return out + (long long)(head * a.G + r % a.G) * a.o_h + (long long)(r / a.G) * a.o_n; };
  const int d_mine = (tid & 15) * kDims;   // of the row tid / 16 that the thread writes
  if(w.part == 0) {
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const int r = row0 + 16 * t + (tid >> 4);
      if(r >= rows && r < a.n * a.G && d_mine < a.dk) {
        const float zeros[kDims] = {};
        store_row<kDims, T>(row_out(r) + d_mine, zeros);
      }
    }
  }
  if(row0 >= rows) return;

  // ---- positions
  const int last_token = min(rows - 1, row0 + 16 * QT - 1) / a.G;
  const int end = min(w.to, w.len + last_token + 1);                              // of what any row sees
  const int open = min(end, w.len + (a.parents ? 0 : row0 / a.G + 1));            // of what all rows see
  const long long first = ((long long)w.s * a.Hk + head) * a.cap;
  const unsigned char *k = a.k + first * a.dk, *v = a.v + first * a.dk;
  const float *ks = a.ks + first, *vs = a.vs + first;
  auto fetch_keys = [&](typename A::Keys& x, int at) __attribute__((always_inline)) {
    if(at + 32 <= end) A::template load<false>(x, k, ks, at, 0, a.dk, lane);
    else if(at < end) A::template load<true>(x, k, ks, at, end - 1, a.dk, lane);
  };
  auto fetch_values = [&](typename A::Values& x, int at) __attribute__((always_inline)) {
    if(at + 32 <= end) A::template load<false>(x, v, vs, at, 0, a.dk, lane);
    else if(at < end) A::template load<true>(x, v, vs, at, end - 1, a.dk, lane);
  };
  // (the first positions are asked for ahead of the queries, the next keys as soon as the last ones are used up, and so the values)
  const int begin = w.from + 32 * wave;
  typename A::Keys key;
  typename A::Values value;
  fetch_keys(key, begin);
  fetch_values(value, begin);

  // ---- queries
  unsigned long long seen = 0;
  if(a.parents) seen = lineage(a.parents + (long long)w.s * a.n, a.n, lane);
  cache_h8 q[QT][kTerms][kSteps];
  float row_scale[QT];          // of a score, to logarithms of base 2
  int token[QT];
  unsigned long long sees[QT];   // drafted tokens
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + c, rr = min(r, rows - 1);
    token[t] = rr / a.G;
    if(a.parents) {
      const unsigned lo = __shfl((unsigned)seen, token[t], 64), hi = __shfl((unsigned)(seen >> 32), token[t], 64);
      sees[t] = (unsigned long long)hi << 32 | lo;
    } else {
      sees[t] = 0;
    }
    const T* row = static_cast<const T*>(a.q) + w.s * a.q_s + (long long)(head * a.G + rr % a.G) * a.q_h + (long long)token[t] * a.q_n;
    float x[kSteps][8];
    unsigned most = 0;   // bits of the row's largest magnitude (NaN above all)
#pragma unroll
    for(int i = 0; i < kSteps; ++i) {
      const int d = 64 * (i / 2) + 16 * g + 8 * (i % 2);
#pragma unroll
      for(int e = 0; e < 8; ++e) x[i][e] = 0.0f;
      if(d < a.dk) load_row<8>(row + d, x[i]);
#pragma unroll
      for(int e = 0; e < 8; ++e) most = max(most, __builtin_bit_cast(unsigned, x[i][e]) & 0x7fffffffu);
    }
    most = max(most, (unsigned)__shfl_xor((int)most, 16, 64));
    most = max(most, (unsigned)__shfl_xor((int)most, 32, 64));
    const int up = clamp_int(127 + 14 + 127 - (int)(most >> 23), 2, 252);   // exponent that brings it to 2^14
    const float factor = __builtin_bit_cast(float, (unsigned)up << 23), back = __builtin_bit_cast(float, (unsigned)(254 - up) << 23);
    row_scale[t] = most >= 0x7f800000u ? __builtin_nanf("") : fmaxf(back * (a.scale_log2 / kCodeUnit<F>), 0x1p-126f);   // (never zero)
#pragma unroll
    for(int i = 0; i < kSteps; ++i) {
      float y[8];
#pragma unroll
      for(int e = 0; e < 8; ++e) y[e] = x[i][e] * factor;
#pragma unroll
      for(int e = 0; e < 8; ++e) q[t][0][i][e] = (_Float16)y[e];
      if constexpr(kTerms == 2) {
#pragma unroll
        for(int e = 0; e < 8; ++e) q[t][1][i][e] = (_Float16)(y[e] - (float)q[t][0][i][e]);
      }
    }
  }

  cache_f4 o[QT][kDims];
  float top[QT], sum[QT], unit[QT];   // carried maximum (base 2), the lane's part of the sum, carried scale
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    top[t] = kNone;
    sum[t] = 0.0f;
    unit[t] = 1e-30f;   // (scales below it are as good as zero)
#pragma unroll
    for(int j = 0; j < kDims; ++j) o[t][j] = cache_f4{0, 0, 0, 0};
  }

  for(int at = begin; at < end; at += kCacheBlock) {
    // scores
    cache_f4 s[QT][2];
#pragma unroll
    for(int t = 0; t < QT; ++t) s[t][0] = s[t][1] = cache_f4{0, 0, 0, 0};
#pragma unroll
    for(int b = 0; b < 2; ++b)
#pragma unroll
      for(int i = 0; i < kSteps; ++i) {
        const cache_u4 piece = key.code[b][i / 2];
        const cache_h8 operand = i % 2 ? half8_of<F>(piece[2], piece[3]) : half8_of<F>(piece[0], piece[1]);
#pragma unroll
        for(int t = 0; t < QT; ++t)
#pragma unroll
          for(int m = kTerms - 1; m >= 0; --m) s[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand, q[t][m][i], s[t][b], 0, 0, 0);
      }
#pragma unroll
    for(int t = 0; t < QT; ++t)
#pragma unroll
      for(int e = 0; e < 8; ++e) s[t][e / 4][e % 4] *= key.scale[e / 4][e % 4];
    fetch_keys(key, at + kCacheBlock);
    // Positions that a row does not see score minus infinity (a weight of zero) and have a scale of zero.
    const bool masked = at + 32 > open;
    unsigned hidden[QT];   // bit e: key e
    float widest = 0.0f;
#pragma unroll
    for(int t = 0; t < QT; ++t) hidden[t] = 0;
    if(masked) {
#pragma unroll
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int e = 0; e < 8; ++e) {
          const int p = at + 16 * (e / 4) + 4 * g + e % 4, j = p - w.len;
          const bool see = p < end && (j < 0 || (a.parents ? (sees[t] >> (j & 63) & 1) != 0 : j <= token[t]));
          hidden[t] |= see ? 0u : 1u << e;
          s[t][e / 4][e % 4] = see ? s[t][e / 4][e % 4] : kNone;
        }
    } else {
#pragma unroll
      for(int e = 0; e < 8; ++e) widest = fmaxf(widest, value.scale[e / 4][e % 4]);
    }
    float high[QT], wide[QT];
    bool grown = false;
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      high[t] = kNone;
#pragma unroll
      for(int e = 0; e < 8; ++e) high[t] = fmaxf(high[t], s[t][e / 4][e % 4]);
      high[t] *= row_scale[t];
      wide[t] = widest;
    }
    if(masked) {
#pragma unroll
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int e = 0; e < 8; ++e) wide[t] = fmaxf(wide[t], hidden[t] >> e & 1 ? 0.0f : value.scale[e / 4][e % 4]);
    }
#pragma unroll
    for(int t = 0; t < QT; ++t) grown |= high[t] > top[t] + kMaximumSlack || wide[t] > unit[t] * kScaleSlack;
    if(__any(grown)) {
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const float m = fmaxf(top[t], over_lanes_max(high[t])), u = fmaxf(unit[t], over_lanes_max(wide[t]));
        const float down = m == top[t] ? 1.0f : __builtin_amdgcn_exp2f(top[t] - m);
        const float both = u == unit[t] ? down : down * (unit[t] / u);
        sum[t] *= down;
#pragma unroll
        for(int j = 0; j < kDims; ++j) o[t][j] *= both;
        top[t] = m;
        unit[t] = u;
      }
    }
    // weights
    float r[QT][8];   // scales over the carried one
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float per = kWeightUnit / unit[t];
#pragma unroll
      for(int e = 0; e < 8; ++e) r[t][e] = value.scale[e / 4][e % 4] * per;
    }
    if(masked) {
#pragma unroll
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int e = 0; e < 8; ++e) r[t][e] = hidden[t] >> e & 1 ? 0.0f : r[t][e];
    }
    cache_h8 p[QT][kTerms];
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float from = top[t] == kNone ? 0.0f : -top[t];   // (nothing seen so far: minus infinity stays that)
#pragma unroll
      for(int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / 4][e % 4], row_scale[t], from)), z = y * r[t][e];
        sum[t] += y;
        p[t][0][e] = (_Float16)z;
        if constexpr(kTerms == 2) p[t][1][e] = (_Float16)(z - (float)p[t][0][e]);
      }
    }
    // weighted values
    unsigned vh[8][A::kWords];
#pragma unroll
    for(int e = 0; e < 8; ++e)
#pragma unroll
      for(int i = 0; i < A::kWords; ++i) vh[e][i] = held<F>(value.code[e][i]);
#pragma unroll
    for(int i = 0; i < A::kWords; ++i) {
      const cache_h8 d[4] = {A::template value_operand<0>(vh, i), A::template value_operand<1>(vh, i), A::template value_operand<2>(vh, i),
                             A::template value_operand<3>(vh, i)};
#pragma unroll
      for(int j = 0; j < 4; ++j)
#pragma unroll
        for(int t = 0; t < QT; ++t)
#pragma unroll
          for(int m = kTerms - 1; m >= 0; --m)
            o[t][4 * i + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(d[j], p[t][m], o[t][4 * i + j], 0, 0, 0);
    }
    fetch_values(value, at + kCacheBlock);
  }

  // ---- the four waves' results
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    sum[t] = over_lanes_sum(sum[t]);
    if(g == 0) {
      row_max[wave][16 * t + c] = top[t];
      row_sum[wave][16 * t + c] = sum[t];
    }
  }
  __syncthreads();
  const bool whole = w.parts == 1;
  const long long place_of_tile = ((long long)w.slot * a.Hk + head) * a.row_tiles + tile, part_stride = (long long)a.Hk * a.row_tiles;
  constexpr int kTileFloats = 16 * QT * (DP + 1);
  float* const part = whole ? nullptr : a.part + (place_of_tile + w.part * part_stride) * kTileFloats;
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    float m = row_max[0][16 * t + c];
#pragma unroll
    for(int i = 1; i < 4; ++i) m = fmaxf(m, row_max[i][16 * t + c]);
    const float mine = top[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f(top[t] - m) * (unit[t] / (kWeightUnit * kCodeUnit<F>));
    const int r = tid >> 4;   // the row whose values the thread adds up
    float m_r = row_max[0][16 * t + r];
#pragma unroll
    for(int i = 1; i < 4; ++i) m_r = fmaxf(m_r, row_max[i][16 * t + r]);
    float total = 0.0f;
#pragma unroll
    for(int i = 0; i < 4; ++i)
      total += row_max[i][16 * t + r] == kNone ? row_sum[i][16 * t + r] : row_sum[i][16 * t + r] * __builtin_amdgcn_exp2f(row_max[i][16 * t + r] - m_r);
    const float per = total == 0.0f ? 0.0f : 1.0f / total;
    const bool there = row0 + 16 * t + r < rows;
#pragma unroll
    for(int h = 0; h < DP / kHalf; ++h) {
      if(h || t) __syncthreads();
      if(DP == kHalf || (g >> 1) == h) {
#pragma unroll
        for(int e = 0; e < 4; ++e)
#pragma unroll
          for(int j = 0; j < kDims; j += 4) {
            const int d = 4 * kDims * g + kDims * e + j - h * kHalf;
            *reinterpret_cast<cache_f4*>(&joined[wave][c][d]) =
                cache_f4{o[t][j][e] * mine, o[t][j + 1][e] * mine, o[t][j + 2][e] * mine, o[t][j + 3][e] * mine};
          }
      }
      __syncthreads();
      constexpr int kEach = kHalf / 16;
      const int d = (tid & 15) * kEach;
      float y[kEach];
#pragma unroll
      for(int j = 0; j < kEach; ++j)
        y[j] = ((joined[0][r][d + j] + joined[1][r][d + j]) + (joined[2][r][d + j] + joined[3][r][d + j])) * per;
      if(there && d + h * kHalf < a.dk) {
        if(whole) {
          store_row<kEach, T>(row_out(row0 + 16 * t + r) + d + h * kHalf, y);
        } else {
          unsigned long long* to = reinterpret_cast<unsigned long long*>(part + (16 * t + r) * DP + d + h * kHalf);
#pragma unroll
          for(int j = 0; j < kEach; j += 2)
            __hip_atomic_store(to + j / 2, (unsigned long long)__builtin_bit_cast(unsigned, y[j + 1]) << 32 | __builtin_bit_cast(unsigned, y[j]),
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    if(!whole && there && (tid & 15) == 0)
      __hip_atomic_store(part + 16 * QT * DP + 16 * t + r, total == 0.0f ? kNone : m_r + __builtin_amdgcn_logf(total), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
  }
  if(whole) return;

  // ---- the parts of a sequence: the workgroup that arrives last joins them, in their order.
  // (Stores and loads of agent scope go past the caches of an XCD; every wave's stores are acknowledged before the count
  // goes up, so whoever reads the last count finds them all.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if(tid == 0) {
    unsigned* const counter = a.counters + place_of_tile;
    const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(w.parts - 1);
    if(last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // (for the next call)
    is_last = last;
  }
  __syncthreads();
  if(!is_last) return;
  const float* const all = a.part + place_of_tile * kTileFloats;
  const long long stride = part_stride * kTileFloats;
#pragma unroll 1
  for(int t = 0; t < QT; ++t) {
    const int r = tid >> 4;
    if(row0 + 16 * t + r >= rows || d_mine >= a.dk) continue;
    const float* logs = all + 16 * QT * DP + 16 * t + r;
    const float* from = all + (16 * t + r) * DP + d_mine;
    float m = kNone;
#pragma unroll 4
    for(int i = 0; i < w.parts; ++i) m = fmaxf(m, __hip_atomic_load(logs + i * stride, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    float total = 0.0f, y[kDims] = {};
#pragma unroll 4
    for(int i = 0; i < w.parts; ++i) {
      const float l = __hip_atomic_load(logs + i * stride, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const float weight = l == kNone ? 0.0f : __builtin_amdgcn_exp2f(l - m);
      total += weight;
#pragma unroll
      for(int j = 0; j < kDims; j += 2) {
        const unsigned long long x = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(from + i * stride + j), __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        y[j] = __builtin_fmaf(weight, __builtin_bit_cast(float, (unsigned)x), y[j]);
        y[j + 1] = __builtin_fmaf(weight, __builtin_bit_cast(float, (unsigned)(x >> 32)), y[j + 1]);
      }
    }
    const float per = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for(int j = 0; j < kDims; ++j) y[j] *= per;
    store_row<kDims, T>(row_out(row0 + 16 * t + r) + d_mine, y);
  }
}

}  // namespace marian_hip
