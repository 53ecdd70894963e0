// Attention of new tokens over pages of keys and values (marian_hip_pages_attention; device code).
//
// For the rows r of an entry (token i of the n new ones, query head g of the group that shares the entry's keys) and
// its positions j:
//   s_rj = scale * q_r . k_j,  p_rj = exp(s_rj - m_r),  out_r = sum_j p_rj v_j / sum_j p_rj
// over the j that token i sees.  One pass: maximum, sum and weighted values are carried along and scaled down when the
// maximum has grown by 2^4 (most turns skip it).  Which workgroup takes which positions, how its waves and the parts of
// a sequence are joined, is what the attention over a quantized cache does (cache_attention_kernel.h).
//
// S^T = K Q^T and O^T = V^T P^T on 16x16 matrix products of the type itself: float16 and bfloat16 32 deep, float32 4 deep, sums in float32.
// A wave takes 32 positions at a time, straight from memory to operands, lane being (c = lane % 16, g = lane / 16):
//   S^T: lane (c, g) loads 16 bytes at 64 i + 16 g of the keys 8 (c / 4) + c % 4 and that + 4; the queries have the same order of values,
//   so none moves between lanes.  The result has row c's scores of the eight positions 8 g ...
//   O^T: ... whose weights are the lane's operand as they are.  V's operand has in lane (c, g) the same eight positions: rows of V of
//   which sixteen lanes take 16 bytes each, side by side, and a dimension's eight values are picked from the registers of eight loads.
// A page holds whole eights of positions, so a lane looks up one page for its keys and one for its values a turn; the numbers of the turn after
// the next are under way with the next one's keys and values.  A page that is none, and positions past the end, are
// read at the start of the cache (one line of memory) and weigh a selected zero: loads need no branches.
//
// Weights enter the product with the values in the type of the values, bfloat16 and float16 in two terms, the second of what the first
// leaves: 16 and 22 bits.  Their sum is of the float32 ones.  They are scaled by a power of two: bfloat16 and float32 2^-24, so that sums over
// 2^20 positions of values next to the largest stay in range; float16 2^11, so that weights down to 2^-25 of the largest keep their bits.
//
// What bounds it: the memory.  One token of 128 sequences of up to 512 positions, 16 heads of 64 values, float32 (360 MB): 71 to 72 us, 5.0 TB/s; of 16
// sequences of up to 32768, 8 heads of 128 values with four rows each, bfloat16 (1.4 GB): 257 to 264 us, 5.4 TB/s; one sequence of 100003 (410 MB) 75
// us, 5.4 TB/s.  Where there is little to read, 6 sequences of up to 120 positions: 5.9 us, a workgroup's start, three dependent loads (length,
// page, keys and values) and its end.
#pragma once

#include <type_traits>

#include "../../include/marian_hip_ops.h"
#include "abi_common.h"
#include "cache_attention_kernel.h"
#include "pages_attention.h"

namespace marian_hip {

typedef __bf16 pages_b8 __attribute__((ext_vector_type(8)));
typedef int cache_i4 __attribute__((ext_vector_type(4)));

static_assert(kPartUnit * kPagesMostParts <= 1.0f, "the parts' weights add up to one at the most");

template <typename T, int DP>
struct Pages {
  static constexpr int kWidth = sizeof(T);
  static constexpr int kKeyPieces = DP * kWidth / 64;              // pieces of 16 bytes of a key to a lane
  static constexpr int kDims = DP / 16;                            // of a value's row to a lane ...
  static constexpr int kTogether = kDims < 16 / kWidth ? kDims : 16 / kWidth;   // ... that lie side by side
  static constexpr int kValuePieces = kDims / kTogether;
  static constexpr int kWords = kTogether * kWidth / 4;            // of a piece of values
  static constexpr int kUp = std::is_same<T, _Float16>::value ? 11 : -24;   // exponent that weights are held with
  static constexpr float kUnit = kUp < 0 ? (float)(1 << -kUp * (kUp < 0)) : 1.0f / (1 << kUp * (kUp > 0));   // 2^-kUp
  struct Keys {
    cache_u4 piece[2][kKeyPieces];
  };
  struct Values {
    unsigned word[8][kValuePieces][kWords];
  };
};

// s += keys . queries over a piece of 16 bytes
template <typename T>
__device__ __forceinline__ cache_f4 pages_product(cache_u4 k, cache_u4 q, cache_f4 s) {
  if constexpr(sizeof(T) == 4) {
    const cache_f4 x = __builtin_bit_cast(cache_f4, k), y = __builtin_bit_cast(cache_f4, q);
#pragma unroll
    for(int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], s, 0, 0, 0);
    return s;
  } else if constexpr(std::is_same<T, _Float16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(cache_h8, k), __builtin_bit_cast(cache_h8, q), s, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pages_b8, k), __builtin_bit_cast(pages_b8, q), s, 0, 0, 0);
  }
}

template <typename T>
__device__ __forceinline__ float pages_half(unsigned bits) {
  const uint16_t b = (uint16_t)bits;
  return to_float(__builtin_bit_cast(T, b));
}

// A word of values, an infinity or NaN in it as zero.
template <typename T>
__device__ __forceinline__ unsigned pages_finite(unsigned w) {
  if constexpr(sizeof(T) == 4) return (w & 0x7f800000u) == 0x7f800000u ? 0 : w;
  constexpr unsigned most = std::is_same<T, _Float16>::value ? 0x7c00u : 0x7f80u;
  return ((w & most) == most ? 0 : w & 0xffffu) | ((w >> 16 & most) == most ? 0 : w & 0xffff0000u);
}

// The number of the page that an eight of positions is in, and the eight's place in it.
struct PagesPlace {
  int id, eight;
};
__device__ __forceinline__ PagesPlace pages_look(const PagesAttentionArgs& a, const int* table, unsigned eight) {
  unsigned within;
  const unsigned j = a.by_eights.of(eight, within);
  return PagesPlace{table[min(j, (unsigned)a.row - 1)] | (j < (unsigned)a.row ? 0 : (int)0x80000000), (int)within};   // (behind the row: none)
}

// The weights of a lane's eight scores, 2^(score * scale + from), in two terms of T, and their sum.
template <typename T>
__device__ __forceinline__ void pages_weights(const cache_f4 (&s)[2], float scale, float from, float& sum, cache_u4 (&w)[2]) {
#pragma unroll
  for(int e = 0; e < 4; ++e) {
    float y[2];
#pragma unroll
    for(int i = 0; i < 2; ++i) {
      const int at = 2 * e + i;
      y[i] = settled(__builtin_amdgcn_exp2f(__builtin_fmaf(s[at / 4][at % 4], scale, from)));
      sum += y[i];
    }
    const unsigned both = pack2<T>(y[0], y[1]);
    w[0][e] = both;
    w[1][e] = pack2<T>(y[0] - pages_half<T>(both & 0xffff), y[1] - pages_half<T>(both >> 16));
  }
}

// A wave's results, written: lane (c, g) holds of row c of each sixteen the values (16 (j / kTogether) + 4 g + e) kTogether + j % kTogether as
// o[t][j][e], unnormalized, the carried maximum and the sum.
template <typename T, int DP, int QT>
__device__ __forceinline__ void pages_write(const CacheOut<T, DP, 16 * QT>& out, const cache_f4 (&o)[QT][DP / 16], const float (&top)[QT],
                                            const float (&sum)[QT], int c, int g) {
  using P = Pages<T, DP>;
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const float factor = sum[t] == 0.0f ? 1.0f : 1.0f / sum[t] * P::kUnit;   // (without weights: zeros, infinities and NaN)
#pragma unroll
    for(int i = 0; i < P::kValuePieces; ++i)
#pragma unroll
      for(int e = 0; e < 4; ++e) {
        float y[P::kTogether];
#pragma unroll
        for(int j = 0; j < P::kTogether; ++j) y[j] = o[t][i * P::kTogether + j][e] * factor;
        out.emit(16 * t + c, (16 * i + 4 * g + e) * P::kTogether, y);
      }
    if(g == 0) out.emit_log(16 * t + c, top[t], sum[t]);
  }
}

// The results of waves that share rows, joined and written; alone: one wave has all of them, and the others have ended; odd: the wave has infinities
// or NaN among them.
template <typename T, int DP, int QT, int WAVES>
__device__ __forceinline__ void pages_finish(const PagesAttentionArgs& a, const CacheTile& x, cache_f4 (&o)[QT][DP / 16], const float (&top)[QT],
                                             float (&sum)[QT], int wave, bool alone, bool odd, CacheJoin<DP, QT, WAVES>& sh) {
  using P = Pages<T, DP>;
  constexpr int kTogether = P::kTogether, kHalf = CacheJoin<DP, QT, WAVES>::kHalf, kPieces = kHalf / (16 * kTogether);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
  for(int t = 0; t < QT; ++t) sum[t] = over_lanes_sum(sum[t]) * P::kUnit;
  const CacheOut<T, DP, 16 * QT> out(a, x);
  if(alone) {
    pages_write<T, DP, QT>(out, o, top, sum, c, g);
    if(WAVES > 1) return;
  } else if constexpr(WAVES > 1) {
#pragma unroll
    for(int t = 0; t < QT; ++t)
      if(g == 0) {
        sh.row_max[wave][16 * t + c] = top[t];
        sh.row_sum[wave][16 * t + c] = sum[t];
      }
    // A row's weights of N positions add up to 2^kMaximumSlack N at the most, and their values to that many times the largest, which may be next
    // to the largest float32: they are summed over a power of two above it, twice as large for the roundings.  (It changes no bit of a result.)
    const int up = 5 + 32 - __builtin_clz((unsigned)max(x.end - x.w.from, 1));
    const float over = __builtin_bit_cast(float, (unsigned)(127 - up) << 23) * P::kUnit, back = __builtin_bit_cast(float, (unsigned)(127 + up) << 23);
    static_assert(kMaximumSlack <= 4.0f, "up counts it");
    const CacheBuffer part(out.part, CacheOut<T, DP, 16 * QT>::kTileFloats * 4);
    __syncthreads();
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      float m = sh.row_max[0][16 * t + c];
#pragma unroll
      for(int i = 1; i < WAVES; ++i) m = fmaxf(m, sh.row_max[i][16 * t + c]);
      float mine = top[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f(top[t] - m) * over;
      if(__builtin_expect(odd, 0)) {
#pragma unroll
        for(int j = 0; j < DP / 16; ++j)
#pragma unroll
          for(int e = 0; e < 4; ++e) o[t][j][e] = times_odd(o[t][j][e], mine);
        mine = 1.0f;
      }
#pragma unroll
      for(int h = 0; h < DP / kHalf; ++h) {
        if(h || t) __syncthreads();
#pragma unroll
        for(int i = 0; i < kPieces; ++i)
#pragma unroll
          for(int e = 0; e < 4; ++e)
#pragma unroll
            for(int j = 0; j < kTogether; j += 4) {
              const int from = (h * kPieces + i) * kTogether + j;
              *reinterpret_cast<cache_f4*>(&sh.joined[wave][c][(16 * i + 4 * g + e) * kTogether + j]) =
                  cache_f4{o[t][from][e] * mine, o[t][from + 1][e] * mine, o[t][from + 2][e] * mine, o[t][from + 3][e] * mine};
            }
        __syncthreads();
        constexpr int kEach = kHalf / 16;
        const int d = (tid & 15) * kEach;
#pragma unroll
        for(int r = tid >> 4; r < 16; r += 4 * WAVES) {   // a row to sixteen threads
          float top_r = sh.row_max[0][16 * t + r], total = 0.0f, y[kEach];
#pragma unroll
          for(int i = 1; i < WAVES; ++i) top_r = fmaxf(top_r, sh.row_max[i][16 * t + r]);
#pragma unroll
          for(int i = 0; i < WAVES; ++i) {
            const float from = sh.row_max[i][16 * t + r];   // (of a wave that saw nothing the sum is 0, or NaN)
            total += sh.row_sum[i][16 * t + r] * (from == kNone ? 1.0f : __builtin_amdgcn_exp2f(from - top_r));
          }
          const float per = total == 0.0f ? 1.0f : 1.0f / total * back;
#pragma unroll
          for(int j = 0; j < kEach; ++j) {
            y[j] = sh.joined[0][r][d + j];
#pragma unroll
            for(int i = 1; i < WAVES; ++i) y[j] += sh.joined[i][r][d + j];
            y[j] *= per;
          }
          if(out.whole) {
            out.emit(16 * t + r, h * kHalf + d, y);
          } else if(x.row0 + 16 * t + r < x.rows) {   // (sixteen bytes at a time)
            const unsigned to = 4u * ((16 * t + r) * DP + h * kHalf + d);
#pragma unroll
            for(int j = 0; j < kEach; j += 4) part.store_through(cache_f4{y[j], y[j + 1], y[j + 2], y[j + 3]}, to + 4u * j);
            if(h == 0 && (tid & 15) == 0)
              part.store_through(total == 0.0f ? kNone : top_r + __builtin_amdgcn_logf(total), 4u * (16 * QT * DP + 16 * t + r));
          }
        }
      }
    }
  }
  if(!out.whole) cache_join_parts<T, DP, 16 * QT, WAVES, true>(a, x, out, sh.parts);
}

// Infinities and NaN among values: a result that sees one is that, of whatever weight, and the sum of them where there are several.  The product
// does not give that - a weight is in two terms, one of which may be zero or below it -, and what a row does not see must not be in
// it.  So where the wave left some out, or has a result that is none, it looks at its positions once more: `eights` of them, `step` apart.  Where
// waves, halves and parts are joined, times_odd and add_odd have them outlive a weight that is zero there: a result does not depend on where
// positions come to lie.  Returns whether it looked.
template <typename T, int DP, int QT>
__device__ __forceinline__ bool pages_odd_values(const PagesAttentionArgs& a, const int* table, const unsigned char* v_head, int row_bytes, int begin, int end,
                                                 int eights, int step, int lane, bool left_out, const CacheSight (&sight)[QT], cache_f4 (&o)[QT][DP / 16]) {
  constexpr int kTogether = Pages<T, DP>::kTogether, kBits = (DP / 4 + 31) / 32;
  float none = 0.0f;   // NaN where a result is none
#pragma unroll
  for(int t = 0; t < QT; ++t)
#pragma unroll
    for(int j = 0; j < DP / 16; ++j)
#pragma unroll
      for(int e = 0; e < 4; ++e) none += o[t][j][e] * 0.0f;
  if(!left_out && !__any(!(none == 0.0f))) return false;
  const int g = lane >> 4;
  unsigned has[QT][kBits] = {};   // results that have seen one
#pragma unroll 1
  for(int at = begin; at < end; at += step)
#pragma unroll 1
    for(int first = at; first < min(at + 8 * eights, end); first += 8) {
      const PagesPlace y = pages_look(a, table, (unsigned)first >> 3);
      if((unsigned)y.id >= (unsigned)a.pages) continue;
      const unsigned char* const rows = v_head + y.id * a.page_bytes + (long long)(8 * y.eight) * row_bytes;
      const int bytes = min(8, end - first) * row_bytes;
      bool odd = false;
#pragma unroll 1
      for(int i = 16 * lane; i < bytes; i += 1024) {
        const cache_u4 w = *reinterpret_cast<const cache_u4*>(rows + i);
#pragma unroll
        for(int e = 0; e < 4; ++e) odd |= pages_finite<T>(w[e]) != w[e];
      }
      if(!__any(odd)) continue;
#pragma unroll 1
      for(int k = 0; k < min(8, end - first); ++k) {
        const T* const v = reinterpret_cast<const T*>(rows + k * row_bytes);
#pragma unroll
        for(int i = 0; i < DP / 16 / kTogether; ++i)
#pragma unroll
          for(int e = 0; e < 4; ++e) {
            const int d = (16 * i + 4 * g + e) * kTogether;
            float z[kTogether];
            load_row<kTogether>(v + (d < a.dk ? d : 0), z);
#pragma unroll
            for(int j = 0; j < kTogether; ++j) {
              const int piece = i * kTogether + j, bit = 4 * piece + e;
              if(__builtin_fabsf(z[j]) < __builtin_huge_valf() || d >= a.dk) continue;
#pragma unroll
              for(int t = 0; t < QT; ++t) {
                if(first + k >= sight[t].limit) continue;
                o[t][piece][e] = has[t][bit / 32] >> (bit % 32) & 1 ? o[t][piece][e] + z[j] : z[j];
                has[t][bit / 32] |= 1u << (bit % 32);
              }
            }
          }
      }
    }
  return true;
}

template <typename T, int DP, bool WHOLE, int QT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, pages_to_a_simd(sizeof(T), DP, QT)) void pages_attention_kernel(PagesAttentionArgs a) {
  using P = Pages<T, DP>;
  constexpr int kWidth = P::kWidth, kDims = P::kDims, kTogether = P::kTogether, kKeyPieces = P::kKeyPieces, kValuePieces = P::kValuePieces;
  constexpr int kTurn = 32 * WAVES;   // positions that the waves take in one turn
  constexpr bool kQueriesInLds = DP == 256;   // (which leaves registers to the rest)
  __shared__ CacheJoin<DP, QT, WAVES> sh;
  __shared__ cache_u4 q_held[kQueriesInLds ? QT : 1][kKeyPieces][kQueriesInLds ? 64 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  CacheTile x;
  if(!cache_tile<T, DP, 16 * QT, WAVES, kPagesMostParts, true>(a, tid, x)) return;
  const int end = x.end, row_bytes = (WHOLE ? DP : a.dk) * kWidth;
  // A sequence of one turn of one wave is that wave's: no join, and the others make room (236 of three positions, 16 heads of 64 values, 11 us and 20).
  const bool alone = WAVES == 1 || (x.w.parts == 1 && end - x.w.from <= 32);
  if(alone && wave > 0) return;
  const int* const table = a.table + (long long)x.w.s * a.row;
  const unsigned char* const k_head = a.k_pages + x.head * a.head_bytes;
  const unsigned char* const v_head = a.v_pages + x.head * a.head_bytes;

  // A lane's page of the eight positions from `at` on, as an offset; whether there is one.
  auto here = [&](const PagesPlace& y, int at, bool& is) __attribute__((always_inline)) -> long long {
    is = (unsigned)y.id < (unsigned)a.pages && at < end;
    return is ? y.id * a.page_bytes + (long long)(8 * y.eight) * row_bytes : 0;
  };
  auto fetch_keys = [&](typename P::Keys& y, const PagesPlace& place, int at) __attribute__((always_inline)) {
    bool is;
    const unsigned char* const p = k_head + here(place, at + 8 * (c >> 2), is);
#pragma unroll
    for(int t = 0; t < 2; ++t) {
      const unsigned char* const key = p + ((c & 3) + 4 * t) * row_bytes;
#pragma unroll
      for(int i = 0; i < kKeyPieces; ++i) {
        const int d = 64 * i + 16 * g;
        y.piece[t][i] = *reinterpret_cast<const cache_u4*>(key + (d < row_bytes ? d : 0));
      }
    }
  };
  auto fetch_values = [&](typename P::Values& y, const PagesPlace& place, int at, bool& is) __attribute__((always_inline)) {
    const unsigned char* const p = v_head + here(place, at + 8 * g, is);
#pragma unroll
    for(int e = 0; e < 8; ++e)
#pragma unroll
      for(int i = 0; i < kValuePieces; ++i) {
        const int d = (16 * i + c) * kTogether * kWidth;
        const unsigned char* const from = p + e * row_bytes + (d < row_bytes ? d : 0);
        if constexpr(P::kWords == 4) {
          const cache_u4 w = *reinterpret_cast<const cache_u4*>(from);
#pragma unroll
          for(int j = 0; j < 4; ++j) y.word[e][i][j] = w[j];
        } else {
          const cache_u2 w = *reinterpret_cast<const cache_u2*>(from);
          y.word[e][i][0] = w[0];
          y.word[e][i][1] = w[1];
        }
      }
  };

  const int begin = x.w.from + 32 * wave;
  auto look_keys = [&](int at) { return pages_look(a, table, (unsigned)(at >> 3) + (c >> 2)); };
  auto look_values = [&](int at) { return pages_look(a, table, (unsigned)(at >> 3) + g); };
  const PagesPlace k_first = look_keys(begin), v_first = look_values(begin);
  PagesPlace k_next = look_keys(begin + kTurn), v_next = look_values(begin + kTurn);
  typename P::Keys key;
  typename P::Values value;
  bool there;   // whether the lane's eight positions have a page
  fetch_keys(key, k_first, begin);
  fetch_values(value, v_first, begin, there);

  cache_u4 q[kQueriesInLds ? 1 : QT][kKeyPieces];
  CacheSight sight[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const int row = min(x.row0 + 16 * t + c, x.rows - 1);
    sight[t] = cache_sight(a, x, row, 0);
    unsigned of_group;
    const unsigned token = a.by_group.of((unsigned)row, of_group);
    const unsigned char* const p =
        reinterpret_cast<const unsigned char*>(static_cast<const T*>(a.q) + x.w.s * a.q_s + (long long)(x.head * a.G + (int)of_group) * a.q_h +
                                               (long long)token * a.q_n);
#pragma unroll
    for(int i = 0; i < kKeyPieces; ++i) {
      const int d = 64 * i + 16 * g;
      const cache_u4 y = *reinterpret_cast<const cache_u4*>(p + (d < row_bytes ? d : 0));
      const cache_u4 z = d < row_bytes ? y : cache_u4{0, 0, 0, 0};
      if constexpr(kQueriesInLds) {
        if(alone || wave == t % WAVES) q_held[t][i][lane] = z;
      } else {
        q[t][i] = z;
      }
    }
  }
  if(kQueriesInLds && !alone) __syncthreads();

  cache_f4 o[QT][kDims];
  float top[QT], sum[QT];   // carried maximum (base 2), the lane's part of the sum
  bool left_out = false;    // whether a value was left out of the product
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    top[t] = kNone;
    sum[t] = 0.0f;
#pragma unroll
    for(int j = 0; j < kDims; ++j) o[t][j] = cache_f4{0, 0, 0, 0};
  }

  for(int at = begin; at < end; at += kTurn) {
    if(!WHOLE) {   // (what was loaded past a row's end is its start again)
#pragma unroll
      for(int i = 0; i < kKeyPieces; ++i)
#pragma unroll
        for(int t = 0; t < 2; ++t) key.piece[t][i] = 64 * i + 16 * g < row_bytes ? key.piece[t][i] : cache_u4{0, 0, 0, 0};
    }
    if constexpr(kQueriesInLds) asm volatile("" ::: "memory");   // (or they would be read ahead of all turns, into registers)
    cache_f4 s[QT][2];
#pragma unroll
    for(int t = 0; t < QT; ++t) s[t][0] = s[t][1] = cache_f4{0, 0, 0, 0};
#pragma unroll
    for(int i = 0; i < kKeyPieces; ++i)
#pragma unroll
      for(int b = 0; b < 2; ++b)
#pragma unroll
        for(int t = 0; t < QT; ++t) s[t][b] = pages_product<T>(key.piece[b][i], kQueriesInLds ? q_held[t][i][lane] : q[t][i], s[t][b]);
    // (Up to sixteen rows of 16-bit values the last turn fetches nothing: 250 sequences of up to 60 positions, 8 heads of 128 values with four rows
    // each, 13 us and 15, 49 of up to 2068, 8 of 256, 125 and 130.  Without the branch 32 rows take 43 us in place of 46, 16 sequences of up
    // to 8192, 4 heads of 128 values, and float32 of one token 2 % less.)
    const bool on = kWidth == 4 || QT == 2 || at + kTurn < end;
    if(on) fetch_keys(key, k_next, at + kTurn);
    const bool is = there;
    const bool masked = at + 32 > x.open || __any(!is);
    const int first = at + 8 * g;
    if(masked) {
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const int sees = is ? sight[t].limit - first : 0;
#pragma unroll
        for(int e = 0; e < 8; ++e) s[t][e / 4][e % 4] = e < sees ? s[t][e / 4][e % 4] : kNone;
      }
      // Values that no row sees weigh zero, whatever they are.
      const int seen = is ? end - first : 0;
#pragma unroll
      for(int e = 0; e < 8; ++e)
#pragma unroll
        for(int i = 0; i < kValuePieces; ++i)
#pragma unroll
          for(int w = 0; w < P::kWords; ++w) value.word[e][i][w] = e < seen ? value.word[e][i][w] : 0;
    }
    float high[QT];
    bool grown = false;
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      high[t] = kNone;
#pragma unroll
      for(int e = 0; e < 8; ++e) high[t] = fmaxf(high[t], s[t][e / 4][e % 4]);
      high[t] *= a.scale_log2;
      grown |= high[t] > top[t] + kMaximumSlack;
    }
    if(__any(grown)) {
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const float m = fmaxf(top[t], over_lanes_max(high[t]));
        const float down = m == top[t] ? 1.0f : __builtin_amdgcn_exp2f(top[t] - m);
        sum[t] *= down;
#pragma unroll
        for(int j = 0; j < kDims; ++j) o[t][j] *= down;
        top[t] = m;
      }
    }
    // Positions that some rows see and others do not: infinities and NaN among their values stay out of the product, see below.
    if(masked && end > x.open) {
      bool odd = false;
#pragma unroll
      for(int e = 0; e < 8; ++e)
#pragma unroll
        for(int i = 0; i < kValuePieces; ++i)
#pragma unroll
          for(int w = 0; w < P::kWords; ++w) {
            const unsigned z = value.word[e][i][w], clean = first + e < x.open ? z : pages_finite<T>(z);
            odd |= z != clean;
            value.word[e][i][w] = clean;
          }
      left_out |= __any(odd) != 0;
    }
    // weighted values
    if constexpr(kWidth == 4) {
      float p[QT][8];
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const float from = top[t] == kNone ? 0.0f : -top[t];   // (nothing seen so far: minus infinity stays that)
        // (Scaled behind the exponential: a weight next to one has an exponent next to zero then, in all its bits.  128 sequences of 513 positions, 64
        // values, are 3.5e-7 off 64 bits, and 6.0e-7 with the scale in the exponent, which takes 1 to 2 us less of 75.)
#pragma unroll
        for(int e = 0; e < 8; ++e) {
          p[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / 4][e % 4], a.scale_log2, from)) * (1.0f / P::kUnit);
          sum[t] += p[t][e];
        }
      }
#pragma unroll
      for(int j = 0; j < kDims; ++j)
#pragma unroll
        for(int e = 0; e < 8; ++e)
#pragma unroll
          for(int t = 0; t < QT; ++t)
            o[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, value.word[e][j / kTogether][j % kTogether]), p[t][e], o[t][j], 0, 0, 0);
    } else {
      cache_u4 weights[QT][2];
#pragma unroll
      for(int t = 0; t < QT; ++t) pages_weights<T>(s[t], a.scale_log2, (top[t] == kNone ? 0.0f : -top[t]) + P::kUp, sum[t], weights[t]);
#pragma unroll
      for(int j = 0; j < kDims; ++j) {
        cache_u4 d;
#pragma unroll
        for(int e = 0; e < 4; ++e)
          d[e] = __builtin_amdgcn_perm(value.word[2 * e + 1][j / kTogether][j % kTogether / 2], value.word[2 * e][j / kTogether][j % kTogether / 2],
                                       j % 2 ? 0x07060302 : 0x05040100);
#pragma unroll
        for(int t = 0; t < QT; ++t)
#pragma unroll
          for(int m = 1; m >= 0; --m) o[t][j] = pages_product<T>(d, weights[t][m], o[t][j]);
      }
    }
    if(!on) break;
    fetch_values(value, v_next, at + kTurn, there);
    k_next = look_keys(at + 2 * kTurn);
    v_next = look_values(at + 2 * kTurn);
  }
  const bool odd = pages_odd_values<T, DP, QT>(a, table, v_head, row_bytes, begin, end, 4, kTurn, lane, left_out, sight, o);
  pages_finish<T, DP, QT, WAVES>(a, x, o, top, sum, wave, alone, odd, sh);
}

// ---- more than 32 rows
// Waves share positions laid out in LDS, 64 at a time, twice: while one is worked on, the next is written and the one after that is on its way
// to registers.  64 rows are taken by eight waves of sixteen, four of them for the first 32 positions of each 64 and four for the second.  128
// rows are taken by eight waves too where rows have 64 values, by four of 32 where they have 128: LDS is read half as often then, and that
// counts by the length of rows (512 new tokens of 4 sequences, 16 heads of 64 values, 42 us by eight and 45 by four; 1024 of them, 32 heads on
// 8, 128 values, 200 and 187).  The last rows go first: a prompt of 4096 tokens, 32 heads on 8, 128 values 262 us and 290; now 225 us, 610 TFLOP/s of what they see.
// Keys lie in LDS as they are, values transposed, a dimension's 64 side by side; pieces of 16 bytes change places within a row (key_place,
// value_place) so that few lanes that read together meet in a bank (a third of the cycles that LDS is busy).  A wave lays out one or two eights
// of positions: sixteen lanes (of rows of 128 bytes eight) to a row of keys; of values a lane has some dimensions of eight positions.
// Products, weights and sums are those above.  float32 is taken by eight waves for 64 and for 128 rows; its values lie in LDS as they are, too, a
// product takes one of them at a time.
//
// What bounds it: latency, of the memory's answers and of the partial results' way to the workgroup that joins them; LDS is busy less than a third of
// the time and the matrix units a fifth.  7 drafted tokens, float16, 24 sequences of up to 8192 positions, 4 heads of 128 values with eight
// rows each (56 rows, 270 MB): 65 to 71 us, 3.9 TB/s; four waves that take all positions and join them 80, waves of the form above with a row
// group each 95.  bfloat16, 64 values, 8 tokens, 16 sequences: 35, by four waves 39.6.  float32, the 56 rows above: 217 us,
// of which the matrix products alone take 110 (17 GFLOP).  __syncthreads in place of the barrier below waits for the loads too.
template <typename T, int DP, int ROWS>
struct PagesMany {
  static constexpr int kWidth = sizeof(T);
  static constexpr int kWaves = pages_many_waves(kWidth, DP, ROWS);
  static constexpr int kSixteens = kWaves == 4 && ROWS == 128 ? 2 : 1;   // of rows, to a wave
  static constexpr int kGroups = ROWS / (16 * kSixteens); // waves that have different rows
  static constexpr int kSplit = kWaves / kGroups;         // shares of the positions
  static constexpr int kTile = 64;                        // positions of a turn
  static constexpr int kRowPieces = DP * kWidth / 16;     // pieces of a row
  static constexpr int kEights = 8 / kWaves;               // of positions that a wave lays out
  static constexpr int kRowLoads = kEights * kRowPieces / 8;       // of a lane, of keys (float32: of values too)
  static constexpr int kLanes = 64 / kEights;             // that have an eight's values, kDimsEach dimensions each
  static constexpr int kDimsEach = DP / kLanes < 2 ? 2 : DP / kLanes;
  static constexpr int kValueWords = kDimsEach / 2;
  // (lanes that read together are, by what was measured, the 16 lanes c, of one half of them with g and of the other with g ^ 1)
  static __device__ __forceinline__ int key_place(int key, int piece) {
    const int c = (key >> 1 & 12) | (key & 3);
    return (key * kRowPieces + (piece ^ (kRowPieces >= 16 ? c : c >> 1))) * 16;
  }
  static __device__ __forceinline__ int value_place(int dim, int eight) {   // (16-bit types)
    const int c = dim / Pages<T, DP>::kTogether, j = dim % Pages<T, DP>::kTogether;
    return (j * 16 + c) * 128 + (eight ^ c >> 1) * 16;
  }
  struct Shared {
    alignas(16) unsigned char keys[2][kTile * DP * kWidth];
    alignas(16) unsigned char values[2][kTile * DP * kWidth];
    int there[2][8];   // of each eight of positions, whether it has a page
    int left_out;
  };
  struct Halves {   // what either half of the waves has for the other
    cache_f4 o[2][4][DP / 32][64];
    float top[2][4][64], sum[2][4][64];
  };
};

// A barrier for what lies in LDS: loads from memory stay under way, which __syncthreads would wait for.
__device__ __forceinline__ void pages_lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <typename T, int DP, bool WHOLE, int ROWS>
__global__ __launch_bounds__(64 * pages_many_waves(sizeof(T), DP, ROWS), pages_many_to_a_simd(sizeof(T), DP, ROWS)) void pages_attention_many_kernel(PagesAttentionArgs a) {
  using P = Pages<T, DP>;
  using M = PagesMany<T, DP, ROWS>;
  constexpr int QT = M::kSixteens, SPLIT = M::kSplit;
  constexpr int kDims = P::kDims, kTogether = P::kTogether, kKeyPieces = P::kKeyPieces, kTile = M::kTile, kEights = M::kEights, kParts = 2 / SPLIT, kWidth = M::kWidth;
  __shared__ struct {
    union {
      typename M::Shared tile;
      typename M::Halves half;
    };
    int is_last;
  } sh;
  const int tid = threadIdx.x, lane = tid & 63, any_wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int wave = any_wave % M::kGroups, half = any_wave / M::kGroups;   // of the rows, of the positions
  CacheTile x;
  if(!cache_tile<T, DP, ROWS, M::kWaves, kPagesMostParts, true>(a, tid, x)) return;
  const int end = x.end, row_bytes = (WHOLE ? DP : a.dk) * kWidth;
  const int* const table = a.table + (long long)x.w.s * a.row;
  const unsigned char* const k_head = a.k_pages + x.head * a.head_bytes;
  const unsigned char* const v_head = a.v_pages + x.head * a.head_bytes;
  if(tid == 0) sh.tile.left_out = 0;

  // ---- what a wave lays out: the eights of a tile from kEights * any_wave on
  struct Fetched {
    cache_u4 key[M::kRowLoads];
    unsigned value[8][M::kValueWords];   // 16-bit types: some dimensions of an eight ...
    cache_u4 value_row[M::kRowLoads];    // ... float32: pieces as of keys
    bool there[kEights];
    PagesPlace next[kEights];   // of the tile that is fetched next
  } fetched;
  auto look = [&](Fetched& y, int at) __attribute__((always_inline)) {
#pragma unroll
    for(int i = 0; i < kEights; ++i) y.next[i] = pages_look(a, table, (unsigned)(at + 8 * (kEights * any_wave + i)) >> 3);
  };
  auto fetch = [&](Fetched& f, int at) __attribute__((always_inline)) {
    long long place[kEights];
#pragma unroll
    for(int i = 0; i < kEights; ++i) {
      const int first = at + 8 * (kEights * any_wave + i);
      const PagesPlace y = f.next[i];
      f.there[i] = (unsigned)y.id < (unsigned)a.pages && first < end;
      place[i] = f.there[i] ? y.id * a.page_bytes + (long long)(8 * y.eight) * row_bytes : 0;
    }
#pragma unroll
    for(int i = 0; i < M::kRowLoads; ++i) {   // (rows past one eight are of the next)
      constexpr int kAtOnce = 64 / M::kRowPieces;
      const int row = kAtOnce * i + lane / M::kRowPieces, piece = lane % M::kRowPieces * 16;
      const long long from = place[kAtOnce * i / 8] + (row & 7) * row_bytes + (piece < row_bytes ? piece : 0);
      f.key[i] = *reinterpret_cast<const cache_u4*>(k_head + from);
      if(kWidth == 4) f.value_row[i] = *reinterpret_cast<const cache_u4*>(v_head + from);
    }
    if constexpr(kWidth == 4) return;
    const int d = lane % M::kLanes * M::kDimsEach * 2;
    const unsigned char* const from = v_head + (lane < M::kLanes ? place[0] : place[kEights - 1]) + (d < row_bytes ? d : 0);
#pragma unroll
    for(int e = 0; e < 8; ++e)
#pragma unroll
      for(int w = 0; w < M::kValueWords; ++w) f.value[e][w] = reinterpret_cast<const unsigned*>(from + e * row_bytes)[w];
  };
  auto lay_out = [&](Fetched& f, int at, int buffer) __attribute__((always_inline)) {
    constexpr int kAtOnce = 64 / M::kRowPieces;
#pragma unroll
    for(int i = 0; i < M::kRowLoads; ++i) {
      const int row = 8 * kEights * any_wave + kAtOnce * i + lane / M::kRowPieces, piece = lane % M::kRowPieces;
      if(!WHOLE) f.key[i] = piece * 16 < row_bytes ? f.key[i] : cache_u4{0, 0, 0, 0};   // (queries are zero there, and so must these be)
      *reinterpret_cast<cache_u4*>(sh.tile.keys[buffer] + M::key_place(row, piece)) = f.key[i];
      if constexpr(kWidth == 4) {
        if(at + kTile > x.open || !f.there[0]) {   // (as below)
          const bool seen = f.there[0] && at + row < end;
#pragma unroll
          for(int w = 0; w < 4; ++w) {
            const unsigned z = seen ? f.value_row[i][w] : 0, clean = at + row < x.open ? z : pages_finite<T>(z);
            if(z != clean) sh.tile.left_out = 1;
            f.value_row[i][w] = clean;
          }
        }
        *reinterpret_cast<cache_u4*>(sh.tile.values[buffer] + (row * M::kRowPieces + piece) * 16) = f.value_row[i];
      }
    }
    if constexpr(kWidth == 4) {
      if(lane == 0) sh.tile.there[buffer][any_wave] = f.there[0];
      return;
    }
    const int eight = kEights * any_wave + lane / M::kLanes, first = at + 8 * eight;
    const bool is = lane < M::kLanes ? f.there[0] : f.there[kEights - 1];
    if(at + kTile > x.open || !(f.there[0] && f.there[kEights - 1])) {
      // Values that no row sees weigh zero, whatever they are; infinities and NaN that some do not see are left out, see below.
      const int seen = is ? end - first : 0;
      bool any = false;
#pragma unroll
      for(int e = 0; e < 8; ++e)
#pragma unroll
        for(int w = 0; w < M::kValueWords; ++w) {
          const unsigned z = e < seen ? f.value[e][w] : 0, clean = first + e < x.open ? z : pages_finite<T>(z);
          any |= z != clean;
          f.value[e][w] = clean;
        }
      if(any) sh.tile.left_out = 1;
    }
    if(lane % M::kLanes == 0) sh.tile.there[buffer][eight] = is;
#pragma unroll
    for(int j = 0; j < M::kDimsEach; ++j) {
      cache_u4 y;
#pragma unroll
      for(int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_perm(f.value[2 * e + 1][j / 2], f.value[2 * e][j / 2], j % 2 ? 0x07060302 : 0x05040100);
      const int dim = lane % M::kLanes * M::kDimsEach + j;
      if(M::kLanes * M::kDimsEach == DP || dim < DP) *reinterpret_cast<cache_u4*>(sh.tile.values[buffer] + M::value_place(dim, eight)) = y;
    }
  };

  const int begin = x.w.from;
  look(fetched, begin);
  fetch(fetched, begin);
  look(fetched, begin + kTile);
  cache_u4 q[QT][kKeyPieces];
  CacheSight sight[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const int row = min(x.row0 + 16 * (QT * wave + t) + c, x.rows - 1);
    sight[t] = cache_sight(a, x, row, 0);
    unsigned of_group;
    const unsigned token = a.by_group.of((unsigned)row, of_group);
    const unsigned char* const p =
        reinterpret_cast<const unsigned char*>(static_cast<const T*>(a.q) + x.w.s * a.q_s + (long long)(x.head * a.G + (int)of_group) * a.q_h +
                                               (long long)token * a.q_n);
#pragma unroll
    for(int i = 0; i < kKeyPieces; ++i) {
      const int d = 64 * i + 16 * g;
      const cache_u4 y = *reinterpret_cast<const cache_u4*>(p + (d < row_bytes ? d : 0));
      q[t][i] = d < row_bytes ? y : cache_u4{0, 0, 0, 0};
    }
  }
  cache_f4 o[QT][kDims];
  float top[QT], sum[QT];   // carried maximum (base 2), the lane's part of the sum
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    top[t] = kNone;
    sum[t] = 0.0f;
#pragma unroll
    for(int j = 0; j < kDims; ++j) o[t][j] = cache_f4{0, 0, 0, 0};
  }
  pages_lds_barrier();   // (left_out is cleared)
  lay_out(fetched, begin, 0);
  fetch(fetched, begin + kTile);
  look(fetched, begin + 2 * kTile);
  pages_lds_barrier();

  int buffer = 0;
  for(int at = begin; at < end; at += kTile, buffer ^= 1) {
    const bool masked = at + kTile > x.open;
    unsigned none = 0;   // the tile's eights without a page
    {
      const cache_i4 lo = *reinterpret_cast<const cache_i4*>(&sh.tile.there[buffer][0]), hi = *reinterpret_cast<const cache_i4*>(&sh.tile.there[buffer][4]);
#pragma unroll
      for(int i = 0; i < 4; ++i) none |= (lo[i] ? 0 : 1u << i) | (hi[i] ? 0 : 16u << i);
    }
    cache_f4 s[QT][2 * kParts];   // two for 32 positions
#pragma unroll
    for(int t = 0; t < QT; ++t)
#pragma unroll
      for(int b = 0; b < 2 * kParts; ++b) s[t][b] = cache_f4{0, 0, 0, 0};
#pragma unroll
    for(int i = 0; i < kKeyPieces; ++i)
#pragma unroll
      for(int b = 0; b < 2 * kParts; ++b) {
        const cache_u4 k = *reinterpret_cast<const cache_u4*>(sh.tile.keys[buffer] + M::key_place(32 * (half + b / 2) + 8 * (c >> 2) + (c & 3) + 4 * (b % 2), 4 * i + g));
#pragma unroll
        for(int t = 0; t < QT; ++t) s[t][b] = pages_product<T>(k, q[t][i], s[t][b]);
      }
    if(masked || none) {
#pragma unroll
      for(int h = 0; h < kParts; ++h) {
        const int first = at + 32 * (half + h) + 8 * g;
#pragma unroll
        for(int t = 0; t < QT; ++t) {
          const int sees = none >> (4 * (half + h) + g) & 1 ? 0 : sight[t].limit - first;
#pragma unroll
          for(int e = 0; e < 8; ++e) s[t][2 * h + e / 4][e % 4] = e < sees ? s[t][2 * h + e / 4][e % 4] : kNone;
        }
      }
    }
    float high[QT];
    bool grown = false;
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      high[t] = kNone;
#pragma unroll
      for(int e = 0; e < 8 * kParts; ++e) high[t] = fmaxf(high[t], s[t][e / 4][e % 4]);
      high[t] *= a.scale_log2;
      grown |= high[t] > top[t] + kMaximumSlack;
    }
    if(__any(grown)) {
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const float m = fmaxf(top[t], over_lanes_max(high[t]));
        const float down = m == top[t] ? 1.0f : __builtin_amdgcn_exp2f(top[t] - m);
        sum[t] *= down;
#pragma unroll
        for(int j = 0; j < kDims; ++j) o[t][j] *= down;
        top[t] = m;
      }
    }
    // (the second half's weights are made while the first half's products run)
    if constexpr(kWidth == 4) {
#pragma unroll
      for(int h = 0; h < kParts; ++h) {
        float p[8];
        const float from = top[0] == kNone ? 0.0f : -top[0];
#pragma unroll
        for(int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][2 * h + e / 4][e % 4], a.scale_log2, from)) * (1.0f / P::kUnit);
          sum[0] += p[e];
        }
#pragma unroll
        for(int i = 0; i < P::kValuePieces; ++i)
#pragma unroll
          for(int e = 0; e < 8; ++e) {
            const cache_f4 v = *reinterpret_cast<const cache_f4*>(sh.tile.values[buffer] + ((32 * (half + h) + 8 * g + e) * M::kRowPieces + 16 * i + c) * 16);
#pragma unroll
            for(int j = 0; j < kTogether; ++j)
              o[0][i * kTogether + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], p[e], o[0][i * kTogether + j], 0, 0, 0);
          }
      }
    } else {
#pragma unroll
      for(int h = 0; h < kParts; ++h) {
        cache_u4 weights[QT][2];
#pragma unroll
        for(int t = 0; t < QT; ++t) {
          const cache_f4 mine[2] = {s[t][2 * h], s[t][2 * h + 1]};
          pages_weights<T>(mine, a.scale_log2, (top[t] == kNone ? 0.0f : -top[t]) + P::kUp, sum[t], weights[t]);
        }
#pragma unroll
        for(int j = 0; j < kDims; ++j) {
          const int dim = (16 * (j / kTogether) + c) * kTogether + j % kTogether;
          const cache_u4 v = *reinterpret_cast<const cache_u4*>(sh.tile.values[buffer] + M::value_place(dim, 4 * (half + h) + g));
#pragma unroll
          for(int t = 0; t < QT; ++t)
#pragma unroll
            for(int m = 1; m >= 0; --m) o[t][j] = pages_product<T>(v, weights[t][m], o[t][j]);
        }
      }
    }
    if(at + kTile < end) lay_out(fetched, at + kTile, buffer ^ 1);
    fetch(fetched, at + 2 * kTile);
    look(fetched, at + 3 * kTile);
    pages_lds_barrier();
  }
  pages_odd_values<T, DP, QT>(a, table, v_head, row_bytes, begin + 32 * half, end, 4 * kParts, kTile, lane, sh.tile.left_out != 0, sight, o);
  // Rows of a sequence in one part go to the output.  Parts go to the workspace as registers have them, 1 KB at a time, and back: whoever
  // arrives last joins them, a wave its own rows (16 parts of 64 rows: 20 us less than by rows of 16 threads, which store and load pieces of 8 bytes).
  const CacheOut<T, DP, ROWS> out(a, x);
#pragma unroll
  for(int t = 0; t < QT; ++t) sum[t] = over_lanes_sum(sum[t]) * P::kUnit;
  // Two halves exchange results: of its rows each has kOwn of the kDims pieces from here on, `shift` the first of them.
  constexpr int kOwn = kDims / SPLIT;
  const int shift = half * kOwn;
  cache_f4 r[QT][kOwn];
  auto none_of = [](const cache_f4 (&y)[kOwn]) {   // whether one of these is an infinity or NaN
    float none = 0.0f;
#pragma unroll
    for(int j = 0; j < kOwn; ++j)
#pragma unroll
      for(int e = 0; e < 4; ++e) none += y[j][e] * 0.0f;
    return !(none == 0.0f);
  };
  if constexpr(SPLIT == 1) {
#pragma unroll
    for(int t = 0; t < QT; ++t)
#pragma unroll
      for(int j = 0; j < kOwn; ++j) r[t][j] = o[t][j];
  } else {
    pages_lds_barrier();   // (left_out has been read)
    if(half == 0) {
#pragma unroll
      for(int j = 0; j < kOwn; ++j) sh.half.o[0][wave][j][lane] = o[0][kOwn + j];
    } else {
#pragma unroll
      for(int j = 0; j < kOwn; ++j) sh.half.o[1][wave][j][lane] = o[0][j];
    }
    sh.half.top[half][wave][lane] = top[0];
    sh.half.sum[half][wave][lane] = sum[0];
    pages_lds_barrier();
    const float other = sh.half.top[1 - half][wave][lane], m = fmaxf(top[0], other);
    const float mine = top[0] == kNone ? 1.0f : __builtin_amdgcn_exp2f(top[0] - m), its = other == kNone ? 1.0f : __builtin_amdgcn_exp2f(other - m);
    // (of a half without positions both are 0, or NaN)
#pragma unroll
    for(int j = 0; j < kOwn; ++j) {
      const cache_f4 y[2] = {o[0][j], o[0][kOwn + j]}, z = sh.half.o[1 - half][wave][j][lane] * its;
#pragma unroll
      for(int e = 0; e < 4; ++e) r[0][j][e] = (half == 0 ? y[0][e] : y[1][e]) * mine + z[e];
    }
    if(__builtin_expect(none_of(r[0]), 0)) {
#pragma unroll
      for(int j = 0; j < kOwn; ++j) {
        const cache_f4 z = sh.half.o[1 - half][wave][j][lane];
#pragma unroll
        for(int e = 0; e < 4; ++e) r[0][j][e] = times_odd(half == 0 ? o[0][j][e] : o[0][kOwn + j][e], mine) + times_odd(z[e], its);
      }
    }
    sum[0] = sum[0] * mine + sh.half.sum[1 - half][wave][lane] * its;
    top[0] = m;
  }
  auto write = [&](int t, float factor) __attribute__((always_inline)) {
    const int row = x.row0 + 16 * (QT * wave + t) + c;
    if(row >= x.rows) return;
    T* const to = cache_row_out<T>(a, x, row);
    constexpr int kRun = kTogether < kOwn ? kTogether : kOwn;   // values side by side
#pragma unroll
    for(int i = 0; i < kOwn / kRun; ++i)
#pragma unroll
      for(int e = 0; e < 4; ++e) {
        const int j0 = shift + i * kRun, d = (16 * (j0 / kTogether) + 4 * g + e) * kTogether + j0 % kTogether;
        float y[kRun];
#pragma unroll
        for(int j = 0; j < kRun; ++j) y[j] = r[t][i * kRun + j][e] * factor;
        if(d < a.dk) {
          if constexpr(kRun == 2 && kWidth == 4) *reinterpret_cast<cache_u2*>(to + d) = cache_u2{__builtin_bit_cast(unsigned, y[0]), __builtin_bit_cast(unsigned, y[1])};
          else if constexpr(kRun == 2) *reinterpret_cast<unsigned*>(to + d) = pack2<T>(y[0], y[1]);
          else store_row<kRun, T>(to + d, y);
        }
      }
  };
  if(out.whole) {
#pragma unroll
    for(int t = 0; t < QT; ++t) write(t, sum[t] == 0.0f ? 1.0f : 1.0f / sum[t] * P::kUnit);   // (without weights: zeros, infinities and NaN)
    return;
  }
  constexpr unsigned kTileBytes = CacheOut<T, DP, ROWS>::kTileFloats * 4;
  const unsigned stride = (unsigned)out.stride * kTileBytes, mine = 1024u * (QT * kDims * wave + shift) + 16u * lane, my_log = 4u * (ROWS * DP + 16 * QT * wave + c);
  const CacheBuffer parts(a.part + out.place * CacheOut<T, DP, ROWS>::kTileFloats, stride * x.w.parts);
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const float factor = sum[t] == 0.0f ? 1.0f : 1.0f / sum[t] * P::kUnit;
    const unsigned to = stride * x.w.part;
#pragma unroll
    for(int j = 0; j < kOwn; ++j) parts.store_through(r[t][j] * factor, to + mine + 1024u * (t * kDims + j));
    if(g == 0 && half == 0) parts.store_through(sum[t] == 0.0f ? kNone : top[t] + __builtin_amdgcn_logf(sum[t]), to + my_log + 64u * t);
  }
  if(!cache_arrived_last(a.counters + out.place, x.w.parts, sh.is_last)) return;
  float weight_sum[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    top[t] = kNone;
    weight_sum[t] = 0.0f;
#pragma unroll
    for(int j = 0; j < kOwn; ++j) r[t][j] = cache_f4{0, 0, 0, 0};
  }
  constexpr int kLogs = 8, kBatch = QT * kOwn > 8 ? 2 : 16 / (QT * kOwn);
#pragma unroll 1
  for(int i = 0; i < x.w.parts; i += kLogs) {   // (behind the last part the buffer gives zeros)
    float l[QT][kLogs];
#pragma unroll
    for(int b = 0; b < kLogs; ++b)
#pragma unroll
      for(int t = 0; t < QT; ++t) l[t][b] = parts.number_through(stride * (unsigned)(i + b) + my_log + 64u * t);
#pragma unroll
    for(int b = 0; b < kLogs; ++b)
#pragma unroll
      for(int t = 0; t < QT; ++t) top[t] = i + b < x.w.parts ? fmaxf(top[t], l[t][b]) : top[t];
  }
  // (a part's weight is at most 1, times kPartUnit: sums stay within the largest value)
  auto weight_of = [](float l, float high) { return l == kNone ? 0.0f : __builtin_amdgcn_exp2f(l - high) * kPartUnit; };
#pragma unroll 1
  for(int i = 0; i < x.w.parts; i += kBatch) {
    float l[QT][kBatch];
    cache_f4 z[kBatch][QT][kOwn];
#pragma unroll
    for(int b = 0; b < kBatch; ++b) {
      const unsigned at = stride * (unsigned)(i + b);
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        l[t][b] = parts.number_through(at + my_log + 64u * t);
#pragma unroll
        for(int j = 0; j < kOwn; ++j) z[b][t][j] = parts.piece_through(at + mine + 1024u * (t * kDims + j));
      }
    }
#pragma unroll
    for(int b = 0; b < kBatch; ++b) {
      if(i + b >= x.w.parts) break;
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const float weight = weight_of(l[t][b], top[t]);
        weight_sum[t] += weight;
#pragma unroll
        for(int j = 0; j < kOwn; ++j)
#pragma unroll
          for(int e = 0; e < 4; ++e) r[t][j][e] = __builtin_fmaf(weight, z[b][t][j][e], r[t][j][e]);
      }
    }
  }
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    if(__builtin_expect(none_of(r[t]), 0)) {
#pragma unroll
      for(int j = 0; j < kOwn; ++j) r[t][j] = cache_f4{0, 0, 0, 0};
#pragma unroll 1
      for(int i = 0; i < x.w.parts; ++i) {
        const unsigned at = stride * (unsigned)i;
        const float weight = weight_of(parts.number_through(at + my_log + 64u * t), top[t]);
#pragma unroll
        for(int j = 0; j < kOwn; ++j) {
          const cache_f4 z = parts.piece_through(at + mine + 1024u * (t * kDims + j));
#pragma unroll
          for(int e = 0; e < 4; ++e) r[t][j][e] = add_odd(r[t][j][e], weight, z[e]);
        }
      }
    }
    write(t, weight_sum[t] == 0.0f ? 1.0f : 1.0f / weight_sum[t]);
  }
}

}  // namespace marian_hip
