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
// leaves: 16 and 22 bits.  Their sum is of the float32 ones.  They are scaled by a power of two: bfloat16 and float32 2^-24, so that sums over 2^20 positions of values next to the largest stay
// in range; float16 2^11, so that weights down to 2^-25 of the largest keep their bits.
#pragma once

#include <type_traits>

#include "../../include/marian_hip_ops.h"
#include "abi_common.h"
#include "cache_attention_kernel.h"
#include "pages_attention.h"

namespace marian_hip {

typedef __bf16 pages_b8 __attribute__((ext_vector_type(8)));

template <typename T, int DP>
struct Pages {
  static constexpr int kWidth = sizeof(T);
  static constexpr int kKeyPieces = DP * kWidth / 64;              // pieces of 16 bytes of a key to a lane
  static constexpr int kDims = DP / 16;                            // of a value's row to a lane ...
  static constexpr int kTogether = kDims < 16 / kWidth ? kDims : 16 / kWidth;   // ... that lie side by side
  static constexpr int kValuePieces = kDims / kTogether;
  static constexpr int kWords = kTogether * kWidth / 4;            // of a piece of values
  static constexpr int kUp = std::is_same<T, _Float16>::value ? 11 : -24;   // exponent that weights are held with
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

// The results of waves that share rows, joined and written.  Lane (c, g) holds of row c of each sixteen the values
// (16 (j / kTogether) + 4 g + e) kTogether + j % kTogether as o[t][j][e], unnormalized, the carried maximum and its part of the sum.
template <typename T, int DP, int QT, int WAVES>
__device__ __forceinline__ void pages_finish(const PagesAttentionArgs& a, const CacheTile& x, const cache_f4 (&o)[QT][DP / 16], const float (&top)[QT],
                                             float (&sum)[QT], int wave, CacheJoin<DP, QT, WAVES>& sh) {
  using P = Pages<T, DP>;
  constexpr int kTogether = P::kTogether, kHalf = CacheJoin<DP, QT, WAVES>::kHalf, kPieces = kHalf / (16 * kTogether);
  constexpr float kUnit = P::kUp < 0 ? (float)(1 << -P::kUp * (P::kUp < 0)) : 1.0f / (1 << P::kUp * (P::kUp > 0));   // 2^-kUp
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    sum[t] = over_lanes_sum(sum[t]) * kUnit;
    if(WAVES > 1 && g == 0) {
      sh.row_max[wave][16 * t + c] = top[t];
      sh.row_sum[wave][16 * t + c] = sum[t];
    }
  }
  const CacheOut<T, DP, 16 * QT> out(a, x);
  if constexpr(WAVES == 1) {
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float factor = sum[t] == 0.0f ? 0.0f : 1.0f / sum[t] * kUnit;
#pragma unroll
      for(int i = 0; i < P::kValuePieces; ++i)
#pragma unroll
        for(int e = 0; e < 4; ++e) {
          float y[kTogether];
#pragma unroll
          for(int j = 0; j < kTogether; ++j) y[j] = o[t][i * kTogether + j][e] * factor;
          out.emit(16 * t + c, (16 * i + 4 * g + e) * kTogether, y);
        }
      if(g == 0) out.emit_log(16 * t + c, top[t], sum[t]);
    }
  } else {
    // A row's weights of N positions add up to 2^kMaximumSlack N at the most, and their values to that many times the largest, which may be next
    // to the largest float32: they are summed over a power of two above it, twice as large for the roundings.  (It changes no bit of a result.)
    const int up = 5 + 32 - __builtin_clz((unsigned)max(x.end - x.w.from, 1));
    const float over = __builtin_bit_cast(float, (unsigned)(127 - up) << 23) * kUnit, back = __builtin_bit_cast(float, (unsigned)(127 + up) << 23);
    static_assert(kMaximumSlack <= 4.0f, "up counts it");
    __syncthreads();
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      float m = sh.row_max[0][16 * t + c];
#pragma unroll
      for(int i = 1; i < WAVES; ++i) m = fmaxf(m, sh.row_max[i][16 * t + c]);
      const float mine = top[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f(top[t] - m) * over;
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
          const float per = total == 0.0f ? 0.0f : 1.0f / total * back;
#pragma unroll
          for(int j = 0; j < kEach; ++j) {
            y[j] = sh.joined[0][r][d + j];
#pragma unroll
            for(int i = 1; i < WAVES; ++i) y[j] += sh.joined[i][r][d + j];
            y[j] *= per;
          }
          out.emit(16 * t + r, h * kHalf + d, y);
          if(h == 0 && (tid & 15) == 0) out.emit_log(16 * t + r, top_r, total);
        }
      }
    }
  }
  if(!out.whole) cache_join_parts<T, DP, 16 * QT, WAVES>(a, x, out, sh.parts);
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
  if(!cache_tile<T, DP, 16 * QT, WAVES>(a, tid, x)) return;
  const int end = x.end, row_bytes = (WHOLE ? DP : a.dk) * kWidth;
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
        if(wave == t % WAVES) q_held[t][i][lane] = z;
      } else {
        q[t][i] = z;
      }
    }
  }
  if constexpr(kQueriesInLds) __syncthreads();

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
    fetch_keys(key, k_next, at + kTurn);
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
    float p[QT][8];
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float from = (top[t] == kNone ? 0.0f : -top[t]) + P::kUp;   // (nothing seen so far: minus infinity stays that)
#pragma unroll
      for(int e = 0; e < 8; ++e) {
        p[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / 4][e % 4], a.scale_log2, from));
        sum[t] += p[t][e];
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
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int e = 0; e < 4; ++e) {
          const float lo = settled(p[t][2 * e]), hi = settled(p[t][2 * e + 1]);
          const unsigned w = pack2<T>(lo, hi);
          weights[t][0][e] = w;
          weights[t][1][e] = pack2<T>(lo - pages_half<T>(w & 0xffff), hi - pages_half<T>(w >> 16));
        }
#pragma unroll
      for(int j = 0; j < kDims; ++j) {
        constexpr unsigned low = 0x05040100, high_half = 0x07060302;
        cache_u4 d;
#pragma unroll
        for(int e = 0; e < 4; ++e)
          d[e] = __builtin_amdgcn_perm(value.word[2 * e + 1][j / kTogether][j % kTogether / 2], value.word[2 * e][j / kTogether][j % kTogether / 2],
                                       j % 2 ? high_half : low);
#pragma unroll
        for(int t = 0; t < QT; ++t)
#pragma unroll
          for(int m = 1; m >= 0; --m) o[t][j] = pages_product<T>(d, weights[t][m], o[t][j]);
      }
    }
    fetch_values(value, v_next, at + kTurn, there);
    k_next = look_keys(at + 2 * kTurn);
    v_next = look_values(at + 2 * kTurn);
  }
  // What was left out goes to the rows that see it: of any weight an infinity is one, and a NaN is one.
  if(left_out) {
#pragma unroll 1
    for(int at = begin; at < end; at += kTurn)
#pragma unroll 1
      for(int k = max(at, x.open); k < min(at + 32, end); ++k) {
        const PagesPlace y = pages_look(a, table, (unsigned)k >> 3);
        if((unsigned)y.id >= (unsigned)a.pages) continue;
        const T* const v = reinterpret_cast<const T*>(v_head + y.id * a.page_bytes + (long long)(8 * y.eight + (k & 7)) * row_bytes);
#pragma unroll
        for(int j = 0; j < kDims; ++j)
#pragma unroll
          for(int e = 0; e < 4; ++e) {
            const int d = (16 * (j / kTogether) + 4 * g + e) * kTogether + j % kTogether;
            const float z = to_float(v[d < a.dk ? d : 0]);
#pragma unroll
            for(int t = 0; t < QT; ++t)
              if(k < sight[t].limit && d < a.dk && !(__builtin_fabsf(z) < __builtin_huge_valf())) o[t][j][e] += z;
          }
      }
  }
  pages_finish<T, DP, QT, WAVES>(a, x, o, top, sum, wave, sh);
}

}  // namespace marian_hip
