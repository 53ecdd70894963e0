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
// instructions.  (The card copies 5.1 TB/s and multiplies large float16 matrices at 1.3 PFLOP/s.)
//
// Three forms, all with S^T = K Q^T or its transpose and O^T = V^T P^T on 16x16x32 float16 products, a row's maximum, sum and
// values in float32 registers, and the next positions' loads under way during the products of the last:
//   cache_attention_kernel: 9 to 32 rows an entry, rows of more than 128 values, and fewer rows over short contexts.  A wave takes 32 positions at
//   a time and 16 * QT rows, all in registers.
//     S^T: lane (c = lane % 16, g = lane / 16) loads sixteen codes at a time of key c - whole 64-byte pieces of a row between four lanes
//     - and uses them as two operands; which codes a step of the product takes is the same for Q, so no code moves between lanes.
//     The result has row c's scores of keys 4 g .. 4 g + 3, for two blocks of 16 keys.
//     O^T: those eight weights of a lane are its operand as they are, if V's operand has the keys in that order: lane (c, g) loads DP / 16
//     codes at c * DP / 16 of each of these eight keys - a row of keys between sixteen lanes - and picks a dimension's eight
//     codes out of its registers, two at a time, while they become float16.
//     So neither keys, values nor weights go through LDS; only the scales do.
//     16 sequences, 4 drafted tokens, 32 heads on 8, up to 4000 positions of 128 values: 26.4 us, 3.5 TB/s; up to 32000 149 us, 5.1 TB/s.
//     Memory bounds the long ones; a part of the short ones is four turns of a workgroup, and its start and the join show.
//   cache_attention_few_kernel: up to 8 rows over long contexts, cache_attention_many_kernel: more than 32 rows; see there.
// Codes are exact in float16.  Q is scaled row by row by a power of two up to 2^14 .. 2^15 and enters in one float16
// (float16 and bfloat16: exact but for values 2^-29 below the row's largest) or two (float32: 22 bits).  A weight is
// p_rj times the value's scale over a running scale S_r (as the maximum runs; of magnitudes, since a scale may be below zero), times
// 2^9: in two float16, rounded to nearest, of what is at most 2^15 and, with normal numbers, down to 2^-14: 22 bits of weights up to
// 2^-24 below the largest.  Their sum is of the weights in float32.  The second float16 costs another product with the values: next to nothing up
// to 32 rows, where memory is waited for (bfloat16; 16 sequences, 32 heads on 8, up to 32768 positions 139.1 us without it, 138.2 with it; 4 drafted
// tokens of them, up to 32000 147.8 and 149.0; 128 sequences' 4 tokens, 32 heads on 16, up to 512 of 64 values 26.6 and 27.8; at the most, in a
// sequence's own few parts, one head of 100000 24.5 and 26.4).  With more rows it does cost: bfloat16 leaves it out there and has 11 bits - 8 trees
// of 64 tokens 82 us, 100 with it, prompts of 1024 tokens 326 and 419 -, for its results are rounded to 8 bits, an error of 1.654e-3 of their
// norm, which such weights make 1.667e-3.  float16's are rounded to 11 bits themselves, 2.08e-4, and would be off by 2.91e-4.
// The sums are scaled down only where a maximum or scale outgrows the carried one by 2^4 (4): most turns skip it.
// Positions that a row does not see, and rows past the end that pad a block, weigh a selected zero; loads go through buffers that end where
// the part does, and give zeros behind it.
#pragma once

#include <type_traits>

#include "cache_attention.h"
#include "cache_codes.h"

namespace marian_hip {

constexpr float kWeightUnit = 512.0f;     // 2^9, see above
constexpr float kMaximumSlack = 4.0f;     // weights may be 2^4 above the carried maximum's ...
constexpr float kScaleSlack = 4.0f;       // ... and scales four times the carried one before the sums are scaled down

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

// Blocks of a part of a sequence of `blocks`, which has up to MOST parts.
template <unsigned MOST>
__device__ __forceinline__ unsigned cache_part_size(unsigned blocks, unsigned each) {
  return max(blocks <= kCacheWhole ? max(each, kCacheWhole) : each, (blocks + MOST - 1) / MOST);
}

// Finds part `item`; false where there are fewer.  All waves do the same, lanes being sequences.
template <unsigned MOST>
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
    for(int i = 0; i < kHeld; ++i) held[i] = 64 * i < a.S ? blocks_of(64 * i + lane) : 0;
#pragma unroll
    for(int i = 0; i < kHeld; ++i) total += held[i];
    for(int base = 64 * kHeld; base < a.S; base += 64) total += blocks_of(base + lane);
    total = (unsigned)__builtin_amdgcn_readlane((int)lanes_sum(total), 63);
    each = max((unsigned)a.least, (total + a.target - 1) / a.target);
    // parts in the lower bits, those of sequences with several in the upper twelve (less than 2 * target)
    unsigned before = 0;
    bool found = false;
    auto look = [&](int base, unsigned mine) __attribute__((always_inline)) {
      const unsigned size = cache_part_size<MOST>(mine, each), parts = base + lane < a.S ? max(1u, (mine + size - 1) / size) : 0;
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
  w.s = __builtin_amdgcn_readfirstlane(w.s);
  w.len = __builtin_amdgcn_readfirstlane(clamp_int(a.lens[w.s], 0, a.cap));
  w.count = a.counts ? __builtin_amdgcn_readfirstlane(clamp_int(a.counts[w.s], 0, a.n)) : a.n;
  w.used = w.count > 0 ? min(w.len + w.count, a.cap) : 0;
  const unsigned mine = (unsigned)(w.used + kCacheBlock - 1) / kCacheBlock;
  const int size = (int)cache_part_size<MOST>(mine, each) * kCacheBlock;
  w.from = a.target > 1 ? w.part * size : 0;
  w.to = a.target > 1 ? min(w.from + size, w.used) : w.used;
  return true;
}

// A product as a number of its own.  Where it becomes a float16 and the rest of it a second one, both have to start from the
// same float32: the compiler would turn the product into float16 in one instruction, with one rounding, for what it subtracts, and in two for
// what it keeps, and the two float16 differ where the first rounding comes to lie half way (a weight in 16000, by 2^-11 of it).
__device__ __forceinline__ float settled(float z) {
  asm("" : "+v"(z));
  return z;
}

template <typename T, CacheFormat F, int DP>
struct CacheAttention {
  static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;   // float16 to a query value ...
  static constexpr int kWeightTerms = 2;                  // ... and to a weight, of up to 32 rows ...
  static constexpr int kManyWeightTerms = __is_same(T, bf16_t) ? 1 : 2;   // ... and of more
  static constexpr int kSteps = DP / 32;                  // of a product over a row
  static constexpr int kPieces = DP / 64;                 // sixteen codes of a key to a lane
  static constexpr int kDims = DP / 16;                   // of a value's row to a lane
  static constexpr int kWords = kDims / 4;

  // 32 positions as they are loaded.
  struct Keys {
    cache_u4 code[2][kPieces];
  };
  struct Values {
    unsigned code[8][kWords];
  };
};

// The codes, or the scales, of an entry's positions up to an end, as a buffer: what lies behind it reads as zeros, so that loads need neither
// branches nor bounds of their own.  (A branch around loads whose registers live on makes the compiler wait for them behind it.)
// All offsets go through the lane's, against which the buffer's size is held; a load lies in one row, whole or not at all inside.
struct CacheBuffer {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ CacheBuffer(const void* p, unsigned bytes)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000)) {}   // (32-bit data, no swizzle)
  __device__ __forceinline__ float number(int i) const {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, (unsigned)i * 4u, 0, 0));
  }
  __device__ __forceinline__ cache_u4 piece(unsigned at) const { return __builtin_bit_cast(cache_u4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0)); }
  // Past the caches of an XCD, as loads and stores of agent scope go.
  static constexpr int kThrough = 16;   // sc1
  __device__ __forceinline__ float number_through(unsigned at) const {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, kThrough));
  }
  __device__ __forceinline__ cache_f4 piece_through(unsigned at) const {
    return __builtin_bit_cast(cache_f4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, kThrough));
  }
  __device__ __forceinline__ void store_through(cache_f4 y, unsigned at) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(cache_u4, y), rsrc, at, 0, kThrough);
  }
  __device__ __forceinline__ void store_through(float y, unsigned at) const {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, y), rsrc, at, 0, kThrough);
  }
  template <int WORDS>
  __device__ __forceinline__ void words(unsigned (&to)[WORDS], unsigned at) const {
    if constexpr(WORDS == 1) {
      to[0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, 0);
    } else if constexpr(WORDS == 2) {
      const cache_u2 x = __builtin_bit_cast(cache_u2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, 0));
      to[0] = x[0];
      to[1] = x[1];
    } else {
      const cache_u4 x = piece(at);
#pragma unroll
      for(int w = 0; w < 4; ++w) to[w] = x[w];
    }
  }
};

// Sixteen codes at a time of rows row, row + 16, ..: lane (c, g) those of row + c from 64 i + 16 g on.  Lanes past a row's end (dk < DP) take
// its start: the queries are zero there, and of values they are not stored.
template <int BLOCKS, int PIECES>
__device__ __forceinline__ void load_keys(cache_u4 (&to)[BLOCKS][PIECES], const CacheBuffer& k, int row, int dk, int lane) {
  const unsigned at = (unsigned)(row + (lane & 15)) * dk;
#pragma unroll
  for(int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for(int i = 0; i < PIECES; ++i) {
      const unsigned d = 64 * i + 16 * (lane >> 4);
      to[b][i] = k.piece(at + (unsigned)(16 * b) * dk + (d < (unsigned)dk ? d : 0));
    }
}

// Dimension B of word w of a lane's values, eight keys.
template <CacheFormat F, int B, int WORDS>
__device__ __forceinline__ cache_h8 value_operand_of(const unsigned (&v)[8][WORDS], int w) {
  const cache_h2 h[4] = {half2_of<F, B, B>(v[0][w], v[1][w]), half2_of<F, B, B>(v[2][w], v[3][w]), half2_of<F, B, B>(v[4][w], v[5][w]),
                         half2_of<F, B, B>(v[6][w], v[7][w])};
  return cache_h8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// Values of lanes that differ in one bit of their number, joined: bits 4 and 5 by an exchange of whole rows of sixteen lanes (in
// assembly, with the wait states around it: the compiler's builtin gives one of the two registers only).
template <typename Join>
__device__ __forceinline__ float over_bit4(float x, Join join) {
  float y = x;
  asm("s_nop 3\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 3" : "+v"(x), "+v"(y));
  return join(x, y);
}
template <typename Join>
__device__ __forceinline__ float over_bit5(float x, Join join) {
  float y = x;
  asm("s_nop 3\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 3" : "+v"(x), "+v"(y));
  return join(x, y);
}
// Over the sixteen lanes of a row, by rotations.
template <typename Join>
__device__ __forceinline__ float over_row(float x, Join join) {
  auto turned = [](float y, auto by) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, y), 0x120 + decltype(by)::value, 0xf, 0xf, false));
  };
  x = join(x, turned(x, std::integral_constant<int, 8>()));
  x = join(x, turned(x, std::integral_constant<int, 4>()));
  x = join(x, turned(x, std::integral_constant<int, 2>()));
  return join(x, turned(x, std::integral_constant<int, 1>()));
}
struct Larger {
  __device__ __forceinline__ float operator()(float x, float y) const { return fmaxf(x, y); }
};
struct Added {
  __device__ __forceinline__ float operator()(float x, float y) const { return x + y; }
};
struct LargerBits {   // (of magnitudes: NaN is above all)
  __device__ __forceinline__ float operator()(float x, float y) const {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y)));
  }
};
// The maximum, and the sum, over the four lanes of a query row.
__device__ __forceinline__ float over_lanes_max(float x) { return over_bit5(over_bit4(x, Larger()), Larger()); }
__device__ __forceinline__ float over_lanes_sum(float x) { return over_bit5(over_bit4(x, Added()), Added()); }
__device__ __forceinline__ float lane_value(float x, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane)); }

constexpr float kNone = -__builtin_huge_valf();

// What a workgroup works on: rows row0 .. of an entry (up to ROWS of them), and its part of the positions.
struct CacheTile {
  CachePart w;
  int head, tile, rows, row0;   // rows: of the sequence that are there
  int end, open;                // of what any row sees, of what all rows see
  const unsigned char *k, *v;   // of the entry
  const float *ks, *vs;
};

template <typename T>
__device__ __forceinline__ T* cache_row_out(const CacheAttentionArgs& a, const CacheTile& x, int r) {
  unsigned of_group;
  const unsigned token = a.by_group.of((unsigned)r, of_group);
  return static_cast<T*>(a.out) + x.w.s * a.o_s + (long long)(x.head * a.G + (int)of_group) * a.o_h + (long long)token * a.o_n;
}

// Finds a workgroup's tile and clears the rows of it that are not there; false where nothing is to be done.  PAGES: an entry's keys and values have no
// place of their own, and the last rows, which see the most positions, go first.
template <typename T, int DP, int ROWS, int WAVES, unsigned MOST = kCacheMostParts, bool PAGES = false>
__device__ __forceinline__ bool cache_tile(const CacheAttentionArgs& a, int tid, CacheTile& x) {
  constexpr int kDims = DP / 16;
  // Workgroups with the same positions follow each other on one XCD (a workgroup to each of the eight in turn).
  unsigned tile, head;
  const int entry = (int)a.by_tiles.of(blockIdx.x >> 3, tile) * 8 + (blockIdx.x & 7);
  if(entry >= a.items * a.Hk) return false;
  const int item = (int)a.by_heads.of((unsigned)entry, head);
  x.tile = PAGES ? a.row_tiles - 1 - (int)tile : (int)tile;
  x.head = (int)head;
  if(!cache_part<MOST>(a, item, tid & 63, x.w)) return false;
  x.rows = x.w.count * a.G;
  x.row0 = x.tile * ROWS;
  if(x.w.part == 0 && x.row0 + ROWS > x.rows) {
    const int d = (tid & 15) * kDims;
    for(int r = x.row0 + (tid >> 4); r < min(x.row0 + ROWS, a.n * a.G); r += 4 * WAVES) {
      const float zeros[kDims] = {};
      if(r >= x.rows && d < a.dk) store_row<kDims, T>(cache_row_out<T>(a, x, r) + d, zeros);
    }
  }
  if(x.row0 >= x.rows) return false;
  const int last_token = (int)a.by_group.of((unsigned)min(x.rows - 1, x.row0 + ROWS - 1));
  x.end = min(x.w.to, x.w.len + last_token + 1);
  x.open = min(x.end, x.w.len + (a.parents ? 0 : (int)a.by_group.of((unsigned)x.row0) + 1));
  if constexpr(!PAGES) {
    const long long first = ((long long)x.w.s * a.Hk + x.head) * a.cap;
    x.k = a.k + first * a.dk;
    x.v = a.v + first * a.dk;
    x.ks = a.ks + first;
    x.vs = a.vs + first;
  }
  return true;
}

// What a row sees: in a chain positions before limit, in a tree the settled ones and the drafted ones of bits sees, before end.
struct CacheSight {
  int limit;
  unsigned long long sees;
};
__device__ __forceinline__ CacheSight cache_sight(const CacheAttentionArgs& a, const CacheTile& x, int row, unsigned long long seen) {
  const int token = (int)a.by_group.of((unsigned)row);
  CacheSight y{min(x.end, x.w.len + token + 1), 0};
  if(a.parents) {
    const unsigned lo = __shfl((unsigned)seen, token, 64), hi = __shfl((unsigned)(seen >> 32), token, 64);
    y.sees = (unsigned long long)hi << 32 | lo;
  }
  return y;
}

// The lane's part of query row `row` as an operand, four lanes (16 apart) to a row; returns the factor of a score, to logarithms of base 2.
template <typename T, CacheFormat F, int DP>
__device__ __forceinline__ float cache_query(const CacheAttentionArgs& a, const CacheTile& x, int row, int g,
                                             cache_h8 (&q)[CacheAttention<T, F, DP>::kTerms][DP / 32]) {
  constexpr int kTerms = CacheAttention<T, F, DP>::kTerms, kSteps = DP / 32;
  unsigned of_group;
  const unsigned token = a.by_group.of((unsigned)row, of_group);
  const T* p = static_cast<const T*>(a.q) + x.w.s * a.q_s + (long long)(x.head * a.G + (int)of_group) * a.q_h + (long long)token * a.q_n;
  float y[kSteps][8];
#pragma unroll
  for(int i = 0; i < kSteps; ++i) {   // (past the row's end its start is read, and dropped: a branch around each load would wait for it)
    const int d = 64 * (i / 2) + 16 * g + 8 * (i % 2);
    load_row<8>(p + (d < a.dk ? d : 0), y[i]);
  }
  unsigned most = 0;   // bits of the row's largest magnitude (NaN above all)
#pragma unroll
  for(int i = 0; i < kSteps; ++i) {
    const int d = 64 * (i / 2) + 16 * g + 8 * (i % 2);
#pragma unroll
    for(int e = 0; e < 8; ++e) {
      y[i][e] = d < a.dk ? y[i][e] : 0.0f;
      most = max(most, __builtin_bit_cast(unsigned, y[i][e]) & 0x7fffffffu);
    }
  }
  most = __builtin_bit_cast(unsigned, over_bit5(over_bit4(__builtin_bit_cast(float, most), LargerBits()), LargerBits()));
  const int up = clamp_int(127 + 14 + 127 - (int)(most >> 23), 2, 252);   // exponent that brings it to 2^14
  const float factor = __builtin_bit_cast(float, (unsigned)up << 23), back = __builtin_bit_cast(float, (unsigned)(254 - up) << 23);
#pragma unroll
  for(int i = 0; i < kSteps; ++i) {
#pragma unroll
    for(int e = 0; e < 8; ++e) {
      const float z = y[i][e] * factor;   // (exact)
      q[0][i][e] = (_Float16)z;
      if constexpr(kTerms == 2) q[1][i][e] = (_Float16)(z - (float)q[0][i][e]);
    }
  }
  return most >= 0x7f800000u ? __builtin_nanf("") : fmaxf(back * (a.scale_log2 / kCodeUnit<F>), 0x1p-126f);   // (never zero)
}

// Where a workgroup's rows go: to the output, or where a sequence has several parts to the workspace.
template <typename T, int DP, int ROWS>
struct CacheOut {
  static constexpr int kTileFloats = ROWS * DP + (ROWS + 3) / 4 * 4;   // (whole pieces of 16 bytes)
  const CacheAttentionArgs& a;
  const CacheTile& x;
  const bool whole;
  const long long place, stride;   // of the tile's first part, of a part to the next, in tiles
  float* const part;
  __device__ __forceinline__ CacheOut(const CacheAttentionArgs& a_, const CacheTile& x_)
      : a(a_), x(x_), whole(x.w.parts == 1), place(((long long)x.w.slot * a.Hk + x.head) * a.row_tiles + x.tile),
        stride((long long)a.Hk * a.row_tiles), part(a.part + (place + x.w.part * stride) * kTileFloats) {}
  // Values d .. of row r of the tile.
  template <int COUNT>
  __device__ __forceinline__ void emit(int r, int d, const float (&y)[COUNT]) const {
    if(x.row0 + r >= x.rows || d >= a.dk) return;
    if(whole) {
      store_row<COUNT, T>(cache_row_out<T>(a, x, x.row0 + r) + d, y);
    } else {
      unsigned long long* to = reinterpret_cast<unsigned long long*>(part + r * DP + d);
#pragma unroll
      for(int j = 0; j < COUNT; j += 2)
        __hip_atomic_store(to + j / 2, (unsigned long long)__builtin_bit_cast(unsigned, y[j + 1]) << 32 | __builtin_bit_cast(unsigned, y[j]),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // The logarithm of the sum of row r's weights, 2^m times total.
  __device__ __forceinline__ void emit_log(int r, float m, float total) const {
    if(!whole && x.row0 + r < x.rows)
      __hip_atomic_store(part + ROWS * DP + r, total == 0.0f ? kNone : m + __builtin_amdgcn_logf(total), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
};

// Counts a workgroup of `parts` that share a counter in, and whether it is the last.  What it has stored for the others is of agent scope, past
// the caches of an XCD: every wave's stores are acknowledged before the count goes up, so whoever reads the last count finds them
// all, with loads of that scope.
__device__ __forceinline__ bool cache_arrived_last(unsigned* counter, int parts, int& is_last) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if(threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(parts - 1);
    if(last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // (for the next call)
    is_last = last;
  }
  __syncthreads();
  return is_last;
}

// What sixteens of threads that share a row's parts join them through.
template <int DP, int WAVES>
struct CacheParts {
  float rest[4 * WAVES][DP];
  float top[4 * WAVES], sum[4 * WAVES];
  int is_last;
};

// A part's weight is at most 1, times this: the sum of their weighted values is no larger than the largest of them, which may be next to the
// largest float32.  (A power of two, which the reciprocal of the weights' sum takes away again: no bit of a result depends on it.)
constexpr float kPartUnit = 1.0f / 64;
static_assert(kPartUnit * kCacheMostParts <= 1.0f, "the parts' weights add up to one at the most");

// A weighted value, and a sum of them, in which infinities and NaN count whatever their weight, zero included.
__device__ __forceinline__ bool is_odd(float z) { return !(__builtin_fabsf(z) < __builtin_huge_valf()); }
__device__ __forceinline__ float times_odd(float z, float weight) { return weight == 0.0f && is_odd(z) ? z : z * weight; }
__device__ __forceinline__ float add_odd(float y, float weight, float z) {
  return weight == 0.0f && is_odd(z) ? y + z : __builtin_fmaf(weight, z, y);
}

// The parts of a sequence: the workgroup that arrives last joins them, in their order.  ODD: an infinity or NaN among a part's results is the
// result, whatever the part weighs; sums that are none are made once more for it.
template <typename T, int DP, int ROWS, int WAVES, bool ODD = false>
__device__ __forceinline__ void cache_join_parts(const CacheAttentionArgs& a, const CacheTile& x, const CacheOut<T, DP, ROWS>& out,
                                                 CacheParts<DP, WAVES>& sh) {
  using Out = CacheOut<T, DP, ROWS>;
  constexpr int kDims = DP / 16;
  const int tid = threadIdx.x;
  if(!cache_arrived_last(a.counters + out.place, x.w.parts, sh.is_last)) return;
  // Sixteen threads to a row; where there are fewer rows than sixteens, several of them share a row's parts.  A batch of parts is
  // asked for at a time, through a buffer that ends behind the last one: the loads come from the memory side, about a microsecond away, and
  // a branch around each would wait for it (2 sequences, 2 heads, 16 rows of 256 values, up to 56618 positions
  // in 48 parts: 51 us, 75 with branches).
  const unsigned stride = (unsigned)(out.stride * Out::kTileFloats), all_parts = x.w.parts;
  const CacheBuffer from(a.part + out.place * Out::kTileFloats, 4u * stride * all_parts);
  constexpr int kGroups = 4 * WAVES, kBatch = 8;
  const int here = min(ROWS, x.rows - x.row0), group = tid >> 4, d_mine = (tid & 15) * kDims;
  int share = 1;
  while(share * here * 2 <= kGroups) share *= 2;
#pragma unroll 1
  for(int r = group / share; r < here; r += kGroups / share) {   // (one turn where parts are shared)
    const unsigned mine = 4u * (r * DP + (d_mine < a.dk ? d_mine : 0)), my_log = 4u * (ROWS * DP + r);
    float m = kNone, total = 0.0f, y[kDims] = {};
#pragma unroll 1
    for(int i = group % share; i < x.w.parts; i += kBatch * share) {
      float l[kBatch];
      cache_f4 z[kBatch][kDims / 4];
#pragma unroll
      for(int b = 0; b < kBatch; ++b) {
        const unsigned at = 4u * stride * (unsigned)(i + b * share);
        l[b] = from.number_through(at + my_log);
#pragma unroll
        for(int j = 0; j < kDims / 4; ++j) z[b][j] = from.piece_through(at + mine + 16u * j);
      }
#pragma unroll
      for(int b = 0; b < kBatch; ++b) l[b] = i + b * share < x.w.parts ? l[b] : kNone;
      float next = m;
#pragma unroll
      for(int b = 0; b < kBatch; ++b) next = fmaxf(next, l[b]);
      const float down = m == kNone ? 0.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      total *= down;
#pragma unroll
      for(int j = 0; j < kDims; ++j) y[j] *= down;
#pragma unroll
      for(int b = 0; b < kBatch; ++b) {
        const float weight = l[b] == kNone ? 0.0f : __builtin_amdgcn_exp2f(l[b] - m) * kPartUnit;
        total += weight;
#pragma unroll
        for(int j = 0; j < kDims; ++j) y[j] = __builtin_fmaf(weight, z[b][j / 4][j % 4], y[j]);
      }
    }
    float none = 0.0f;
    if constexpr(ODD) {
#pragma unroll
      for(int j = 0; j < kDims; ++j) none += y[j] * 0.0f;
    }
    if(ODD && __builtin_expect(!(none == 0.0f), 0)) {
      float again[kDims] = {};
#pragma unroll 1
      for(int i = group % share; i < x.w.parts; i += share) {
        const unsigned at = 4u * stride * (unsigned)i;
        const float log = from.number_through(at + my_log), weight = log == kNone ? 0.0f : __builtin_amdgcn_exp2f(log - m) * kPartUnit;
#pragma unroll
        for(int j = 0; j < kDims / 4; ++j) {
          const cache_f4 z = from.piece_through(at + mine + 16u * j);
#pragma unroll
          for(int e = 0; e < 4; ++e) again[4 * j + e] = add_odd(again[4 * j + e], weight, z[e]);
        }
      }
#pragma unroll
      for(int j = 0; j < kDims; ++j) y[j] = is_odd(y[j]) ? again[j] : y[j];
    }
    if(share > 1) {   // (r is the only row of all threads: sixteens beyond the rows have left)
      float* const rest = &sh.rest[group][(tid & 15) * kDims];
#pragma unroll
      for(int j = 0; j < kDims; ++j) rest[j] = y[j];
      if((tid & 15) == 0) {
        sh.top[group] = m;
        sh.sum[group] = total;
      }
    }
    if(share == 1 && d_mine < a.dk) {
      const float per = total == 0.0f ? ODD : 1.0f / total;   // (without weights: zeros, infinities and NaN)
#pragma unroll
      for(int j = 0; j < kDims; ++j) y[j] *= per;
      store_row<kDims, T>(cache_row_out<T>(a, x, x.row0 + r) + d_mine, y);
    }
  }
  if(share == 1) return;
  __syncthreads();
  const int r = group / share;
  if(group % share != 0 || r >= here || d_mine >= a.dk) return;
  float m = kNone, total = 0.0f, y[kDims] = {};
  for(int i = 0; i < share; ++i) m = fmaxf(m, sh.top[group + i]);
  for(int i = 0; i < share; ++i) {
    const float from = sh.top[group + i], weight = from == kNone ? 1.0f : __builtin_amdgcn_exp2f(from - m);   // (of none: 0, or NaN)
    const float* const rest = &sh.rest[group + i][(tid & 15) * kDims];
    total += sh.sum[group + i] * weight;
#pragma unroll
    for(int j = 0; j < kDims; ++j) y[j] = __builtin_fmaf(rest[j], weight, y[j]);
  }
  float none = 0.0f;
  if constexpr(ODD) {
#pragma unroll
    for(int j = 0; j < kDims; ++j) none += y[j] * 0.0f;
  }
  if(ODD && __builtin_expect(!(none == 0.0f), 0)) {
    float again[kDims] = {};
#pragma unroll 1
    for(int i = 0; i < share; ++i) {
      const float from = sh.top[group + i], weight = from == kNone ? 0.0f : __builtin_amdgcn_exp2f(from - m);
#pragma unroll
      for(int j = 0; j < kDims; ++j) again[j] = add_odd(again[j], weight, sh.rest[group + i][(tid & 15) * kDims + j]);
    }
#pragma unroll
    for(int j = 0; j < kDims; ++j) y[j] = is_odd(y[j]) ? again[j] : y[j];
  }
  const float per = total == 0.0f ? ODD : 1.0f / total;
#pragma unroll
  for(int j = 0; j < kDims; ++j) y[j] *= per;
  store_row<kDims, T>(cache_row_out<T>(a, x, x.row0 + r) + d_mine, y);
}

// What the waves of a workgroup join their results through.  (Rows are written in pieces of 16 bytes.)
template <int DP, int QT, int WAVES>
struct alignas(16) CacheJoin {
  static constexpr int kHalf = DP < 128 ? DP : 128;   // dimensions that are joined at a time
  static_assert((kHalf + 4) % 4 == 0, "whole pieces to a row");
  union {
    float joined[WAVES][16][kHalf + 4];
    CacheParts<DP, WAVES> parts;
  };
  float row_max[WAVES][16 * QT], row_sum[WAVES][16 * QT];
};

// The results of waves that share rows, joined and written.  Lane (c, g) holds values 4 * kDims * g .. of row c of each sixteen,
// unnormalized, the carried maximum and scale and its part of the sum.
template <typename T, CacheFormat F, int DP, int QT, int WAVES>
__device__ __forceinline__ void cache_finish(const CacheAttentionArgs& a, const CacheTile& x, const cache_f4 (&o)[QT][DP / 16], const float (&top)[QT],
                                             float (&sum)[QT], const float (&unit)[QT], CacheJoin<DP, QT, WAVES>& sh) {
  constexpr int kDims = DP / 16, kHalf = CacheJoin<DP, QT, WAVES>::kHalf;
  const int tid = threadIdx.x, lane = tid & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    sum[t] = over_lanes_sum(sum[t]);
    if(WAVES > 1 && g == 0) {
      sh.row_max[wave][16 * t + c] = top[t];
      sh.row_sum[wave][16 * t + c] = sum[t];
    }
  }
  const CacheOut<T, DP, 16 * QT> out(a, x);
  constexpr float kUnit = 1.0f / (kWeightUnit * kCodeUnit<F>);
  if constexpr(WAVES == 1) {
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float factor = (sum[t] == 0.0f ? 0.0f : 1.0f / sum[t]) * (unit[t] * kUnit);
#pragma unroll
      for(int e = 0; e < 4; ++e) {
        float y[kDims];
#pragma unroll
        for(int j = 0; j < kDims; ++j) y[j] = o[t][j][e] * factor;
        out.emit(16 * t + c, kDims * (4 * g + e), y);
      }
      if(g == 0) out.emit_log(16 * t + c, top[t], sum[t]);
    }
  } else {
    // A row's weights of N positions add up to 2^kMaximumSlack N at the most, and their values to that many times the largest, which may be next
    // to the largest float32: they are summed over a power of two above it, twice as large for the roundings.  (It changes no bit of a result.)
    const int up = 5 + 32 - __builtin_clz((unsigned)max(x.end - x.w.from, 1));
    const float over = __builtin_bit_cast(float, (unsigned)(127 - up) << 23), back = __builtin_bit_cast(float, (unsigned)(127 + up) << 23);
    static_assert(kMaximumSlack <= 4.0f, "up counts it");
    __syncthreads();
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      float m = sh.row_max[0][16 * t + c];
#pragma unroll
      for(int i = 1; i < WAVES; ++i) m = fmaxf(m, sh.row_max[i][16 * t + c]);
      const float mine = top[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f(top[t] - m) * (unit[t] * kUnit) * over;
#pragma unroll
      for(int h = 0; h < DP / kHalf; ++h) {
        if(h || t) __syncthreads();
        if(DP == kHalf || (g >> 1) == h) {
#pragma unroll
          for(int e = 0; e < 4; ++e)
#pragma unroll
            for(int j = 0; j < kDims; j += 4)
              *reinterpret_cast<cache_f4*>(&sh.joined[wave][c][4 * kDims * g + kDims * e + j - h * kHalf]) =
                  cache_f4{o[t][j][e] * mine, o[t][j + 1][e] * mine, o[t][j + 2][e] * mine, o[t][j + 3][e] * mine};
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

// ---- sixteen rows and more to a wave
// Between two barriers of LDS there is nothing to wait for but memory; the loads of the next 32 positions are out while these are worked on.
// The workgroup's waves take turns of 32 positions of the same rows and join in LDS in the end, so a short context is one turn.
template <typename T, CacheFormat F, int DP, int QT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (DP == 64 ? 5 - QT : DP == 128 ? 4 - QT : 2)) void cache_attention_kernel(CacheAttentionArgs a) {
  using A = CacheAttention<T, F, DP>;
  constexpr int kTerms = A::kTerms, kWeightTerms = A::kWeightTerms, kSteps = A::kSteps, kDims = A::kDims;
  constexpr int kTurn = 32 * WAVES;   // positions that the waves take in one turn
  __shared__ struct {
    CacheJoin<DP, QT, WAVES> join;
    alignas(16) float scales[WAVES][64];
  } sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  CacheTile x;
  if(!cache_tile<T, DP, 16 * QT, WAVES>(a, tid, x)) return;
  const int end = x.end;
  const CacheBuffer k_codes(x.k, (unsigned)end * a.dk), v_codes(x.v, (unsigned)end * a.dk);
  // (a position's scales are loaded to one lane, and go through LDS to those that have its scores)
  const CacheBuffer k_scales(x.ks, 4u * end), v_scales(x.vs, 4u * end);
  float scale_k, scale_v;
  auto fetch_keys = [&](typename A::Keys& y, int at) __attribute__((always_inline)) {
    load_keys(y.code, k_codes, at, a.dk, lane);
    scale_k = k_scales.number(at + (lane & 31));
  };
  auto fetch_values = [&](typename A::Values& y, int at) __attribute__((always_inline)) {
    const unsigned d = (unsigned)(kDims * c) < (unsigned)a.dk ? kDims * c : 0, row = (unsigned)(at + 4 * g) * a.dk + d;
#pragma unroll
    for(int e = 0; e < 8; ++e) v_codes.words(y.code[e], row + (unsigned)(16 * (e / 4) + e % 4) * a.dk);
    scale_v = v_scales.number(at + (lane & 31));
  };
  // (the first positions are asked for ahead of the queries, the next keys as soon as the last ones are used up, and so the values)
  const int begin = x.w.from + 32 * wave;
  typename A::Keys key;
  typename A::Values value;
  fetch_keys(key, begin);
  fetch_values(value, begin);
  unsigned long long seen = 0;
  if(a.parents) seen = lineage(a.parents + (long long)x.w.s * a.n, a.n, lane);
  cache_h8 q[QT][kTerms][kSteps];
  float row_scale[QT];
  CacheSight sight[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const int row = min(x.row0 + 16 * t + c, x.rows - 1);
    sight[t] = cache_sight(a, x, row, seen);
    row_scale[t] = cache_query<T, F, DP>(a, x, row, g, q[t]);
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

  for(int at = begin; at < end; at += kTurn) {
    if(lane < 32) {
      sh.scales[wave][lane] = scale_k;
      sh.scales[wave][32 + lane] = scale_v;
    }
    __builtin_amdgcn_wave_barrier();   // (a wave's accesses to LDS are done in their order)
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
    cache_f4 ks[2], vs[2];
#pragma unroll
    for(int b = 0; b < 2; ++b) {
      ks[b] = *reinterpret_cast<const cache_f4*>(&sh.scales[wave][16 * b + 4 * g]);
      vs[b] = *reinterpret_cast<const cache_f4*>(&sh.scales[wave][32 + 16 * b + 4 * g]);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for(int t = 0; t < QT; ++t)
#pragma unroll
      for(int e = 0; e < 8; ++e) s[t][e / 4][e % 4] *= ks[e / 4][e % 4];
    fetch_keys(key, at + kTurn);
    // Positions that a row does not see score minus infinity (a weight of zero) and have a scale of zero.
    const bool masked = at + 32 > x.open;
    unsigned seen_here[QT];   // bit e: key e
    float widest = 0.0f;
#pragma unroll
    for(int t = 0; t < QT; ++t) seen_here[t] = 0xff;
    if(masked) {
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        unsigned bits = 0;
#pragma unroll
        for(int b = 0; b < 2; ++b) {
          const int from = at + 16 * b + 4 * g;
          unsigned four = (1u << clamp_int((a.parents ? end : sight[t].limit) - from, 0, 4)) - 1;
          if(a.parents) {   // settled positions, then the drafted ones from bit 0 on
            const int j = from - x.w.len, settled = clamp_int(-j, 0, 4);
            four &= j < 0 ? ((unsigned)sight[t].sees << settled | ((1u << settled) - 1)) : (unsigned)(sight[t].sees >> min(j, 63));
          }
          bits |= four << (4 * b);
        }
        seen_here[t] = bits;
#pragma unroll
        for(int e = 0; e < 8; ++e) s[t][e / 4][e % 4] = bits >> e & 1 ? s[t][e / 4][e % 4] : kNone;
      }
    } else {
#pragma unroll
      for(int e = 0; e < 8; ++e) widest = fmaxf(widest, __builtin_fabsf(vs[e / 4][e % 4]));
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
        for(int e = 0; e < 8; ++e) wide[t] = fmaxf(wide[t], seen_here[t] >> e & 1 ? __builtin_fabsf(vs[e / 4][e % 4]) : 0.0f);
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
      for(int e = 0; e < 8; ++e) r[t][e] = vs[e / 4][e % 4] * per;
    }
    if(masked) {
#pragma unroll
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int e = 0; e < 8; ++e) r[t][e] = seen_here[t] >> e & 1 ? r[t][e] : 0.0f;
    }
    cache_h8 p[QT][kWeightTerms];
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float from = top[t] == kNone ? 0.0f : -top[t];   // (nothing seen so far: minus infinity stays that)
#pragma unroll
      for(int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / 4][e % 4], row_scale[t], from)), z = settled(y * r[t][e]);
        sum[t] += y;
        p[t][0][e] = (_Float16)z;
        p[t][1][e] = (_Float16)(z - (float)p[t][0][e]);
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
      const cache_h8 d[4] = {value_operand_of<F, 0>(vh, i), value_operand_of<F, 1>(vh, i), value_operand_of<F, 2>(vh, i),
                             value_operand_of<F, 3>(vh, i)};
#pragma unroll
      for(int j = 0; j < 4; ++j)
#pragma unroll
        for(int t = 0; t < QT; ++t)
#pragma unroll
          for(int m = kWeightTerms - 1; m >= 0; --m)
            o[t][4 * i + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(d[j], p[t][m], o[t][4 * i + j], 0, 0, 0);
    }
    fetch_values(value, at + kTurn);
  }

  cache_finish<T, F, DP, QT, WAVES>(a, x, o, top, sum, unit, sh.join);
}

// ---- up to eight rows to a wave
// Scores of a few rows would leave most columns of the form above empty, and weights cost more instructions than codes do.  Here
// 64 positions are taken at a time, S = Q K^T with the rows repeated over the sixteen of an operand, so that every lane has, of
// one of the four products' sixteen keys each, scores of up to four rows - of one key (ROWS up to 4) or two (8) - and each
// score is in one lane only.  A key's scales are a value to a lane, whole lines of memory.  The weights go
// through LDS, a row of 64 a query, to where they are an operand: lane (c, g) takes eight of row c, those of positions
// 4 e + g of 32, so that four rows of values that follow each other in memory are loaded at a time.
// Memory bounds it: 16 sequences, 32 heads on 8, up to 32768 positions of 128 values in e4m3 139 us, 5.5 TB/s (the form above 148), 64 of up to
// 4096 in int8 74.3 us, 5.0 TB/s (83.8); 128 sequences, 16 heads, up to 512 of 64 values, float32, 20.3 us, 4.7 TB/s (22.0).  Not so one sequence
// with few heads: its parts are few (kCacheMostParts), a head of 100000 positions takes 26.4 us, 1.0 TB/s.
// Its start costs more, so short contexts are left to the form above.
template <typename T, CacheFormat F, int DP, int ROWS>
struct CacheFew {
  using A = CacheAttention<T, F, DP>;
  static constexpr int kRegs = ROWS < 4 ? ROWS : 4;    // rows whose scores a lane has
  static constexpr int kKeys = ROWS <= 4 ? 1 : 2;      // keys whose scores a lane has
  static constexpr int kStride = 72;                   // weights of a row in LDS, and eight more
  typedef _Float16 Weights[A::kWeightTerms][ROWS][kStride];

  struct Keys {
    cache_u4 code[4][A::kPieces];
    float scale[kKeys];
  };
  struct Values {
    unsigned code[2][8][A::kWords];
    float scale[kKeys];
  };
  // The position, of 64, whose scores lane (c, g) has.
  static __device__ __forceinline__ int key_of(int i, int lane) { return kKeys == 1 ? lane : 32 * i + 16 * (lane >> 5) + (lane & 15); }
  static_assert(kStride % 8 == 0, "weights are read in pieces of 16 bytes");
};

// Weights until the last turn, then what the waves join through.
template <typename T, CacheFormat F, int DP, int ROWS, int WAVES>
union CacheFewShared {
  CacheJoin<DP, 1, WAVES> join;
  alignas(16) typename CacheFew<T, F, DP, ROWS>::Weights weights[WAVES];
};

template <typename T, CacheFormat F, int DP, int ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (DP == 128 ? 2 : ROWS <= 2 ? 4 : 3)) void cache_attention_few_kernel(CacheAttentionArgs a) {
  using A = CacheAttention<T, F, DP>;
  using B = CacheFew<T, F, DP, ROWS>;
  constexpr int kTerms = A::kTerms, kWeightTerms = A::kWeightTerms, kSteps = A::kSteps, kDims = A::kDims, kRegs = B::kRegs, kKeys = B::kKeys;
  constexpr int kTurn = 64 * WAVES;   // positions that the waves take in one turn
  __shared__ CacheFewShared<T, F, DP, ROWS, WAVES> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  CacheTile x;
  if(!cache_tile<T, DP, ROWS, WAVES>(a, tid, x)) return;
  const int end = x.end;
  const CacheBuffer k_codes(x.k, (unsigned)end * a.dk), v_codes(x.v, (unsigned)end * a.dk), k_scales(x.ks, 4u * end), v_scales(x.vs, 4u * end);
  auto fetch_keys = [&](typename B::Keys& y, int at) __attribute__((always_inline)) {
    load_keys(y.code, k_codes, at, a.dk, lane);
#pragma unroll
    for(int i = 0; i < kKeys; ++i) y.scale[i] = k_scales.number(at + B::key_of(i, lane));
  };
  auto fetch_values = [&](typename B::Values& y, int at) __attribute__((always_inline)) {
    const unsigned d = (unsigned)(kDims * c) < (unsigned)a.dk ? kDims * c : 0, row = (unsigned)(at + g) * a.dk + d;
#pragma unroll
    for(int e = 0; e < 16; ++e) v_codes.words(y.code[e / 8][e % 8], row + (unsigned)(4 * e) * a.dk);
#pragma unroll
    for(int i = 0; i < kKeys; ++i) y.scale[i] = v_scales.number(at + B::key_of(i, lane));
  };
  const int begin = x.w.from + 64 * wave;
  typename B::Keys key;
  typename B::Values value;
  fetch_keys(key, begin);
  fetch_values(value, begin);
  unsigned long long seen = 0;
  if(a.parents) seen = lineage(a.parents + (long long)x.w.s * a.n, a.n, lane);
  cache_h8 q[kTerms][kSteps];
  const float query_scale = cache_query<T, F, DP>(a, x, min(x.row0 + c % ROWS, x.rows - 1), g, q);
  const int mine0 = ROWS == 8 ? 4 * (g & 1) : 0;   // the first of the rows whose scores the lane has
  float row_scale[kRegs];
  CacheSight sight[kRegs];
#pragma unroll
  for(int t = 0; t < kRegs; ++t) {
    row_scale[t] = lane_value(query_scale, t);
    if constexpr(ROWS == 8) row_scale[t] = g & 1 ? lane_value(query_scale, t + 4) : row_scale[t];
    sight[t] = cache_sight(a, x, min(x.row0 + mine0 + t, x.rows - 1), seen);
  }
  cache_f4 o[1][kDims];
#pragma unroll
  for(int j = 0; j < kDims; ++j) o[0][j] = cache_f4{0, 0, 0, 0};
  float top[kRegs], sum[kRegs], unit[kRegs], per[kRegs];
#pragma unroll
  for(int t = 0; t < kRegs; ++t) {
    top[t] = kNone;
    sum[t] = 0.0f;
    unit[t] = 1e-30f;
    per[t] = kWeightUnit / unit[t];
  }
  // of row c, what the lanes that have its scores hold
  auto of_row = [&](const float(&y)[kRegs]) __attribute__((always_inline)) {
    float z = 0.0f;
#pragma unroll
    for(int r = 0; r < ROWS; ++r) {
      const float it = lane_value(y[r % 4], r < 4 ? 0 : 16);
      z = r == 0 || c % ROWS == r ? it : z;
    }
    return z;
  };
  auto over_rows_lanes = [&](float y, auto join) __attribute__((always_inline)) {   // over the lanes that have scores of the same rows
    y = over_bit5(over_row(y, join), join);
    if constexpr(ROWS != 8) y = over_bit4(y, join);
    return y;
  };

  for(int at = begin; at < end; at += kTurn) {
    // scores
    float s[kKeys][kRegs];
    {
      cache_f4 p[4];
#pragma unroll
      for(int b = 0; b < 4; ++b) {
        p[b] = cache_f4{0, 0, 0, 0};
#pragma unroll
        for(int i = 0; i < kSteps; ++i) {
          const cache_u4 piece = key.code[b][i / 2];
          const cache_h8 operand = i % 2 ? half8_of<F>(piece[2], piece[3]) : half8_of<F>(piece[0], piece[1]);
#pragma unroll
          for(int m = kTerms - 1; m >= 0; --m) p[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[m][i], operand, p[b], 0, 0, 0);
        }
      }
#pragma unroll
      for(int t = 0; t < kRegs; ++t) {
        if(kKeys == 1) {
          s[0][t] = g & 2 ? (g & 1 ? p[3][t] : p[2][t]) : (g & 1 ? p[1][t] : p[0][t]);
        } else {
          s[0][t] = g & 2 ? p[1][t] : p[0][t];
          s[kKeys - 1][t] = g & 2 ? p[3][t] : p[2][t];
        }
      }
    }
#pragma unroll
    for(int i = 0; i < kKeys; ++i)
#pragma unroll
      for(int t = 0; t < kRegs; ++t) s[i][t] *= key.scale[i];
    fetch_keys(key, at + kTurn);
    // Positions that a row does not see score minus infinity (a weight of zero) and have a scale of zero.
    float scale[kKeys][kRegs];
#pragma unroll
    for(int i = 0; i < kKeys; ++i)
#pragma unroll
      for(int t = 0; t < kRegs; ++t) scale[i][t] = value.scale[i];
    if(at + 64 > x.open) {
#pragma unroll
      for(int i = 0; i < kKeys; ++i) {
        const int p = at + B::key_of(i, lane), j = p - x.w.len;
#pragma unroll
        for(int t = 0; t < kRegs; ++t) {
          const bool see = a.parents ? p < end && (j < 0 || (sight[t].sees >> (j & 63) & 1) != 0) : p < sight[t].limit;
          s[i][t] = see ? s[i][t] : kNone;
          scale[i][t] = see ? scale[i][t] : 0.0f;
        }
      }
    }
    float high[kRegs], wide[kRegs];
    bool grown = false;
#pragma unroll
    for(int t = 0; t < kRegs; ++t) {
      high[t] = (kKeys == 1 ? s[0][t] : fmaxf(s[0][t], s[kKeys - 1][t])) * row_scale[t];
      wide[t] = kKeys == 1 ? __builtin_fabsf(scale[0][t]) : fmaxf(__builtin_fabsf(scale[0][t]), __builtin_fabsf(scale[kKeys - 1][t]));
      grown |= high[t] > top[t] + kMaximumSlack || wide[t] > unit[t] * kScaleSlack;
    }
    if(__any(grown)) {
      float both[kRegs];
#pragma unroll
      for(int t = 0; t < kRegs; ++t) {
        // (a NaN is left out by both maxima, its row by its sum)
        const float m = fmaxf(top[t], over_rows_lanes(high[t], Larger())), u = fmaxf(unit[t], over_rows_lanes(wide[t], Larger()));
        const float down = m == top[t] ? 1.0f : __builtin_amdgcn_exp2f(top[t] - m);
        both[t] = u == unit[t] ? down : down * (unit[t] / u);
        sum[t] *= down;
        top[t] = m;
        unit[t] = u;
        per[t] = kWeightUnit / u;
      }
      const float factor = of_row(both);
#pragma unroll
      for(int j = 0; j < kDims; ++j) o[0][j] *= factor;
    }
    // weights
#pragma unroll
    for(int i = 0; i < kKeys; ++i) {
      const int p = B::key_of(i, lane), slot = (p & 32) + 8 * (p & 3) + (p >> 2 & 7);
#pragma unroll
      for(int t = 0; t < kRegs; ++t) {
        const float from = top[t] == kNone ? 0.0f : -top[t];   // (nothing seen so far: minus infinity stays that)
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][t], row_scale[t], from)), z = settled(y * (scale[i][t] * per[t]));
        sum[t] += y;
        const _Float16 hi = (_Float16)z;
        sh.weights[wave][0][mine0 + t][slot] = hi;
        sh.weights[wave][1][mine0 + t][slot] = (_Float16)(z - (float)hi);
      }
    }
    __builtin_amdgcn_wave_barrier();   // (a wave's accesses to LDS are done in their order)
    // weighted values
#pragma unroll
    for(int h = 0; h < 2; ++h) {
      cache_h8 p[kWeightTerms];
#pragma unroll
      for(int m = 0; m < kWeightTerms; ++m) p[m] = *reinterpret_cast<const cache_h8*>(&sh.weights[wave][m][c % ROWS][32 * h + 8 * g]);
      unsigned vh[8][A::kWords];
#pragma unroll
      for(int e = 0; e < 8; ++e)
#pragma unroll
        for(int i = 0; i < A::kWords; ++i) vh[e][i] = held<F>(value.code[h][e][i]);
#pragma unroll
      for(int i = 0; i < A::kWords; ++i) {
        const cache_h8 d[4] = {value_operand_of<F, 0>(vh, i), value_operand_of<F, 1>(vh, i), value_operand_of<F, 2>(vh, i),
                               value_operand_of<F, 3>(vh, i)};
#pragma unroll
        for(int j = 0; j < 4; ++j)
#pragma unroll
          for(int m = kWeightTerms - 1; m >= 0; --m) o[0][4 * i + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(d[j], p[m], o[0][4 * i + j], 0, 0, 0);
      }
    }
    __builtin_amdgcn_wave_barrier();
    fetch_values(value, at + kTurn);
  }
#pragma unroll
  for(int t = 0; t < kRegs; ++t) sum[t] = over_rows_lanes(sum[t], Added());
  float row_top[1] = {of_row(top)}, row_sum[1] = {of_row(sum) * 0.25f}, row_unit[1] = {of_row(unit)};   // (four lanes of a row add up in the end)
  if(WAVES > 1) __syncthreads();   // (the weights' memory is taken for the results)
  cache_finish<T, F, DP, 1, WAVES>(a, x, o, row_top, row_sum, row_unit, sh.join);
}

// ---- many rows to an entry
// 16 * QT rows to a wave, whose waves share 64 positions at a time: these are loaded once, turned into float16 and laid into LDS as the
// operands that every wave then reads, piece after piece of 64 lanes.  Wave w turns the keys of block w of sixteen, and of
// half w / 2 of the positions half the dimensions of the values; the next codes are on their way meanwhile.  The products are those
// of the first form, but for the dimensions, lane (c, g) having 64 i + 16 g + 4 e + j.  While a wave lays positions out it goes ahead of those in
// products (the others wait for it): 81.3 us against 84.8 (the trees below).  A second buffer in LDS, with one barrier a turn, gained nothing.
// 4 sequences, 1024 tokens behind 3072 positions, 32 heads on 8, 128 values, bfloat16: 328 us, 730 TFLOP/s of what the tokens see; 8 trees of 64
// tokens, 32 heads on 4, behind 8192 positions 113 us, 610 TFLOP/s, up to 8192 82 us, 550 TFLOP/s: products and exponentials take turns in
// the issue slots, and with lengths that differ parts do, too, and results go through memory to the workgroup that joins them.  The first form:
// 8 sequences of 16 tokens, 32 heads on 8, up to 8192 positions 53.9 us, this one 42.8; 64 sequences of 50 rows, 16 heads, up to
// 500 positions 53.0 and 37.2.  (Few entries of a few thousand positions leave most of the card idle, a part being 512 of them: 64 tokens of 8 heads
// of 256 values, 4000 positions, 64 workgroups, 34 us, 62 TFLOP/s.)
template <typename T, CacheFormat F, int DP, int QT>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void cache_attention_many_kernel(CacheAttentionArgs a) {
  using A = CacheAttention<T, F, DP>;
  constexpr int kTerms = A::kTerms, kWeightTerms = A::kManyWeightTerms, kSteps = A::kSteps, kDims = A::kDims, kPieces = A::kPieces;
  constexpr int kTile = 64, kRows = 16 * QT * 4;
  constexpr int kMine = kDims / 2;                      // dimensions' operands that a wave makes ...
  constexpr int kMineWords = kMine < 4 ? 1 : kMine / 4;   // ... of so many words of a row
  __shared__ union {
    struct {
      cache_h8 k[4 * kSteps][64], v[2 * kDims][64];
      cache_f4 ks[kTile / 4], vs[kTile / 4];
    } tile;
    CacheParts<DP, 4> parts;
  } sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  CacheTile x;
  if(!cache_tile<T, DP, kRows, 4>(a, tid, x)) return;

  // ---- what the wave loads
  const int half = wave >> 1, side = wave & 1;
  cache_u4 k_code[1][kPieces];
  unsigned v_code[8][kMineWords];
  float scale;   // of a position's key, or, in waves 1 and 3, value
  const CacheBuffer k_codes(x.k, (unsigned)x.end * a.dk), v_codes(x.v, (unsigned)x.end * a.dk), scales(side ? x.vs : x.ks, 4u * x.end);
  auto fetch = [&](int at) __attribute__((always_inline)) {
    load_keys(k_code, k_codes, at + 16 * wave, a.dk, lane);
    const unsigned row = (unsigned)(at + 32 * half + 4 * g) * a.dk;
#pragma unroll
    for(int i = 0; i < kMineWords; ++i) {
      const unsigned d = 64 * (DP == 64 ? 0 : side * kMineWords + i) + 4 * c, from = row + (d < (unsigned)a.dk ? d : 0);
#pragma unroll
      for(int e = 0; e < 8; ++e) {
        unsigned word[1];
        v_codes.words(word, from + (unsigned)(16 * (e / 4) + e % 4) * a.dk);
        v_code[e][i] = word[0];
      }
    }
    scale = scales.number(at + lane);
  };
  auto lay = [&]() __attribute__((always_inline)) {
#pragma unroll
    for(int i = 0; i < kPieces; ++i) {
      sh.tile.k[wave * kSteps + 2 * i][lane] = half8_of<F>(k_code[0][i][0], k_code[0][i][1]);
      sh.tile.k[wave * kSteps + 2 * i + 1][lane] = half8_of<F>(k_code[0][i][2], k_code[0][i][3]);
    }
    unsigned vh[8][kMineWords];
#pragma unroll
    for(int e = 0; e < 8; ++e)
#pragma unroll
      for(int i = 0; i < kMineWords; ++i) vh[e][i] = held<F>(v_code[e][i]);
    cache_h8(*to)[64] = &sh.tile.v[half * kDims + side * kMine];
    if constexpr(DP == 64) {   // two of the four dimensions of the only word
      to[0][lane] = side ? value_operand_of<F, 2>(vh, 0) : value_operand_of<F, 0>(vh, 0);
      to[1][lane] = side ? value_operand_of<F, 3>(vh, 0) : value_operand_of<F, 1>(vh, 0);
    } else {
#pragma unroll
      for(int i = 0; i < kMineWords; ++i) {
        to[4 * i][lane] = value_operand_of<F, 0>(vh, i);
        to[4 * i + 1][lane] = value_operand_of<F, 1>(vh, i);
        to[4 * i + 2][lane] = value_operand_of<F, 2>(vh, i);
        to[4 * i + 3][lane] = value_operand_of<F, 3>(vh, i);
      }
    }
    if(tid < 128) (tid < 64 ? reinterpret_cast<float*>(sh.tile.ks) : reinterpret_cast<float*>(sh.tile.vs))[lane] = scale;
  };
  fetch(x.w.from);

  // ---- the wave's rows
  unsigned long long seen = 0;
  if(a.parents) seen = lineage(a.parents + (long long)x.w.s * a.n, a.n, lane);
  const int row0 = x.row0 + 16 * QT * wave;
  cache_h8 q[QT][kTerms][kSteps];
  float row_scale[QT];
  CacheSight sight[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const int row = min(row0 + 16 * t + c, x.rows - 1);
    sight[t] = cache_sight(a, x, row, seen);
    row_scale[t] = cache_query<T, F, DP>(a, x, row, g, q[t]);
  }
  // of what any of them see (trees: as the workgroup's)
  const int end = row0 >= x.rows ? 0 : a.parents ? x.end : min(x.end, x.w.len + (int)a.by_group.of((unsigned)min(x.rows - 1, row0 + 16 * QT - 1)) + 1);
  cache_f4 o[QT][kDims];
  float top[QT], sum[QT], unit[QT], per[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    top[t] = kNone;
    sum[t] = 0.0f;
    unit[t] = 1e-30f;   // (scales below it are as good as zero)
    per[t] = kWeightUnit / unit[t];
#pragma unroll
    for(int j = 0; j < kDims; ++j) o[t][j] = cache_f4{0, 0, 0, 0};
  }

  // Positions at .. at + 31, half h of the block.  MASKED: not all of them are seen by all rows.  Up to the first such block the carried
  // scale is the same for all rows.
  auto take = [&](int at, int h, auto masked) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked)::value;
    cache_f4 s[QT][2], vs[2];
#pragma unroll
    for(int b = 0; b < 2; ++b)
#pragma unroll
      for(int t = 0; t < QT; ++t) s[t][b] = cache_f4{0, 0, 0, 0};
    {
      cache_h8 operand[2][kSteps];
#pragma unroll
      for(int i = 0; i < kSteps; ++i)
#pragma unroll
        for(int b = 0; b < 2; ++b) operand[b][i] = sh.tile.k[(2 * h + b) * kSteps + i][lane];
#pragma unroll
      for(int i = 0; i < kSteps; ++i)
#pragma unroll
        for(int m = kTerms - 1; m >= 0; --m)
#pragma unroll
          for(int b = 0; b < 2; ++b)
#pragma unroll
            for(int t = 0; t < QT; ++t) s[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[b][i], q[t][m][i], s[t][b], 0, 0, 0);
    }
    // (the first values are on their way while the weights are made)
    constexpr int kAhead = 4;
    cache_h8 ahead[kAhead];
#pragma unroll
    for(int j = 0; j < kAhead; ++j) ahead[j] = sh.tile.v[h * kDims + j][lane];
#pragma unroll
    for(int b = 0; b < 2; ++b) {
      const cache_f4 ks = sh.tile.ks[4 * (2 * h + b) + g];
      vs[b] = sh.tile.vs[4 * (2 * h + b) + g];
#pragma unroll
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int e = 0; e < 4; ++e) s[t][b][e] *= ks[e];
    }
    unsigned seen_here[QT];   // bit 4 b + e
    float widest = 0.0f;
    if constexpr(MASKED) {
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        seen_here[t] = 0;
#pragma unroll
        for(int b = 0; b < 2; ++b) {
          const int from = at + 16 * b + 4 * g;
          unsigned four = (1u << clamp_int((a.parents ? end : sight[t].limit) - from, 0, 4)) - 1;
          if(a.parents) {   // settled positions, then the drafted ones from bit 0 on
            const int j = from - x.w.len, settled = clamp_int(-j, 0, 4);
            four &= j < 0 ? ((unsigned)sight[t].sees << settled | ((1u << settled) - 1)) : (unsigned)(sight[t].sees >> min(j, 63));
          }
          seen_here[t] |= four << (4 * b);
#pragma unroll
          for(int e = 0; e < 4; ++e) s[t][b][e] = four >> e & 1 ? s[t][b][e] : kNone;
        }
      }
    } else {
#pragma unroll
      for(int e = 0; e < 8; ++e) widest = fmaxf(widest, __builtin_fabsf(vs[e / 4][e % 4]));
    }
    float high[QT], wide[QT];
    bool grown = false;
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      high[t] = kNone;
      wide[t] = widest;
#pragma unroll
      for(int e = 0; e < 8; ++e) {
        high[t] = fmaxf(high[t], s[t][e / 4][e % 4]);
        if constexpr(MASKED) wide[t] = fmaxf(wide[t], seen_here[t] >> e & 1 ? __builtin_fabsf(vs[e / 4][e % 4]) : 0.0f);
      }
      high[t] *= row_scale[t];
      grown |= high[t] > top[t] + kMaximumSlack || wide[t] > unit[t] * kScaleSlack;
    }
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
        per[t] = kWeightUnit / u;
      }
    }
    cache_h8 p[QT][kWeightTerms];
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float from = top[t] == kNone ? 0.0f : -top[t];   // (nothing seen so far: minus infinity stays that)
#pragma unroll
      for(int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / 4][e % 4], row_scale[t], from));
        float r = vs[e / 4][e % 4] * per[MASKED ? t : 0];
        if constexpr(MASKED) r = seen_here[t] >> e & 1 ? r : 0.0f;
        const float z = kWeightTerms == 2 ? settled(y * r) : y * r;
        sum[t] += y;
        p[t][0][e] = (_Float16)z;
        if constexpr(kWeightTerms == 2) p[t][kWeightTerms - 1][e] = (_Float16)(z - (float)p[t][0][e]);
      }
    }
#pragma unroll
    for(int j = 0; j < kDims; ++j) {
      const cache_h8 operand = ahead[j % kAhead];
      if(j + kAhead < kDims) ahead[j % kAhead] = sh.tile.v[h * kDims + j + kAhead][lane];
#pragma unroll
      for(int t = 0; t < QT; ++t)
#pragma unroll
        for(int m = kWeightTerms - 1; m >= 0; --m) o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand, p[t][m], o[t][j], 0, 0, 0);
    }
  };
  auto turn = [&](int at) __attribute__((always_inline)) {   // the positions in hand into LDS, the next ones asked for
    __syncthreads();   // (nobody reads the last ones any more)
    __builtin_amdgcn_s_setprio(2);
    lay();
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    fetch(at + kTile);
  };
  int at = x.w.from;
  for(; at + kTile <= x.open; at += kTile) {
    turn(at);
#pragma unroll 1
    for(int h = 0; h < 2; ++h) take(at + 32 * h, h, std::false_type());
  }
  for(; at < x.end; at += kTile) {
    turn(at);
#pragma unroll 1
    for(int h = 0; h < 2; ++h)
      if(at + 32 * h < end) take(at + 32 * h, h, std::true_type());
  }

  // A sequence in several parts: a part's values go to the workspace as the registers have them, whole lines at a time, a lane's where the
  // same lane of the workgroup that arrives last finds them, the logarithms of the rows' sums behind them.
  constexpr float kUnit = 1.0f / (kWeightUnit * kCodeUnit<F>);
  float factor[QT], log[QT];
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    sum[t] = over_lanes_sum(sum[t]);
    factor[t] = (sum[t] == 0.0f ? 0.0f : 1.0f / sum[t]) * (unit[t] * kUnit);
    log[t] = sum[t] == 0.0f ? kNone : top[t] + __builtin_amdgcn_logf(sum[t]);
#pragma unroll
    for(int j = 0; j < kDims; ++j) o[t][j] *= factor[t];
  }
  if(x.w.parts > 1) {
    constexpr int kTileFloats = kRows * (DP + 1);
    const long long place = ((long long)x.w.slot * a.Hk + x.head) * a.row_tiles + x.tile, stride = (long long)a.Hk * a.row_tiles * kTileFloats;
    float* const first = a.part + place * kTileFloats;
    const unsigned mine = wave * (16 * QT * DP) + 4 * lane, my_log = kRows * DP + wave * 16 * QT + c;
    {
      const CacheBuffer to(first + x.w.part * stride, 4u * kTileFloats);
#pragma unroll
      for(int t = 0; t < QT; ++t) {
#pragma unroll
        for(int j = 0; j < kDims; ++j) to.store_through(o[t][j], 4u * (mine + 256u * (t * kDims + j)));
        if(g == 0) to.store_through(log[t], 4u * (my_log + 16u * t));
      }
    }
    if(!cache_arrived_last(a.counters + place, x.w.parts, sh.parts.is_last)) return;
    float most[QT], total[QT];
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      most[t] = kNone;
      total[t] = 0.0f;
#pragma unroll
      for(int j = 0; j < kDims; ++j) o[t][j] = cache_f4{0, 0, 0, 0};
    }
#pragma unroll 1
    for(int i = 0; i < x.w.parts; ++i) {
      const CacheBuffer from(first + i * stride, 4u * kTileFloats);
      cache_f4 y[QT][kDims];
      float l[QT];
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        l[t] = from.number_through(4u * (my_log + 16u * t));
#pragma unroll
        for(int j = 0; j < kDims; ++j) y[t][j] = from.piece_through(4u * (mine + 256u * (t * kDims + j)));
      }
#pragma unroll
      for(int t = 0; t < QT; ++t) {
        const float m = fmaxf(most[t], l[t]), down = most[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f(most[t] - m);
        const float weight = l[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f(l[t] - m) * kPartUnit;
        most[t] = m;
        total[t] = total[t] * down + weight;
#pragma unroll
        for(int j = 0; j < kDims; ++j)
#pragma unroll
          for(int e = 0; e < 4; ++e) o[t][j][e] = __builtin_fmaf(weight, y[t][j][e], o[t][j][e] * down);
      }
    }
#pragma unroll
    for(int t = 0; t < QT; ++t) {
      const float all = total[t] == 0.0f ? 0.0f : 1.0f / total[t];
#pragma unroll
      for(int j = 0; j < kDims; ++j) o[t][j] *= all;
    }
  }
#pragma unroll
  for(int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + c;
    if(r >= x.rows) continue;
    T* const out = cache_row_out<T>(a, x, r);
#pragma unroll
    for(int e = 0; e < 4; ++e)
#pragma unroll
      for(int i = 0; i < kDims / 4; ++i) {
        const int d = 64 * i + 16 * g + 4 * e;
        const float y[4] = {o[t][4 * i][e], o[t][4 * i + 1][e], o[t][4 * i + 2][e], o[t][4 * i + 3][e]};
        if(d < a.dk) store_row<4, T>(out + d, y);
      }
  }
}

}  // namespace marian_hip
