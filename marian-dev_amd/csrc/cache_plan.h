// How marian_hip_cache_attention deals its rows and positions to workgroups (host code, no HIP).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace marian_hip {

constexpr int kCacheBlock = 128;    // positions that parts are counted in: four waves take as many in one turn
constexpr unsigned kCacheWhole = 4;        // blocks that are not worth splitting
// Of a sequence.  One token of one sequence, 128 values, bfloat16 over int8, with 32, with these, with 64: a head of keys with 32000 positions 15.5,
// 13.7, 12.2 us, 100000 34.4, 26.4, 22.4; 8 heads with four rows each 20.0, 21.8, 22.4 and 45.3, 50.3, 45.3; 2 sequences, 2 heads with 16
// rows of 256 values, up to 56618 positions 45.3, 46.9, 52.8.  No number is best for all of them.
constexpr unsigned kCacheMostParts = 48;
constexpr int kCacheMost = 8192;    // counters of a workspace: two for each of the workgroups that positions are split for

struct CacheAttentionPlan {
  int dp;              // values of a row as the kernel holds it: dk rounded up to 64, 128 or 256
  int qt;              // sixteens of query rows to a workgroup
  int few;             // the rows of an entry, up to 1, 2, 4 or 8 of them (0: more, or values too long for that form)
  int many;            // rows of a workgroup of four waves that share positions laid out in LDS (0: fewer rows)
  int waves;           // of a workgroup, which share its positions
  int tile_rows;       // of a workgroup
  int64_t row_tiles;   // workgroups that share an entry's positions
  int least;           // blocks of a part
  int64_t target;      // parts that the positions of all sequences together are split into
  int64_t items;       // the most parts there can be, a sequence having at least one
  int64_t slots;       // the most parts of sequences that have more than one: these leave partial results
  int64_t grid;
  int64_t row_floats;  // of a partial result: dp values and the logarithm of the sum of its weights
};

// A part is a whole number of blocks of positions, as many as all sequences have divided by target: then the parts of the
// sequences that have several are less than 2 * target, whatever the lengths.
inline CacheAttentionPlan cache_attention_plan(int64_t sequences, int64_t heads, int64_t q_heads, int64_t capacity, int64_t n, int64_t dk) {
  CacheAttentionPlan p{};
  p.dp = dk <= 64 ? 64 : dk <= 128 ? 128 : 256;
  const int64_t rows = n * (q_heads / heads);
  // The form for few rows takes 64 positions a turn and has the memory busier, the other starts faster.  One token; 64 sequences of 8 heads with
  // four rows each, up to 4096 positions of 128 values: 74.3 us in the first, 83.8 in the second; one sequence of 60: 8.2 and 6.0, eight of 4000
  // 21.4 and 19.1; 64 values, float32: 32 sequences of 8 heads, up to 2000 positions 16.4 and 17.6, 1000 11.7 and 12.9.  What sequences hold
  // only the device knows: the capacity stands for it, and is wrong where a large cache holds little (64 sequences of up to 60 in room for 4096:
  // 9.9 us here, 7.5 in the other; one of 4000 in room for 60000: 12.9 and 10.8).
  p.few = rows > 8 || p.dp == 256 || sequences * heads * capacity < 400000 ? 0 : rows > 4 ? 8 : rows > 2 ? 4 : (int)rows;
  p.qt = rows <= 16 || p.dp == 256 ? 1 : 2;   // (what the registers hold)
  // More than 32 rows: a workgroup of 128 takes less time a row than one of 64, unless the last of several is half empty
  // (300 rows of 16 sequences, 16 heads, up to 4000 positions of 128 values: 215 us in 64s, 230 us in 128s; 440 rows: 325 and 314)
  // or there are too few to keep the card busy (256 rows of 4000 positions, 8 heads: 23 us in 64s, 31 us in 128s).
  const int64_t sixtyfours = (rows + 63) / 64, wide_tiles = (rows + 127) / 128;
  if(rows > 32 && (8 * sixtyfours < 14 * wide_tiles || sequences * heads * wide_tiles < 128)) p.qt = 1;
  p.many = rows > 32 ? 64 * p.qt : 0;   // (33 .. 64 rows: 42.8 us against 53.9 of the form for fewer, see the kernel)
  p.tile_rows = p.many ? p.many : 16 * p.qt;
  p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t entries = sequences * heads * p.row_tiles;
  // Where single workgroups of two waves or one keep the card busy, fewer have to join: one token, 16 heads of 64 values, 400 sequences of up to
  // 300 positions 40.3 us with one wave, 45.1 with four; 128 of up to 512 20.2 with two, 20.3 with four.
  p.waves = p.many ? 4 : entries >= 4096 ? 1 : entries >= 2048 ? 2 : 4;
  // Parts for one round of the workgroups that run at a time, by the registers of their form: a second round runs half empty, and a sequence's
  // last part is half as long as the others on average, so half a part for each is left out (16 sequences, up to 32768 positions: 139 us, with
  // parts for all 154; 64 of up to 4096: 74 and 86).
  const int to_a_simd = p.many ? (p.dp == 256 ? 1 : p.qt == 1 ? 3 : 2) : p.few ? (p.dp == 128 ? 2 : p.few <= 2 ? 4 : 3) : p.dp == 64 ? 5 - p.qt : p.dp == 128 ? 4 - p.qt : 2;
  const int64_t at_a_time = 1024 * to_a_simd / p.waves;
  p.target = std::max<int64_t>(1, at_a_time / (heads * p.row_tiles) - sequences / 2);
  // Joining parts takes some 2.5 us, four blocks of one wave's turn each as long: with few entries parts go down to two blocks, a sequence of
  // up to four stays whole (one sequence, 8 heads, 128 values: 1000 positions 10.0 us, 11.9 in fours, 500 8.8 whole, 9.9 in two).
  p.least = !p.many && entries <= 32 ? 2 : 4;
  p.items = p.target == 1 ? sequences : p.target + sequences;
  p.slots = p.target == 1 ? 0 : 2 * p.target;
  p.grid = (p.items * heads + 7) / 8 * 8 * p.row_tiles;
  p.row_floats = p.dp + 1;
  return p;
}

// The workspace: a counter for each row tile of a sequence with several parts (at most slots * heads * row_tiles, kCacheMost of
// them), in the same place for all sizes, then the partial results.
constexpr int64_t kCacheCounterBytes = kCacheMost * 4;
inline int64_t cache_attention_bytes(const CacheAttentionPlan& p, int64_t heads) {
  return p.slots == 0 ? 0 : kCacheCounterBytes + p.slots * heads * p.row_tiles * p.tile_rows * p.row_floats * 4;
}

}  // namespace marian_hip
