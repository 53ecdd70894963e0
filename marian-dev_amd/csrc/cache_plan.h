// How marian_hip_cache_attention deals its rows and positions to workgroups (host code, no HIP).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace marian_hip {

constexpr int kCacheBlock = 128;    // positions that parts are counted in: four waves take as many in one turn
constexpr unsigned kCacheWhole = 4;        // blocks that are not worth splitting
// of a sequence: one with 8 heads of 32000 positions would take 25.7 us with 32 and 28.2 with 64, one head of 100000 41.6 and 34.1
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
  // four rows each, 4096 positions of 128 values: 73.5 us in the first, 84.7 in the second; one sequence of 60: 8.1 and 5.4, eight of 4000
  // 19.4 and 16.1; 64 values, float32: 32 sequences of 8 heads, 2000 positions 16.4 and 16.7, 1000 14.4 and 12.6.  (What sequences hold only
  // the device knows: the capacity stands for it.)
  p.few = rows > 8 || p.dp == 256 || sequences * heads * capacity < 400000 ? 0 : rows > 4 ? 8 : rows > 2 ? 4 : (int)rows;
  p.qt = rows <= 16 || p.dp == 256 ? 1 : 2;   // (what the registers hold)
  // More than 32 rows: a workgroup of 128 takes 11 to 15 % less time a row than one of 64, unless the last of several is half empty
  // (300 rows of 16 sequences, 16 heads, 4000 positions of 128 values: 239 us in 64s, 254 us in 128s; 440 rows: 329 and 312)
  // or there are too few to keep the card busy (256 rows of 4000 positions, 8 heads: 23 us in 64s, 31 us in 128s).
  const int64_t sixtyfours = (rows + 63) / 64, wide_tiles = (rows + 127) / 128;
  if(rows > 32 && (8 * sixtyfours < 14 * wide_tiles || sequences * heads * wide_tiles < 128)) p.qt = 1;
  p.many = rows > 32 ? 64 * p.qt : 0;   // (33 .. 64 rows: 45.2 us against 47.3 of the form for fewer, see the kernel)
  p.tile_rows = p.many ? p.many : 16 * p.qt;
  p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t entries = sequences * heads * p.row_tiles;
  // Where single workgroups of two waves or one keep the card busy, fewer have to join: one token, 16 heads of 64 values, 400 sequences of up to
  // 300 positions 42.2 us with one wave, 45.2 with four; 128 of 512 22.5 with two, 23.0 with four.
  p.waves = p.many ? 4 : entries >= 4096 ? 1 : entries >= 2048 ? 2 : 4;
  // Parts for one round of the workgroups that run at a time, by the registers of their form: a second round runs half empty, and a sequence's
  // last part is half as long as the others on average, so half a part for each is left out (16 sequences, up to 32768 positions: 157 us, with
  // parts for all 181; with a fixed 1024 168).
  const int to_a_simd = p.many ? (p.dp == 256 ? 1 : p.qt == 1 ? 3 : 2) : p.few ? (p.dp == 128 ? 2 : p.few <= 2 ? 4 : 3) : p.dp == 64 ? 5 - p.qt : p.dp == 128 ? 4 - p.qt : 2;
  const int64_t at_a_time = 1024 * to_a_simd / p.waves;
  p.target = std::max<int64_t>(1, at_a_time / (heads * p.row_tiles) - sequences / 2);
  // Joining parts takes some 2.5 us, four blocks of one wave's turn each as long: with few entries parts go down to two blocks, a sequence of
  // up to four stays whole (one sequence, 8 heads, 128 values: 1000 positions 9.2 us, 10.4 in fours, 500 7.8 whole, 8.9 in two).
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
