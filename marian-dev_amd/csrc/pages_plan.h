// How marian_hip_pages_attention deals its rows and positions to workgroups (host code, no HIP).
#pragma once

#include <stdint.h>

#include <algorithm>

#include "cache_plan.h"

namespace marian_hip {

// Registers of a form (an estimate).  Of float32 rows of 65 to 127 values, up to sixteen rows, it is nine too low, and as many go to memory;
// with one wave to a SIMD none do: one token, 16 sequences of up to 2000 positions, 16 heads of 80 values 74.1 us so and 78.3, of up to 8192, 8 of
// 112 with four rows each 140.4 and 138.1.
constexpr int pages_registers(int width, int dp, int qt) {
  const int words = width * dp / 8;   // of keys and of values, each: 32 positions' bytes over 64 lanes
  return 2 * words + qt * (dp / 4 + words / 2 + 16) + 48;   // results, queries, scores and weights; addresses
}

// Of a sequence.  One token, bfloat16, 128 values, with 48 and with these: a sequence of 100003 positions, 8 heads of keys, 87.1 and 79.9 us; 32000,
// two heads 17.7 and 16.2; one head of 100000 33.2 and 29.4.
constexpr unsigned kPagesMostParts = 64;

// Sixteens of query rows that a wave takes over the same positions, at the most.
constexpr int pages_most_qt(int width, int dp) { return width == 4 && dp == 256 ? 1 : 2; }
// Whether rows past that have a form in which waves with rows of their own share positions in LDS, for 64 or 128 rows.  float32 without and with it: 7
// tokens of 24 sequences of up to 8192 positions, 4 heads with eight rows each, 128 values 268 and 220 us, 64 values 118 and 117; 9 of 11 of
// up to 64, 16 heads with four rows, 128 values 24 and 18; 256 of 4 of up to 512, 16 heads, 64 values 39 and 48.
constexpr bool pages_has_many(int width, int dp) { return dp == 128 || (width == 2 && dp == 64); }
constexpr int pages_many_waves(int width, int dp, int rows) { return width == 2 && dp == 128 && rows == 128 ? 4 : 8; }
// (a workgroup of float32, 128 values, has 128 KB of LDS)
constexpr int pages_many_to_a_simd(int width, int dp, int rows) { return width == 4 && dp == 128 ? 2 : pages_many_waves(width, dp, rows) / 2; }

// Positions up to which a sequence is short: eight turns of a wave.  (Where rows of the table have no room for more, sequences are not split: so one wave
// to an entry, which leaves room for more parts, never needs a larger workspace than what is asked for without knowing the rows.)
constexpr int64_t kPagesShort = 256;
static_assert(kPagesShort <= (int64_t)kCacheWhole * kCacheBlock, "short sequences have one part");
// Positions up to which sequences are taken to differ little.
constexpr int64_t kPagesEven = 1024;

// Waves of a form that fit a SIMD, by its registers.
constexpr int pages_to_a_simd(int width, int dp, int qt) {
  const int all = pages_registers(width, dp, qt);
  return all <= 128 ? 4 : all <= 168 ? 3 : all <= 256 ? 2 : 1;
}

struct PagesAttentionPlan {
  int dp;              // values of a row as the kernel holds it: dk rounded up to 64, 128 or 256
  bool many;           // the waves have rows of their own and share positions laid out in LDS
  int qt;              // if not: sixteens of query rows to a workgroup
  int waves;           // of a workgroup; if not, they share its rows and take turns of 32 positions
  int tile_rows;       // of a workgroup
  int64_t row_tiles;   // workgroups that share an entry's positions
  int least;           // blocks of a part
  int64_t target;      // parts that the positions of all sequences together are split into
  int64_t items;       // the most parts there can be, a sequence having at least one
  int64_t slots;       // the most parts of sequences that have more than one: these leave partial results
  int64_t grid;
};

inline PagesAttentionPlan pages_attention_plan(int64_t sequences, int64_t heads, int64_t q_heads, int64_t n, int64_t dk, int width, int64_t capacity = 1 << 30) {
  PagesAttentionPlan p{};
  p.dp = dk <= 64 ? 64 : dk <= 128 ? 128 : 256;
  const int64_t rows = n * (q_heads / heads);
  p.many = rows > 32 && pages_has_many(width, p.dp);
  p.qt = std::min(rows <= 16 ? 1 : 2, pages_most_qt(width, p.dp));
  p.tile_rows = p.many ? (rows > 64 ? 128 : 64) : 16 * p.qt;
  p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t entries = sequences * heads * p.row_tiles;
  const int form = pages_to_a_simd(width, p.dp, p.qt);
  // One wave to an entry where the entries fill the card with that, or in four rounds and are short for certain: four waves of which most find no
  // position cost a start and a join for it.  One token, four waves - of which three end at once where positions are 32 at the most - and one:
  // 241 sequences of two positions, 16 heads of 256 values, float16 102 and 30 us; 182 of up to 192, 16 of 80, float32 97 and 82; 250 of up to 60, 8
  // of 128 with four rows each, bfloat16 19.8 and 12.4; but in room for 512, 128 of up to 512, 16 of 64, float32 74 and 84.
  const bool one = entries >= 1024 * form || (entries >= 256 * form && capacity <= kPagesShort);
  p.waves = p.many ? pages_many_waves(width, p.dp, p.tile_rows) : one ? 1 : 4;
  // Parts for one round of the workgroups that run at a time, by the registers of their form, half a part for each sequence left out.  Of 16-bit values
  // half of them have the memory as busy, and leave fewer parts to join: where that makes two parts of a sequence.  One token, 8 heads with four
  // rows each, 128 values, all and half, over ten sets of lengths: 100003 positions 80.2 and 77.6 us, 4 sequences of up to 16000 44.2 and 42.0, 8
  // 75.1 and 72.4, but 16 of up to 32768 264 and 291; 4 drafted tokens, 4 heads with eight rows each, 16 of up to 16384 81.3 and 77.2, 40 of up to
  // 8192 96.9 and 101.  Not where rows leave many lanes without a load (80 values, 16 of up to 8192: 51.8 and 57.0), nor of float32 (64 values,
  // 16384: 83.4 and 88.2), nor of the form that shares positions in LDS (7 tokens, 24 of up to 8192: 75 and 108).
  const int to_a_simd = p.many ? pages_many_to_a_simd(width, p.dp, p.tile_rows) : form;
  // Many sequences leave few parts or none, and one of them may still have most of the positions: half of the parts there are anyway, where a row of
  // the table has room for that to show.  8 heads of 128 values with four rows each, 128 sequences, one of 4096 positions and the others of
  // 80: 55 and 22 us, all of up to 4096 269 and 269; but 200 of up to 700 76 and 79, by the look at all lengths.
  auto parts_of = [&](int64_t at_a_time) {
    const int64_t parts = at_a_time / (heads * p.row_tiles);
    return std::max<int64_t>({1, parts - sequences / 2, capacity > kPagesEven ? parts / 2 : 0});
  };
  const int64_t all = parts_of(1024 * to_a_simd / p.waves), half = parts_of(512 * to_a_simd / p.waves);
  p.target = width == 2 && !p.many && to_a_simd > 1 && 4 * dk > 3 * p.dp && half >= 2 * sequences ? half : all;
  // A sequence of up to four blocks stays whole, and where no row of the table has room for more nobody looks at the others' lengths (6 sequences
  // of up to 120 positions, 8 heads of 64 values, float32: 6.7 and 6.0 us).  Nor where these are many: their parts would be few, and a look at them
  // costs every workgroup a load for 64 of them (8 heads of 128 values with four rows each, all of 80 positions: 1024 sequences 95 us, 1025 72).  That is
  // wrong where one of many is long (one of 32768: 173 us, and 1729), and so is row_tiles where only one sequence has many new tokens: in a
  // batch with a prompt of 4096 tokens no sequence has parts (16 sequences, one token behind 80 positions 301 us, of one of them behind 32768 1538).
  if(capacity <= kCacheWhole * kCacheBlock || sequences > 1024) p.target = 1;
  p.least = entries <= 32 ? 2 : 4;
  p.items = p.target == 1 ? sequences : p.target + sequences;
  p.slots = p.target == 1 ? 0 : 2 * p.target;
  p.grid = (p.items * heads + 7) / 8 * 8 * p.row_tiles;
  return p;
}

// The workspace: counters as in that of the attention over a quantized cache, then the partial results: rows of dp values and a logarithm.
inline int64_t pages_attention_bytes(const PagesAttentionPlan& p, int64_t heads) {
  return p.slots == 0 ? 0 : kCacheCounterBytes + p.slots * heads * p.row_tiles * p.tile_rows * (p.dp + 1) * 4;
}

}  // namespace marian_hip
