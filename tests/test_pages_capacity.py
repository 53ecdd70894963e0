"""The plan of an attention over pages for the rows of the table that a call brings, against the workspace that was asked for without them."""
import os
import subprocess

from conftest import PKG, ROOT

SWEEP = r"""
#include "pages_plan.h"
#include <cstdio>
#include <random>
using namespace marian_hip;
int main() {
  std::mt19937_64 rng(5);
  auto one_of = [&](std::initializer_list<int64_t> x) { return x.begin()[rng() % x.size()]; };
  int64_t split = 0;
  for(int i = 0; i < 400000; ++i) {
    const int64_t few[] = {1, 2, 3, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1023, 1024, 1025, 4096, 65535};
    const int64_t s = rng() % 2 ? few[rng() % (sizeof(few) / 8)] : 1 + rng() % 1100, h = one_of({1, 2, 3, 4, 7, 8, 16, 32, 64, 128}), hq = h * one_of({1, 2, 3, 4, 8, 16, 64});
    const int64_t n = one_of({1, 1, 1, 2, 4, 7, 8, 16, 17, 64, 100, 1000, 5000}), dk = one_of({16, 48, 64, 80, 96, 128, 144, 256});
    const int width = rng() % 2 ? 2 : 4;
    const int64_t capacity = rng() % 2 ? one_of({8, 64, 120, 128, 136, 248, 256, 264, 504, 512, 520, 1016, 1024, 1032, 2048, 4096, (1 << 30) - 8}) : 8 * (1 + rng() % 2000);
    const PagesAttentionPlan p = pages_attention_plan(s, h, hq, n, dk, width, capacity), asked = pages_attention_plan(s, h, hq, n, dk, width);
    const int64_t bytes = pages_attention_bytes(p, h), room = pages_attention_bytes(asked, h);
    bool good = bytes <= room && p.row_tiles * p.tile_rows >= n * (hq / h) && p.grid >= p.items * h * p.row_tiles;
    if(p.target > 1) {
      ++split;
      // sequences of all positions that a row has room for, and one of all among empty ones: parts, as the kernel counts them
      const int64_t blocks = (capacity + kCacheBlock - 1) / kCacheBlock;
      for(int64_t full : {s, (int64_t)1, s / 2 + 1}) {
        const int64_t each = std::max<int64_t>(p.least, (full * blocks + p.target - 1) / p.target);
        const int64_t size = std::max<int64_t>(blocks <= (int64_t)kCacheWhole ? std::max<int64_t>(each, kCacheWhole) : each, (blocks + kPagesMostParts - 1) / kPagesMostParts);
        const int64_t parts = (blocks + size - 1) / size, several = parts > 1 ? parts * full : 0, all = parts * full + s - full;
        good = good && all <= p.items && several <= p.slots && several < 4096 && all < 1 << 20 && several * h * p.row_tiles <= kCacheMost;
      }
    }
    if(!good) {
      std::printf("%lld %lld %lld %lld %lld %d %lld: %lld of %lld\n", (long long)s, (long long)h, (long long)hq, (long long)n, (long long)dk, width, (long long)capacity,
                  (long long)bytes, (long long)room);
      return 1;
    }
  }
  std::printf("%lld\n", (long long)split);
  return split > 20000 ? 0 : 2;
}
"""


def test_a_call_needs_no_more_than_it_was_told(tmp_path):
    """Plans of random calls with rows of all sizes: their workspace is no larger than what the query, which knows no rows, says; the parts of
    full and of single long sequences stay within the launch, the workspace, the counters and the bits that they are counted in"""
    (tmp_path / "sweep.cpp").write_text(SWEEP)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, PKG, "csrc"), "-o", str(tmp_path / "sweep"), str(tmp_path / "sweep.cpp")], check=True)
    got = subprocess.run([str(tmp_path / "sweep")], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout
