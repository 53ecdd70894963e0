"""What the attention over a quantized cache keeps in LDS is read and written 16 bytes at a time: its types say that they begin
there (nothing else would, of members of two and four bytes)."""
import os
import subprocess

import pytest

from conftest import PKG, ROOT

HIPCC = "/opt/rocm/bin/hipcc"
TYPES = """
#include "cache_attention_kernel.h"
using namespace marian_hip;
template <int DP, int QT>
constexpr bool joins() { return alignof(CacheJoin<DP, QT, 1>) % 16 == 0 && alignof(CacheJoin<DP, QT, 2>) % 16 == 0 && alignof(CacheJoin<DP, QT, 4>) % 16 == 0; }
static_assert(joins<64, 1>() && joins<64, 2>() && joins<128, 1>() && joins<128, 2>() && joins<256, 1>(), "rows of results");
template <typename T, CacheFormat F, int DP, int ROWS, int WAVES>
constexpr bool shared() {
  using U = CacheFewShared<T, F, DP, ROWS, WAVES>;
  return alignof(U) % 16 == 0 && sizeof(typename CacheFew<T, F, DP, ROWS>::Weights) % 16 == 0;
}
template <typename T, CacheFormat F, int DP, int WAVES>
constexpr bool rows() { return shared<T, F, DP, 1, WAVES>() && shared<T, F, DP, 2, WAVES>() && shared<T, F, DP, 4, WAVES>() && shared<T, F, DP, 8, WAVES>(); }
template <typename T, CacheFormat F>
constexpr bool all() { return rows<T, F, 64, 1>() && rows<T, F, 64, 2>() && rows<T, F, 64, 4>() && rows<T, F, 128, 1>() && rows<T, F, 128, 2>() && rows<T, F, 128, 4>(); }
static_assert(all<float, CacheFormat::int8>() && all<_Float16, CacheFormat::e4m3>() && all<bf16_t, CacheFormat::int8>(), "weights");
"""


def test_lds_begins_on_16_bytes(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    (tmp_path / "types.hip").write_text(TYPES)
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-std=c++17", "--cuda-host-only", "-fsyntax-only", "-I", os.path.join(ROOT, PKG, "csrc"),
                        str(tmp_path / "types.hip")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
