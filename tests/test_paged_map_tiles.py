"""The key ranges of a paged batch's row tiles, tiles of 256 rows among them, walked on the
CPU: a split's ranges cover every key that a tile's rows see once, whatever the lengths."""
import shutil
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include "paged_map.hpp"
using namespace sm;
static unsigned long long z = 88172645463325252ull;
static unsigned rnd() { z ^= z << 13; z ^= z >> 7; z ^= z << 17; return (unsigned)(z >> 16); }
#define CHECK(x) do { if (!(x)) { printf("failed: %s line %d\n", #x, __LINE__); return 1; } } while (0)
int main() {
  const int tiles[] = {16, 128, 256};
  for (int it = 0; it < 300000; ++it) {
    const int tile = tiles[it % 3], G = 1 + rnd() % 16, n = 1 + rnd() % 700;
    const int pos0 = it % 7 ? (int)(rnd() % 40000) - 300 : 0x7fffffff - (int)(rnd() % 1000);
    const int cb = 16 * (2 + rnd() % 30), nsplit = 1 + rnd() % 40, most = 1 + rnd() % 3000;
    for (int row0 = 0; row0 < n * G; row0 += tile) {
      const PagedKeys k(pos0, n, G, row0, tile, cb, nsplit, most);
      // the tile's last row and, one by one, what its rows see
      long last = 0;
      for (int r = row0; r < row0 + tile && r < n * G; ++r) {
        const long sees = (long)pos0 + r / G + 1;
        last = sees > last ? sees : last;
      }
      const long held = (long)most * 16;
      if (last > held) last = held;
      if (last > 0x7fffffff) last = 0x7fffffff;
      CHECK(k.keys == last && k.blocks == (last + 15) / 16 && k.blocks <= most);
      CHECK(k.splits <= nsplit && (k.splits == 0) == (last == 0));
      int at = 0;
      for (int i = 0; i < k.splits; ++i) {
        CHECK(k.begin(i, cb) == at && k.end(i, cb) > at);
        CHECK(i + 1 == k.splits || k.end(i, cb) - at == cb);
        at = k.end(i, cb);
      }
      CHECK(at == k.blocks);
      // the join finds a row's tile, and with it the same ranges, from the row alone
      const int row = row0 + (int)(rnd() % (unsigned)tile);
      if (row < n * G) {
        const Divide by(tile);
        const PagedKeys j(pos0, n, G, by.div(row) * tile, tile, cb, nsplit, most);
        CHECK(j.splits == k.splits && j.blocks == k.blocks);
      }
    }
  }
  printf("ok\n");
  return 0;
}
"""


def test_key_ranges_of_row_tiles(tmp_path):
    src, exe = tmp_path / "map.cpp", tmp_path / "map"
    src.write_text(PROGRAM)
    cxx = shutil.which("g++") or shutil.which("c++")
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(ROOT / "summa_amd" / "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
