"""The splits that a tree batch's sequences share, walked on the CPU: every length has its splits, no more
than there are, and they cover each sequence's keys once."""
import shutil
import subprocess
from pathlib import Path

from summa_amd import _lib

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "paged_map.hpp"
using namespace sm;
static unsigned long long z = 88172645463325252ull;
static unsigned rnd() { z ^= z << 13; z ^= z >> 7; z ^= z << 17; return (unsigned)(z >> 16); }
#define CHECK(x) do { if (!(x)) { printf("failed: %s line %d\n", #x, __LINE__); return 1; } } while (0)
int main() {
  for (unsigned by = 1; by < 3000; ++by)
    for (unsigned x : {0u, 1u, by - 1, by, by + 1, 7 * by, 7 * by + 1, (1u << 21) / by * by,
                       (1u << 21) / by * by - by, (1u << 21) / by * by - by + 1, (1u << 21) - 1,
                       rnd() % (1u << 21), 1u << 24, rnd() % (1u << 25)})
      CHECK(share_ceil(x, by) == (unsigned)(((unsigned long long)x + by - 1) / by));
  for (int it = 0; it < 20000; ++it) {
    const int S = 1 + rnd() % (it % 5 ? 40 : 256), share = S + 1 + rnd() % (it % 3 ? 20 : 1000);
    const int slots = 2 + rnd() % 40, G = 1 + rnd() % 8;
    const int most = it % 4 ? 1 << (rnd() % 20) : 1 << 27;
    std::vector<PagedKeys> keys;
    std::vector<int> pos, n;
    float all = 0;
    for (int s = 0; s < S; ++s) {
      const unsigned span = 1u << (rnd() % (it % 11 ? 18 : 31));
      pos.push_back((int)(rnd() % span) - (int)(rnd() % 50));
      n.push_back(rnd() % 9 ? 1 + rnd() % 64 : 0);
      keys.push_back(PagedKeys(pos[s], n[s], G, 0, n[s] * G, 1, 1, most));
      all += (float)((keys[s].blocks + kUnit - 1) / kUnit);
    }
    int lo, hi;
    PagedShare::bounds(all, S, share, lo, hi);
    CHECK(lo >= kShare && hi >= lo);
    auto units = [](const PagedKeys& k) { return (unsigned)(k.blocks + kUnit - 1) / kUnit; };
    auto total = [&](int cb) {
      long t = 0;
      for (auto& k : keys) t += PagedShare::most(units(k), cb, slots);
      return t;
    };
    CHECK(total(hi) <= share);
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (total(mid) <= share) hi = mid; else lo = mid + 1;
    }
    CHECK(total(lo) <= share);
    for (int s = 0; s < S; ++s) {
      const PagedShare ps(units(keys[s]), lo, slots);
      CHECK(ps.splits <= (int)PagedShare::most(units(keys[s]), lo, slots));
      CHECK(ps.splits >= 1 && ps.splits <= slots && ps.cb % kUnit == 0 && ps.cb > 0);
      const PagedKeys k(pos[s], n[s], G, 0, n[s] * G, ps.cb, ps.splits, most);
      CHECK(k.blocks == keys[s].blocks && k.splits == (k.blocks ? ps.splits : 0));
      int at = 0;
      for (int i = 0; i < k.splits; ++i) {
        CHECK(k.begin(i, ps.cb) == at && k.end(i, ps.cb) > at && k.end(i, ps.cb) - at <= ps.cb);
        at = k.end(i, ps.cb);
      }
      CHECK(at == k.blocks);
    }
  }
  printf("ok\n");
  return 0;
}
"""


def test_shared_splits(tmp_path):
    src, exe = tmp_path / "map.cpp", tmp_path / "map"
    src.write_text(PROGRAM)
    cxx = shutil.which("g++") or shutil.which("c++")
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(ROOT / "summa_amd" / "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_workspace():
    size = _lib.lib().sm_paged_tree_attention_workspace_bytes
    args = (2, 128, 64, 16, 4, 128)
    assert size(*args, 512) == 0 and size(*args, 1 << 17) > 0
    assert size(0, 0, 0, 16, 4, 128, 1 << 17) == 0
    assert size(2, 128, 64, 16, 4, 96, 1 << 17) == -1
    # a split more than sequences: two a row, and the counts
    assert size(255, 255, 1, 4, 4, 64, 1 << 20) == 255 * 4 * 2 * 66 * 4 + 1024
    assert size(257, 257, 1, 2, 2, 64, 513) == 257 * 2 * 2 * 66 * 4  # not shared
