"""The paged batch's map (csrc/paged_map.hpp) walked on the CPU - rows whatever row_start
holds, pages outside the pool, key splits - and the refusals of the paged calls, which
come before any device work."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from summa_amd import _lib

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged_map.hpp"
using namespace sm;
static unsigned long long z = 88172645463325252ull;
static unsigned rnd() { z ^= z << 13; z ^= z >> 7; z ^= z << 17; return (unsigned)(z >> 16); }
#define CHECK(x) do { if (!(x)) { printf("failed: %s line %d\n", #x, __LINE__); return 1; } } while (0)
int main() {
  // rows: whatever row_start holds, they lie inside [0, rows) and number at most max_rows
  for (int it = 0; it < 200000; ++it) {
    const int rows = rnd() % 1000, most = rows ? rnd() % (rows + 1) : 0;
    int32_t st[2] = {(int32_t)rnd(), (int32_t)rnd()};
    if (it % 3 == 0) { st[0] = rnd() % 1200 - 100; st[1] = rnd() % 1200 - 100; }
    const PagedRows p(st, 0, rows, most);
    CHECK(p.n >= 0 && p.n <= most && p.first >= 0 && p.first + p.n <= rows);
    if (st[0] >= 0 && st[1] >= st[0] && st[1] <= rows && st[1] - st[0] <= most)
      CHECK(p.first == st[0] && p.n == st[1] - st[0]);
  }
  const PagedRows even(nullptr, 3, 20, 5);
  CHECK(even.first == 15 && even.n == 5);
  // blocks: inside the cache or -1
  for (int it = 0; it < 200000; ++it) {
    const int cols = 1 + rnd() % 6, pages = 1 + rnd() % 9, KVH = 1 + rnd() % 5, bpp = 1 + rnd() % 9;
    int32_t row[6];
    for (int i = 0; i < 6; ++i) row[i] = it % 2 ? (int)(rnd() % (pages + 4)) - 2 : (int32_t)rnd();
    const int blk = (int)(rnd() % (cols * bpp + 20)) - 5, kvh = rnd() % KVH;
    const int b = paged_block(row, cols, pages, KVH, kvh, bpp, blk);
    const bool ok = blk >= 0 && blk / bpp < cols && row[blk / bpp] >= 0 && row[blk / bpp] < pages;
    CHECK(ok ? b == (row[blk / bpp] * KVH + kvh) * bpp + blk % bpp : b == -1);
    CHECK(b < pages * KVH * bpp);
  }
  // blocks that n tokens touch, wherever they start
  for (int n = 1; n < 100; ++n) {
    int most = 0;
    for (int p = 0; p < 16; ++p) {
      const int t = (p + n - 1) / 16 - p / 16 + 1;
      most = t > most ? t : most;
    }
    CHECK(paged_touched(n) == most);
  }
  // division by a known divisor
  const int ds[] = {1, 2, 3, 5, 7, 10, 12, 48, 641, 65535, 65536, 1 << 24, 0x3fffffff, 0x40000001, 0x7fffffff};
  for (int d : ds) {
    const Divide by(d);
    for (int it = 0; it < 20000; ++it) {
      int n = it < 4 ? 0x7fffffff - it : it < 8 ? it - 4 : (int)(rnd() & 0x7fffffff) >> (it % 31);
      CHECK(by.div(n) == n / d);
      int q = n;
      CHECK(by.mod(q) == n % d && q == n / d);
    }
  }
  // workgroups: every (group, place) once; whole eights of groups one XCD each, every XCD
  // every group of a set in some set
  for (int wide = 0; wide < 2; ++wide)
    for (uint32_t groups : {1u, 3u, 4u, 8u, 16u, 23u, 128u, 1000u})
      for (uint32_t per : {1u, 2u, 7u, 16u, 33u}) {
        const PagedMap map(groups, per, wide != 0);
        std::vector<int> seen(groups * per, 0), home(groups, -1);
        uint32_t last = 0;
        for (long w = 0; w < map.map.workgroups(); ++w) {
          uint32_t g, p;
          if (!map.at((uint32_t)w, g, p)) continue;
          CHECK(g < groups && p < per);
          seen[g * per + p]++;
          if (g < groups / 8 * 8) {
            CHECK(home[g] < 0 || home[g] == w % 8);
            home[g] = (int)(w % 8);
            if (wide) {
              CHECK(p >= last);
              last = p;
            }
          }
        }
        for (int n : seen) CHECK(n == 1);
      }
  // splits: every key block of a tile exactly once, none beyond the last key
  for (int it = 0; it < 100000; ++it) {
    const int G = 1 + rnd() % 9, n = 1 + rnd() % 40, tile = it % 2 ? 16 : 128;
    const int pos0 = it % 5 ? (int)(rnd() % 3000) - 20 : 0x7fffffff - (int)(rnd() % 3);
    const int cb = 16 * (1 + rnd() % 8), nsplit = 1 + rnd() % 12;
    const int row0 = rnd() % (n * G) / tile * tile;
    const PagedKeys k(pos0, n, G, row0, tile, cb, nsplit);
    int last = row0 + tile - 1;
    if (last >= n * G) last = n * G - 1;
    long keys = (long)pos0 + last / G + 1;
    if (keys < 0) keys = 0;
    if (keys > 0x7fffffff) keys = 0x7fffffff;
    CHECK(k.keys == keys && k.blocks == (keys + 15) / 16 && k.splits <= nsplit);
    CHECK((k.splits == 0) == (keys == 0));
    int at = 0;
    for (int i = 0; i < k.splits; ++i) {
      CHECK(k.begin(i, cb) == at && k.end(i, cb) > at);
      at = k.end(i, cb);
    }
    CHECK(at == k.blocks);
    // no more blocks than a table row holds and one
    const int most = 1 + rnd() % 200;
    const PagedKeys c(pos0, n, G, row0, tile, cb, nsplit, most);
    CHECK(c.blocks == (k.blocks < most ? k.blocks : most) && c.keys <= k.keys);
    CHECK(c.keys == (k.blocks <= most ? k.keys : most * 16) && c.splits <= k.splits);
    CHECK(c.splits == 0 || c.end(c.splits - 1, cb) == c.blocks);
  }
  printf("ok\n");
  return 0;
}
"""


def test_paged_map(tmp_path):
    src, exe = tmp_path / "map.cpp", tmp_path / "map"
    src.write_text(PROGRAM)
    cxx = shutil.which("g++") or shutil.which("c++")
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(ROOT / "summa_amd" / "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


D = 1 << 20  # a device pointer that is never dereferenced: each call fails its checks first


def cache(**kw):
    v = dict(k=D, v=D, k_scales=D, v_scales=D, pages=4, kv_heads=2, page_tokens=32, head_dim=64,
             dtype=_lib.SM_F8E4M3)
    v.update(kw)
    return _lib.PagedCache(*v.values())


def append(c, **kw):
    v = dict(table=D, cols=4, pos0=D, starts=None, S=2, rows=2, most=1, q=None, ldq=0, k=D, ldk=128,
             v=D, ldv=128, dt=_lib.SM_BF16, H=0, rope=None, rope_rows=0, rot=0, layout=0, out=None,
             qd=_lib.SM_F16)
    v.update(kw)
    st = _lib.lib().sm_paged_append(c if c is None else ctypes.addressof(c), *v.values(), None)
    return st, _lib.lib().sm_last_error().decode()


def attention(c, **kw):
    v = dict(table=D, cols=4, pos0=D, starts=None, S=2, rows=2, most=1, tokens=128, q=D,
             dt=_lib.SM_BF16, ldq=256, H=4, out=D, lse=None, ws=None, wsb=0)
    v.update(kw)
    st = _lib.lib().sm_paged_attention(c if c is None else ctypes.addressof(c), *v.values(), None)
    return st, _lib.lib().sm_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=_lib.SM_F32), "cache dtype must be"), (dict(head_dim=96), "head_dim must be 64 or 128"),
    (dict(page_tokens=24), "multiple of 16"), (dict(page_tokens=0), "multiple of 16"),
    (dict(pages=0), "need pages"), (dict(kv_heads=0), "need pages"),
    (dict(pages=1 << 30, kv_heads=8), "2^31 blocks"), (dict(k=None), "null cache pages"),
    (dict(v=D + 8), "16-byte aligned"), (dict(k_scales=None), "needs k_scales"),
    (dict(v_scales=None), "needs k_scales and v_scales"),
])
def test_cache_descriptors_refused(kw, msg):
    for call in (append, attention):
        st, err = call(cache(**kw))
        assert st == -1 and msg in err


def test_null_cache_refused():
    for call in (append, attention):
        st, err = call(None)
        assert st == -1 and "null cache" in err


@pytest.mark.parametrize("kw,msg", [
    (dict(dt=7), "dtype must be"), (dict(S=-1), "need S >= 0"), (dict(most=3), "max_rows <= rows"),
    (dict(rows=3, most=1), "rows must be S * max_rows"), (dict(ldk=64), "hold their heads"),
    (dict(ldv=132), "16-byte aligned"), (dict(k=D + 2), "16-byte aligned"),
    (dict(k=None), "null buffer"), (dict(pos0=None), "null buffer"), (dict(cols=0), "table_cols"),
    (dict(q=D, ldq=256, H=0, out=D), "query heads"), (dict(q=D, ldq=256, H=4), "null buffer"),
    (dict(q=D, ldq=128, H=4, out=4 * D), "hold their heads"),
    (dict(q=D, ldq=256, H=4, out=4 * D, qd=_lib.SM_F32), "q_dtype must be"),
    (dict(q=D, ldq=256, H=4, out=D + 512), "must not overlap"),
    (dict(q=D, ldq=256, H=4, out=8 * D, k=8 * D + 64), "must not overlap q, k or v"),
    (dict(q=D, ldq=256, H=4, out=8 * D, v=8 * D - 128), "must not overlap q, k or v"),
    (dict(rot=32), "rot_dim without"), (dict(rope=D, rot=32), "have rows"),
    (dict(rope=D, rot=24, rope_rows=8), "multiple of 16 up to head_dim"),
    (dict(rope=D, rot=128, rope_rows=8), "multiple of 16 up to head_dim"),
    (dict(rope=D, rot=32, rope_rows=8, layout=2), "layout must be"), (dict(rope=D + 4, rot=32), "rope_table must"),
])
def test_append_refusals(kw, msg):
    st, err = append(cache(), **kw)
    assert st == -1 and msg in err, err


@pytest.mark.parametrize("kw,msg", [
    (dict(dt=_lib.SM_F32), "dtype must be"), (dict(H=5), "multiple of KVH"), (dict(H=0), "multiple of KVH"),
    (dict(most=3), "max_rows <= rows"), (dict(rows=3), "rows must be S * max_rows"),
    (dict(ldq=128), "ldq >= H * head_dim"), (dict(ldq=260), "16-byte aligned"),
    (dict(q=D + 8), "16-byte aligned"), (dict(out=D + 8), "16-byte aligned"),
    (dict(out=None), "null buffer"), (dict(table=None), "null buffer"), (dict(cols=0), "table_cols"),
    (dict(tokens=-1), "max_tokens"), (dict(tokens=1 << 31), "max_tokens"),
    (dict(tokens=1 << 20), "needed"), (dict(tokens=1 << 20, ws=D + 8, wsb=1 << 40), "16-byte aligned"),
])
def test_attention_refusals(kw, msg):
    st, err = attention(cache(), **kw)
    assert st == -1 and msg in err, err


def test_more_refusals():
    for kw in (dict(out=D), dict(out=D + 512), dict(out=D - 512), dict(q=D + 256, ldq=512)):
        st, err = attention(cache(), **kw)
        assert st == -1 and "out must not overlap q" in err, err
    st, err = attention(cache(), ldq=1 << 31)
    assert st == -1 and "ldq < 2^31" in err
    for kw in (dict(ldk=1 << 31), dict(ldv=1 << 40), dict(q=D, ldq=1 << 62, H=4, out=4 * D)):
        st, err = append(cache(), **kw)
        assert st == -1 and "hold their heads" in err
    # workspace bytes that no card holds, and no 64-bit sum
    assert _lib.lib().sm_paged_attention_workspace_bytes(1, (1 << 31) - 2, 1, 65535, 1, 128, 1 << 30) == -1


def test_attention_types_have_to_agree():
    for c, q in ((_lib.SM_F16, _lib.SM_BF16), (_lib.SM_BF16, _lib.SM_F16)):
        st, err = attention(cache(dtype=c), dt=q)
        assert st == -1 and "must have the query's dtype" in err


def test_problems_beyond_a_grid_are_refused():
    st, err = attention(cache(), S=1 << 23, rows=1 << 24, most=2)
    assert st == -3 and "too large" in err
    st, err = append(cache(), S=1 << 25, rows=1 << 25, most=1)
    assert st == -3 and "too large" in err
    assert _lib.lib().sm_paged_attention_workspace_bytes(1 << 23, 1 << 24, 2, 4, 2, 64, 64) == -1


def test_empty_batches_do_nothing():
    for call in (append, attention):
        assert call(cache(), S=0, rows=0, most=0)[0] == 0
        assert call(cache(), rows=0, most=0)[0] == 0
    assert _lib.lib().sm_paged_attention_workspace_bytes(0, 0, 0, 4, 2, 64, 64) == 0
    assert _lib.lib().sm_paged_attention_workspace_bytes(1, 1, 1, 4, 2, 96, 64) == -1


def test_rope_host_refusals():
    L = _lib.lib()
    bad = [((float("nan"), 64, 8, 0, 1, 0, 0, 0, 1), "theta"), ((1e4, 63, 8, 0, 1, 0, 0, 0, 1), "even"),
           ((1e4, 64, -1, 0, 1, 0, 0, 0, 1), "positions"), ((1e4, 64, 8, 9, 1, 0, 0, 0, 1), "scaling"),
           ((1e4, 64, 8, 1, 0, 0, 0, 0, 1), "factor"), ((1e4, 2, 8, 2, 2, 0, 0, 0, 1), "rot_dim > 2"),
           ((1e4, 64, 8, 3, 2, 0, 1, 8, 1), "original_positions"),
           ((1e4, 64, 8, 3, 2, 64, 8, 8, 1), "low_turns"), ((1e4, 64, 8, 0, 1, 0, 0, 0, 0), "magnitude")]
    for args, msg in bad:
        st = L.sm_rope_table(*args, D, None)
        assert st == -1 and msg in L.sm_last_error().decode(), args
    assert L.sm_rope_table(1e4, 64, 0, 0, 1, 0, 0, 0, 1, None, None) == 0
    ok = dict(x=D, ldx=128, y=2 * D, ldy=128, dt=0, t=D, tr=8, p=D, rows=4, heads=2, hd=64, rot=32,
              layout=0, back=0)
    for kw, msg in [(dict(dt=3), "dtype"), (dict(layout=5), "layout"), (dict(rows=-1), "rows"),
                    (dict(rows=(1 << 26) - 4), "rows"), (dict(tr=0), "no rows"),
                    (dict(heads=0), "heads"), (dict(hd=72), "head_dim"), (dict(rot=8), "rot_dim"),
                    (dict(rot=80), "rot_dim"), (dict(ldx=64), "hold heads"), (dict(ldy=130), "aligned"),
                    (dict(x=D + 4), "aligned"), (dict(t=D + 8), "aligned"), (dict(y=D + 64), "overlap"),
                    (dict(y=D, ldy=192), "overlap"), (dict(p=None), "null")]:
        v = dict(ok)
        v.update(kw)
        st = L.sm_rope(*v.values(), None)
        assert st == -1 and msg in L.sm_last_error().decode(), (kw, L.sm_last_error())
