"""Paged attention with many row tiles, long key spans and ragged batches: both workgroup sizes
of the tile kernel past their first rows and past the first 64 cache blocks of a split."""
import math

import pytest
import torch

import _paged as P
from test_paged_gpu import Batch, tolerance

pytestmark = pytest.mark.gpu
BF16, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def check_rows(b, q, got, lse, rows, dtype, cdt, kv=slice(None)):
    """Rows `rows` [(sequence, row of it)] against the definition, the heads of KV heads `kv`."""
    cached = tuple(x if x is None else x[:, kv] for x in b.store())
    q, got, lse = (x.unflatten(1, (b.KVH, -1))[:, kv].flatten(1, 2) for x in (q, got.cpu(), lse.cpu()))
    for s, i in rows:
        r = b.starts[s] + i
        ref, rl, mag, err, unit = P.attend(q[r:r + 1], cached, [b.table[s]], [b.pos0[s] + i], [0, 1],
                                           b.page)
        g, l = got[r:r + 1].double(), lse[r:r + 1].double()
        where = (s, i)
        assert torch.equal(torch.isnan(g), torch.isnan(ref)), where
        inf = torch.isinf(ref)
        assert torch.equal(g[inf], ref[inf]), where
        fin = torch.isfinite(ref)
        tol = tolerance(dtype, cdt, ref, mag, err, unit, b.hd)
        assert bool(((g - ref).abs() <= tol)[fin].all()), where
        f = torch.isfinite(rl)
        t = err.double() * (b.hd + 6) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * rl.abs()
        assert torch.equal(torch.isnan(l), torch.isnan(rl)) and bool(((l - rl).abs() <= t)[f].all()), where


def make(dev, pos0, n, H, KVH, hd, page, dtype, cdt, odd=()):
    """A filled batch and its queries; `odd`: (sequence, token, head, dim, value) of V."""
    b = Batch(dev, pos0, n, KVH, hd, page, cdt, pad_rows=1)
    k, v = (torch.randn(b.rows, KVH, hd) for _ in range(2))
    b.fill()
    for s, t, h, d, x in odd:
        if t >= pos0[s]:
            v[b.starts[s] + t - pos0[s], h, d] = x
    b.append(k.to(dev), v.to(dev))
    for s, t, h, d, x in odd:  # (earlier tokens: where they lie)
        if t < pos0[s]:
            flat = b.cache.v.view(torch.uint8 if cdt == F8 else b.cache.v.dtype).flatten(3)
            at = int(P.v_index(hd, 4 if cdt == F8 else 2)[t % 16, d])
            flat[b.table[s][t // page], h, t % page // 16, at] = 0x7f if cdt == F8 else x
    return b, torch.randn(b.rows, H, hd).to(dtype)


WIDE = [  # pos0, n, H, KVH
    ([2500, 1900, 2300, 2450], [512, 450, 333, 512], 32, 8),  # one split, 8 tiles of 256 rows
    ([18000, 9000], [256, 131], 16, 4),                       # 8 splits of 2304 keys, 4 tiles
]


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, F8), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("case", range(len(WIDE)))
def test_many_tiles_of_256_rows(dev, case, dtype, cdt):
    """Heads of 128, four to a KV head: a row of every tile and the rows at its edges, with
    more than 128 cache blocks to a split."""
    pos0, n, H, KVH = WIDE[case]
    print(f"case wide {case} {dtype} {cdt}", flush=True)
    b, q = make(dev, pos0, n, H, KVH, 128, 64, dtype, cdt)
    out, lse = b.attention(q.to(dev), want_lse=True, max_tokens=max(p + m for p, m in zip(pos0, n)))
    rows = [(s, i) for s, m in enumerate(n) for i in
            sorted({0, m - 1} | {x for x in range(0, m, 64)} | {x + 63 for x in range(0, m - 63, 128)})]
    check_rows(b, q, out, lse, rows, dtype, cdt, [0, KVH // 2, KVH - 1])


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, BF16)])
def test_tiles_of_256_rows_with_odd_values_and_pages(dev, dtype, cdt):
    """As above in one split: a page that is none in the second 64 blocks of one sequence and in
    the third of another, values that are not finite in each 64 blocks, seen by all, some or no
    rows, and (8 bits) scales beyond 2^17 from the second 64 on."""
    pos0, n = [1000, 2100, 2300, 2100], [512, 512, 300, 512]
    print(f"case wide odd {dtype} {cdt}", flush=True)
    odd = [(0, 3, 0, 5, math.inf), (0, 1200, 1, 100, -math.inf), (1, 1100, 2, 64, math.nan),
           (1, 2300, 3, 127, math.inf), (2, 2100, 4, 0, math.inf), (2, 2599, 5, 33, math.inf)]
    b, q = make(dev, pos0, n, 32, 8, 128, 64, dtype, cdt, odd)
    for s, t in ((0, 1408), (3, 2432)):
        b.t[s, t // 64] = -1
        b.table[s][t // 64] = -1
    if cdt == F8:
        b.cache.v_scales[torch.tensor(b.table[2][20:30]).to(dev)] += 60
    out, lse = b.attention(q.to(dev), want_lse=True, max_tokens=2612)
    rows = [(0, 0), (0, 199), (0, 200), (0, 407), (0, 408), (0, 511), (1, 0), (1, 130), (1, 199), (1, 200),
            (1, 511), (2, 0), (2, 100), (2, 298), (2, 299), (3, 0), (3, 331), (3, 332), (3, 511)]
    if dtype == F16:  # (values of 2^60 leave f16)
        rows = [r for r in rows if cdt != F8 or r[0] != 2]
    check_rows(b, q, out, lse, rows, dtype, cdt)


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, F8), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [40, 200])
def test_long_sweeps_of_128_rows(dev, n, hd, dtype, cdt):
    """More than 128 cache blocks in one split (the longest sequence understated): a page that is
    none in the second and in the third 64 blocks, values that are not finite in both."""
    print(f"case sweep {n} {hd} {dtype} {cdt}", flush=True)
    pos0 = [2150, 1100, 2150 + n, 3000]
    odd = [(0, 1500, 0, 3, math.inf), (0, 2100, 1, 60, math.nan), (0, 2150 + n // 2, 2, 9, -math.inf),
           (1, 1090, 0, 11, -math.inf), (1, 1100 + n - 1, 1, 12, math.inf), (2, 2140, 2, 13, math.inf)]
    b, q = make(dev, pos0, [n] * 4, 3, 3, hd, 32, dtype, cdt, odd)
    for s, t in ((1, 1100 + n // 2), (2, 2150 + n + n // 2)):
        col = -(-t // 32)
        if col < len(b.table[s]):
            b.t[s, col] = b.pages
            b.table[s][col] = -1
    out, lse = b.attention(q.to(dev), want_lse=True, max_tokens=1)
    rows = [(s, i) for s in range(4) for i in sorted({0, n // 2 - 1, n // 2, n // 2 + 1, n - 1, n - 2,
                                                      min(n - 1, 127), min(n - 1, 128)})]
    check_rows(b, q, out, lse, rows, dtype, cdt)


def test_one_long_sequence_among_many(dev):
    """128 sequences, one of 32768 rows and the others of one: the longest's rows count for all
    in the grid, and 128 x 32768 x 16 is 2^26."""
    S, most = 128, 32768
    n = [1] * S
    n[17] = most
    pos0 = [5] * S
    pos0[17] = 0
    b, q = make(dev, pos0, n, 16, 1, 64, 256, F16, F8)
    out, lse = b.attention(q.to(dev), want_lse=True, max_tokens=most)
    check_rows(b, q, out, lse, [(0, 0), (16, 0), (17, 0), (17, 1), (17, 8191), (17, 20000), (17, most - 1),
                                (18, 0), (127, 0)], F16, F8)


@pytest.mark.parametrize("cdt", [F8, BF16])
@pytest.mark.parametrize("hd,n", [(64, 60), (128, 300)])
def test_a_captured_chunk(dev, hd, n, cdt):
    """A chunk's append and attention captured once and replayed as the sequences grow, its rows
    fewer than max_rows at times, with eager work between: bit for bit the eager calls."""
    from summa_amd import ops, paged
    H, KVH, page, S = 8, 2, 64, 2
    cache = paged.PagedKVCache(48, KVH, hd, page, cdt, dev)
    table = torch.randperm(48, device=dev).int().view(S, 24).contiguous()
    rope = ops.rope_table(24 * page, hd, device=dev)
    cur = torch.empty(S * n, H + 2 * KVH, hd, dtype=BF16, device=dev)
    pos = torch.zeros(S, dtype=torch.int32, device=dev)
    st = torch.zeros(S + 1, dtype=torch.int32, device=dev)
    out = torch.empty(S * n, H, hd, dtype=BF16, device=dev)
    chunks = []
    at = [0, 0]
    for m in ([n, n], [n - 7, 1], [1, n], [n // 2, 0], [n, n - 1]):
        chunks.append((torch.randn_like(cur), list(at), m))
        at = [x + y for x, y in zip(at, m)]
    assert max(at) <= 24 * page

    def set_up(x, at, m):
        cur.copy_(x)
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        st.copy_(torch.tensor([0, m[0], m[0] + m[1]], dtype=torch.int32))
        out.zero_()

    def chunk():
        q, k, v = cur.split([H, KVH, KVH], 1)
        qr = paged.paged_append(cache, k, v, table, pos, st, q=q, rope_table=rope, layout="half",
                                max_rows=n, q_dtype=BF16)
        paged.paged_attention(cache, qr, table, pos, st, max_rows=n, out=out)

    def clear():
        for x in (cache.k, cache.v):
            x.view(torch.uint8).zero_()
        if cdt == F8:
            cache.k_scales.zero_()
            cache.v_scales.zero_()

    eager = []
    for c in chunks:
        set_up(*c)
        chunk()
        eager.append(out.clone())
    assert all(bool(torch.isfinite(x).all()) for x in eager)
    set_up(*chunks[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chunk()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chunk()
    for again in range(2):
        clear()
        for c, want in zip(chunks, eager):
            set_up(*c)
            g.replay()
            assert torch.equal(out, want), (again, c[1:])
            torch.cuda.synchronize()
