"""Trees of drafted tokens over the paged cache against 64-bit definitions: masks, attention, the
confirmed path and its tokens moved together."""
import math

import pytest
import torch

import _paged as P
import _tree as R
from test_paged_gpu import BF16, F16, F32, F8, Batch, tolerance

pytestmark = pytest.mark.gpu
PAIRS = [(F16, F8), (BF16, F8), (F16, F16), (BF16, BF16)]


def tree_batch(dev, pos0, n, KVH, hd, page, cdt, pad_rows=0, ragged=None):
    b = Batch(dev, pos0, n, KVH, hd, page, cdt, pad_rows=pad_rows, ragged=ragged)
    b.fill()
    k, v = torch.randn(2, b.rows, KVH, hd)
    b.append(k.to(dev), v.to(dev))
    return b


def random_masks(b, gen, kind):
    """Sets of rows that each row sees."""
    sees = []
    for n in b.n:
        if kind == "tree":
            sees += R.masks(R.random_tree(n, gen))[0]
        elif kind == "any":
            sees += [{j for j in range(n) if torch.rand(1, generator=gen) < 0.3} for _ in range(n)]
        else:
            sees += [set() if i % 2 else {n - 1} for i in range(n)]
    return sees + [set()] * (b.rows - b.starts[-1])


def attention(b, q, mask, **kw):
    from summa_amd import paged
    kw.setdefault("max_rows", b.most)
    return paged.paged_tree_attention(b.cache, q, mask, b.t, b.p, b.rs, **kw)


def check(b, q, sees, got, lse=None, heads=None):
    cached = b.store() if heads is None else tuple(x if x is None else x[:, heads] for x in b.store())
    n = b.starts[-1]
    ref, rl, mag, err, unit = (x[:n] for x in R.attend(q[:b.rows], cached, b.table, b.pos0, b.starts,
                                                       b.page, sees))
    got = got.cpu().double()[:n]
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    fin = torch.isfinite(ref)
    tol = tolerance(q.dtype, b.dtype, ref, mag, err, unit, b.hd)
    assert bool(((got - ref).abs() <= tol)[fin].all()), float(((got - ref).abs() - tol)[fin].max())
    if lse is not None:
        lse = lse.cpu().double()[:n]
        assert torch.equal(torch.isneginf(lse), torch.isneginf(rl))
        f = torch.isfinite(rl)
        t = err.double() * (b.hd + 6) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * rl.abs()
        assert bool(((lse - rl).abs() <= t)[f].all())


CASES = [  # pos0, n, H, KVH, hd, page
    ([0], [1], 1, 1, 64, 16),
    ([0, 5, 16, 33], [4, 4, 4, 4], 4, 4, 128, 16),
    ([70, 0, 333], [6, 6, 6], 8, 2, 64, 32),
    ([5, 0, 130, 15], [40, 1, 17, 33], 8, 2, 64, 32),
    ([200, 64], [64, 64], 4, 1, 128, 64),
    ([600, 1], [65, 31], 2, 2, 64, 48),
    ([40], [150], 6, 2, 128, 64),
    ([-3, -40, 0, 7], [20, 12, 33, 2], 4, 2, 64, 16),
    ([30, 0], [300, 7], 3, 3, 64, 128),
    ([128, 100], [20, 20], 64, 2, 128, 64),   # 640 rows a KV head
]


@pytest.mark.parametrize("dtype,cdt", PAIRS)
@pytest.mark.parametrize("kind", ["tree", "any", "few"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_tree_attention(dev, case, kind, dtype, cdt):
    pos0, n, H, KVH, hd, page = CASES[case]
    print(f"case tree {case} {kind} {dtype} {cdt}", flush=True)
    b = tree_batch(dev, pos0, n, KVH, hd, page, cdt, pad_rows=2 if len(set(n)) > 1 else 0)
    gen = torch.Generator().manual_seed(case)
    sees = random_masks(b, gen, kind)
    w = (max(n) + 31) // 32 + (case % 2)      # a word more than needed
    mask = R.words(sees, w)
    junk = torch.randint(-2 ** 31, 2 ** 31, mask.shape, generator=gen).to(torch.int32)
    for s, m in enumerate(n):                 # bits of rows that the sequence does not have
        for j in range(m, 32 * w):
            bit = torch.tensor(1 << (j % 32), dtype=torch.int64)
            sl = mask[b.starts[s]:b.starts[s + 1], j // 32]
            sl |= (junk[b.starts[s]:b.starts[s + 1], j // 32].long() & bit).where(
                torch.tensor(j % 32 < 31), torch.tensor(0)).to(torch.int32)
    wide = (torch.randn(b.rows, H + 3, hd) * 1.5).to(dtype)
    q, qd = wide[:, :H], wide.to(dev)[:, :H]
    out = torch.full((b.rows, H, hd), 5.0, dtype=dtype, device=dev)
    got, lse = attention(b, qd, mask.to(dev), want_lse=True, out=out)
    assert bool((out[b.starts[-1]:] == 5).all())
    check(b, q, sees, got, lse)
    got = attention(b, qd, mask.to(dev), max_tokens=1)
    check(b, q, sees, got)


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, BF16)])
@pytest.mark.parametrize("H,KVH,n", [(4, 1, 3), (2, 1, 24), (3, 3, 40), (4, 2, 200)])
def test_long_context(dev, H, KVH, n, dtype, cdt):
    """Keys split over many workgroups and joined."""
    b = tree_batch(dev, [5003, 10], [n, n], KVH, 64, 64, cdt)
    gen = torch.Generator().manual_seed(n)
    sees = random_masks(b, gen, "tree")
    q = torch.randn(b.rows, H, 64).to(dtype)
    got, lse = attention(b, q.to(dev), R.words(sees, (n + 31) // 32).to(dev), want_lse=True)
    cached = b.store()
    for r in sorted({0, 1, n - 1, n, 2 * n - 1}):
        s = r // n
        ref, rl, mag, err, unit = R.attend(q[r:r + 1], cached, [b.table[s]], [b.pos0[s]], [0, 1],
                                           b.page, [set()])
        full = R.attend(q[s * n:s * n + n], cached, [b.table[s]], [b.pos0[s]], [0, n], b.page,
                        sees[s * n:s * n + n]) if n <= 3 else None
        if full is None:  # one row: its keys as a chain of its own
            keys = sorted(sees[r])
            ids = list(range(b.pos0[s])) + [b.pos0[s] + j for j in keys]
            sub = [None] * 4
            K, V, _, evs = cached
            pg = torch.tensor([b.table[s][i // b.page] for i in ids])
            at = torch.tensor(ids) % b.page
            G = H // KVH
            for a in range(H):
                k, v = K[pg, a // G, at], V[pg, a // G, at]
                sc = k @ q[r, a].double() / 8.0
                p = torch.softmax(sc, 0)
                vs = torch.ones(len(ids), 1, dtype=torch.float64) if evs is None else \
                    2.0 ** evs[pg, a // G, at // 16].double()[:, None]
                e = float((k.abs() @ q[r, a].double().abs()).max()) / 8.0
                tol = tolerance(dtype, cdt, (p @ v)[None, None], (p @ v.abs())[None, None],
                                torch.tensor([[e]]), ((p[:, None] * vs).max() * (v / vs).abs().sum(0)), 64)
                assert bool(((got[r, a].cpu().double() - p @ v).abs() <= tol[0, 0]).all())
                assert abs(float(lse[r, a]) - float(torch.logsumexp(sc, 0))) <= \
                    e * 70 * 2.0 ** -24 + 2.0 ** -20
        else:
            tol = tolerance(dtype, cdt, full[0], full[2], full[3], full[4], 64)
            i = r - s * n
            assert bool(((got[r].cpu().double() - full[0][i]).abs() <= tol[i]).all())


def test_chain_is_the_causal_form(dev):
    """A tree without branches gives what paged_attention gives, bit for bit where the keys are
    met in the same order."""
    for n, H, KVH, cdt in ((4, 4, 1, F8), (9, 2, 2, F16), (70, 4, 2, F8)):
        b = tree_batch(dev, [100, 17], [n, n], KVH, 64, 32, cdt)
        q = torch.randn(b.rows, H, 64).to(F16).to(dev)
        sees = [set(range(i + 1)) for i in range(n)] * 2
        got, lse = attention(b, q, R.words(sees, (n + 31) // 32).to(dev), want_lse=True)
        ref, rl = b.attention(q, want_lse=True)
        assert float((got.float() - ref.float()).abs().max()) <= 2.0 ** -9 * float(ref.abs().max())
        assert float((lse - rl).abs().max()) <= 1e-5


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("n,KVH", [(4, 2), (20, 2), (90, 2), (130, 64)])
def test_values_that_a_row_does_not_see(dev, n, KVH, dtype, cdt):
    """Infinities and NaN in keys and values of other branches have no effect; those that a row
    sees have; a page that is none gives NaN to the rows that see a token of it."""
    hd = 128 if KVH > 2 else 64
    b = Batch(dev, [30, 0, 64], [n] * 3, KVH, hd, 16, cdt)
    b.fill()
    k, v = torch.randn(2, b.rows, KVH, hd)
    v[1, 0, 3], v[n + n - 1, 1, 7], k[2 * n + n // 2, 0, 9] = math.inf, math.nan, math.nan
    b.append(k.to(dev), v.to(dev))
    if cdt != F8:
        b.cache.v[b.table[0][0], 1, 0, 0, 0, 3, 0, 2] = -math.inf  # a context token's
    if n >= 20:
        b.t[1, 1] = -1
        b.table[1][1] = -1
    gen = torch.Generator().manual_seed(n)
    sees = random_masks(b, gen, "any" if n < 90 else "tree")
    q = torch.randn(b.rows, KVH, hd).to(dtype)
    got, lse = attention(b, q.to(dev), R.words(sees, (n + 31) // 32).to(dev), want_lse=True)
    heads = torch.tensor([0, 1])
    cached = tuple(x if x is None else x[:, heads] for x in b.store())
    ref, rl, mag, err, unit = R.attend(q[:, heads], cached, b.table, b.pos0, b.starts, b.page, sees)
    got, lse = got[:, heads].cpu().double(), lse[:, heads].cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    fin = torch.isfinite(ref)
    tol = tolerance(dtype, cdt, ref, mag, err, unit, hd)
    assert bool(((got - ref).abs() <= tol)[fin].all())
    assert torch.equal(torch.isnan(lse), torch.isnan(rl))


@pytest.mark.parametrize("n", [[1], [8, 8], [1, 0, 31, 32, 33, 64, 200], [1024, 3]])
def test_masks(dev, n):
    from summa_amd import tree
    gen = torch.Generator().manual_seed(sum(n))
    parents, sees, depth, pos0 = [], [], [], [7 * i for i in range(len(n))]
    for s, m in enumerate(n):
        t = R.random_tree(m, gen, window=1 if m == 1024 else 9) if m else []
        if m > 40:                     # not parents: the context alone
            t[20], t[21], t[22] = -5, 21, 30
        parents += t
        a, d = R.masks(t) if m else ([], [])
        sees += a
        depth += [pos0[s] + x for x in d]
    even = len(set(n)) == 1
    p = torch.tensor(parents, dtype=torch.int32, device=dev)
    starts = torch.tensor([0] + n).cumsum(0).to(torch.int32).to(dev)
    mask, pos = tree.tree_masks(p.view(len(n), -1) if even else p,
                                torch.tensor(pos0, dtype=torch.int32, device=dev),
                                None if even else starts, max_rows=None if even else max(n))
    assert torch.equal(mask.cpu(), R.words(sees, (max(n) + 31) // 32))
    assert pos.cpu().tolist() == depth


@pytest.mark.parametrize("n", [[1], [6, 6, 6], [1, 0, 31, 64, 65, 130], [1024, 5]])
def test_accept(dev, n):
    from summa_amd import tree
    gen = torch.Generator().manual_seed(sum(n))
    rnd = lambda m, hi: torch.randint(0, hi, (m,), generator=gen).tolist()  # noqa: E731
    for hi in (1, 2, 3, 50):           # few tokens: long paths, equal siblings
        parents, toks, smp, ref = [], [], [], []
        for m in n:
            t, a, c = R.random_tree(m, gen) if m else [], rnd(m, hi), rnd(m, hi)
            if m > 40:
                t[20] = 25
            parents, toks, smp = parents + t, toks + a, smp + c
            ref.append(R.accept(t, a, c))
        even = len(set(n)) == 1
        x = [torch.tensor(v, dtype=torch.int32, device=dev) for v in (parents, toks, smp)]
        starts = torch.tensor([0] + n).cumsum(0).to(torch.int32).to(dev)
        path, count, emitted = tree.tree_accept(
            *[v.view(len(n), -1) if even else v for v in x], None if even else starts,
            max_rows=None if even else max(n))
        assert path.shape == emitted.shape == (len(n), max(n))
        for s, (p, e) in enumerate(ref):
            pad = [-1] * (max(n) - len(p))
            assert int(count[s]) == len(p)
            assert path[s].tolist() == p + pad and emitted[s].tolist() == e + pad


KEEPS = [  # pos0, path, KVH, hd, page
    ([0], [[0]], 1, 64, 16),
    ([5, 0, 16, 40], [[0, 1, 3], [2], [1, 4, 6, 20], []], 2, 64, 16),
    ([14, 31, 100], [[3, 4, 9, 17, 18, 40], [0, 1, 2, 3], [1, 2, 3, 4, 5, 6, 7, 8]], 3, 128, 32),
    ([3, 60], [list(range(0, 90, 2)), list(range(40, 100))], 2, 128, 48),
    ([7, 7, 7, 7, -2, 9], [[4, 4, 6], [3, 2, 1], [2, 500, 501], [-1, 3], [1, 2], [5, 9]], 2, 64, 16),
]


@pytest.mark.parametrize("cdt", [F8, BF16, F16])
@pytest.mark.parametrize("layers", [1, 3, 35])
@pytest.mark.parametrize("case", range(len(KEEPS)))
def test_keep(dev, case, layers, cdt):
    from summa_amd import paged
    pos0, path, KVH, hd, page = KEEPS[case]
    most = max(max((len(p) for p in path)), 1)
    b = Batch(dev, pos0, [100] * len(pos0), KVH, hd, page, cdt)
    if case == 4:                      # a page that is none under a path's third token
        b.t[5, 1] = -1
        b.table[5][1] = -1
    batches = []
    for i in range(min(layers, 3)):
        c = paged.PagedKVCache(b.pages, KVH, hd, page, cdt, dev)
        raw = torch.uint8 if cdt == F8 else torch.int16
        for x in (c.k, c.v):           # any bits, NaN and infinities among them
            x.view(raw).copy_(torch.randint(-2 ** 15, 2 ** 15, x.shape).to(raw))
        if cdt == F8:
            for x in (c.k_scales, c.v_scales):
                x.copy_(torch.randint(118 - 20 * i, 124, x.shape).to(torch.uint8))
        batches.append(c)
    caches = [batches[i % 3] if i < 3 else paged.PagedKVCache(b.pages, KVH, hd, page, cdt, dev)
              for i in range(layers)]

    def raw(c):
        b.cache = c
        return b.raw()
    before = [raw(c) for c in caches[:3]]
    t = torch.full((len(pos0), most), 77, dtype=torch.int32)
    for s, p in enumerate(path):
        t[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    count = torch.tensor([len(p) for p in path], dtype=torch.int32, device=dev)
    paged.paged_keep(caches if layers > 1 else caches[0], t.to(dev), count, b.t, b.p)
    for c, old in zip(caches, before):
        ref = R.keep(old, b.table, pos0, path, page, hd)
        for x, y in zip(raw(c), ref):
            assert torch.equal(x, y)


def test_keep_counts_past_the_path(dev):
    """count beyond max_rows is max_rows; nothing else is read."""
    from summa_amd import paged
    b = Batch(dev, [4], [60], 2, 64, 16, F16)
    before = b.raw()
    paged.paged_keep(b.cache, torch.tensor([[3, 5]], dtype=torch.int32, device=dev),
                     torch.tensor([9], dtype=torch.int32, device=dev), b.t, b.p)
    for x, y in zip(b.raw(), R.keep(before, b.table, [4], [[3, 5]], 16, 64)):
        assert torch.equal(x, y)


def test_graph_of_a_step(dev):
    """Masks, attention, acceptance and keeping, captured and replayed with other trees, lengths
    and queries, eager work between."""
    from summa_amd import paged, tree
    n, H, KVH, hd = 9, 4, 2, 64
    b = tree_batch(dev, [50, 3, 700], [n] * 3, KVH, hd, 32, F8)
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(b.rows, H, hd).to(F16).to(dev)
    parents = torch.zeros(3, n, dtype=torch.int32, device=dev)
    toks, smp = torch.zeros_like(parents), torch.zeros_like(parents)
    first = [x.clone() for x in (b.cache.k.view(torch.uint8), b.cache.v.view(torch.uint8),
                                 b.cache.k_scales, b.cache.v_scales)]

    def restore():
        for x, y in zip((b.cache.k.view(torch.uint8), b.cache.v.view(torch.uint8),
                         b.cache.k_scales, b.cache.v_scales), first):
            x.copy_(y)

    def fill(seed):
        gen.manual_seed(seed)
        parents.copy_(torch.tensor([R.random_tree(n, gen) for _ in range(3)], dtype=torch.int32))
        toks.copy_(torch.randint(0, 2, (3, n), generator=gen))
        smp.copy_(torch.randint(0, 2, (3, n), generator=gen))
        b.p.copy_(torch.tensor([50 - seed, 3 + seed, 700 - 60 * seed], dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=gen))

    def step():
        mask, pos = tree.tree_masks(parents, b.p)
        o, lse = attention(b, q, mask, want_lse=True, max_tokens=800)
        path, count, emitted = tree.tree_accept(parents, toks, smp)
        paged.paged_keep(b.cache, path, count, b.t, b.p)
        return mask, pos, o, lse, path, count, emitted

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        fill(seed)
        restore()
        graph.replay()
        torch.cuda.synchronize()
        moved = b.raw()
        restore()
        for x, y in zip(out, step()):  # (bits: what was never stored may be NaN)
            bits = {2: torch.int16, 4: torch.int32}[x.dtype.itemsize]
            assert torch.equal(x.view(bits), y.view(bits))
        for x, y in zip(moved, b.raw()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("pos0,n,H,KVH,dtype,cdt", [
    ([9000, 0, 700, 31, 4100], [3, 1, 2, 3, 3], 4, 2, F16, F8),          # 16 rows a KV head
    ([20000, 0, -9, 513, 130], [40, 3, 9, 33, 64], 2, 1, BF16, BF16),    # 128
    ([9000, 8000, 1], [150, 2, 70], 4, 2, F16, F16),                     # several tiles
    ([60 * (i % 9) + (4000 if i == 70 else 0) for i in range(100)], [2] * 100, 2, 2, F16, F8),
    ([40 * (i % 5) + 600 * (i % 64 == 63) for i in range(256)], [1] * 256, 2, 1, BF16, F8),
    ([40 * (i % 5) + 600 * (i % 64 == 63) for i in range(257)], [1] * 257, 2, 1, F16, F16),
])
def test_unequal_contexts(dev, pos0, n, H, KVH, dtype, cdt):
    """Splits shared by sequences of very different lengths, whatever max_tokens says, and captured
    with other lengths than it is replayed with."""
    print(f"case unequal {len(n)} {dtype} {cdt}", flush=True)
    b = tree_batch(dev, pos0, n, KVH, 64, 32, cdt)
    gen = torch.Generator().manual_seed(len(n))
    sees = random_masks(b, gen, "tree")
    mask = R.words(sees, (max(n) + 31) // 32).to(dev)
    q = torch.randn(b.rows, H, 64).to(dtype)
    qd = q.to(dev)
    results = {}
    for tokens in (None, max(pos0) + max(n), 513, 1, 2 ** 31 - 1):
        got, lse = attention(b, qd, mask, want_lse=True, max_tokens=tokens)
        check(b, q, sees, got, lse)
        results[tokens] = got
    out = torch.empty_like(results[None])
    right = b.p.clone()
    graph = torch.cuda.CUDAGraph()
    b.p.zero_()
    with torch.cuda.graph(graph):
        attention(b, qd, mask, out=out)
    for turn in range(4):
        b.p.copy_(right if turn % 2 else torch.zeros_like(right))
        graph.replay()
        again = attention(b, qd, mask)
        torch.cuda.synchronize()
        # (bits: at position 0 a sequence without a page has NaN)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    assert torch.equal(out, results[None])
