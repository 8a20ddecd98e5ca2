"""The paged KV cache (sm_paged_append, sm_paged_attention) against 64-bit definitions."""
import math

import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu
BF16, F16, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11, F8: 2.0 ** -4}
LEAST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F8: 2.0 ** -10}  # half the least subnormal


class Batch:
    """A pool with the sequences' pages in random order and garbage in all of it."""

    def __init__(self, dev, pos0, n, KVH, hd, page, dtype, pad_rows=0, spare=2, ragged=None):
        from summa_amd import paged
        self.pos0, self.n, self.page, self.hd, self.KVH, self.dtype = pos0, n, page, hd, KVH, dtype
        need = [max(0, -(-(p + m) // page)) for p, m in zip(pos0, n)]
        self.cols = max(max(need), 1)
        order = torch.randperm(sum(need) + spare).tolist()
        self.table = []
        for x in need:
            self.table.append([order.pop() for _ in range(x)])
        t = torch.full((len(n), self.cols), -1, dtype=torch.int32)
        for i, r in enumerate(self.table):
            t[i, : len(r)] = torch.tensor(r, dtype=torch.int32)
        self.t = t.to(dev)
        self.pages = sum(need) + spare
        self.cache = paged.PagedKVCache(self.pages, KVH, hd, page, dtype, dev)
        raw = torch.uint8 if dtype == F8 else torch.int16
        for x in (self.cache.k, self.cache.v):  # any bits, NaN and infinities among them
            x.view(raw).copy_(torch.randint(-2 ** 15, 2 ** 15, x.shape).to(raw))
        if dtype == F8:
            for x in (self.cache.k_scales, self.cache.v_scales):
                x.copy_(torch.randint(0, 256, x.shape).to(torch.uint8))
        self.starts = [0]
        for m in n:
            self.starts.append(self.starts[-1] + m)
        self.rows = self.starts[-1] + pad_rows
        self.p = torch.tensor(pos0, dtype=torch.int32, device=dev)
        ragged = len(set(n)) > 1 or pad_rows > 0 if ragged is None else ragged
        self.rs = torch.tensor(self.starts, dtype=torch.int32, device=dev) if ragged else None
        self.most = max(n)
        self.dev = dev

    def fill(self, fresh=True):
        """Every token before pos0 through the append itself; returns (k, v) f32."""
        from summa_amd import paged
        old = [max(0, p) for p in self.pos0]
        if sum(old) == 0:
            return
        k, v = (torch.randn(sum(old), self.KVH, self.hd) for _ in range(2))
        st = torch.tensor([0] + old, dtype=torch.int32).cumsum(0).to(torch.int32)
        paged.paged_append(self.cache, k.to(self.dev), v.to(self.dev), self.t,
                           torch.zeros_like(self.p), st.to(self.dev), max_rows=max(old))

    def store(self):
        c = self.cache
        return P.read(c.k, c.v, c.k_scales, c.v_scales)

    def raw(self):
        c = self.cache
        view = torch.uint8 if self.dtype == F8 else torch.int16
        return [x.cpu().clone() for x in [c.k.view(view), c.v.view(view)] +
                ([c.k_scales, c.v_scales] if c.k_scales is not None else [])]

    def append(self, k, v, **kw):
        from summa_amd import paged
        return paged.paged_append(self.cache, k, v, self.t, self.p, self.rs, max_rows=self.most, **kw)

    def attention(self, q, **kw):
        from summa_amd import paged
        kw.setdefault("max_rows", self.most)
        return paged.paged_attention(self.cache, q, self.t, self.p, self.rs, **kw)


def check_append(b, before, k, v, cs_rows, layout, dtype):
    """Stored values against the 64-bit rotation, scales and untouched places bit for bit.
    k, v [rows, KVH, hd] on the CPU in the call's dtype."""
    K, V, eks, evs = b.store()
    raw = b.raw()
    oldraw = before
    T = 4 if dtype == F8 else 2
    idx = P.v_index(b.hd, T)
    touched_k = torch.zeros(raw[0].shape, dtype=torch.bool)
    touched_v = torch.zeros(raw[1].shape, dtype=torch.bool).reshape(*raw[1].shape[:3], -1)
    touched_s = torch.zeros(b.pages, b.KVH, b.page // 16, dtype=torch.bool)
    for s, n in enumerate(b.n):
        done = {}
        for i in range(n):
            p = b.pos0[s] + i
            if p < 0 or p // b.page >= len(b.table[s]):
                continue
            done.setdefault(p // 16, []).append((p, b.starts[s] + i))
        for blk, toks in done.items():
            pg, lb = b.table[s][blk * 16 // b.page], blk * 16 % b.page // 16
            for h in range(b.KVH):
                for which, new, stored in ((0, k, K), (1, v, V)):
                    x32 = new[[r for _, r in toks], h].float()
                    ex = x32.double()
                    if which == 0 and cs_rows is not None:
                        cs = cs_rows[[p for p, _ in toks]]
                        x32, ex = P.rotate(x32, cs, layout), P.rotate(ex, cs.double(), layout)
                    at = torch.tensor([p % b.page for p, _ in toks])
                    got = stored[pg, h, at]
                    if dtype == F8:
                        e = P.need_exp(float(x32.abs().nan_to_num(0, 0, 0).max()))
                        old = int(oldraw[2 + which][pg, h, lb]) - 127
                        part = toks[0][0] % 16
                        if part:
                            e = max(e, old)
                        assert int((eks, evs)[which][pg, h, lb]) == e, (s, blk, h, which)
                        unit = 2.0 ** e
                    else:
                        unit = 1.0
                    fin = torch.isfinite(x32)
                    # the f32 rotation (three roundings), the type's rounding, its least step
                    tol = HALF[dtype] * ex.abs() * 1.001 + LEAST[dtype] * unit + \
                        4 * 2.0 ** -24 * ex.abs().nan_to_num(0, 0, 0).max()
                    assert bool(((got - ex).abs() <= tol)[fin].all()), (s, blk, h, which)
                    if dtype == F8:
                        assert bool(torch.isnan(got[~fin]).all())
                    if dtype == F8 and toks[0][0] % 16:  # earlier tokens of the block
                        t0 = toks[0][0] % 16
                        a = torch.arange(toks[0][0] % b.page - t0, toks[0][0] % b.page)
                        if which == 0:
                            was = oldraw[0][pg, h, a].view(F8).float()
                            now = raw[0][pg, h, a].view(F8).float()
                        else:
                            sel = idx[:t0]
                            was = oldraw[1].reshape(touched_v.shape)[pg, h, lb][sel].view(F8).float()
                            now = raw[1].reshape(touched_v.shape)[pg, h, lb][sel].view(F8).float()
                        want = (was * 2.0 ** (old - e)).to(F8).float()
                        same = (now == want) | (torch.isnan(now) & torch.isnan(want))
                        assert bool(same.all()), (s, blk, h, which)
                t0 = toks[0][0] % 16
                rows = torch.arange(lb * 16 + (0 if dtype == F8 else t0),
                                    lb * 16 + toks[-1][0] % 16 + 1)
                touched_k[pg, h, rows] = True
                touched_v[pg, h, lb, idx[(0 if dtype == F8 else t0): toks[-1][0] % 16 + 1].flatten()] = True
                touched_s[pg, h, lb] = True
    assert torch.equal(raw[0][~touched_k], oldraw[0][~touched_k])
    assert torch.equal(raw[1].reshape(touched_v.shape)[~touched_v],
                       oldraw[1].reshape(touched_v.shape)[~touched_v])
    if dtype == F8:
        for w in (2, 3):
            assert torch.equal(raw[w][~touched_s], oldraw[w][~touched_s])


APPENDS = [  # pos0, n, H, KVH, hd, page, rot
    ([0], [1], 1, 1, 64, 16, 64),
    ([0, 15, 16, 31], [1, 1, 1, 1], 4, 2, 128, 16, 128),
    ([5, 0, 47, 130], [3, 40, 17, 1], 6, 3, 64, 32, 32),
    ([7, 100], [16, 16], 8, 1, 128, 64, 96),
    ([0, 0, 0], [33, 0, 129], 4, 4, 128, 48, 16),
    ([1000, 3, 250], [5, 5, 5], 5, 5, 64, 256, 48),
]


@pytest.mark.parametrize("cdt", [F8, BF16, F16])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(dev, case, layout, dt, cdt):
    pos0, n, H, KVH, hd, page, rot = APPENDS[case]
    print(f"case append {case} {layout} {dt} {cdt}", flush=True)
    b = Batch(dev, pos0, n, KVH, hd, page, cdt, pad_rows=2)
    b.fill()
    qkv = torch.randn(b.rows, H + 2 * KVH, hd)
    qkv[torch.rand(b.rows) < 0.3] *= 30  # scales grow within blocks
    qkv = qkv.to(dt)
    q, k, v = qkv.split([H, KVH, KVH], 1)
    qd, kd, vd = qkv.to(dev).split([H, KVH, KVH], 1)
    table = P.angles(rot, 2048)
    qdt = F16 if dt == F32 else dt
    out = torch.full((b.rows, H, hd), 5.0, dtype=qdt, device=dev)
    before = b.raw()
    got = b.append(kd, vd, q=qd, rope_table=table.to(dev), layout=layout, out=out)
    assert got is out
    check_append(b, before, k, v, table, layout, cdt)
    got = out.cpu().double()
    for s, m in enumerate(n):
        for i in range(m):
            r = b.starts[s] + i
            ref = P.rotate(q[r].double(), table[pos0[s] + i].double(), layout)
            tol = HALF[qdt] * ref.abs() * 1.001 + 4 * 2.0 ** -24 * ref.abs().max() + 2.0 ** -25
            assert bool(((got[r] - ref).abs() <= tol).all())
    assert bool((out[b.starts[-1]:] == 5).all())  # rows of no sequence
    # once more with the same rows: the same cache (the scales have grown already)
    after = b.raw()
    b.append(kd, vd, rope_table=table.to(dev), layout=layout)
    for x, y in zip(after, b.raw()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("cdt", [F8, BF16])
def test_append_without_rotation_or_queries(dev, cdt):
    b = Batch(dev, [3, 0], [20, 20], 2, 64, 32, cdt)
    b.fill()
    k, v = torch.randn(2, 40, 2, 64)
    before = b.raw()
    assert b.append(k.to(dev), v.to(dev)) is None
    check_append(b, before, k, v, None, "half", cdt)


@pytest.mark.parametrize("cdt", [F8, F16])
def test_append_odd_values(dev, cdt):
    """Infinities, NaN, zeros, the largest and the least values; and positions outside the
    rotary table."""
    b = Batch(dev, [0, 21], [17, 17], 2, 64, 32, cdt)
    b.fill()
    k, v = torch.randn(2, 34, 2, 64)
    k[3, 0, 5], k[4, 0, 6], v[3, 1, 7], v[20, 0, 1] = math.inf, math.nan, -math.inf, math.nan
    if cdt == F8:
        v[0:16, 0] = 0.0                    # a block of zeros: the least scale
        v[16, 0] = 3e38                     # and of the largest values
        v[16, 1] = 1e-30
        k[17 + 11, 1] = 448.0 * 4           # right at a scale's border
        k[17 + 12, 1] = 448.1 * 4
    before = b.raw()
    b.append(k.to(dev), v.to(dev))
    check_append(b, before, k, v, None, "half", cdt)
    short = P.angles(64, 10)
    b.append(k.to(dev), v.to(dev), rope_table=short.to(dev))
    K, V = b.store()[:2]
    pg = b.table[0][0]
    assert bool(torch.isnan(K[pg, :, 10:16]).all())  # no angle for these positions
    assert bool(torch.isfinite(K[pg, :, 0:3]).all())


def test_append_token_by_token_is_the_block_at_once(dev):
    """Tokens appended one at a time end at the scale of the block at once; the codes differ
    by the second rounding among e4m3's subnormals only: one step there."""
    ks = torch.randn(48, 2, 64) * (2.0 ** torch.randint(-6, 6, (48, 1, 1)))
    caches = []
    for step in (48, 1, 5):
        b = Batch(dev, [0], [48], 2, 64, 32, F8, ragged=True)
        b.table, b.t = [[1, 0]], torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
        for i in range(0, 48, step):
            part = ks[i:i + step].to(dev)
            b.p = torch.tensor([i], dtype=torch.int32, device=dev)
            b.rs = torch.tensor([0, len(part)], dtype=torch.int32, device=dev)
            b.most = len(part)
            b.append(part, part)
        caches.append((b.store(), b.raw()))
    used = torch.tensor([0, 1])
    for (K, V, ek, ev), raw in caches[1:]:
        (K0, V0, ek0, ev0), raw0 = caches[0]
        for w in (2, 3):
            assert torch.equal(raw[w][1], raw0[w][1]) and torch.equal(raw[w][0, :, :1], raw0[w][0, :, :1])
        for X, X0, e in ((K, K0, ek0), (V, V0, ev0)):
            step = (2.0 ** -9 * 2.0 ** e.double()).repeat_interleave(16, 2)[..., None]
            small = X0.abs() <= step * 8
            d = (X - X0).abs()
            for sl in ((1, slice(None), slice(0, 32)), (0, slice(None), slice(0, 16))):
                assert bool((d[sl] <= torch.where(small, step, step * 0).expand_as(d)[sl]).all())


def test_append_skips_what_has_no_place(dev):
    """Negative positions, a table entry outside the pool, tokens past the table: not stored,
    nothing else touched."""
    b = Batch(dev, [-3, 0, 30], [6, 40, 6], 2, 64, 32, F8)
    k, v = torch.randn(2, b.rows, 2, 64)
    b.t[1, 1] = b.pages                       # sequence 1: its second page is no page
    b.t[2, 1] = -7
    b.table[1], b.table[2] = b.table[1][:1], b.table[2][:1]
    before = b.raw()
    q = torch.randn(b.rows, 2, 64, device=dev)
    out = torch.full((b.rows, 2, 64), 5.0, dtype=F16, device=dev)
    b.append(k.to(dev), v.to(dev), q=q, out=out)
    check_append(b, before, k, v, None, "half", F8)
    assert bool((out[:3] == 5).all()) and torch.equal(out[3:], q[3:].half())


def tolerance(dtype, cdt, ref, mag, err, unit, hd):
    """|out - ref|: the output's rounding, P's rounding (f16 for f16 and 8-bit values, bf16
    for bf16 ones) against sum p |v|, P's f16 subnormals (half a step of 2^-24 for every
    key, where the largest weight times scale is one or more), and the f32 scores: products exact, hd + 2 roundings of up to |q| . |k|, and
    exp2 with its argument's rounding (score * log2 e: up to 2^-23 of the score, err bounds
    it) and 2^-22 of its own."""
    p = HALF[BF16] if cdt == BF16 else HALF[F16]
    score = err.double()[..., None] * (hd + 6) * 2.0 ** -24
    sub = 0.0 if cdt == BF16 else unit * 2.0 ** -25
    return (HALF[dtype] * ref.abs() + (p + 2 * score + 2.0 ** -20) * mag) * 1.01 + sub + 1e-30 + \
        (2.0 ** -25 if dtype == F16 else 0.0)


def check_attention(b, q, got, lse=None):
    ref, rl, mag, err, unit = P.attend(q, b.store(), b.table, b.pos0, b.starts, b.page)
    n = b.starts[-1]
    got, ref, mag, err, unit = (x[:n] for x in (got.cpu().double(), ref, mag, err, unit))
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fin = torch.isfinite(ref)
    tol = tolerance(q.dtype, b.dtype, ref, mag, err, unit, b.hd)
    if q.dtype == F16:  # what rounds past the largest f16, 65504 + half a step, is an infinity
        over = torch.isinf(got)
        assert bool((ref.abs() + tol >= 65520.0)[over].all()) and bool((ref * got > 0)[over].all())
        assert bool((ref.abs() - tol <= 65520.0)[~over & fin].all())
        fin &= ~over
    d = (got - ref).abs()
    assert bool((d <= tol)[fin].all()), float((d - tol)[fin].max())
    if lse is not None:
        lse, rl = lse.cpu().double()[:n], rl[:n]
        assert torch.equal(torch.isneginf(lse), torch.isneginf(rl))
        f = torch.isfinite(rl)
        t = err.double() * (b.hd + 6) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * rl.abs()
        assert bool(((lse - rl).abs() <= t)[f].all()), float((lse - rl).abs()[f].max())


STEPS = [  # pos0, n, H, KVH, hd, page
    ([0], [1], 1, 1, 64, 16),
    ([0, 15, 16, 17, 1], [1] * 5, 4, 4, 128, 16),
    ([200, 3, 64, 511], [1] * 4, 16, 4, 128, 64),
    ([1500, 900], [1, 1], 12, 2, 64, 32),
    ([70, 0, 333], [4, 4, 4], 4, 1, 128, 48),
    ([40, 7], [3, 3], 6, 2, 64, 256),
    ([300], [1], 40, 1, 128, 32),             # more heads to a KV head than a tile has rows
    ([0, 5, 130], [40, 1, 17], 8, 2, 64, 32),
    ([0, 0], [130, 300], 4, 2, 128, 64),
    ([600], [150], 3, 3, 64, 128),
]


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, F8), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_attention(dev, case, dtype, cdt):
    pos0, n, H, KVH, hd, page = STEPS[case]
    print(f"case attention {case} {dtype} {cdt}", flush=True)
    b = Batch(dev, pos0, n, KVH, hd, page, cdt, pad_rows=1 if len(set(n)) > 1 else 0)
    b.fill()
    k, v = torch.randn(2, b.rows, KVH, hd)
    b.append(k.to(dev), v.to(dev))
    wide = (torch.randn(b.rows, H + 3, hd) * 1.5).to(dtype)
    q, qd = wide[:, :H], wide.to(dev)[:, :H]
    out, lse = b.attention(qd, want_lse=True)
    check_attention(b, q, out, lse)
    # however the keys are split: the longest sequence understated and exact
    for most in (1, max(p + m for p, m in zip(pos0, n))):
        out, lse = b.attention(qd, want_lse=True, max_tokens=most)
        check_attention(b, q, out, lse)


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, F8), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("pos0,n", [
    ([1200, 900], [200, 131]),                          # keys in two splits
    ([1100, -40, 0, 1024, 77], [200, 131, 256, 190, 0]),  # whole
    ([2100, 1000], [130, 256])])
def test_attention_of_many_heads_and_long_sequences(dev, pos0, n, dtype, cdt):
    """Enough heads, rows and keys for the largest workgroups (256 rows, heads of 128), the
    definition checked for some heads: ragged rows, rows without keys, a page that is none,
    values that are not finite among those that all rows, some or none see."""
    KVH = 64
    b = Batch(dev, pos0, n, KVH, 128, 32, cdt, pad_rows=3)
    b.fill()
    k, v = torch.randn(2, b.rows, KVH, 128)
    heads = torch.tensor([0, 1, 31, 63])
    v[0, 1, 5], v[100, 31, 127], v[b.starts[1] + 5, 63, 64] = math.inf, math.nan, -math.inf
    b.append(k.to(dev), v.to(dev))
    if cdt != F8:  # seen by all rows of sequence 0; and behind sequence 1, seen by none
        b.cache.v[b.table[0][0], 31, 0, 0, 0, 3, 0, 2] = math.inf
    if len(n) == 2:
        b.t[1, -(-(pos0[1] + 60) // 32)] = -1
        b.table[1][-(-(pos0[1] + 60) // 32)] = -1
    q = torch.randn(b.rows, KVH, 128).to(dtype)
    out = torch.full((b.rows, KVH, 128), 5.0, dtype=dtype, device=dev)
    _, lse = b.attention(q.to(dev), want_lse=True, out=out)
    assert bool((out[b.starts[-1]:] == 5).all())
    cached = tuple(x if x is None else x[:, heads] for x in b.store())
    m = b.starts[-1]
    ref, rl, mag, err, unit = (x[:m] for x in P.attend(q[:, heads], cached, b.table, b.pos0,
                                                       b.starts, b.page))
    got, lse = (x[:, heads].cpu().double()[:m] for x in (out, lse))
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    fin = torch.isfinite(ref)
    tol = tolerance(dtype, cdt, ref, mag, err, unit, 128)
    assert bool(((got - ref).abs() <= tol)[fin].all())
    assert torch.equal(torch.isneginf(lse), torch.isneginf(rl))
    f = torch.isfinite(rl)
    t = err.double() * (128 + 6) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * rl.abs()
    assert torch.equal(torch.isnan(lse), torch.isnan(rl)) and bool(((lse - rl).abs() <= t)[f].all())


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, BF16)])
@pytest.mark.parametrize("H,KVH,n", [(4, 1, 1), (2, 1, 24), (4, 2, 200)])
def test_attention_split_over_many_keys(dev, dtype, cdt, H, KVH, n):
    """One long and one short sequence: the long one's keys go to many workgroups."""
    b = Batch(dev, [6000, 10], [n, n], KVH, 64, 64, cdt)
    b.fill()
    k, v = torch.randn(2, b.rows, KVH, 64)
    b.append(k.to(dev), v.to(dev))
    q = torch.randn(b.rows, H, 64).to(dtype)
    rows = sorted({0, n - 1, n, n + n // 2, 2 * n - 1})
    out, lse = b.attention(q.to(dev), want_lse=True)
    cached = b.store()
    for r in rows:
        s = r // n
        ref, rl, mag, err, unit = P.attend(q[r:r + 1], cached, [b.table[s]],
                                           [b.pos0[s] + r % n], [0, 1], b.page)
        tol = tolerance(dtype, cdt, ref, mag, err, unit, 64)
        assert bool(((out[r:r + 1].cpu().double() - ref).abs() <= tol).all())
        t = err.double() * 70 * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * rl.abs()
        assert bool(((lse[r:r + 1].cpu().double() - rl).abs() <= t).all())


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("n", [2, 5, 90])
def test_values_a_row_does_not_see(dev, dtype, cdt, n):
    """A token's infinity or NaN, in its key or its value, reaches the rows that see it and
    no earlier row; what lies behind the last token reaches nobody (the pool is garbage)."""
    b = Batch(dev, [30, 0, 64], [n] * 3, 2, 64, 32, cdt)
    b.fill()
    k, v = torch.randn(2, b.rows, 2, 64)
    v[1, 0, 3], v[n + n - 1, 1, 7], k[2 * n + n // 2, 0, 9] = math.inf, math.nan, math.nan
    if n > 40:
        v[n + 37, 0, 11] = -math.inf
    b.append(k.to(dev), v.to(dev))
    q = torch.randn(b.rows, 4, 64).to(dtype)
    out = b.attention(q.to(dev))
    ref, _, mag, err, unit = P.attend(q, b.store(), b.table, b.pos0, b.starts, b.page)
    got = out.cpu().double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin)
    tol = tolerance(dtype, cdt, ref, mag, err, unit, 64)
    assert bool(((got - ref).abs() <= tol)[fin].all())
    assert not bool(fin.all()) and bool(fin[0].all())


@pytest.mark.parametrize("dtype,cdt", [(F16, F8), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("pos0,n", [(40, 1), (40, 60), (1400, 3), (1400, 90)])
def test_infinite_values_that_rows_see(dev, pos0, n, dtype, cdt):
    """An infinity has a positive weight in every row that sees it, however small: the sum is
    infinite, of both signs or with a NaN it is NaN, and other dims are left alone. (8 bits:
    an infinity is stored as NaN.)"""
    b = Batch(dev, [0], [pos0 + n], 1, 64, 32, cdt)
    k, v = torch.randn(2, pos0 + n, 1, 64)
    k[:pos0 * 2 // 5] = -60.0  # weights that 32 bits round to zero: whole splits, or steps
    v[0, 0, 1], v[pos0 - 1, 0, 2], v[pos0 // 2, 0, 3] = math.inf, -math.inf, math.inf
    v[1, 0, 4], v[pos0 - 2, 0, 4] = math.inf, -math.inf
    v[2, 0, 5], v[pos0 // 2, 0, 6], v[pos0 + n // 2, 0, 7] = math.nan, math.nan, math.inf
    v[3, 0, 8] = v[pos0 + n - 1, 0, 8] = math.inf
    b.append(k.to(dev), v.to(dev))
    b.pos0, b.n, b.starts, b.rows, b.most = [pos0], [n], [0, n], n, n
    b.p = torch.tensor([pos0], dtype=torch.int32, device=dev)
    q = torch.randn(n, 4, 64).abs().to(dtype)
    got = b.attention(q.to(dev)).cpu().double()
    ref, _, mag, err, unit = P.attend(q, b.store(), b.table, b.pos0, b.starts, b.page)
    assert bool((ref[..., 1].isnan() if cdt == F8 else ref[..., 1] == math.inf).all())
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]) and bool(torch.isfinite(got[~odd]).all())
    tol = tolerance(dtype, cdt, ref, mag, err, unit, 64)
    assert bool(((got - ref).abs() <= tol)[~odd].all())


@pytest.mark.parametrize("cdt", [F8, F16])
def test_lengths_beyond_the_table(dev, cdt):
    """A length that no table row holds is read no further than the first token without a
    page: its rows are NaN, and the call ends as soon as one over a full table."""
    from summa_amd import paged
    cache = paged.PagedKVCache(4, 2, 64, 32, cdt, dev)
    t = torch.tensor([[0, 1], [2, 3], [1, 0]], dtype=torch.int32, device=dev)
    k = torch.randn(3 * 64, 2, 64, device=dev)
    paged.paged_append(cache, k, k, t, torch.zeros(3, dtype=torch.int32, device=dev))
    for n in (1, 40):
        pos0 = torch.tensor([1 << 30, 64 - n, 2 ** 31 - 50], dtype=torch.int32, device=dev)
        q = torch.randn(3 * n, 4, 64, device=dev).half()
        out = paged.paged_attention(cache, q, t, pos0, max_tokens=4096)
        assert bool(out[:n].isnan().all()) and bool(out[2 * n:].isnan().all())
        assert torch.equal(out[n:2 * n], paged.paged_attention(cache, q[n:2 * n], t[1:2], pos0[1:2],
                                                               max_tokens=4096))


@pytest.mark.parametrize("cdt", [F8, F16])
def test_rows_without_keys_or_pages(dev, cdt):
    """Negative positions: zero and -inf. A row that needs a page that is none: NaN, the rows
    before it in the same tile are whole."""
    b = Batch(dev, [-2, 0, 28], [4, 8, 8], 2, 64, 32, cdt, pad_rows=3)
    k, v = torch.randn(2, b.rows, 2, 64)
    b.fill()
    b.append(k.to(dev), v.to(dev))
    b.t[2, 1] = b.pages + 5
    b.table[2][1] = -1
    q = torch.randn(b.rows, 6, 64).to(F16)
    out = torch.full((b.rows, 6, 64), 5.0, dtype=F16, device=dev)
    got, lse = b.attention(q.to(dev), want_lse=True, out=out)
    assert got is out and bool((out[-3:] == 5).all())
    check_attention(b, q, out, lse)
    assert bool((out[:2] == 0).all()) and bool(torch.isneginf(lse[:2]).all())
    assert bool(torch.isfinite(out[12:16]).all()) and bool(torch.isnan(out[16:20]).all())


def test_scales_far_apart(dev):
    """Blocks whose scales differ by 2^40 in K or V: each block's weight and values keep
    their accuracy (the running maximum is that of weight times scale)."""
    b = Batch(dev, [160], [1], 1, 64, 32, F8)
    k, v = torch.randn(2, 161, 1, 64)
    k[:16] *= 2.0 ** -30
    v[32:48] *= 2.0 ** -20
    v[64:80] *= 2.0 ** 20
    k[64:80] *= 8.0
    st = torch.tensor([0, 161], dtype=torch.int32, device=dev)
    from summa_amd import paged
    paged.paged_append(b.cache, k.to(dev), v.to(dev), b.t, torch.zeros_like(b.p), st, max_rows=161)
    for scale in (0.1, 1.0, 20.0):
        q = (torch.randn(1, 3, 64) * scale).to(F16)
        out, lse = b.attention(q.to(dev), want_lse=True)
        check_attention(b, q, out, lse)


def test_offsets_past_32_bits(dev):
    """Pages 4 GiB and more into the pool."""
    from summa_amd import paged
    hd, KVH, page = 128, 1, 256
    pages = (5 << 30) // (hd * KVH * page)
    cache = paged.PagedKVCache(pages, KVH, hd, page, F8, dev)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=dev)
    k, v = torch.randn(2, 700, KVH, hd)
    p0 = torch.zeros(1, dtype=torch.int32, device=dev)
    paged.paged_append(cache, k.to(dev), v.to(dev), table, p0)
    q = torch.randn(1, 4, hd).to(BF16)
    p1 = torch.full((1,), 699, dtype=torch.int32, device=dev)
    out = paged.paged_attention(cache, q.to(dev), table, p1)
    small = paged.PagedKVCache(3, KVH, hd, page, F8, dev)
    t2 = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev)
    paged.paged_append(small, k.to(dev), v.to(dev), t2, p0)
    assert torch.equal(out, paged.paged_attention(small, q.to(dev), t2, p1))
    assert torch.equal(small.k.view(torch.uint8)[0], cache.k.view(torch.uint8)[pages - 1])


@pytest.mark.parametrize("cdt", [F8, F16])
def test_a_rollout(dev, cdt):
    """Prefill, then decode steps, as a rollout runs them: ragged prompts, each step appends
    one token a sequence and attends; two sequences share their prompt's full pages. Each
    step against the definition over what the cache holds, and, captured in a graph whose
    positions a kernel advances, bit for bit the same on every replay."""
    from summa_amd import ops, paged
    H, KVH, hd, page, S, steps = 8, 2, 64, 32, 3, 6
    lens = [70, 70, 9]
    cache = paged.PagedKVCache(16, KVH, hd, page, cdt, dev)
    rope = ops.rope_table(256, 32, device=dev)
    # sequences 0 and 1 share pages 4 and 9 (64 tokens)
    table = torch.tensor([[4, 9, 2, 7], [4, 9, 11, 0], [5, 1, 3, 6]], dtype=torch.int32, device=dev)
    prompt = torch.randn(79, H + 2 * KVH, hd, device=dev).half()
    st = torch.tensor([0, 70, 79], dtype=torch.int32, device=dev)
    q, k, v = prompt.split([H, KVH, KVH], 1)
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    owners = table[[0, 2]].contiguous()
    qr = paged.paged_append(cache, k, v, owners, zero, st, q=q, rope_table=rope, layout="half",
                            q_dtype=F16, max_rows=70)
    out = paged.paged_attention(cache, qr, owners, zero, st, max_rows=70)
    # sequence 1's own page takes the last 6 prompt tokens
    paged.paged_append(cache, k[64:70], v[64:70], table[1:2].contiguous(),
                       torch.tensor([64], dtype=torch.int32, device=dev), rope_table=rope,
                       layout="half")
    toks = torch.randn(steps, S, H + 2 * KVH, hd, device=dev).half()
    keep = [x.clone() for x in (cache.k.view(torch.uint8), cache.v.view(torch.uint8))]
    scales = [x.clone() for x in (cache.k_scales, cache.v_scales)] if cdt == F8 else []

    pos = torch.tensor(lens, dtype=torch.int32, device=dev)
    cur = torch.empty_like(toks[0])

    def step():
        q, k, v = cur.split([H, KVH, KVH], 1)
        qr = paged.paged_append(cache, k, v, table, pos, q=q, rope_table=rope, layout="half",
                                q_dtype=F16)
        o = paged.paged_attention(cache, qr, table, pos, max_tokens=128)
        pos.add_(1)
        return qr, o

    def reset():
        for x, y in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8)), keep):
            x.copy_(y)
        for x, y in zip((cache.k_scales, cache.v_scales), scales):
            x.copy_(y)
        pos.copy_(torch.tensor(lens, dtype=torch.int32))

    eager = []
    for i in range(steps):
        cur.copy_(toks[i])
        at = [p + i for p in lens]
        qr, o = step()
        cached = P.read(cache.k, cache.v, cache.k_scales, cache.v_scales)
        ref, _, mag, err, unit = P.attend(qr.cpu(), cached, table.cpu().tolist(), at,
                                          list(range(S + 1)), page)
        tol = tolerance(F16, cdt, ref, mag, err, unit, hd)
        assert bool(((o.cpu().double() - ref).abs() <= tol).all())
        eager.append(o.clone())
    g = torch.cuda.CUDAGraph()
    reset()
    cur.copy_(toks[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        qr, o = step()
    for again in range(2):
        reset()
        for i in range(steps):
            cur.copy_(toks[i])
            g.replay()
            assert torch.equal(o, eager[i]), (again, i)
            torch.cuda.synchronize()


@pytest.mark.parametrize("cdt", [F8, F16])
def test_many_sequences(dev, cdt):
    """70000 sequences of one token: more than one grid dimension's 65535. The one weight is
    1, so the output is V as the cache holds it."""
    from summa_amd import paged
    S = 70000
    cache = paged.PagedKVCache(S, 1, 64, 16, cdt, dev)
    table = torch.randperm(S, device=dev).to(torch.int32)[:, None].contiguous()
    zero = torch.zeros(S, dtype=torch.int32, device=dev)
    v = torch.randint(-8, 9, (S, 1, 64), device=dev).half() / 4  # (exact in either type)
    q = torch.randn(S, 2, 64, device=dev).half()
    got = paged.paged_append(cache, v, v, table, zero, q=q)
    assert torch.equal(got, q)
    out, lse = paged.paged_attention(cache, q, table, zero, max_tokens=1, want_lse=True)
    assert torch.equal(out, v.expand(S, 2, 64))
    score = (q.double() * v.double()).sum(-1) / 8
    tol = (q.double().abs() * v.double().abs()).sum(-1) / 8 * 70 * 2.0 ** -24 + 2.0 ** -21 + \
        2.0 ** -22 * score.abs()
    assert bool(((lse.double() - score).abs() <= tol).all())


def test_two_calls_at_once(dev):
    """Two attention calls over one cache on two streams, each with its own workspace."""
    b = Batch(dev, [3000, 3000], [1, 1], 2, 64, 64, F8)
    b.fill()
    k, v = torch.randn(2, 2, 2, 64)
    b.append(k.to(dev), v.to(dev))
    q1, q2 = (torch.randn(2, 4, 64, device=dev).half() for _ in range(2))
    want = b.attention(q1), b.attention(q2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = b.attention(q1)
        with torch.cuda.stream(s2):
            c = b.attention(q2)
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(c, want[1])


def test_a_cache_keeps_its_storage(dev):
    """The descriptor holds addresses: the tensors behind it cannot be exchanged."""
    from summa_amd import paged
    c = paged.PagedKVCache(4, 2, 64, 32, F8, dev)
    with pytest.raises(AttributeError):
        c.k = torch.zeros_like(c.v)
    again = paged.PagedKVCache.from_tensors(c.k, c.v, c.k_scales, c.v_scales)
    assert again.nbytes == c.nbytes == 4 * 2 * 32 * 64 * 2 + 2 * 4 * 2 * 2


def test_python_refusals(dev):
    from summa_amd import SummaError, paged
    with pytest.raises(TypeError):
        paged.PagedKVCache(4, 2, 64, 32, F32, dev)
    with pytest.raises(ValueError):
        paged.PagedKVCache(4, 2, 96, 32, F8, dev)
    with pytest.raises(ValueError):
        paged.PagedKVCache(4, 2, 64, 24, F8, dev)
    b = Batch(dev, [0, 0], [4, 4], 2, 64, 32, F8)
    k, v = torch.randn(2, 8, 2, 64, device=dev)
    q = torch.randn(8, 4, 64, device=dev)
    with pytest.raises(ValueError, match="needs max_rows"):
        paged.paged_append(b.cache, k, v, b.t, b.p, torch.tensor([0, 4, 8], dtype=torch.int32,
                                                                device=dev))
    with pytest.raises(ValueError, match="rows / sequences"):
        paged.paged_append(b.cache, k[:7], v[:7], b.t, b.p)
    with pytest.raises(TypeError, match="int32"):
        paged.paged_append(b.cache, k, v, b.t.long(), b.p)
    with pytest.raises(TypeError, match="one dtype"):
        paged.paged_append(b.cache, k, v.half(), b.t, b.p)
    with pytest.raises(ValueError, match="contiguous heads"):
        paged.paged_append(b.cache, k.transpose(1, 2), v, b.t, b.p)
    with pytest.raises(ValueError, match="rotary table"):
        paged.paged_append(b.cache, k, v, b.t, b.p, rope_table=torch.zeros(4, 8, device=dev))
    with pytest.raises(ValueError, match="table is empty"):
        paged.paged_append(b.cache, k, v, b.t, b.p, rope_table=torch.zeros(0, 8, 2, device=dev))
    with pytest.raises(ValueError, match="device"):
        paged.paged_append(b.cache, k.cpu(), v, b.t, b.p)
    with pytest.raises(TypeError, match="q must be"):
        paged.paged_attention(b.cache, q, b.t, b.p)
    with pytest.raises(ValueError, match="out must be"):
        paged.paged_attention(b.cache, q.half(), b.t, b.p, out=torch.empty(8, 4, 64, device=dev))
    with pytest.raises(SummaError, match="multiple of KVH"):
        paged.paged_attention(b.cache, torch.zeros(8, 3, 64, device=dev).half(), b.t, b.p)
    half = paged.PagedKVCache(4, 2, 64, 32, F16, dev)
    with pytest.raises(SummaError, match="query's dtype"):
        paged.paged_attention(half, q.bfloat16(), b.t, b.p)
