"""Next tokens from given random numbers (sm_sample_rows) against a 64-bit definition: tokens have
to be equal, log-probs within the roundings of an f32 sum."""
import math

import numpy as np
import pytest
import torch

import _tree as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(x, u, T=1.0, k=None, p=1.0, m=0.0, dev="cuda:0", where=""):
    """x [rows, vocab] on the CPU; options as numbers or CPU tensors."""
    from summa_amd import sampling
    to = lambda o: o.to(dev) if torch.is_tensor(o) else o  # noqa: E731
    tok, lp = sampling.sample_rows(to(x), to(u), temperature=to(T), top_k=to(k), top_p=to(p),
                                   min_p=to(m))
    tok, lp = tok.cpu().tolist(), lp.cpu().double().tolist()
    rows, vocab = x.shape
    x64 = x.double().numpy()
    f32 = lambda o, r: float(o[r]) if torch.is_tensor(o) else float(np.float32(o))  # noqa: E731
    for r in range(rows):
        kk = -1 if k is None else int(k[r]) if torch.is_tensor(k) else k
        ref, rl = R.sample(x64[r], float(u[r]), f32(T, r), kk, f32(p, r), f32(m, r))
        assert tok[r] == ref, (where, r, tok[r], ref)
        if math.isinf(rl):
            assert lp[r] == rl
            continue
        # x - max and the result (half a step each); the sum's relative error: exponentials of up
        # to 20 octaves below the largest where it has its weight (30 * 2^-24), chains of up to
        # 200 additions (200 * 2^-24), together below 2^-16
        tol = 2.0 ** -23 * abs(rl) + 2.0 ** -16
        assert abs(lp[r] - rl) <= tol, (where, r, lp[r], rl)
    return tok


VOCABS = [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1025, 4096, 4099, 16384, 20001, 32768, 50001, 65536,
          65537, 100003, 131072, 131073, 200001]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_sizes_and_filters(dev, vocab, dtype):
    """Every size with every combination of filters, a row each."""
    print(f"case sample {vocab} {dtype}", flush=True)
    g = torch.Generator().manual_seed(vocab)
    combos = [(T, k, p, m) for T in (0.0, 0.7, 1.0) for k in (-1, 1, 40, 3000) for p in (0.6, 1.0)
              for m in (0.0, 0.1)]
    rows = len(combos)
    x = torch.randn(rows, vocab, generator=g) * 2.5
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 6
    x = x.to(dtype)
    u = torch.rand(rows, generator=g)
    T, k, p, m = (torch.tensor(c) for c in zip(*combos))
    check(x, u, T, k.to(torch.int32), p, m)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(3, 262144), (5, 262143), (3, 262145), (2, 700001)])
def test_the_largest_vocabularies(dev, rows, vocab, dtype):
    """Where the sums of 512 logits fill their place, and past it."""
    print(f"case sample {rows} {vocab} {dtype}", flush=True)
    x = (torch.randn(rows, vocab) * 2.5).to(dtype)
    x[:, 7] += 8
    u = torch.rand(rows)
    for kw in (dict(), dict(k=40), dict(p=0.9), dict(m=0.01), dict(T=0.0), dict(k=700, p=0.8)):
        check(x, u, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 3, 8, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("vocab", [49153, 98305, 131071])
def test_rows_shared_out_over_the_chip(dev, rows, vocab, dtype):
    """Every number of parts to a row and its neighbours, filters mixed over the rows."""
    print(f"case sample {rows} {vocab} {dtype}", flush=True)
    x = (torch.randn(rows, vocab) * 2).to(dtype)
    u = torch.rand(rows)
    T = torch.tensor([1.0, 0.0, 0.7, 1.3])[torch.arange(rows) % 4]
    k = torch.tensor([-1, 50, 1, -1, 400, 600])[torch.arange(rows) % 6].to(torch.int32)
    p = torch.tensor([0.95, 1.0, 0.5, 0.99, 1.0])[torch.arange(rows) % 5]
    m = torch.tensor([0.0, 0.05, 0.0])[torch.arange(rows) % 3]
    x[rows // 2, 5:] = -math.inf
    if rows > 4:
        x[4], x[3, 9], x[2, 100:90000] = -math.inf, math.inf, torch.finfo(dtype).min
    check(x, u, T, k, p, m)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 151), (700, 61), (300, 4097), (37, 32768)])
def test_many_rows_one_setting(dev, rows, vocab, dtype):
    x = (torch.randn(rows, vocab) * 3).to(dtype)
    u = torch.rand(rows)
    for kw in (dict(), dict(k=5), dict(p=0.9), dict(m=0.05), dict(T=0.0),
               dict(T=1.3, k=200, p=0.95, m=0.01)):
        check(x, u, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_equal_logits(dev, vocab, dtype):
    """Ties everywhere: all logits equal, two values, a few values; cuts inside a tie go to
    the lowest indexes."""
    x = torch.zeros(6, vocab)
    x[1] = 3.0
    x[1, ::3] = 5.0
    x[2] = torch.randint(0, 4, (vocab,)).float()
    x[3, 7:] = -1.0
    x[4] = torch.randint(0, 2, (vocab,)).float() * 20
    x[5, -1] = 1e-3
    x = x.to(dtype)
    for u in (0.0, 0.25, 0.5, 0.999999):
        for kw in (dict(), dict(k=10), dict(p=0.5), dict(k=51, p=0.3), dict(m=1.0), dict(m=0.2, p=0.7),
                   dict(T=30.0), dict(T=0.01), dict(T=0.0)):
            check(x, torch.full((6,), u), where=(u, kw), **kw)


def test_masked_and_odd_logits(dev):
    """-inf, the type's lowest value, +inf, NaN; rows with nothing to choose."""
    x = torch.randn(12, 3001)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, :3000] = -math.inf
    x[4, ::2] = math.nan
    x[5, 17], x[5, 2000] = math.inf, math.inf
    x[6] = torch.finfo(F32).min
    x[7, 100:] = torch.finfo(F32).min
    x[8, 5] = 1e30
    x[9] = -1e30
    x[9, 77:79] = -0.99e30
    x[10] = -math.inf
    x[10, 3] = -0.0
    x[10, 2000] = 0.0
    x[11] = -math.inf
    x[11, ::100] = math.nan
    for u in (0.0, 0.3, 0.99):
        for kw in (dict(), dict(k=2), dict(k=700), dict(p=0.5), dict(m=0.5), dict(T=0.0),
                   dict(T=math.inf), dict(k=1, p=0.1, m=1.0)):
            check(x, torch.full((12,), u), where=(u, kw), **kw)
            y = x.clone()
            y[8, 5], y[9], y[9, 77:79] = 100.0, -1000.0, -900.0
            check(y.to(BF16), torch.full((12,), u), where=(u, kw), **kw)


def test_options_outside_their_range(dev):
    """In an array nothing is refused: each value's meaning is stated."""
    x = torch.randn(8, 2000) * 2
    u = torch.rand(8)
    T = torch.tensor([math.nan, -1.0, math.inf, 1e-30, 1e30, 1.0, 1.0, 1.0])
    got = check(x, u, T=T)
    assert got[0] == int(x[0].argmax()) and got[3] == int(x[3].argmax())
    p = torch.tensor([-1.0, 0.0, 1e-9, math.nan, 2.0, 1.0, 0.5, 0.9])
    check(x, u, p=torch.where(torch.isnan(p), torch.tensor(1.0), p))
    from summa_amd import sampling
    a = sampling.sample_rows(x.to(dev), u.to(dev), top_p=p.to(dev))[0]
    b = sampling.sample_rows(x.to(dev), u.to(dev), top_p=p.nan_to_num(1.0).to(dev))[0]
    assert torch.equal(a, b)
    k = torch.tensor([-5, 0, 1, 2, 1999, 2000, 2001, 2 ** 31 - 1], dtype=torch.int32)
    check(x, u, k=k)
    m = torch.tensor([-1.0, 0.0, 1e-20, 0.5, 1.0, 2.0, 0.01, 0.3])
    check(x, u, m=m)
    over = torch.tensor([-0.5, 1.0, 1.5, 0.0, math.nan, 0.99999994, 0.5, 2.0 ** -30])
    got = check(x[:4], over[:4])
    assert got[1] == 1999 and got[2] == 1999  # past the end: the last


def test_small_numbers_and_their_neighbours(dev):
    """u right at, below and above borders of whole weights."""
    x = torch.zeros(64, 64)
    u = torch.arange(64) / 64.0
    for v in (u, torch.nextafter(u, torch.tensor(1.0)), torch.nextafter(u, torch.tensor(0.0)).clamp(min=0)):
        check(x, v)
    x[:, 0] = 40.0
    check(x, torch.linspace(0, 1, 65)[:64])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_strided_rows_and_alignment(dev, dtype):
    """Rows of a wider tensor, from any column on."""
    from summa_amd import sampling
    wide = (torch.randn(33, 9001) * 2).to(dtype)
    u = torch.rand(33)
    wd = wide.to(dev)
    for first, vocab in ((0, 9001), (1, 9000), (3, 8191), (7, 130), (2, 4096)):
        x = wide[:, first:first + vocab].contiguous()
        for kw in (dict(top_k=30), dict(top_p=0.8), dict()):
            a = sampling.sample_rows(wd[:, first:first + vocab], u.to(dev), **kw)
            b = sampling.sample_rows(x.to(dev), u.to(dev), **kw)
            assert torch.equal(a[0], b[0])
        check(x, u, k=30, p=0.9)


def test_a_row_does_not_depend_on_its_batch(dev):
    from summa_amd import sampling
    x = (torch.randn(300, 33001) * 2).to(dev)
    u = torch.rand(300, device=dev)
    kw = dict(temperature=0.9, top_k=500, top_p=0.9, min_p=0.001)
    tok, lp = sampling.sample_rows(x, u, **kw)
    for r in (0, 1, 150, 299):
        t, l = sampling.sample_rows(x[r:r + 1], u[r:r + 1], **kw)
        assert int(t) == int(tok[r]) and abs(float(l) - float(lp[r])) <= 2.0 ** -16
    alone = sampling.sample_rows(x, u, want_logprobs=False, **kw)
    assert torch.equal(alone, tok)
    t, l = sampling.sample_rows(x[:0], u[:0])
    assert t.shape == (0,) and l.shape == (0,)


def test_streams_and_graphs(dev):
    """Captured once, replayed with other logits, numbers and options, eager work between."""
    from summa_amd import sampling
    rows, vocab = 20, 40001
    x, u = torch.empty(rows, vocab, device=dev), torch.empty(rows, device=dev)
    T, p = torch.empty(rows, device=dev), torch.empty(rows, device=dev)
    k = torch.empty(rows, dtype=torch.int32, device=dev)
    x2 = torch.empty(3, 131072, dtype=BF16, device=dev)

    def fill(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        x.normal_(0, 2, generator=g)
        x2.normal_(0, 2, generator=g)
        u.uniform_(generator=g)
        T.uniform_(0.3, 1.5, generator=g)
        p.uniform_(0.3, 1.0, generator=g)
        k.random_(-1, 3000, generator=g)

    def step():
        return (*sampling.sample_rows(x, u, temperature=T, top_k=k, top_p=p),
                *sampling.sample_rows(x2, u[:3], top_p=p[:3]))

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
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
