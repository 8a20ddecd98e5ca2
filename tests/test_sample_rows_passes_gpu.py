"""Rows that the sampler does not hold in its lists: what many small weights together come to."""
import math
from fractions import Fraction

import pytest
import torch

from test_sample_rows_gpu import BF16, F16, F32, check

pytestmark = pytest.mark.gpu


def peak_and_tail(vocab, octaves, at):
    """One large logit and a flat rest, 2^-octaves of its weight each."""
    x = torch.full((1, vocab), -octaves * math.log(2.0))
    x[0, at] = 0.0
    w = math.exp(float(x[0, at - 1 if at else 1]))
    return x, w


def behind_the_peak(n, w, u, p=1.0):
    """Tokens that sampling may give where the first of n + 1 weighs 1 and the others w, in exact
    arithmetic. (Running sums in f64 drift: 2^-53 at each of millions of additions to 1, against a w of
    2^-42 to 2^-46.) The kernel's own sums may be off by what 36 additions of up to 1 and the product with u
    round: of its first 4096 logits four in a thread, six over a wave, sixteen over the waves, for the
    thread's sum and again for the step's, and four within the thread; what lies behind them adds up
    small numbers. Its border is off by two roundings."""
    w, u, p = Fraction(w), Fraction(u), Fraction(p)
    whole = 1 + n * w
    tokens = set()
    for border in (p * whole * (1 - Fraction(2) ** -51), p * whole * (1 + Fraction(2) ** -51)):
        kept = n if p >= 1 else min(n, max(0, math.ceil((border - 1) / w)))
        aim = u * (1 + kept * w)
        for off in (-37 * Fraction(2) ** -53, 37 * Fraction(2) ** -53):
            tokens.add(0 if aim + off < 1 else min(kept, math.floor((aim + off - 1) / w) + 1))
    return min(tokens), max(tokens)


@pytest.mark.parametrize("vocab,octaves", [(2 ** 22, 42.1), (2 ** 20 + 7, 44.05), (300001, 46.3), (300001, 60.0)])
def test_flat_tails_of_large_vocabularies(dev, vocab, octaves):
    """Every weight of the tail is nothing beside the largest, and their sum is not."""
    from summa_amd import sampling
    print(f"case tail {vocab} {octaves}", flush=True)
    # behind the peak: the last numbers below one (where the tail has 2^-24 of the whole)
    x, w = peak_and_tail(vocab, octaves, 0)
    tail, xd = w * (vocab - 1), x.to(dev)
    for u in (1 - 2.0 ** -24, 1 - 2.0 ** -22, 1 - 2.0 ** -23):
        for p in (1.0, 1 - 2.0 ** -24, 1 - 2.0 ** -22):
            tok, lp = sampling.sample_rows(xd, torch.tensor([u], device=dev), top_p=p)
            least, most = behind_the_peak(vocab - 1, w, u, p)
            assert least <= int(tok) <= most and most - least <= 2, (u, p, int(tok), least, most)
            assert abs(float(lp) - (float(x[0, int(tok)]) - math.log1p(tail))) <= 2.0 ** -16 + 2.0 ** -23 * 45
            if p == 1:
                assert (most > 0) == (1 - u < tail / (1 + tail))
    # before it: small numbers
    x, w = peak_and_tail(vocab, octaves, vocab - 1)
    for j in (0, 1, 1000, vocab // 2):
        u = torch.tensor([(j + 0.5) * w / (1 + tail)])
        assert check(x, u) == [j]


@pytest.mark.parametrize("vocab,k", [(7, 5), (20000, 9000), (65536, 60000), (131072, 1500)])
@pytest.mark.parametrize("octaves", [47.5, 70.0, 200.0, 800.0])
def test_small_numbers_of_rows_with_a_large_top_k(dev, vocab, k, octaves):
    """A small u is an answer of its own, however small the weights are that it falls in."""
    print(f"case small u {vocab} {k} {octaves}", flush=True)
    x, w = peak_and_tail(vocab, octaves, vocab - 1)
    for T in (1.0, 8.0):
        y = x * T                                    # (exact: a power of two)
        for j in (0, 2, k // 2):
            u = (j + 0.5) * w
            if u < 1e-45:                            # (below the least f32: u is zero)
                u, j = 0.0, 0
            got = check(y, torch.tensor([u]), T=T, k=k, where=(T, j))
            if u == 0.0 or u > 1e-37:
                assert got == [j]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [65536, 131072, 262145, 1 << 20])
def test_flat_rows(dev, vocab, dtype):
    """Spreads from nothing to one: most logits are near the border."""
    print(f"case flat {vocab} {dtype}", flush=True)
    g = torch.Generator().manual_seed(vocab)
    spread = torch.tensor([0.0, 0.01, 0.1, 0.3, 1.0])
    x = (torch.randn(5, vocab, generator=g) * spread[:, None]).to(dtype)
    u = torch.rand(5, generator=g)
    for kw in (dict(), dict(p=0.5), dict(p=0.9, T=2.0), dict(p=0.9, k=vocab // 2), dict(m=0.7, T=0.5)):
        check(x, u, where=kw, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", [(5, 9000), (5, 16384), (5, 32768), (70, 65536), (70, 131072), (2, 131072)])
@pytest.mark.parametrize("order", ["falling", "rising", "together"])
def test_borders_in_one_stretch_of_the_vocabulary(dev, rows, vocab, dtype, order):
    """A vocabulary in the order of its frequencies, and one whose border's logits lie side by side: more of
    them in one wave's range than its part of the list holds, up to the list's 512 or 1024 and past it."""
    print(f"case stretch {rows} {vocab} {dtype} {order}", flush=True)
    g = torch.Generator().manual_seed(vocab)
    if order == "together":
        x = torch.randn(rows, vocab, generator=g) * 2 - 12
        near = [40, 60, 130, 500, 900, 1500, 0][: rows]
        for r in range(rows):
            at = vocab // 3 + 17 * r
            x[r, at:at + near[r % len(near)]] = 2e-4 * torch.rand(near[r % len(near)], generator=g)
            x[r, 11] = 3.0
    else:
        x = torch.sort(torch.randn(rows, vocab, generator=g) * 2, 1, descending=order == "falling")[0]
    x = x.to(dtype)
    u = torch.rand(rows, generator=g)
    for kw in (dict(p=0.97), dict(p=0.6, T=1.3), dict(p=0.9, m=1e-3)):
        check(x, u, where=(order, kw), **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [49153, 65536, 131072])
def test_a_row_is_the_same_in_every_batch(dev, vocab, dtype):
    """Shared out over the chip in small batches, in one workgroup in large ones: the rows' tokens are the
    definition's and each other's, log-probs the same within their f32 sums."""
    from summa_amd import sampling
    print(f"case batches {vocab} {dtype}", flush=True)
    x = (torch.randn(300, vocab) * 2).to(dtype)
    u = torch.rand(300)
    xd, ud = x.to(dev), u.to(dev)
    for kw in (dict(), dict(top_k=300), dict(top_p=0.9), dict(top_k=400, top_p=0.8, min_p=1e-3),
               dict(temperature=0.0), dict(min_p=0.05, temperature=1.4)):
        tok, lp = sampling.sample_rows(xd, ud, **kw)
        for rows in (1, 3, 8, 31, 32, 33, 63, 64, 65, 128):
            t, l = sampling.sample_rows(xd[:rows], ud[:rows], **kw)
            assert torch.equal(t, tok[:rows]), (kw, rows)
            assert float((l - lp[:rows]).abs().max()) <= 2.0 ** -15, (kw, rows)
        names = dict(top_k="k", top_p="p", min_p="m", temperature="T")
        got = check(x[:4], u[:4], **{names[k]: v for k, v in kw.items()})
        assert got == tok[:4].tolist()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_logits_of_a_very_large_vocabulary(dev, dtype):
    """Counts past 2^24: every token, border and draw follows from the number of logits."""
    from summa_amd import sampling
    n = 2 ** 25 + 3
    print(f"case equal {n} {dtype}", flush=True)
    x = torch.full((1, n), -3.0, dtype=dtype, device=dev)
    for u in (0.0, 2.0 ** -26, 0.7, 1 - 2.0 ** -24):
        for kw, kept in ((dict(), n), (dict(top_k=2 ** 24 + 5), 2 ** 24 + 5), (dict(top_p=0.75), math.ceil(0.75 * n)),
                         (dict(top_k=2 ** 24 + 5, top_p=0.5), math.ceil((2 ** 24 + 5) * 0.5)),
                         (dict(min_p=1.0, temperature=0.3), n)):
            ud = torch.tensor([u], device=dev)
            tok, lp = sampling.sample_rows(x, ud, **kw)
            # the first at which i + 1 > u kept, in 64 bits exact up to one rounding (2^-27 of a token)
            assert int(tok) == int(Fraction(float(ud)) * kept), (u, kw)
            assert abs(float(lp) + math.log(n)) <= 2.0 ** -20 * math.log(n)
