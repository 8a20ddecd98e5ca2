"""Paged attention where the weights or the scales of the values are far apart: the softmax
sum and its parts of other waves and splits, against 64-bit definitions."""
import math

import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu
BF16, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def stored(hd, page, keys, vals, ev):
    """Storage (k, v, k_scales, v_scales) of one sequence's e4m3 keys and values [tokens, hd]
    (whole pages, kept in reverse order) with the exponents ev of V's blocks and 0 of K's,
    and its page table."""
    pages = keys.shape[0] // page
    k = keys.view(pages, 1, page, hd).flip(0).contiguous()
    v = torch.empty(pages, 1, page // 16, 16 * hd, dtype=torch.uint8)
    v[..., P.v_index(hd, 4)] = vals.view(torch.uint8).view(pages, 1, page // 16, 16, hd)
    v = v.flip(0).contiguous().view(pages, 1, page // 16, hd // 64, 4, 16, 4, 4).view(F8)
    vs = (torch.tensor(ev) + 127).to(torch.uint8).view(pages, 1, page // 16).flip(0).contiguous()
    return (k, v, torch.full_like(vs, 127), vs), torch.arange(pages - 1, -1, -1)[None].int()


def attend(dev, tensors, table, q, pos0, most):
    from summa_amd import paged
    cache = paged.PagedKVCache.from_tensors(*(x.to(dev) for x in tensors))
    return paged.paged_attention(cache, q.to(dev), table.to(dev),
                                 torch.tensor([pos0], dtype=torch.int32, device=dev),
                                 max_tokens=most, want_lse=True)


def check(got, lse, ref, rl, mag, err, unit, hd, dtype):
    """The output's rounding; P's, 2^-11 of each weight; P's f16 subnormals: weights are held
    so that the largest weight times scale is at least 2^10, so half a step of 2^-24 is
    2^-35 of it for every key; scores in f32, products exact, hd + 2 roundings of up to
    |q| . |k|; and the exponents of scales, up to 127 + 63 beside a score in f32: half a step
    of values below 256 is 2^-17, once in the weights and once in their sum, with what a sum
    leaves out of keys 33 and more binary orders below the largest (fewer than 2^10 keys:
    2^-23)."""
    score = err.double()[..., None] * (hd + 6) * 2.0 ** -24 + 2.0 ** -17
    tol = (HALF[dtype] * ref.abs() + (2.0 ** -11 + 2 * score + 2.0 ** -20) * mag) * 1.01 + \
        unit * 2.0 ** -35 + (2.0 ** -25 if dtype == F16 else 2.0 ** -134)
    d = (got.cpu().double() - ref).abs()
    assert bool((d <= tol).all()), (float((d - tol).max()), float((d / ref.abs()).max()))
    t = err.double() * (hd + 6) * 2.0 ** -24 + 2 * 2.0 ** -17 + 2.0 ** -22 * rl.abs()
    assert bool(((lse.cpu().double() - rl).abs() <= t).all()), (lse.cpu().double() - rl).abs().max()


def one_large(hd, n, G, small, big, place, gap):
    """(storage, table, q) with one block of values near 2^big, its score about `gap` binary
    orders above the others'."""
    keys = torch.randn(640, hd).clamp(-3, 3) * 0.02
    vals = torch.randn(640, hd).clamp(-4, 4) * 100
    at = slice(place * 16, place * 16 + 16)
    if gap:
        keys[at] += 1.0
    if small == "zeros":
        large, vals = vals, torch.zeros_like(vals)
        vals[at] = large[at]
    ev = [-63] * 40
    ev[place] = big
    q = torch.randn(n, G, hd) * 0.1 + gap * math.log(2) / math.sqrt(hd)
    return *stored(hd, 32, keys.to(F8), vals.to(F8), ev), q.to(BF16)


def any_scales(hd, n, G, dtype, slope):
    """(storage, table, q) with any scale bytes from 64 to 245 for V; a block's score falls by
    `slope` binary orders, about, for each by which its scale passes 1."""
    ev = torch.randint(-63, 119, (48,))
    keys = torch.randn(768, hd).clamp(-3, 3) * 0.02
    vals = torch.randn(768, hd).clamp(-4, 4) * 60
    keys -= (ev.clamp(min=0) * slope / 8).repeat_interleave(16)[:, None]
    q = torch.randn(n, G, hd) * 0.01 + 8 * math.log(2) / math.sqrt(hd)
    return *stored(hd, 32, keys.to(F8), vals.to(F8), ev.tolist()), q.to(dtype)


SHAPES = [(64, 1, 3), (128, 2, 4), (64, 9, 3), (128, 40, 1)]  # hd, rows, heads


# Places of the large block among 40: blocks 2 w, 2 w + 1 of every eight are wave w's of the
# 16-row kernel, a split is 32 blocks.
@pytest.mark.parametrize("place", [0, 1, 3, 31, 33, 39])
@pytest.mark.parametrize("big", [41, 70, 91, 118])
@pytest.mark.parametrize("small", ["zeros", "values"])
@pytest.mark.parametrize("hd,n,G", SHAPES)
def test_one_block_of_large_values(dev, hd, n, G, small, big, place):
    """One block of values near 2^big among blocks of the least scale, zeros or values near
    2^-57: every block's share of the sum stays, with equal scores and with the large block's
    far above and below."""
    for gap in (0, 20, -20, -70):
        tensors, table, q = one_large(hd, n, G, small, big, place, gap)
        ref = P.attend(q, P.read(*tensors), table.tolist(), [640 - n], [0, n], 32)
        for most in (1, 640):  # one split, and two
            print(f"case large {hd} {n} {G} {small} {big} {place} {gap} {most}", flush=True)
            check(*attend(dev, tensors, table, q, 640 - n, most), *ref, hd, BF16)


@pytest.mark.parametrize("dtype,slope", [(BF16, 0.0), (BF16, 0.5), (BF16, 1.0), (BF16, 1.25), (F16, 1.25)])
@pytest.mark.parametrize("hd,n,G", SHAPES)
def test_scales_anywhere_in_their_range(dev, hd, n, G, dtype, slope):
    for it in range(3):
        tensors, table, q = any_scales(hd, n, G, dtype, slope)
        ref = P.attend(q, P.read(*tensors), table.tolist(), [768 - n], [0, n], 32)
        for most in (1, 768):
            print(f"case any {hd} {n} {G} {dtype} {slope} {it} {most}", flush=True)
            check(*attend(dev, tensors, table, q, 768 - n, most), *ref, hd, dtype)
