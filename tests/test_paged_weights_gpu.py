"""Paged attention where one key dominates and the rest of the weight lies in very many small
weights, as behind the first token of a long context."""
import math

import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu
BF16, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
TOKENS = 1 << 17


@pytest.mark.parametrize("dtype,cdt", [(F16, F16), (F16, F8), (BF16, F8), (BF16, BF16)])
@pytest.mark.parametrize("n,H", [(1, 2), (12, 2)])  # the 16-row kernel, the tile kernel
@pytest.mark.parametrize("below", [16, 24, 26, 30])
@pytest.mark.parametrize("split", [False, True])
def test_one_key_before_many_small_weights(dev, split, below, n, H, dtype, cdt):
    """The first key's score is `below` binary orders above 131 k others', and its value zero:
    the output is what the others have.

    Tolerance: the output's rounding; each weight's, half a step of its type, and in f16 at
    most half of 2^-24 where the largest weight is 2^11 or more (2^-36 of it for every key);
    scores: products exact, hd + 2 roundings of up to |q| . |k|; 2^-20 for exp2; and the f32
    sums, of some thousand terms a lane: a wave's 16 or 32 keys of TOKENS, less than 2^13
    additions in a row, each off by 2^-24 of the sum."""
    from summa_amd import paged
    print(f"case dominant {split} {below} {n} {H} {dtype} {cdt}", flush=True)
    hd, page = 64, 64
    cache = paged.PagedKVCache(TOKENS // page, 1, hd, page, cdt, dev)
    table = torch.randperm(TOKENS // page).int()[None].contiguous()
    k = torch.randn(TOKENS, 1, hd) * 0.02
    v = 1.0 + 0.25 * torch.randn(TOKENS, 1, hd)
    k[0], v[0] = 1.0, 0.0
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    paged.paged_append(cache, k.to(dev), v.to(dev), table.to(dev), zero)
    q = torch.full((n, H, hd), below * math.log(2) / math.sqrt(hd)) + 0.001 * torch.randn(n, H, hd)
    q = q.to(dtype)
    out, lse = paged.paged_attention(cache, q.to(dev), table.to(dev), zero + (TOKENS - n),
                                     max_tokens=TOKENS if split else 1, want_lse=True)
    ref, rl, mag, err, unit = P.attend(q, P.read(cache.k, cache.v, cache.k_scales, cache.v_scales),
                                       table.tolist(), [TOKENS - n], [0, n], page)
    p = HALF[BF16] if cdt == BF16 else HALF[F16]
    score = err.double()[..., None] * (hd + 6) * 2.0 ** -24
    tol = (HALF[dtype] * ref.abs() + (p + 2 * score + 2.0 ** -20 + 2.0 ** -11) * mag) * 1.01 + \
        (0.0 if cdt == BF16 else unit * 2.0 ** -36) + (2.0 ** -25 if dtype == F16 else 0.0)
    d = (out.cpu().double() - ref).abs()
    assert bool((d <= tol).all()), (float((d - tol).max()), float((d / ref).max()))
    t = err.double() * (hd + 6) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * rl.abs() + 2.0 ** -11
    assert bool(((lse.cpu().double() - rl).abs() <= t).all())
