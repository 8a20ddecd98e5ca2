"""What a 16-bit paged cache holds of values that are not finite, and of those that its type
does not: the append stores what one rounding to the type gives."""
import math

import pytest
import torch

import _paged as P
from test_paged_gpu import Batch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("cdt", [BF16, F16])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_values_that_are_not_finite(dev, hd, dt, cdt):
    b = Batch(dev, [0, 21, 3], [17, 17, 1], 2, hd, 32, cdt)
    b.fill()
    k, v = torch.randn(2, b.rows, 2, hd)
    for x in (k, v):
        for r in range(0, b.rows, 3):
            x[r, r % 2, 5], x[r, r % 2, 6], x[r, 0, hd - 1] = math.inf, math.nan, -math.inf
        x[1, 0, :8] = torch.tensor([65504.0, 65519.0, 65520.0, -65520.0, 1e5, -1e30, 3.39e38, -3.4e38])
    k, v = k.to(dt), v.to(dt)
    before = b.raw()
    b.append(k.to(dev), v.to(dev))
    K, V = b.store()[:2]
    for s, n in enumerate(b.n):
        for i in range(n):
            p = b.pos0[s] + i
            for new, got in ((k, K), (v, V)):
                got = got[b.table[s][p // 32], :, p % 32]
                want = new[b.starts[s] + i].to(cdt).double()
                same = (got == want) | (torch.isnan(got) & torch.isnan(want))
                assert bool(same.all()), (s, i, got[~same], want[~same])
    touched = sum(int((x != y).sum()) for x, y in zip(before, b.raw()))
    assert touched <= 2 * sum(b.n) * 2 * hd


@pytest.mark.parametrize("cdt", [BF16, F16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotated_values_that_are_not_finite(dev, layout, cdt):
    """An infinity or NaN reaches the two dims of its pair, as products and sums have it, and no
    other; V is not rotated."""
    b = Batch(dev, [7], [20], 1, 64, 32, cdt)
    k, v = torch.randn(2, 20, 1, 64)
    k[2, 0, 4], k[5, 0, 9], k[9, 0, 50] = math.inf, math.nan, -math.inf
    table = P.angles(32, 64)
    b.fill()
    b.append(k.to(dev), v.to(dev), rope_table=table.to(dev), layout=layout)
    K, V = b.store()[:2]
    for i in range(20):
        p = 7 + i
        got = K[b.table[0][p // 32], 0, p % 32]
        want = P.rotate(k[i, 0], table[p], layout).to(cdt).double()
        assert torch.equal(torch.isfinite(got), torch.isfinite(want)), i
        assert torch.equal(torch.isnan(got), torch.isnan(want)), i
        inf = torch.isinf(want)
        assert torch.equal(got[inf], want[inf]), i
        assert torch.equal(V[b.table[0][p // 32], 0, p % 32], v[i, 0].to(cdt).double())
