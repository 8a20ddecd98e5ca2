"""Copies of more pieces than a launch takes, and those refused as too many."""
import ctypes

import pytest
import torch

from summa_amd import _lib

D = 1 << 20  # a device pointer that is never dereferenced


def test_refused_sizes():
    def go(n, layers=1, pages=4, page=32):
        c = (_lib.PagedCache * layers)(*[_lib.PagedCache(D, D, D, D, pages, 1, page, 128, _lib.SM_F16)
                                         for _ in range(layers)])
        st = _lib.lib().sm_paged_copy(c, layers, D, D, n, None)
        return st, _lib.lib().sm_last_error().decode()
    # 2^31 pieces in all; a page of more pieces than a launch has
    for st, err in (go(1 << 30), go(1 << 25, 32), go(1, 1, 1, 2 ** 31 - 16)):
        assert st == -3 and "too large" in err


@pytest.mark.gpu
@pytest.mark.parametrize("n,layers", [(2 ** 23 - 1, 1), (2 ** 23, 1), (2 ** 23 + 5, 1), (300001, 35)])
def test_pairs_of_several_launches(dev, n, layers):
    """A compaction's lists are half the pool's pages, most of them -1: the pairs that there are may lie in any
    of the launches."""
    from summa_amd import paged
    caches = [paged.PagedKVCache(9, 1, 64, 16, torch.float8_e4m3fn, dev) for _ in range(layers)]
    for c in caches:
        for x in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scales, c.v_scales):
            x.copy_(torch.randint(0, 256, x.shape))
    src = torch.full((n,), -1, dtype=torch.int32, device=dev)
    dst = src.clone()
    each = (2 ** 24 - 1) // (2 * min(layers, 32))
    at = sorted({0, min(each, n) - 1, min(each, n - 1), n - 1})
    ref = [[x.clone() for x in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scales, c.v_scales)]
           for c in caches]
    for i, a in enumerate(at):
        src[a], dst[a] = i, 8 - i
    paged.paged_copy(caches, src, dst)
    for c, old in zip(caches, ref):
        for x, y in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scales, c.v_scales), old):
            for i in range(len(at)):
                y[8 - i] = y[i].clone()
            assert torch.equal(x, y)
