"""What the calls of drafted trees, pages and row sampling refuse, without a device: arguments are
settled before anything is launched, and what is empty launches nothing."""
import ctypes

import pytest
import torch

from summa_amd import _lib

D = 1 << 20  # a device pointer that is never dereferenced
F8, F16, BF16, F32 = _lib.SM_F8E4M3, _lib.SM_F16, _lib.SM_BF16, _lib.SM_F32


def call(name, *args):
    st = getattr(_lib.lib(), name)(*args)
    return st, _lib.lib().sm_last_error().decode()


def cache(dtype=F16, pages=4, heads=2, page=32, hd=64, k=D):
    return _lib.PagedCache(k, D, D, D, pages, heads, page, hd, dtype)


def test_masks_and_accept():
    for n in ("sm_tree_masks", "sm_tree_accept"):
        def go(S, rows, most, starts=None, words=64, parents=D, pos0=D):
            if n == "sm_tree_masks":
                return call(n, parents, pos0, starts, S, rows, most, D, words, D, None)
            return call(n, parents, D, D, starts, S, rows, most, D, D, None, None)
        assert "at most 1024 rows" in go(2, 4096, 1025, D)[1]
        assert "rows must be S * max_rows" in go(2, 9, 4)[1]
        assert go(-1, 4, 4)[0] == -1 and go(1 << 24, 0, 0)[0] == -1 and go(2, 4, 5, D)[0] == -1
        assert "null buffer" in go(2, 8, 4, parents=None)[1]
        assert go(0, 0, 0)[0] == 0
    assert "words must be" in call("sm_tree_masks", D, D, None, 2, 80, 40, D, 1, D, None)[1]
    assert "null buffer" in call("sm_tree_masks", D, None, None, 2, 80, 40, D, 2, D, None)[1]


def test_keep_and_copy():
    c = (_lib.PagedCache * 2)(cache(), cache(heads=3))
    for n, rest in (("sm_paged_keep", (D, D, 2, 8, D, 4, D, None)), ("sm_paged_copy", (D, D, 8, None))):
        assert "one geometry" in call(n, c, 2, *rest)[1]
        assert "page_tokens a positive multiple of 16" in call(n, (_lib.PagedCache * 1)(cache(page=24)), 1, *rest)[1]
        assert "null cache pages" in call(n, (_lib.PagedCache * 1)(cache(k=0)), 1, *rest)[1]
        assert "0 to 65535 caches" in call(n, c, -1, *rest)[1]
        assert call(n, None, 0, *rest)[0] == 0
    one = (_lib.PagedCache * 1)(cache())
    assert "null buffer" in call("sm_paged_keep", one, 1, D, None, 2, 8, D, 4, D, None)[1]
    assert "table_cols" in call("sm_paged_keep", one, 1, D, D, 2, 8, D, 0, D, None)[1]
    assert call("sm_paged_keep", one, 1, None, None, 0, 8, None, 0, None, None)[0] == 0
    big = (_lib.PagedCache * 1)(cache(heads=2000))
    st, err = call("sm_paged_keep", big, 1, D, D, 1 << 23, 8, D, 4, D, None)
    assert st == -3 and "too large" in err
    st, err = call("sm_paged_copy", one, 1, D, D, 1 << 30, None)
    assert st == -3 and "too large" in err
    assert "null buffer" in call("sm_paged_copy", one, 1, None, D, 3, None)[1]
    assert call("sm_paged_copy", one, 1, None, None, 0, None)[0] == 0


def test_pages():
    for pages in (0, -1, 2 ** 31 - 1):
        assert "pages must be positive" in call("sm_page_reserve", D, pages, D, 2, 4, D, 16, None, None)[1]
        assert "pages must be positive" in call("sm_page_compact", D, pages, D, D, D, D, None)[1]
    assert "page_tokens" in call("sm_page_reserve", D, 9, D, 2, 4, D, 0, None, None)[1]
    assert "table_cols" in call("sm_page_reserve", D, 9, D, 2, 0, D, 16, None, None)[1]
    assert "null buffer" in call("sm_page_reserve", D, 9, D, 2, 4, None, 16, None, None)[1]
    assert "null refs" in call("sm_page_free", None, 9, D, 2, 4, None, 16, None)[1]
    assert "null buffer" in call("sm_page_free", D, 9, None, 2, 4, None, 16, None)[1]
    assert call("sm_page_free", D, 9, None, 0, 4, None, 16, None)[0] == 0

    def fork(table=D, out=2 * D, P=3, C=5, src=D):
        return call("sm_page_fork", D, 9, table, P, 4, D, D, C, 16, out, src, D, None, None)
    assert "overlap" in fork(out=D) [1] and "overlap" in fork(out=D + 44)[1] and \
        "overlap" in fork(out=D - 76)[1]
    assert "null buffer" in fork(src=None)[1] and "null buffer" in fork(table=None)[1]
    assert fork(P=-1)[0] == -1 and fork(C=(1 << 24) + 1)[0] == -1
    assert "null buffer" in call("sm_page_remap", None, 4, D, 9, D, None)[1]
    assert call("sm_page_remap", None, 0, D, 9, D, None)[0] == 0
    assert call("sm_page_remap", D, -1, D, 9, D, None)[0] == -1


def test_tree_attention():
    def go(cdt=F16, dtype=F16, mask=D, words=2, rows=80, most=40, q=D, out=1 << 24, ldq=256, tokens=100):
        c = cache(cdt)
        return call("sm_paged_tree_attention", ctypes.addressof(c), D, 4, D, None, 2, rows, most, tokens,
                    mask, words, q, dtype, ldq, 4, out, None, None, 0, None)
    assert "null buffer" in go(mask=None)[1]
    assert "words must be at least" in go(words=1)[1]
    assert "16-bit cache must have the query's dtype" in go(cdt=BF16)[1]
    assert "dtype must be SM_BF16 or SM_F16" in go(dtype=F32)[1]
    assert "without row_start" in go(rows=81)[1]
    assert "must not overlap q" in go(out=D + 64)[1]
    assert "16-byte aligned" in go(ldq=257)[1]
    assert "workspace of 0 bytes" in go(tokens=1 << 20)[1]
    assert go(rows=0, most=0, mask=None)[0] == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=F8), "dtype must be SM_F32, SM_BF16 or SM_F16"),
    (dict(vocab=0), "1 to 2^30 - 1 logits"),
    (dict(vocab=1 << 30, ld=1 << 30), "1 to 2^30 - 1 logits"),
    (dict(rows=1 << 22), "0 to 2^22 - 1 rows"),
    (dict(ld=99), "ld must be at least vocab"),
    (dict(temperature=float("nan")), "temperature must not be NaN"),
    (dict(top_p=0.0), "top_p must be in (0, 1]"), (dict(top_p=1.5), "top_p must be in (0, 1]"),
    (dict(top_p=float("nan")), "top_p must be in (0, 1]"),
    (dict(min_p=-0.1), "min_p must be in [0, 1]"), (dict(min_p=1.1), "min_p must be in [0, 1]"),
    (dict(logits=None), "null buffer"), (dict(tokens=None), "null buffer"),
    (dict(uniforms=None), "null buffer"),
])
def test_sample_rows(kw, msg):
    from summa_amd.sampling import RowSamplingC
    a = dict(logits=D, dtype=F32, rows=4, ld=100, vocab=100, uniforms=D, tokens=D, temperature=1.0,
             top_p=1.0, min_p=0.0)
    a.update(kw)
    o = RowSamplingC(None, None, None, None, a["temperature"], -1, a["top_p"], a["min_p"])
    st, err = call("sm_sample_rows", a["logits"], a["dtype"], a["rows"], a["ld"], a["vocab"], a["uniforms"],
                   ctypes.addressof(o), a["tokens"], None, None, 0, None)
    assert st == -1 and msg in err


def test_sample_rows_of_no_rows():
    from summa_amd.sampling import RowSamplingC
    o = RowSamplingC(None, None, None, None, 1.0, -1, 1.0, 0.0)
    assert call("sm_sample_rows", None, F32, 0, 100, 100, None, ctypes.addressof(o), None, None, None, 0,
                None)[0] == 0
    assert "null options" in call("sm_sample_rows", D, F32, 1, 100, 100, D, None, D, None, None, 0, None)[1]
    assert _lib.lib().sm_sample_rows_workspace_bytes(4, 0, F32) == -1
    assert _lib.lib().sm_sample_rows_workspace_bytes(4, 100, F8) == -1


def test_host_tensors_are_refused():
    """The Python calls take device tensors only."""
    from summa_amd import paged, pages, sampling, tree
    t, i = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32)
    one = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: sampling.sample_rows(t, torch.zeros(2)), lambda: tree.tree_masks(i, one),
              lambda: tree.tree_accept(i, i, i), lambda: pages.page_free(one, i, 16),
              lambda: pages.page_reserve(one, i, one, 16), lambda: pages.page_fork(one, i, one, one, 16),
              lambda: pages.page_compact(one), lambda: pages.page_remap(i, one)):
        with pytest.raises(ValueError, match="on the device"):
            f()
    with pytest.raises(ValueError):
        pages.page_refs(0)
    with pytest.raises(TypeError):
        sampling.sample_rows(t.double(), torch.zeros(2))
    with pytest.raises(ValueError, match="at least one cache"):
        paged.paged_copy([], one, one)
