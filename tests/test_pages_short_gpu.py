"""Pools that are too small and tables that are too narrow: what a fork shares, copies and counts."""
import pytest
import torch

from test_pages_gpu import Pool, i32

pytestmark = pytest.mark.gpu


def fork(pool, table, tokens, source, page):
    """The definition: a child holds what its prompt's row holds, and a page of its own for an unfinished
    last page that is there to be copied."""
    cols, pages = len(table[0]), len(pool.refs)
    out, src, dst, missing = [], [], [], 0
    for s in source:
        row, a = [-1] * cols, -1
        if 0 <= s < len(table):
            n = max(0, tokens[s])
            full, need = n // page, -(-n // page)
            held = [p if 0 <= p < pages else -1 for p in table[s]]
            missing += sum(p < 0 for p in held[:need]) + max(0, need - cols)
            row[:full] = held[:full][:cols]
            if need > full and full < cols:
                a = held[full]
        else:
            missing += 1
        out.append(row)
        src.append(a)
        dst.append(-1)
    free = sorted((p for p, r in enumerate(pool.refs) if r <= 0), reverse=True)
    for row in out:
        for p in row:
            if p >= 0:
                pool.refs[p] += 1
    for c, s in enumerate(source):
        if src[c] >= 0:
            if free:
                dst[c] = out[c][tokens[s] // page] = free.pop()
                pool.refs[dst[c]] = 1
            else:
                src[c] = -1
                missing += 1
    return out, src, dst, missing


@pytest.mark.parametrize("pages,S,cols,page", [(1, 1, 1, 16), (6, 3, 4, 16), (30, 9, 7, 32), (900, 40, 70, 16),
                                               (3000, 1100, 5, 48)])
def test_forks_of_prompts_without_all_their_pages(dev, pages, S, cols, page):
    from summa_amd import pages as pg
    gen = torch.Generator().manual_seed(pages)
    rnd = lambda hi, n=1: torch.randint(0, hi, (n,), generator=gen).tolist()  # noqa: E731
    short = 0
    for turn in range(6):
        pool, refs = Pool([0] * pages), pg.page_refs(pages, dev)
        table = [[-1] * cols for _ in range(S)]
        t = torch.full((S, cols), -1, dtype=torch.int32, device=dev)
        tokens = rnd(cols * page + 3 * page, S)
        room = [min(x, y) for x, y in zip(tokens, rnd(2 * cols * page, S))] if turn % 2 else tokens
        pg.page_reserve(refs, t, i32(room, dev), page)
        pool.reserve(table, room, page)
        if turn > 3:   # and entries that name no page
            table[S // 2][0] = pages + 3
            t[S // 2, 0] = pages + 3
        if turn > 1:   # room for some of the children
            for s in range(0, S, 2):
                keep = [x if i != s else 0 for i, x in enumerate(room)]
                pool.free(table[s:s + 1], [0], page)
                pg.page_free(refs, t[s:s + 1], page)
                room = keep
        kids = [k - 1 for k in rnd(S + 2, 50)]
        missing = torch.full((1,), 77, dtype=torch.int32, device=dev)
        c, src, dst = pg.page_fork(refs, t, i32(tokens, dev), i32(kids, dev), page, missing=missing)
        rc, rs, rd, rm = fork(pool, table, tokens, kids, page)
        assert c.tolist() == rc and src.tolist() == rs and dst.tolist() == rd
        assert refs.tolist() == pool.refs and int(missing) == rm
        assert all((a < 0) == (b < 0) for a, b in zip(rs, rd))
        short += rm
    assert short > 0


def test_a_child_never_shows_anothers_tokens(dev):
    """A prompt whose reserve ran short in its last page: its children have no page there, free or not."""
    from summa_amd import pages as pg
    refs = pg.page_refs(5, dev)
    other = torch.full((1, 2), -1, dtype=torch.int32, device=dev)
    pg.page_reserve(refs, other, i32([32], dev), 16)
    table = torch.full((1, 4), -1, dtype=torch.int32, device=dev)
    missing = torch.zeros(1, dtype=torch.int32, device=dev)
    pg.page_reserve(refs, table, i32([60], dev), 16, missing)
    assert int(missing) == 1 and table.tolist() == [[2, 3, 4, -1]]
    pg.page_free(refs, other, 16)
    kids, src, dst = pg.page_fork(refs, table, i32([60], dev), i32([0, 0], dev), 16, missing=missing)
    assert kids.tolist() == [[2, 3, 4, -1]] * 2
    assert src.tolist() == [-1, -1] and dst.tolist() == [-1, -1]
    assert int(missing) == 2 and refs.tolist() == [0, 0, 3, 3, 3]


def test_missing_does_not_wrap(dev):
    """Counts past 2^31 - 1 stay there."""
    from summa_amd import pages as pg
    refs = pg.page_refs(4, dev)
    missing = torch.zeros(1, dtype=torch.int32, device=dev)
    table = torch.full((3, 2), -1, dtype=torch.int32, device=dev)
    most = i32([2 ** 31 - 1] * 3, dev)
    pg.page_fork(refs, table, most, i32([0, 1, 2, 5], dev), 1, missing=missing)
    assert int(missing) == 2 ** 31 - 1
    pg.page_fork(refs, table, most, i32([0, 9, 9], dev), 2 ** 20, missing=missing)
    assert int(missing) == 2 ** 11 + 2


def test_missing_of_a_reserve_does_not_wrap(dev):
    """Columns that narrow tables lack, past 2^31 together; the pages that there are are given all the same."""
    from summa_amd import pages as pg
    for S, page, most in ((3, 1, 2 ** 31 - 1), (1200, 16, 2 ** 31 - 1), (1, 16, 2 ** 27 - 2)):
        refs = pg.page_refs(4, dev)
        missing = torch.zeros(1, dtype=torch.int32, device=dev)
        table = torch.full((S, 2), -1, dtype=torch.int32, device=dev)
        pg.page_reserve(refs, table, torch.full((S,), 2 ** 31 - 1, dtype=torch.int32, device=dev), page,
                        missing)
        assert int(missing) == most
        got = [p for row in table.tolist() for p in row]
        given = min(4, 2 * S)
        assert got == list(range(given)) + [-1] * (2 * S - given) and int(refs.sum()) == given
