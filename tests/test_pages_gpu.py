"""The pages of a paged cache against a simulation: reserve, fork, free, compact, remap, copy; and a
drafted rollout that uses all of it."""
import math

import pytest
import torch

import _paged as P
import _tree as R
from test_paged_gpu import BF16, F16, F8, tolerance

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Pool:
    """The definition: lowest free page first."""

    def __init__(self, refs):
        self.refs = list(refs)

    def take(self):
        for p, r in enumerate(self.refs):
            if r <= 0:
                self.refs[p] = 1
                return p
        return -1

    def reserve(self, table, tokens, page):
        missing = 0
        for row, t in zip(table, tokens):
            need = max(0, -(-t // page))
            held = next((j for j, p in enumerate(row) if p < 0), len(row))
            for j in range(held, min(need, len(row))):
                row[j] = self.take()
                missing += row[j] < 0
            missing += max(0, need - len(row))
        return missing

    def fork(self, table, tokens, source, page):
        out, src, dst, missing = [], [], [], 0
        cols = len(table[0]) if table else 1
        pending = []
        for s in source:
            row, a = [-1] * cols, -1
            if not 0 <= s < len(table):
                missing += 1
            else:
                t = max(0, tokens[s])
                full = t // page
                for j in range(min(full, cols)):
                    row[j] = table[s][j]
                if full >= cols:
                    missing += t > cols * page
                elif t % page:
                    a = table[s][full]
                    pending.append((len(out), full))
            out.append(row)
            src.append(a)
            dst.append(-1)
        for c, full in pending:
            out[c][full] = dst[c] = self.take()
            missing += dst[c] < 0
        for c in range(len(out)):
            for j, p in enumerate(out[c]):
                if p >= 0 and p != dst[c]:
                    self.refs[p] += 1
            if dst[c] < 0:
                src[c] = -1
        return out, src, dst, missing

    def free(self, table, tokens, page):
        for row, t in zip(table, tokens):
            for j in range(max(0, -(-t // page)), len(row)):
                if 0 <= row[j] < len(self.refs):
                    self.refs[row[j]] = max(0, self.refs[row[j]] - 1)
                row[j] = -1


@pytest.mark.parametrize("pages,S,cols,page", [(1, 1, 1, 16), (50, 5, 7, 16), (4097, 70, 40, 32),
                                               (20000, 1500, 9, 64), (300, 2, 200, 16)])
def test_reserve_fork_free(dev, pages, S, cols, page):
    """A pool's life at random: growth, forks, release, more than there is."""
    from summa_amd import pages as pg
    gen = torch.Generator().manual_seed(pages)
    rnd = lambda hi, n=1: torch.randint(0, hi, (n,), generator=gen).tolist()  # noqa: E731
    pool = Pool([0] * pages)
    refs = pg.page_refs(pages, dev)
    table = [[-1] * cols for _ in range(S)]
    t = torch.full((S, cols), -1, dtype=torch.int32, device=dev)
    missing = torch.zeros(1, dtype=torch.int32, device=dev)
    tokens = [0] * S
    for step in range(6):
        tokens = [min(x + y, cols * page + page) for x, y in zip(tokens, rnd(cols * page // 3 + 2, S))]
        pg.page_reserve(refs, t, i32(tokens, dev), page, missing)
        assert pool.reserve(table, tokens, page) == int(missing)
        assert t.tolist() == table and refs.tolist() == pool.refs
        kids = rnd(S + 2, min(2 * S, 40))
        kids = [k - 1 for k in kids]   # sources that do not exist among them
        out = None if step % 2 else torch.full((len(kids), cols), 12345, dtype=torch.int32, device=dev)
        c, src, dst = pg.page_fork(refs, t, i32(tokens, dev), i32(kids, dev), page, out=out,
                                   missing=missing)
        rc, rs, rd, rm = pool.fork(table, tokens, kids, page)
        assert c.tolist() == rc and src.tolist() == rs and dst.tolist() == rd and int(missing) == rm
        assert refs.tolist() == pool.refs
        keep = [x // 2 for x in tokens]
        pg.page_free(refs, c, page)
        pool.free(rc, [0] * len(rc), page)
        assert c.tolist() == rc and refs.tolist() == pool.refs
        pg.page_free(refs, t, page, i32(keep, dev))
        pool.free(table, keep, page)
        assert t.tolist() == table and refs.tolist() == pool.refs
        tokens = keep
    pg.page_free(refs, t, page)
    assert not refs.any() and bool((t == -1).all())
    # entries too many: no count below zero
    t.fill_(min(3, pages - 1))
    pg.page_free(refs, t, page)
    assert not refs.any()


@pytest.mark.parametrize("pages", [1, 2, 31, 1000, 4096, 4097, 9000])
@pytest.mark.parametrize("live", [0.0, 0.01, 0.3, 0.9, 1.0])
def test_compact(dev, pages, live):
    from summa_amd import pages as pg
    gen = torch.Generator().manual_seed(pages)
    refs = torch.where(torch.rand(pages, generator=gen) < live,
                       torch.randint(1, 5, (pages,), generator=gen), 0).to(torch.int32)
    r = refs.tolist()
    L = sum(x > 0 for x in r)
    frm = [p for p in range(L, pages) if r[p] > 0]
    to = [p for p in range(L) if r[p] <= 0]
    where = [p if x > 0 else -1 for p, x in enumerate(r)]
    new = r[:L] + [0] * (pages - L)
    for a, b in zip(frm, to):
        where[a], new[b] = b, r[a]
    pad = [-1] * (pages // 2 - len(frm))
    d = refs.to(dev)
    for out in (None, d):
        got, m, src, dst = pg.page_compact(d if out is not None else refs.to(dev), out)
        assert got.tolist() == new and m.tolist() == where
        assert src.tolist() == frm + pad and dst.tolist() == to + pad
    t = torch.randint(-2, pages + 2, (7, 11), generator=gen).to(torch.int32)
    moved = [[where[p] if 0 <= p < pages else -1 for p in row] for row in t.tolist()]
    td = t.to(dev)
    assert pg.page_remap(td, m).tolist() == moved
    assert pg.page_remap(td, m, out=td) is td and td.tolist() == moved


@pytest.mark.parametrize("cdt", [F8, BF16])
@pytest.mark.parametrize("KVH,hd,page,layers", [(1, 64, 16, 1), (3, 128, 48, 2), (5, 128, 256, 3),
                                               (2, 64, 32, 40)])
def test_copy(dev, KVH, hd, page, layers, cdt):
    from summa_amd import paged
    caches = [paged.PagedKVCache(11, KVH, hd, page, cdt, dev) for _ in range(layers)]
    raw = torch.uint8 if cdt == F8 else torch.int16

    def parts(c):
        return [c.k.view(raw), c.v.view(raw)] + ([c.k_scales, c.v_scales] if cdt == F8 else [])
    for c in caches:
        for x in parts(c):
            x.copy_(torch.randint(-2 ** 15, 2 ** 15, x.shape).to(x.dtype))
    src, dst = [3, 0, -1, 5, 11, 2, 7, 3], [1, 9, 4, -1, 6, 11, 7, 10]
    ref = [[x.clone() for x in parts(c)] for c in caches]
    paged.paged_copy(caches if layers > 1 else caches[0], i32(src, dev), i32(dst, dev))
    for c, old in zip(caches, ref):
        for x, y in zip(parts(c), old):
            for a, b in zip(src, dst):
                if 0 <= a < 11 and 0 <= b < 11:
                    y[b] = y[a].clone()
            assert torch.equal(x, y)


@pytest.mark.parametrize("cdt", [F8, F16])
def test_drafted_rollouts_as_they_run(dev, cdt):
    """Two prompts, three rollouts each that share its pages, trees of drafted tokens for
    five steps in a model of two layers: the caches hold at the end what one token after
    the other would have put there, and each step's attention is that over these tokens."""
    from summa_amd import ops, paged, pages as pg, sampling, tree
    H, KVH, hd, page, layers, group, n, vocab = 4, 2, 64, 16, 2, 3, 7, 40
    gen = torch.Generator().manual_seed(11)
    prompts = [21, 48]
    refs = pg.page_refs(60, dev)
    caches = [paged.PagedKVCache(60, KVH, hd, page, cdt, dev) for _ in range(layers)]
    rope = P.angles(hd, 256).to(dev)
    # a token's key, value and query in a layer depend on the token and its position alone
    emb = torch.randn(layers, vocab, H + 2 * KVH, hd, generator=gen).to(F16)
    embd = emb.to(dev)
    W = torch.randn(H * hd, vocab, generator=gen).to(dev) * 0.2

    table = torch.full((2, 8), -1, dtype=torch.int32, device=dev)
    pg.page_reserve(refs, table, i32(prompts, dev), page)
    text = [torch.randint(0, vocab, (p,), generator=gen).tolist() for p in prompts]
    for layer, c in enumerate(caches):
        x = embd[layer, torch.tensor(sum(text, []), device=dev)]
        paged.paged_append(c, x[:, H:H + KVH], x[:, H + KVH:], table, i32([0, 0], dev),
                           i32([0, prompts[0], sum(prompts)], dev), max_rows=max(prompts),
                           rope_table=rope)
    S = 2 * group
    source = i32([0] * group + [1] * group, dev)
    kids, src, dst = pg.page_fork(refs, table, i32(prompts, dev), source, page)
    paged.paged_copy(caches, src, dst)
    assert int((refs > 1).sum()) == prompts[0] // page + prompts[1] // page
    pos = i32([prompts[0]] * group + [prompts[1]] * group, dev)
    said = [list(text[0])] * group + [list(text[1])] * group
    said = [list(x) for x in said]
    last = torch.randint(0, vocab, (S,), generator=gen).to(torch.int32).to(dev)
    for step in range(5):
        parents = torch.tensor([R.random_tree(n, gen, 3) for _ in range(S)], dtype=torch.int32)
        toks = torch.randint(0, vocab, (S, n), generator=gen).to(torch.int32).to(dev)
        toks[:, 0] = last
        pg.page_reserve(refs, kids, pos + n, page)
        mask, at = tree.tree_masks(parents.to(dev), pos)
        rows = toks.flatten().long()
        for layer, c in enumerate(caches):
            x = embd[layer, rows]
            qk = ops.rope(x[:, :H + KVH], rope, at)
            paged.paged_append(c, qk[:, H:], x[:, H + KVH:], kids, pos)
            o = paged.paged_tree_attention(c, qk[:, :H], mask, kids, pos)
        # every row's result over its own path alone
        got = o.cpu().double()
        K, V, _, evs = P.read(c.k, c.v, c.k_scales, c.v_scales)
        sees = [R.masks(t)[0] for t in parents.tolist()]
        ref, _, mag, err, unit = R.attend(qk[:, :H].cpu(), (K, V, None, evs), kids.tolist(), pos.tolist(),
                                          [n * s for s in range(S + 1)], page, sum(sees, []))
        assert bool(((got - ref).abs() <= tolerance(F16, cdt, ref, mag, err, unit, hd)).all())
        logits = o.float().flatten(1) @ W
        u = torch.rand(S * n, generator=gen).to(dev)
        sampled, lp = sampling.sample_rows(logits, u, temperature=0.7, top_k=20, top_p=0.95)
        ref_tok = [R.sample(logits[r].double().cpu().numpy(), float(u[r]), float(torch.tensor(0.7)), 20,
                            float(torch.tensor(0.95)))[0] for r in range(S * n)]
        assert sampled.tolist() == ref_tok
        # drafts that are right now and then
        lucky = torch.rand(S, n, generator=gen).to(dev) < 0.6
        up = parents.clamp(min=0).long().to(dev)
        toks[:, 1:] = torch.where(lucky, sampled.view(S, n).gather(1, up), toks)[:, 1:]
        rows = toks.flatten().long()   # (the drafter's choice, made anew: written again)
        for layer, c in enumerate(caches):
            x = embd[layer, rows]
            qk = ops.rope(x[:, :H + KVH], rope, at)
            paged.paged_append(c, qk[:, H:], x[:, H + KVH:], kids, pos)
        path, count, emitted = tree.tree_accept(parents.to(dev), toks, sampled.view(S, n))
        paged.paged_keep(caches, path, count, kids, pos)
        for s in range(S):
            m = int(count[s])
            assert m >= 1
            said[s] += [int(toks[s, i]) for i in path[s, :m].tolist()]
        last = emitted.gather(1, (count - 1).long()[:, None])[:, 0].contiguous()
        pos = pos + count
        pg.page_free(refs, kids, page, pos)
    # what the caches hold, token by token; 8 bits: half a step of the block's scale at most at
    # each of up to three roundings (append, a scale that grew, moved)
    for layer, c in enumerate(caches):
        K, V, ek, ev = P.read(c.k, c.v, c.k_scales, c.v_scales)
        for s in range(S):
            assert len(said[s]) == int(pos[s])
            x = emb[layer, torch.tensor(said[s])].double()
            k = P.rotate(x[:, H:H + KVH], P.angles(hd, 256)[:len(said[s])].double()[:, None], "interleaved")
            for ref, X, e in ((k, K, ek), (x[:, H + KVH:], V, ev)):
                row = kids[s].tolist()
                idx = torch.tensor([row[i // page] for i in range(len(said[s]))])
                off = torch.arange(len(said[s])) % page
                have = X[idx, :, off]
                if cdt == F8:
                    sc = 2.0 ** e[idx, :, off // 16].double()[..., None]
                    tol = ref.abs() * (1.1 * 2.0 ** -4) + 3 * 2.0 ** -10 * sc + 2.0 ** -20
                else:
                    tol = ref.abs() * 2.0 ** -10 + 2.0 ** -20
                assert bool(((have - ref).abs() <= tol).all()), (layer, s)
    # and the pool after the rollouts: compact, then free
    new, where, src, dst = pg.page_compact(refs)
    moved = pg.page_remap(kids, where)
    before = [P.read(c.k, c.v, c.k_scales, c.v_scales) for c in caches]
    paged.paged_copy(caches, src, dst)
    L = int((refs > 0).sum())
    assert bool((new[:L] > 0).all()) and not new[L:].any()
    for c, (K, V, *_) in zip(caches, before):
        K2, V2 = P.read(c.k, c.v, c.k_scales, c.v_scales)[:2]
        for a, b in zip(kids.flatten().tolist(), moved.flatten().tolist()):
            assert (a < 0) == (b < 0)
            if a >= 0:
                assert torch.equal(K[a], K2[b]) and torch.equal(V[a], V2[b])
    table = pg.page_remap(table, where)
    pg.page_free(new, moved, page)
    pg.page_free(new, table, page)
    assert not new.any()


def test_graph_of_the_page_calls(dev):
    """A batch's turn captured once - the old rollouts freed, prompts forked, pages copied, room
    reserved, the pool compacted - and replayed with other prompts and lengths, eager work between."""
    from summa_amd import paged, pages as pg
    pages, page, P, group, cols = 200, 16, 3, 4, 12
    cache = paged.PagedKVCache(pages, 2, 64, page, F16, dev)
    cache.k.normal_(generator=torch.Generator(device=dev).manual_seed(1))
    cache.v.copy_(cache.k.view(cache.v.shape))
    refs = pg.page_refs(pages, dev)
    prompts = torch.full((P, cols), -1, dtype=torch.int32, device=dev)
    kids = torch.full((P * group, cols), -1, dtype=torch.int32, device=dev)
    source = torch.arange(P, dtype=torch.int32, device=dev).repeat_interleave(group)
    tokens, room = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (P, P * group))
    new = torch.empty_like(refs)

    def turn():
        pg.page_free(refs, kids, page)
        pg.page_free(refs, prompts, page)
        pg.page_reserve(refs, prompts, tokens, page)
        _, src, dst = pg.page_fork(refs, prompts, tokens, source, page, out=kids)
        paged.paged_copy(cache, src, dst)
        pg.page_reserve(refs, kids, room, page)
        _, where, a, b = pg.page_compact(refs, new)
        paged.paged_copy(cache, a, b)
        return pg.page_remap(kids, where), src, dst, where

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = turn()
    gen = torch.Generator().manual_seed(5)
    for _ in range(5):
        tokens.copy_(torch.randint(0, 6 * page, (P,), generator=gen))
        room.copy_(tokens[source.long()] + torch.randint(0, 5 * page, (P * group,), generator=gen).to(dev))
        state = [x.clone() for x in (refs, prompts, kids, cache.k, cache.v)]
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*out, refs, prompts, kids, new, cache.k, cache.v)]
        for x, y in zip((refs, prompts, kids, cache.k, cache.v), state):
            x.copy_(y)
        again = turn()
        for x, y in zip(got, (*again, refs, prompts, kids, new, cache.k, cache.v)):
            assert torch.equal(x, y)
        used = -(-room // page)
        assert torch.equal((kids >= 0).sum(1), used.clamp(max=cols).long())


def test_two_streams_at_once(dev):
    """Calls on two streams share nothing: sampling in parts, trees and attention."""
    from summa_amd import sampling
    xs = [torch.randn(4, 131072, device=dev) for _ in range(2)]
    us = [torch.rand(4, device=dev) for _ in range(2)]
    alone = [sampling.sample_rows(x, u, top_p=0.9) for x, u in zip(xs, us)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(sampling.sample_rows(xs[i], us[i], top_p=0.9))
    torch.cuda.synchronize()
    for i in range(2):
        for tok, lp in outs[i]:
            assert torch.equal(tok, alone[i][0]) and torch.equal(lp, alone[i][1])
