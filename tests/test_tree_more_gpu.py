"""Further tests of drafted trees: every layer of a call over many caches, chains bit for bit, calls that repeat
themselves, and calls of all kinds on two streams at once."""
import pytest
import torch

import _tree as R
from test_paged_gpu import BF16, F16, F8, Batch
from test_tree_gpu import KEEPS, attention, random_masks, tree_batch

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.dtype.itemsize])


@pytest.mark.parametrize("cdt", [F8, F16])
@pytest.mark.parametrize("layers", [32, 33, 35, 65])
@pytest.mark.parametrize("case", range(len(KEEPS)))
def test_keep_in_every_layer(dev, case, layers, cdt):
    """Caches of a launch of their own (from the 33rd on) among them, each with other contents."""
    from summa_amd import paged
    print(f"case keep {case} {layers} {cdt}", flush=True)
    pos0, path, KVH, hd, page = KEEPS[case]
    most = max(max(len(p) for p in path), 1)
    b = Batch(dev, pos0, [100] * len(pos0), KVH, hd, page, cdt)
    if case == 4:
        b.t[5, 1] = -1
        b.table[5][1] = -1
    raw = torch.uint8 if cdt == F8 else torch.int16
    caches, before = [], []
    for i in range(layers):
        c = paged.PagedKVCache(b.pages, KVH, hd, page, cdt, dev)
        for x in (c.k, c.v):
            x.view(raw).copy_(torch.randint(-2 ** 15, 2 ** 15, x.shape).to(raw))
        if cdt == F8:
            for x in (c.k_scales, c.v_scales):
                x.copy_(torch.randint(118 - i % 40, 124, x.shape).to(torch.uint8))
        caches.append(c)
        b.cache = c
        before.append(b.raw())
    t = torch.full((len(pos0), most), 77, dtype=torch.int32)
    for s, p in enumerate(path):
        t[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    paged.paged_keep(caches, t.to(dev), i32([len(p) for p in path], dev), b.t, b.p)
    compared = 0
    for i, (c, old) in enumerate(zip(caches, before)):
        b.cache = c
        now = b.raw()
        if i in (0, 31, 32, layers - 1):  # (the definition walks token by token: the launches' ends)
            for x, y in zip(now, R.keep(old, b.table, pos0, path, page, hd)):
                assert torch.equal(x, y), i
        else:
            # the others by a call of their own
            for x, y in zip((c.k.view(raw), c.v.view(raw), c.k_scales, c.v_scales), old):
                x.copy_(y)
            paged.paged_keep(c, t.to(dev), i32([len(p) for p in path], dev), b.t, b.p)
            for x, y in zip(now, b.raw()):
                assert torch.equal(x, y), i
        compared += 1
    assert compared == layers


@pytest.mark.parametrize("n,H,KVH,hd,dtype,cdt", [
    (4, 4, 1, 64, F16, F8), (1, 2, 2, 128, BF16, BF16), (9, 2, 2, 64, F16, F16),      # 16 rows a KV head
    (16, 1, 1, 128, BF16, F8), (70, 4, 2, 64, F16, F8), (40, 2, 1, 128, BF16, BF16),  # tiles of 128
    (64, 4, 2, 128, F16, F16)])
def test_a_chain_is_the_causal_form_bit_for_bit(dev, n, H, KVH, hd, dtype, cdt):
    """Where one workgroup has a sequence's rows and keys, masked keys are the only difference: they weigh
    nothing in either form."""
    print(f"case chain {n} {H} {hd} {dtype} {cdt}", flush=True)
    b = tree_batch(dev, [100, 17, 0], [n] * 3, KVH, hd, 32, cdt)
    q = torch.randn(b.rows, H, hd).to(dtype).to(dev)
    sees = [set(range(i + 1)) for i in range(n)] * 3
    got, lse = attention(b, q, R.words(sees, (n + 31) // 32).to(dev), want_lse=True, max_tokens=256)
    ref, rl = b.attention(q, want_lse=True, max_tokens=256)
    assert torch.equal(bits(got), bits(ref)) and torch.equal(bits(lse), bits(rl))


@pytest.mark.parametrize("n,H,KVH,hd,dtype,cdt", [(24, 4, 1, 128, F16, F8), (3, 4, 2, 64, BF16, BF16),
                                                  (150, 4, 2, 128, BF16, F8)])
def test_attention_repeats_itself(dev, n, H, KVH, hd, dtype, cdt):
    """Splits of keys are joined in a fixed order: one call is as good as the next, in other memory too."""
    b = tree_batch(dev, [4000, 30, 1700], [n] * 3, KVH, hd, 64, cdt)
    q = torch.randn(b.rows, H, hd).to(dtype).to(dev)
    mask = R.words(random_masks(b, torch.Generator().manual_seed(n), "tree"), (n + 31) // 32).to(dev)
    first, lse = attention(b, q, mask, want_lse=True)
    hold = []
    for _ in range(10):
        hold.append(torch.full((1 << 20,), 3e38, device=dev))
        got, again = attention(b, q.clone(), mask.clone(), want_lse=True)
        assert torch.equal(bits(got), bits(first)) and torch.equal(bits(again), bits(lse))


def test_trees_and_pages_on_two_streams(dev):
    """Split tree attention of different lengths, and a pool's turn on refs of their own: calls on two streams
    share nothing."""
    from summa_amd import pages as pg, paged, tree
    n, H, KVH, hd = 20, 4, 2, 64
    work = []
    for i, pos0 in enumerate(([9000, 40, 700], [300, 5000, 2500])):
        b = tree_batch(dev, pos0, [n] * 3, KVH, hd, 32, (F8, F16)[i])
        gen = torch.Generator().manual_seed(i)
        parents = torch.tensor([R.random_tree(n, gen) for _ in range(3)], dtype=torch.int32, device=dev)
        toks, smp = (torch.randint(0, 2, (3, n), generator=gen).to(torch.int32).to(dev) for _ in range(2))
        q = torch.randn(b.rows, H, hd).to(F16).to(dev)
        refs = pg.page_refs(900 + 7 * i, dev)
        prompts = torch.full((5, 30), -1, dtype=torch.int32, device=dev)
        tokens = torch.randint(1, 400, (5,), generator=gen).to(torch.int32).to(dev)
        source = torch.randint(0, 5, (24,), generator=gen).to(torch.int32).to(dev)
        work.append((b, parents, toks, smp, q, refs, prompts, tokens, source))

    def step(b, parents, toks, smp, q, refs, prompts, tokens, source):
        mask, at = tree.tree_masks(parents, b.p)
        o, lse = attention(b, q, mask, want_lse=True)
        path, count, emitted = tree.tree_accept(parents, toks, smp)
        missing = torch.zeros(1, dtype=torch.int32, device=dev)
        pg.page_free(refs, prompts, 16)
        pg.page_reserve(refs, prompts, tokens, 16)
        kids, src, dst = pg.page_fork(refs, prompts, tokens, source, 16, missing=missing)
        pg.page_reserve(refs, kids, tokens[source.long()] + 50, 16, missing)
        new, where, a, c = pg.page_compact(refs)
        moved = pg.page_remap(kids, where)
        pg.page_free(refs, kids, 16)
        return mask, at, o, lse, path, count, emitted, kids, src, dst, missing, new, where, a, c, moved, refs.clone()

    alone = [step(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(step(*work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for turn in outs[i]:
            for k, (x, y) in enumerate(zip(turn, alone[i])):
                assert torch.equal(bits(x), bits(y)), (i, k)
    # each keeps its own paths meanwhile
    first = [w[0].raw() for w in work]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            b = work[i][0]
            paged.paged_keep(b.cache, alone[i][4], alone[i][5], b.t, b.p)
    torch.cuda.synchronize()
    for i, w in enumerate(work):
        b, path, count = w[0], alone[i][4].tolist(), alone[i][5].tolist()
        ref = R.keep(first[i], b.table, b.pos0, [p[:c] for p, c in zip(path, count)], b.page, hd)
        for x, y in zip(b.raw(), ref):
            assert torch.equal(x, y)
