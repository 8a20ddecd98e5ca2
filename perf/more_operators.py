"""Tree-drafted rollouts over the paged cache: the operators' cases and plain forms.

What a loop runs that drafts several tokens a step and keeps the confirmed ones:

- ``sample``: the next token of every row from a given random number, each row with its
  own temperature, top-k, top-p and min-p, and its log-probability.
- ``tree``: attention of a tree of drafted tokens over the paged cache: a row sees the
  context and those drafted tokens that its mask names (its ancestors and itself).
- ``keep``: the longest drafted path that the sampled tokens confirm, and its tokens moved
  together behind the context in the caches of all layers.
- ``fork`` / ``compact``: a finished batch's pages freed, prompts' pages shared by the next
  rollouts with the unfinished last page copied; live pages moved to the pool's front.

The cache's layout is that of ``paged.PagedKVCache``: ``k`` [pages, KVH, page, hd]; ``v``
[pages, KVH, page / 16, hd / 16T, 4, 16, T, 4] with T = 4 (8-bit) or 2 (16-bit): token
4 g + j and dim 16 (c T + t) + r of a 16-token block at [c, g, r, t, j]; scales of 8-bit
caches [pages, KVH, page / 16] uint8: exponent + 127.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn}
BLOCK = 16
# heads, KV heads, head_dim and layers of summa_amd.configs' decoders
GEOMETRY = {"d256": (4, 4, 64, 2), "d768": (12, 12, 64, 12), "d2048": (16, 4, 128, 24),
            "moe2048": (16, 16, 128, 16)}


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # A step of four short requests with one setting: the smallest call, all latency.
        dict(name="sample_step_small", kind="sample", rows=4, vocab=4096, dtype="f32",
             filters="k", mixed=False, peak=6.0),
        # The rollout step of 32 prompts x 8 rollouts, nucleus of the whole vocabulary.
        dict(name="sample_rollouts", kind="sample", rows=256, vocab=65536, dtype="f32",
             filters="p", mixed=False, peak=6.0),
        # Every node of 32 sequences' trees, bf16 logits over an odd vocabulary, each row
        # with a request's own options (some greedy, some with all filters, some with none).
        dict(name="sample_verify", kind="sample", rows=768, vocab=50001, dtype="bf16",
             filters="kpm", mixed=True, peak=8.0),
        # A few requests over a large vocabulary: one row is more than a compute unit holds.
        dict(name="sample_large_vocab", kind="sample", rows=6, vocab=131072, dtype="f32",
             filters="pm", mixed=False, peak=4.0),
        # Three short requests, trees of eight drafted tokens, masks made from the parents.
        dict(name="tree_small", kind="tree", seqs=3, rows_lo=8, rows_hi=8, ctx_lo=60, ctx_hi=200,
             geometry="d256", dtype="f16", cache="f16", page=16, lse=False, plan=True),
        # One verification step of a serving batch: 32 sequences, 24 drafted tokens each.
        dict(name="tree_verify", kind="tree", seqs=32, rows_lo=24, rows_hi=24, ctx_lo=1000,
             ctx_hi=4000, geometry="d2048", dtype="f16", cache="e4m3", page=64, lse=False,
             plan=False),
        # Ragged trees, one sequence without a context among them, no head shared, small
        # pages, bf16, masks and log-sum-exp.
        dict(name="tree_ragged", kind="tree", seqs=17, rows_lo=1, rows_hi=63, ctx_lo=0,
             ctx_hi=3000, geometry="moe2048", dtype="bf16", cache="bf16", page=16, lse=True,
             plan=True),
        # Two very long contexts with wide trees: the work is split over the keys.
        dict(name="tree_long", kind="tree", seqs=2, rows_lo=48, rows_hi=64, ctx_lo=90000,
             ctx_hi=131000, geometry="d2048", dtype="bf16", cache="e4m3", page=256, lse=False,
             plan=False),
        # Four short requests' accepted paths in a two-layer model: latency.
        dict(name="keep_small", kind="keep", seqs=4, rows_lo=8, rows_hi=8, ctx_lo=40, ctx_hi=200,
             geometry="d256", layers=2, cache="f16", page=16),
        # The same of 64 sequences in all 24 layers, trees of unequal size, 8-bit cache.
        dict(name="keep_rollouts", kind="keep", seqs=64, rows_lo=12, rows_hi=40, ctx_lo=100,
             ctx_hi=500, geometry="d2048", layers=24, cache="e4m3", page=64),
        # The next 32 prompts x 8 rollouts: the last batch's pages freed, prompts shared.
        dict(name="fork_rollouts", kind="fork", seqs=32, group=8, ctx_lo=257, ctx_hi=512,
             geometry="d2048", layers=24, cache="e4m3", page=64),
        # A pool of which a third is in use, moved to its front before the rest is given
        # back; 16-bit cache, twelve layers.
        dict(name="compact_pool", kind="compact", pages=1001, live=0.34, geometry="d768",
             layers=12, cache="f16", page=32),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "tree", "tree", "keep", "pages"])
    if kind == "sample":
        vocab = _log(rng, 100, 131072)
        return dict(kind=kind, rows=_log(rng, 1, min(1024, 38000000 // vocab)), vocab=vocab,
                    dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                    filters=rng.choice(["", "k", "p", "m", "kp", "pm", "kpm"]),
                    mixed=rng.random() < 0.4, peak=rng.uniform(0.5, 10.0))
    geometry = rng.choice(sorted(GEOMETRY))
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "tree":
        dtype = rng.choice(["bf16", "f16"])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 2, min(128, 1024 // seqs + 1))
        ctx = _log(rng, 1, max(2, min(131000, 131072 // seqs, 6000000 // (seqs * hi))))
        return dict(kind=kind, seqs=seqs, rows_lo=max(1, hi // 2), rows_hi=hi, ctx_lo=ctx // 2,
                    ctx_hi=ctx, geometry=geometry, dtype=dtype,
                    cache=rng.choice(["e4m3", "e4m3", dtype]), page=page,
                    lse=rng.random() < 0.3, plan=rng.random() < 0.4)
    H, KVH, hd, layers = GEOMETRY[geometry]
    layers = rng.randint(1, layers)
    cache = rng.choice(["e4m3", "e4m3", "bf16", "f16"])
    token = 2 * KVH * hd * layers * DTYPES[cache].itemsize
    if kind == "keep":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, 64)
        ctx = _log(rng, 1, max(2, min(500, 500000000 // (seqs * token) - hi)))
        return dict(kind=kind, seqs=seqs, rows_lo=max(1, hi // 3), rows_hi=hi, ctx_lo=ctx // 2,
                    ctx_hi=ctx, geometry=geometry, layers=layers, cache=cache, page=page)
    if rng.random() < 0.5:
        most = 400000000 // (page * token)  # rollouts
        seqs = _log(rng, 1, min(32, most))
        group = rng.randint(1, min(8, most // seqs))
        ctx = _log(rng, 1, max(2, min(512, 400000000 // (seqs * token))))
        return dict(kind="fork", seqs=seqs, group=group, ctx_lo=(ctx + 1) // 2, ctx_hi=ctx,
                    geometry=geometry, layers=layers, cache=cache, page=page)
    return dict(kind="compact", pages=_log(rng, 2, max(3, min(4000, 1000000000 // (page * token)))),
                live=rng.uniform(0.0, 1.0), geometry=geometry, layers=layers, cache=cache,
                page=page)


def _lengths(case, seed):
    """(new rows, cached tokens) of each sequence: the case's own, in the seed's order; the
    ends of both ranges among them."""
    rng = random.Random(29)
    n = [rng.randint(case.get("rows_lo", 0), case.get("rows_hi", 0)) for _ in range(case["seqs"])]
    c = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    n[-1], c[0] = case.get("rows_hi", 0), case["ctx_hi"]
    if len(c) > 1:
        c[-1] = case["ctx_lo"]
    both = list(zip(n, c))
    random.Random(seed).shuffle(both)
    return [a for a, _ in both], [b for _, b in both]


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["rows"] * 12, "flops": 4 * n}
    H, KVH, hd, _ = GEOMETRY[case["geometry"]]
    csize = DTYPES[case["cache"]].itemsize
    token = 2 * KVH * (hd * csize + (1.0 / BLOCK if csize == 1 else 0.0))  # of one layer
    if case["kind"] == "tree":
        n, c = _lengths(case, 0)
        rows, words = sum(n), (max(n) + 31) // 32
        size = DTYPES[case["dtype"]].itemsize
        keys = sum(a + b for a, b in zip(n, c))
        moved = keys * token + 2 * rows * H * hd * size + rows * words * 4
        if case["plan"]:
            moved += rows * 8 + rows * words * 4
        seen = sum(a * b for a, b in zip(n, c)) + 4 * rows  # context, and about four ancestors
        return {"bytes": moved, "flops": 4 * seen * H * hd}
    if case["kind"] == "keep":
        n, _ = _lengths(case, 0)
        return {"bytes": sum(n) * 12 + case["seqs"] * 4 * 2 * token * case["layers"], "flops": 0}
    page_bytes = case["page"] * token * case["layers"]
    if case["kind"] == "fork":
        _, c = _lengths(case, 0)
        copied = case["group"] * sum(1 for t in c if t % case["page"])
        entries = sum(-(-t // case["page"]) for t in c) * (1 + case["group"])
        return {"bytes": 2 * copied * page_bytes + 8 * entries, "flops": 0}
    live = int(case["live"] * case["pages"])
    moves = live * (case["pages"] - live) / case["pages"]  # as they lie at random
    return {"bytes": 2 * moves * page_bytes + 12 * case["pages"], "flops": 0}


# ----------------------------------------------------------------- inputs --

def _caches(case, pages, g, layers):
    """k, v and scales [layers, ..] of all layers: values of about one."""
    _, KVH, hd, _ = GEOMETRY[case["geometry"]]
    page, cdt = case["page"], DTYPES[case["cache"]]
    T = 4 if cdt.itemsize == 1 else 2
    shapes = ((pages, KVH, page, hd), (pages, KVH, page // BLOCK, hd // (16 * T), 4, 16, T, 4))

    def values(shape):
        t = torch.empty((layers, *shape), dtype=cdt, device=DEV).flatten(0, 1)
        step = max(1, (1 << 27) // max(1, t[0].numel()))
        for i in range(0, t.shape[0], step):
            x = torch.randn(t[i:i + step].shape, generator=g, device=DEV)
            t[i:i + step] = (x * 100).clamp_(-448, 448).to(cdt) if cdt.itemsize == 1 else x.to(cdt)
        return t.unflatten(0, (layers, -1))

    ks = vs = None
    if cdt.itemsize == 1:
        ks, vs = (torch.randint(119, 122, (layers, pages, KVH, page // BLOCK), generator=g,
                                device=DEV, dtype=torch.uint8) for _ in range(2))
    return dict(k=values(shapes[0]), v=values(shapes[1]), ks=ks, vs=vs)


def _layer(caches, i):
    return {name: None if t is None else t[i] for name, t in caches.items()}


def _table(need, pages, g):
    """Block table with `need` pages a sequence, of `pages` in a random order; what is left."""
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
    cols = max(1, max(need))
    table = torch.full((len(need), cols), -1, dtype=torch.int32)
    table[torch.arange(cols)[None, :] < torch.tensor(need)[:, None]] = order[: sum(need)]
    return table.to(DEV), order[sum(need):]


def _tree(n, rng):
    """Parents of n drafted tokens: the first is the root, others hang on one of the eight before."""
    return [-1] + [rng.randint(max(0, i - 8), i - 1) for i in range(1, n)]


def _starts(n):
    return torch.tensor(np.concatenate([[0], np.cumsum(n)]).astype(np.int32), device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    st = dict(case=dict(case), seed=seed)
    if case["kind"] == "sample":
        return _prepare_sample(st, case, g)
    if case["kind"] == "compact":
        pages = case["pages"]
        live = torch.randperm(pages, generator=g, device=DEV)[: int(case["live"] * pages)]
        st["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
        st["refs"][live] = torch.randint(1, 9, live.shape, generator=g, device=DEV,
                                         dtype=torch.int32)
        # the tables of 33 sequences: live pages, in rows that end at different lengths
        cols = max(1, len(live) // 33 + 1)
        table = torch.full((33 * cols,), -1, dtype=torch.int32, device=DEV)
        table[: len(live)] = live.to(torch.int32)
        st["table"] = table.view(33, cols)
        st["caches"] = _caches(case, pages, g, case["layers"])
        return _own_caches(st)
    n, c = _lengths(case, seed)
    page = case["page"]
    if case["kind"] == "fork":
        return _prepare_fork(st, case, c, g)
    need = [(a + b + page - 1) // page for a, b in zip(n, c)]
    pages = sum(need) + 3
    st["table"], _ = _table(need, pages, g)
    st["pos0"] = torch.tensor(c, dtype=torch.int32, device=DEV)
    ragged = len(set(n)) > 1
    st["row_start"] = _starts(n) if ragged else None
    st["max_rows"], st["max_tokens"] = max(n), max(a + b for a, b in zip(n, c))
    trees = [_tree(a, rng) for a in n]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=DEV)
    st["parents"] = parents if ragged else parents.view(len(n), -1)
    if case["kind"] == "tree":
        H, _, hd, _ = GEOMETRY[case["geometry"]]
        st["caches"] = _caches(case, pages, g, 1)
        st["q"] = (torch.randn(sum(n), H, hd, generator=g, device=DEV) * 1.5).to(
            DTYPES[case["dtype"]])
        st["mask"] = None if case["plan"] else _masks(st)[0]
        return _own_caches(st)
    # Drafted tokens, and sampled ones that confirm a path. The path's tokens that move come
    # from behind its length, so that a pass can be repeated.
    drafted, sampled = [], []
    for t in trees:
        best = [0]
        for v in [rng.randrange(len(t)) for _ in range(16)]:
            path = [v]
            while t[path[0]] >= 0:
                path.insert(0, t[path[0]])
            if len(path) > len(best) and \
                    all(x == i or x >= len(path) for i, x in enumerate(path)):
                best = path
        tok = [rng.randrange(0, 30000) * 2 for _ in t]
        for i in range(1, len(t)):  # the draft's best token twice among siblings never happens
            tok[i] += 60000 * (i - t[i])
        smp = [2 * rng.randrange(0, 30000) + 1 for _ in t]
        for a, b in zip(best, best[1:]):
            smp[a] = tok[b]
        drafted += tok
        sampled += smp
    st["tokens"] = torch.tensor(drafted, dtype=torch.int32, device=DEV).view(st["parents"].shape)
    st["sampled"] = torch.tensor(sampled, dtype=torch.int32, device=DEV).view(st["parents"].shape)
    st["caches"] = _caches(case, pages, g, case["layers"])
    return _own_caches(st)


def _prepare_sample(st, case, g):
    rows, vocab = case["rows"], case["vocab"]
    # logits of a language model: a wide middle, and a few tokens far above it
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.0
    tops = torch.randint(0, vocab, (rows, 12), generator=g, device=DEV)
    lift = torch.rand(rows, 12, generator=g, device=DEV) * case["peak"] + 2.0
    x.scatter_add_(1, tops, lift)
    st["logits"] = x.to(DTYPES[case["dtype"]])
    st["u"] = torch.rand(rows, generator=g, device=DEV)

    def option(on, one, values, off):
        if not on:
            return off
        if not case["mixed"]:
            return one
        pick = torch.randint(0, len(values), (rows,), generator=g, device=DEV)
        return torch.tensor(values, device=DEV)[pick]

    st["T"] = option(True, 0.8, [0.0, 0.6, 0.8, 1.0, 1.0, 1.5], None)
    st["k"] = option("k" in case["filters"], 50, [-1, 1, 20, 50, 400], None)
    st["p"] = option("p" in case["filters"], 0.95, [0.5, 0.9, 0.95, 1.0], 1.0)
    st["m"] = option("m" in case["filters"], 0.05, [0.0, 0.02, 0.1, 0.3], 0.0)
    if torch.is_tensor(st["k"]):
        st["k"] = st["k"].to(torch.int32)
    return st


def _prepare_fork(st, case, c, g):
    """Prompts, and the tables of the last batch's rollouts, which share them; these hold
    pages of their own behind the prompt."""
    page, group = case["page"], case["group"]
    need = [(t + page - 1) // page for t in c]
    kids = len(c) * group
    pages = sum(need) + 2 * kids + 3
    table, left = _table(need, pages, g)
    cols = table.shape[1] + 1
    st["table"] = torch.cat([table, torch.full_like(table[:, :1], -1)], 1).contiguous()
    st["tokens"] = torch.tensor(c, dtype=torch.int32, device=DEV)
    st["source"] = torch.arange(len(c), dtype=torch.int32, device=DEV).repeat_interleave(group)
    old = st["table"][st["source"].long()].clone()
    full = (st["tokens"] // page).long()[st["source"].long()]
    left = left.to(DEV)
    old[torch.arange(kids, device=DEV), full] = left[:kids]
    st["children"] = old.contiguous()
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    for t in (st["table"], old):
        held = t[t >= 0].long()
        refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    st["refs"] = refs
    st["caches"] = _caches(case, pages, g, case["layers"])
    return _own_caches(st)


def _own_caches(st):
    if own:
        from summa_amd import paged
        layers = [_layer(st["caches"], i) for i in range(st["caches"]["k"].shape[0])]
        st["paged"] = [paged.PagedKVCache.from_tensors(x["k"], x["v"], x["ks"], x["vs"])
                       for x in layers]
    return st


# ------------------------------------------------------------------- pass --

def run(st):
    kind = st["case"]["kind"]
    if own:
        return _OWN[kind](st, st["case"])
    return _PLAIN[kind](st, st["case"])


def _own_sample(st, case):
    from summa_amd import sampling
    return sampling.sample_rows(st["logits"], st["u"], temperature=st["T"], top_k=st["k"],
                                top_p=st["p"], min_p=st["m"])


def _own_tree(st, case):
    from summa_amd import paged, tree
    mask, positions = st["mask"], None
    if case["plan"]:
        mask, positions = tree.tree_masks(st["parents"], st["pos0"], st["row_start"],
                                          max_rows=st["max_rows"])
    o = paged.paged_tree_attention(st["paged"][0], st["q"], mask, st["table"], st["pos0"],
                                   st["row_start"], max_rows=st["max_rows"],
                                   max_tokens=st["max_tokens"], want_lse=case["lse"])
    return {"o": o, "mask": mask if case["plan"] else None, "positions": positions}


def _own_keep(st, case):
    from summa_amd import paged, tree
    path, count, emitted = tree.tree_accept(st["parents"], st["tokens"], st["sampled"],
                                            st["row_start"], max_rows=st["max_rows"])
    paged.paged_keep(st["paged"], path, count, st["table"], st["pos0"])
    return {"path": path, "count": count, "emitted": emitted, "caches": st["caches"]}


def _own_fork(st, case):
    from summa_amd import paged, pages
    pages.page_free(st["refs"], st["children"], case["page"])
    table, src, dst = pages.page_fork(st["refs"], st["table"], st["tokens"], st["source"],
                                      case["page"], out=st["children"])
    paged.paged_copy(st["paged"], src, dst)
    return {"table": table, "refs": st["refs"], "src": src, "dst": dst, "caches": st["caches"]}


def _own_compact(st, case):
    from summa_amd import paged, pages
    refs, where, src, dst = pages.page_compact(st["refs"])
    table = pages.page_remap(st["table"], where)
    paged.paged_copy(st["paged"], src, dst)
    return {"refs": refs, "table": table, "src": src, "dst": dst, "caches": st["caches"]}


# ------------------------------------------------------------ plain forms --

def _per_row(x, rows, off, dtype):
    if x is None:
        x = off
    return x.to(dtype) if torch.is_tensor(x) else torch.full((rows,), x, dtype=dtype, device=DEV)


def _sample(st, case):
    """Weights and sums in 64 bits: a token's place between two sums is decided by them."""
    rows, vocab = st["logits"].shape
    T = _per_row(st["T"], rows, 1.0, torch.float64)
    k = _per_row(st["k"], rows, -1, torch.int64)
    p = _per_row(st["p"], rows, 1.0, torch.float32).double()
    mp = _per_row(st["m"], rows, 0.0, torch.float32).double()
    if not torch.is_tensor(st["T"]):  # (as the call takes it)
        T = T.float().double()
    tokens, lps = [], []
    step = max(1, (1 << 25) // vocab)
    at = torch.arange(vocab, device=DEV)
    for i in range(0, rows, step):
        x = st["logits"][i:i + step].float()
        t = T[i:i + step, None]
        d = x.double() - x.amax(-1, keepdim=True).double()
        w = torch.exp(d / torch.where(t > 0, t, 1.0))
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        kk = k[i:i + step, None]
        ws = ws * ((kk < 1) | (at < kk))
        before = torch.cumsum(ws, -1)
        total = before[:, -1:].clone()
        before = before - ws
        keep = ws > 0
        pp = p[i:i + step, None]
        keep &= (pp >= 1) | (before < pp * total)
        keep &= (mp[i:i + step, None] <= 0) | (ws >= mp[i:i + step, None])
        keep[:, 0] = True
        w = w * torch.zeros_like(keep).scatter_(1, order, keep)
        upto = torch.cumsum(w, -1)
        aim = st["u"][i:i + step, None].double() * upto[:, -1:]
        tok = torch.where(upto > aim, at, vocab).amin(-1)
        tok = torch.where(t[:, 0] > 0, tok, torch.where(d == 0, at, vocab).amin(-1))
        lp = d.gather(1, tok[:, None])[:, 0] - torch.exp(d).sum(-1).log()
        tokens.append(tok.to(torch.int32))
        lps.append(lp.float())
    return torch.cat(tokens), torch.cat(lps)


def _rows(st, rows):
    """Sequence and place in it of every row."""
    r = torch.arange(rows, device=DEV)
    if st["row_start"] is None:
        return r // st["max_rows"], r % st["max_rows"]
    seq = torch.searchsorted(st["row_start"][1:].long(), r, right=True)
    return seq, r - st["row_start"].long()[seq]


def _masks(st):
    """Mask words [rows, words] and positions of every drafted token."""
    parents = st["parents"].reshape(-1).long()
    rows, L = parents.shape[0], st["max_rows"]
    seq, i = _rows(st, rows)
    first = torch.arange(rows, device=DEV) - i
    sees = torch.zeros(rows, (L + 31) // 32 * 32, dtype=torch.bool, device=DEV)
    depth = torch.full((rows,), -1, dtype=torch.int64, device=DEV)
    cur, on = i.clone(), torch.ones(rows, dtype=torch.bool, device=DEV)
    for _ in range(L):  # (a path has no more tokens than the tree)
        sees.scatter_(1, cur[:, None], sees.gather(1, cur[:, None]) | on[:, None])
        depth += on
        up = parents[first + cur]
        on = on & (up >= 0)
        cur = torch.where(on, up, cur)
    weight = torch.ones(32, dtype=torch.int64, device=DEV) << torch.arange(32, device=DEV)
    words = (sees.view(rows, -1, 32).long() * weight).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return words, (st["pos0"].long()[seq] + depth).to(torch.int32)


def _cached(st, case):
    """Keys and values [S, KVH, tokens, hd] f32 of every sequence's pages."""
    x = _layer(st["caches"], 0)
    at = st["table"].clamp(min=0).long()
    S, cols = at.shape
    KVH, page, hd = x["k"].shape[1:]

    def take(t):
        if t.dtype.itemsize == 1:
            return t.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        return t[at].float()

    k = take(x["k"]).view(S, cols, KVH, page // BLOCK, BLOCK, hd)
    v = take(x["v"]).permute(0, 1, 2, 3, 5, 8, 4, 7, 6).reshape(k.shape)
    if x["ks"] is not None:
        k, v = (torch.ldexp(t, (s[at].int() - 127)[..., None, None])
                for t, s in ((k, x["ks"]), (v, x["vs"])))
    return tuple(t.permute(0, 2, 1, 3, 4, 5).reshape(S, KVH, cols * page, hd) for t in (k, v))


def _attend(st, case):
    q = st["q"]
    rows, H, hd = q.shape
    S, L = st["table"].shape[0], case["rows_hi"]
    mask, positions = _masks(st) if case["plan"] else (st["mask"], None)
    k, v = _cached(st, case)
    KVH, T = k.shape[1:3]
    G = H // KVH
    seq, i = _rows(st, rows)
    bits = mask[:, :, None] >> torch.arange(32, dtype=torch.int32, device=DEV) & 1
    drafted = bits.view(rows, -1)[:, :L].bool()
    key = torch.arange(T, device=DEV)
    sees = torch.zeros(S, L, T, dtype=torch.bool, device=DEV)
    rel = key[None, :] - st["pos0"].long()[seq][:, None]
    sees[seq, i] = (rel < 0) | (drafted.gather(1, rel.clamp(0, L - 1)) & (rel >= 0) & (rel < L))
    qp = torch.zeros(S, L, H, hd, device=DEV)
    qp[seq, i] = q.float()
    qp = qp.view(S, L, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(S, KVH, L * G, hd)
    sc = torch.matmul(qp, k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    sc.masked_fill_(~sees.repeat_interleave(G, 1)[:, None], float("-inf"))
    m = sc.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(sc - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total
    o = o.view(S, KVH, L, G, hd).permute(0, 2, 1, 3, 4).reshape(S, L, H, hd)[seq, i].to(q.dtype)
    if case["lse"]:
        lse = (m + total.log()).view(S, KVH, L, G).permute(0, 2, 1, 3).reshape(S, L, H)[seq, i]
        o = (o, lse)
    return {"o": o, "mask": mask if case["plan"] else None, "positions": positions}


def _accept(st):
    """path [S, L], count [S] and the sampled tokens along it, -1 behind their ends."""
    parents, tokens, sampled = (st[x].reshape(-1).long() for x in ("parents", "tokens", "sampled"))
    rows, S, L = parents.shape[0], st["table"].shape[0], st["max_rows"]
    seq, i = _rows(st, rows)
    pad = torch.full((S, L), -2, dtype=torch.int64, device=DEV)
    par, tok, smp = pad.clone(), pad.clone(), pad.clone()
    par[seq, i], tok[seq, i], smp[seq, i] = parents, tokens, sampled
    path, emitted = (torch.full((S, L), -1, dtype=torch.int64, device=DEV) for _ in range(2))
    count = torch.zeros(S, dtype=torch.int64, device=DEV)
    cur = torch.zeros(S, dtype=torch.int64, device=DEV)
    on = torch.ones(S, dtype=torch.bool, device=DEV)
    place = torch.arange(L, device=DEV)
    for j in range(L):
        want = smp.gather(1, cur[:, None])
        path[:, j] = torch.where(on, cur, -1)
        emitted[:, j] = torch.where(on, want[:, 0], -1)
        count += on
        fits = (par == cur[:, None]) & (tok == want)
        nxt = torch.where(fits, place, L).amin(-1)
        on = on & (nxt < L)
        cur = torch.where(on, nxt, cur)
    return path.to(torch.int32), count.to(torch.int32), emitted.to(torch.int32)


def _keep(st, case):
    path, count, emitted = _accept(st)
    page = case["page"]
    s, j = torch.nonzero(torch.arange(path.shape[1], device=DEV) < count[:, None], as_tuple=True)
    pos0 = st["pos0"].long()[s]
    frm, to = pos0 + path[s, j], pos0 + j
    for x in (_layer(st["caches"], i) for i in range(case["layers"])):
        KVH, hd = x["k"].shape[1], x["k"].shape[3]
        T = x["v"].shape[6]
        heads = torch.arange(KVH, device=DEV)
        d = torch.arange(hd, device=DEV)
        raw = torch.uint8 if T == 4 else x["k"].dtype
        kr = x["k"].view(raw)
        vl = x["v"].view(raw).permute(0, 1, 2, 4, 7, 3, 6, 5)

        def where(pos):
            pid = st["table"][s, pos // page].long()[:, None]
            blk = (pos % page // BLOCK)[:, None]
            t = pos % BLOCK
            return ((pid, heads, (pos % page)[:, None]),
                    (pid[..., None], heads[:, None], blk[..., None], (t // 4)[:, None, None],
                     (t % 4)[:, None, None], d // (16 * T), d // 16 % T, d % 16),
                    (pid, heads, blk))

        kf, vf, bf = where(frm)
        kt, vt, bt = where(to)
        k, v = kr[kf], vl[vf]
        if T == 4:
            for name, old_rows, blocks in (("ks", k, None), ("vs", v, vl)):
                sc = x[name]
                was = sc.clone()
                flat = (bt[0] * KVH + bt[1]) * sc.shape[2] + bt[2]
                sc.view(-1).scatter_reduce_(0, flat.flatten(), was[bf].flatten(), "amax")
                up = (was[bf].int() - sc[bt].int())[..., None]
                new = torch.ldexp(old_rows.view(torch.float8_e4m3fn).float(), up).to(
                    torch.float8_e4m3fn).view(torch.uint8)
                # the other tokens of a block whose scale grew
                page_id, h, b = torch.nonzero(sc != was, as_tuple=True)
                fall = (was.int() - sc.int())[page_id, h, b]
                if blocks is None:
                    kb = kr.view(kr.shape[0], KVH, page // BLOCK, BLOCK, hd)
                    kb[page_id, h, b] = torch.ldexp(
                        kb[page_id, h, b].view(torch.float8_e4m3fn).float(),
                        fall[:, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
                    kr[kt] = new
                else:
                    vb = x["v"].view(torch.uint8)
                    vb[page_id, h, b] = torch.ldexp(
                        vb[page_id, h, b].view(torch.float8_e4m3fn).float(),
                        fall[:, None, None, None, None, None]).to(torch.float8_e4m3fn).view(
                            torch.uint8)
                    vl[vt] = new
        else:
            kr[kt] = k
            vl[vt] = v
    return {"path": path, "count": count, "emitted": emitted, "caches": st["caches"]}


def _copy(caches, src, dst):
    for t in caches.values():
        if t is not None:
            raw = t.view(torch.uint8) if t.dtype.itemsize == 1 else t
            raw[:, dst] = raw[:, src]


def _fork(st, case):
    page, refs, kids = case["page"], st["refs"], st["children"]
    held = kids[kids >= 0].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    s = st["source"].long()
    tokens = st["tokens"].long()[s]
    full, part = tokens // page, tokens % page > 0
    col = torch.arange(kids.shape[1], device=DEV)
    kids[:] = torch.where(col < full[:, None], st["table"][s], -1)
    shared = kids[kids >= 0].long()
    free = torch.nonzero(refs == 0)[:, 0]
    refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    which = torch.nonzero(part)[:, 0]
    fresh = free[: which.shape[0]]
    refs[fresh] = 1
    src, dst = (torch.full_like(st["source"], -1) for _ in range(2))
    src[which] = st["table"][s[which], full[which]]
    dst[which] = fresh.to(torch.int32)
    kids[which, full[which]] = fresh.to(torch.int32)
    _copy(st["caches"], src[which].long(), fresh)
    return {"table": kids, "refs": refs, "src": src, "dst": dst, "caches": st["caches"]}


def _compact(st, case):
    refs, table = st["refs"], st["table"]
    pages = refs.shape[0]
    live = refs > 0
    at = torch.arange(pages, device=DEV)
    front = at < live.sum()
    frm, to = torch.nonzero(live & ~front)[:, 0], torch.nonzero(~live & front)[:, 0]
    where = torch.where(live, at, -1).to(torch.int32)
    where[frm] = to.to(torch.int32)
    new = torch.where(front, refs, 0)
    new[to] = refs[frm]
    src, dst = (torch.full((pages // 2,), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    src[: frm.shape[0]], dst[: to.shape[0]] = frm.to(torch.int32), to.to(torch.int32)
    moved = torch.where(table >= 0, where[table.clamp(min=0).long()], -1)
    _copy(st["caches"], frm, to)
    return {"refs": new, "table": moved, "src": src, "dst": dst, "caches": st["caches"]}


_PLAIN = dict(sample=_sample, tree=_attend, keep=_keep, fork=_fork, compact=_compact)
_OWN = dict(sample=_own_sample, tree=_own_tree, keep=_own_keep, fork=_own_fork,
            compact=_own_compact)


# ---------------------------------------------------- 64-bit definitions --

def exact(case, seed):
    """None for the page calls and for accepted paths: whole numbers and values moved as they are."""
    if case["kind"] not in ("sample", "tree"):
        return None
    st = prepare(case, seed)
    return _sample_exact(st) if case["kind"] == "sample" else _tree_exact(st, case)


def _sample_exact(st):
    x = st["logits"].double().cpu().numpy()
    u = st["u"].double().cpu().numpy()
    rows, vocab = x.shape

    def each(o, off):
        if o is None:
            o = off
        return o.cpu().numpy() if torch.is_tensor(o) else np.full(rows, o)

    T, p, mp = (each(o, f).astype(np.float32).astype(np.float64)
                for o, f in ((st["T"], 1.0), (st["p"], 1.0), (st["m"], 0.0)))
    k = each(st["k"], -1)
    tokens, lps = np.empty(rows, np.int32), np.empty(rows)
    for r in range(rows):
        row, top = x[r], x[r].max()
        if T[r] <= 0:
            tok = int(np.flatnonzero(row == top)[0])
        else:
            kept = np.argsort(-row, kind="stable")
            if k[r] >= 1:
                kept = kept[: k[r]]
            w = np.exp(((row[kept] - top) / T[r]).astype(np.longdouble))
            if p[r] < 1:
                kept = kept[: int(np.searchsorted(np.cumsum(w), p[r] * w.sum())) + 1]
            kept = kept[w[: len(kept)] >= min(mp[r], 1.0)]
            kept = np.sort(kept)
            c = np.cumsum(np.exp(((row[kept] - top) / T[r]).astype(np.longdouble)))
            tok = int(kept[min(int(np.searchsorted(c, u[r] * c[-1], side="right")), len(kept) - 1)])
        tokens[r] = tok
        lps[r] = row[tok] - top - np.log(np.exp(row - top).sum())
    return torch.from_numpy(tokens).to(DEV), torch.from_numpy(lps).to(DEV)


def _tree_exact(st, case):
    n, c = _lengths(case, seed=st["seed"])
    H, KVH, hd, _ = GEOMETRY[case["geometry"]]
    x, page = _layer(st["caches"], 0), case["page"]
    parents = st["parents"].reshape(-1).cpu().tolist()
    table = st["table"].cpu().tolist()
    T = x["v"].shape[6]
    # value of (token j, dim d) in a 16-token block of v, by its address
    j, d = torch.meshgrid(torch.arange(BLOCK, device=DEV), torch.arange(hd, device=DEV),
                          indexing="ij")
    place = (((d // (16 * T)) * 4 + j // 4) * 16 + d % 16) * 4 * T + d // 16 % T * 4 + j % 4
    outs, lses, positions, row = [], [], [], 0
    words = (max(n) + 31) // 32
    mask = np.zeros((sum(n), words), np.uint32)
    for s in range(case["seqs"]):
        total = n[s] + c[s]
        ids = torch.tensor(table[s][: (total + page - 1) // page], device=DEV)
        hide = torch.zeros(n[s], total, dtype=torch.bool)
        hide[:, c[s]:] = True
        for a in range(n[s]):
            at, depth = a, -1
            while at >= 0:
                hide[a, c[s] + at] = False
                mask[row + a, at // 32] |= np.uint32(1 << (at % 32))
                depth += 1
                at = parents[row + at]
            positions.append(c[s] + depth)
        hide = hide.to(DEV)
        out = torch.empty(n[s], H, hd, dtype=torch.float64, device=DEV)
        lse = torch.empty(n[s], H, dtype=torch.float64, device=DEV)
        for h in range(KVH):
            k = x["k"][:, h].view(torch.uint8 if T == 4 else x["k"].dtype)[ids]
            v = x["v"][:, h].flatten(2).view(torch.uint8 if T == 4 else x["v"].dtype)[ids]
            if T == 4:
                k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
            k = k.double().view(-1, BLOCK, hd)
            v = v.double().view(-1, BLOCK * hd)[:, place.flatten()].view(-1, BLOCK, hd)
            if T == 4:
                k = k * 2.0 ** (x["ks"][ids, h].double().view(-1, 1, 1) - 127)
                v = v * 2.0 ** (x["vs"][ids, h].double().view(-1, 1, 1) - 127)
            k, v = k.reshape(-1, hd)[:total], v.reshape(-1, hd)[:total]
            for a in range(h * (H // KVH), (h + 1) * (H // KVH)):
                z = st["q"][row:row + n[s], a].double() @ k.t().contiguous() / hd ** 0.5
                z.masked_fill_(hide, float("-inf"))
                lse[:, a] = torch.logsumexp(z, -1)
                out[:, a] = torch.exp(z - lse[:, a:a + 1]) @ v
        outs.append(out)
        lses.append(lse)
        row += n[s]
    o = (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)
    if not case["plan"]:
        return {"o": o, "mask": None, "positions": None}
    return {"o": o, "mask": torch.from_numpy(mask.view(np.int32)).to(DEV),
            "positions": torch.tensor(positions, dtype=torch.int32, device=DEV)}
