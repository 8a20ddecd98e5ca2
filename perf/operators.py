"""Paged key/value cache with rotary positions: the operators' cases and plain forms.

Three operators that a rollout or serving loop of this engine runs together:

- ``rope``: rotary positions of query and key heads inside fused qkv rows, forward
  and gradient, adjacent pairs or half-split, part of the head, any position.
- ``append``: new keys and values into a paged cache, keys and queries rotated on the
  way; the cache in 16 bits, or in 8 (e4m3) with a power-of-two scale for every 16
  tokens of a head.
- ``attn``: attention over that cache, from one query a sequence (a rollout step) to
  ragged chunks of queries (prefill, verification of drafted tokens).

Cache layout: ``k`` [pages, KVH, page, hd]; ``v`` [pages, KVH, page / 16, hd / 16T, 4, 16,
T, 4] with T = 4 (8-bit) or 2 (16-bit): token 4 g + j and dim 16 (c T + t) + r of a
16-token block at [c, g, r, t, j]. Scales [pages, KVH, page / 16] uint8: exponent + 127.
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
BLOCK = 16       # tokens of a scale
MIN_EXP = -63    # the least scale an append writes
# heads, KV heads and head_dim of summa_amd.configs' decoders
GEOMETRY = {"d256": (4, 4, 64), "d768": (12, 12, 64), "d2048": (16, 4, 128),
            "moe2048": (16, 16, 128)}


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # Rotation of one decode step's eight rows: the smallest call, all latency.
        dict(name="rope_step", kind="rope", rows=8, geometry="d2048", rot=128,
             layout="interleaved", dtype="bf16", backward=False, far=4096),
        # Queries and keys of a policy update's 8 x 1024 positions, f32 as it trains.
        dict(name="rope_train", kind="rope", rows=8192, geometry="d2048", rot=128,
             layout="interleaved", dtype="f32", backward=False, far=1024),
        # Its gradient in bf16 with the half-split layout over half of a 64-wide head,
        # at the far positions of a long context; an odd number of rows.
        dict(name="rope_grad_half", kind="rope", rows=16381, geometry="d768", rot=32,
             layout="half", dtype="bf16", backward=True, far=1000000),
        # One rollout step of 32 prompts x 8 rollouts: the f32 rows of the 4-bit qkv
        # projection, one token a sequence, into the 8-bit cache.
        dict(name="append_step", kind="append", seqs=256, rows_lo=1, rows_hi=1, ctx_lo=512,
             ctx_hi=1023, geometry="d2048", rot=128, layout="interleaved", dtype="f32",
             cache="e4m3", page=64),
        # Prefill of 32 prompts of unequal length, bf16 rows, small pages.
        dict(name="append_prefill", kind="append", seqs=32, rows_lo=257, rows_hi=512, ctx_lo=0,
             ctx_hi=0, geometry="d2048", rot=128, layout="half", dtype="bf16", cache="e4m3",
             page=16),
        # Chunks of three long prompts that continue inside a block, 16-bit cache, half
        # of the head rotated.
        dict(name="append_chunk", kind="append", seqs=3, rows_lo=1000, rows_hi=2047, ctx_lo=1,
             ctx_hi=5000, geometry="d768", rot=32, layout="half", dtype="f16", cache="f16",
             page=128),
        # A decode step of three short requests: latency.
        dict(name="attn_step_small", kind="attn", seqs=3, rows_lo=1, rows_hi=1, ctx_lo=60,
             ctx_hi=200, geometry="d256", dtype="f16", cache="f16", page=16, lse=False),
        # The rollout step of 256 sequences half way through 512 + 512 tokens.
        dict(name="attn_step", kind="attn", seqs=256, rows_lo=1, rows_hi=1, ctx_lo=512,
             ctx_hi=1023, geometry="d2048", dtype="f16", cache="e4m3", page=64, lse=False),
        # A few requests with very long contexts: the work is split over the keys.
        dict(name="attn_step_long", kind="attn", seqs=4, rows_lo=1, rows_hi=1, ctx_lo=100000,
             ctx_hi=131071, geometry="d2048", dtype="bf16", cache="e4m3", page=256, lse=False),
        # Four drafted tokens a sequence verified at once, no head shared, bf16 cache.
        dict(name="attn_verify", kind="attn", seqs=48, rows_lo=4, rows_hi=4, ctx_lo=1000,
             ctx_hi=4000, geometry="moe2048", dtype="bf16", cache="bf16", page=32, lse=False),
        # Prefill of 32 prompts of unequal length, with the log-sum-exp.
        dict(name="attn_prefill", kind="attn", seqs=32, rows_lo=257, rows_hi=512, ctx_lo=0,
             ctx_hi=0, geometry="d2048", dtype="bf16", cache="e4m3", page=64, lse=True),
        # Two prompts' next 1024 tokens against what is cached of them: the largest.
        dict(name="attn_chunk", kind="attn", seqs=2, rows_lo=1024, rows_hi=1024, ctx_lo=24000,
             ctx_hi=32767, geometry="d2048", dtype="f16", cache="e4m3", page=64, lse=False),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attn"])
    geometry = rng.choice(sorted(GEOMETRY))
    hd = GEOMETRY[geometry][2]
    rot = rng.choice([r for r in (16, 32, 64, 96, 128) if r <= hd])
    layout = rng.choice(["interleaved", "half"])
    if kind == "rope":
        return dict(kind=kind, rows=_log(rng, 1, 16384), geometry=geometry, rot=rot,
                    layout=layout, dtype=rng.choice(["f32", "bf16", "f16"]),
                    backward=rng.random() < 0.5, far=_log(rng, 64, 2000000))
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        seqs = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, 16384 // seqs))
        ctx = _log(rng, 1, max(2, min(20000, 262144 // seqs)))
        return dict(kind=kind, seqs=seqs, rows_lo=max(1, hi // 2), rows_hi=hi, ctx_lo=ctx // 2,
                    ctx_hi=ctx, geometry=geometry, rot=rot, layout=layout,
                    dtype=rng.choice(["f32", "bf16", "f16"]),
                    cache=rng.choice(["e4m3", "e4m3", "bf16", "f16"]), page=page)
    dtype = rng.choice(["bf16", "f16"])
    cache = rng.choice(["e4m3", "e4m3", dtype])
    shape = rng.choice(["step", "verify", "chunk"])
    if shape == "step":
        seqs, hi = _log(rng, 1, 256), 1
        ctx = _log(rng, 16, max(17, 262144 // seqs if seqs > 2 else 131071))
    elif shape == "verify":
        seqs, hi = _log(rng, 1, 64), rng.randint(2, 8)
        ctx = _log(rng, 16, max(17, 131072 // seqs))
    else:
        seqs = _log(rng, 1, 16)
        hi = _log(rng, 9, max(10, 2048 // seqs))
        ctx = _log(rng, 1, max(2, 16384 // seqs))
    return dict(kind=kind, seqs=seqs, rows_lo=max(1, hi // 2), rows_hi=hi, ctx_lo=ctx // 2,
                ctx_hi=ctx, geometry=geometry, dtype=dtype, cache=cache, page=page,
                lse=rng.random() < 0.25)


def _lengths(case, seed):
    """(new rows, cached tokens) of each sequence: the case's own, in the seed's order; the
    largest of both ranges among them."""
    rng = random.Random(13)
    n = [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    c = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    n[-1], c[0] = case["rows_hi"], case["ctx_hi"]
    both = list(zip(n, c))
    random.Random(seed).shuffle(both)
    return [a for a, _ in both], [b for _, b in both]


def work(case):
    H, KVH, hd = GEOMETRY[case["geometry"]]
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "rope":
        moved = case["rows"] * (H + KVH) * hd * size
        pairs = case["rows"] * (H + KVH) * case["rot"] / 2
        return {"bytes": 2 * moved + case["rows"] * (case["rot"] // 2 * 8 + 4), "flops": 6 * pairs}
    n, c = _lengths(case, 0)
    rows, csize = sum(n), DTYPES[case["cache"]].itemsize
    if case["kind"] == "append":
        read = rows * ((H + 2 * KVH) * hd * size + case["rot"] // 2 * 8)
        wrote = rows * (H * hd * 2 + 2 * KVH * hd * csize)
        if csize == 1:
            wrote += rows * 2 * KVH / BLOCK
        return {"bytes": read + wrote, "flops": rows * (H + KVH) * case["rot"] * 3}
    keys = sum(a + b for a, b in zip(n, c))
    kv = keys * 2 * KVH * (hd * csize + (1.0 / BLOCK if csize == 1 else 0.0))
    pairs = sum(a * b + a * (a + 1) / 2 for a, b in zip(n, c))
    return {"bytes": kv + 2 * rows * H * hd * size, "flops": 4 * pairs * H * hd}


# ----------------------------------------------------------------- inputs --

def _rope_table(far, rot):
    """[far, rot / 2, 2] f32 cosines and sines, angles in 64 bits (theta 10000)."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(far, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    H, KVH, hd = GEOMETRY[case["geometry"]]
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    st = dict(case=dict(case), seed=seed)
    if case["kind"] == "rope":
        rows, far = case["rows"], case["far"]
        qkv = randn(rows, (H + 2 * KVH) * hd).to(dtype)
        st["x"] = qkv[:, : (H + KVH) * hd].unflatten(1, (H + KVH, hd))  # q | k of fused rows
        st["table"] = _rope_table(far, case["rot"])
        st["positions"] = torch.randint(0, far, (rows,), generator=g, device=DEV,
                                        dtype=torch.int32)
        return st
    n, c = _lengths(case, seed)
    S, page, cdt = case["seqs"], case["page"], DTYPES[case["cache"]]
    need = [(a + b + page - 1) // page for a, b in zip(n, c)]
    pages, cols = sum(need) + 3, max(need)
    order = torch.randperm(pages, generator=g, device=DEV)[: sum(need)].to(torch.int32).cpu()
    table = torch.full((S, cols), -1, dtype=torch.int32)
    table[torch.arange(cols)[None, :] < torch.tensor(need)[:, None]] = order
    st["table"] = table.to(DEV)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    rows = int(start[-1])
    st["pos0"] = torch.tensor(c, dtype=torch.int32, device=DEV)
    st["row_start"] = torch.from_numpy(start).to(DEV) if len(set(n)) > 1 else None
    st["max_rows"], st["max_tokens"] = max(n), max(a + b for a, b in zip(n, c))
    T = 4 if cdt.itemsize == 1 else 2
    vshape = (pages, KVH, page // BLOCK, hd // (16 * T), 4, 16, T, 4)
    if cdt.itemsize == 1:  # codes and scales of values of about one
        def codes(*shape):
            t = torch.empty(shape, dtype=cdt, device=DEV)
            step = max(1, (1 << 28) // t[0].numel())
            for i in range(0, shape[0], step):
                t[i:i + step] = (randn(*t[i:i + step].shape) * 100).clamp_(-448, 448).to(cdt)
            return t
        st["k"], st["v"] = codes(pages, KVH, page, hd), codes(*vshape)
        st["ks"], st["vs"] = (torch.randint(119, 122, (pages, KVH, page // BLOCK), generator=g,
                                            device=DEV, dtype=torch.uint8) for _ in range(2))
    else:
        st["k"], st["v"] = randn(pages, KVH, page, hd).to(cdt), randn(*vshape).to(cdt)
        st["ks"] = st["vs"] = None
    if case["kind"] == "append":
        qkv = randn(rows, H + 2 * KVH, hd)
        # a few tokens much larger than the others, as keys and values have them
        big = torch.rand(rows, 1, 1, generator=g, device=DEV) < 0.01
        qkv = torch.where(big, qkv * 16, qkv).to(dtype)
        st["q"], st["kn"], st["vn"] = qkv.split([H, KVH, KVH], 1)
        st["rope"] = _rope_table(cols * page, case["rot"])
        st["q_dtype"] = torch.float16 if dtype == torch.float32 else dtype
    else:
        st["q"] = (randn(rows, H, hd) * 1.5).to(dtype)
    if own:
        from summa_amd import paged
        st["cache"] = paged.PagedKVCache.from_tensors(st["k"], st["v"], st["ks"], st["vs"])
    return st


# ------------------------------------------------------------------- pass --

def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    if case["kind"] == "rope":
        return _rotate(st["x"].float(), st["table"][st["positions"].long()][:, None],
                       case["layout"], -1.0 if case["backward"] else 1.0).to(st["x"].dtype)
    return _append(st, case) if case["kind"] == "append" else _attend(st, case)


def _run_own(st, case):
    from summa_amd import ops, paged
    if case["kind"] == "rope":
        return ops.rope(st["x"], st["table"], st["positions"], layout=case["layout"],
                        backward=case["backward"])
    if case["kind"] == "append":
        q = paged.paged_append(st["cache"], st["kn"], st["vn"], st["table"], st["pos0"],
                               st["row_start"], q=st["q"], rope_table=st["rope"],
                               layout=case["layout"], q_dtype=st["q_dtype"],
                               max_rows=st["max_rows"])
        return {"q": q, "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}
    return paged.paged_attention(st["cache"], st["q"], st["table"], st["pos0"], st["row_start"],
                                 max_rows=st["max_rows"], max_tokens=st["max_tokens"],
                                 want_lse=case["lse"])


# ------------------------------------------------------------ plain forms --

def _rotate(x, cs, layout, sign):
    """x [..., hd] f32 rotated by cs [..., rot / 2, 2]; dims past rot pass through."""
    rot = 2 * cs.shape[-2]
    c, s = cs[..., 0], cs[..., 1] * sign
    a, b = ((x[..., 0:rot:2], x[..., 1:rot:2]) if layout == "interleaved" else
            (x[..., : rot // 2], x[..., rot // 2:rot]))
    ra, rb = a * c - b * s, b * c + a * s
    y = torch.stack([ra, rb], -1).flatten(-2) if layout == "interleaved" else \
        torch.cat([ra, rb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _rows(st, rows):
    """Sequence and place in it of every row."""
    r = torch.arange(rows, device=DEV)
    if st["row_start"] is None:
        each = rows // st["table"].shape[0]
        return r // each, r % each
    seq = torch.searchsorted(st["row_start"][1:].long(), r, right=True)
    return seq, r - st["row_start"].long()[seq]


def _need_exp(amax):
    """The least e with amax <= 448 * 2^e, from MIN_EXP up."""
    m, ex = torch.frexp(amax)
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    return torch.where(amax > 0, e, MIN_EXP).clamp(min=MIN_EXP)


def _append(st, case):
    S, page = st["table"].shape[0], case["page"]
    rows, KVH, hd = st["kn"].shape
    seq, i = _rows(st, rows)
    pos = st["pos0"].long()[seq] + i
    pid = st["table"][seq, pos // page].long()
    cs = st["rope"][pos][:, None]
    q = _rotate(st["q"].float(), cs, case["layout"], 1.0).to(st["q_dtype"])
    kn = _rotate(st["kn"].float(), cs, case["layout"], 1.0)
    vn = st["vn"].float()
    blk, tok = pos % page // BLOCK, pos % BLOCK
    heads = torch.arange(KVH, device=DEV)
    T = st["v"].shape[6]
    # v as [pages, KVH, block, 16 tokens, hd] without moving it
    v_logical = st["v"].view(torch.uint8 if T == 4 else st["v"].dtype).permute(
        0, 1, 2, 4, 7, 3, 6, 5)
    d = torch.arange(hd, device=DEV)
    v_at = (pid[:, None, None], heads[:, None], blk[:, None, None], (tok // 4)[:, None, None],
            (tok % 4)[:, None, None], d // (16 * T), d // 16 % T, d % 16)
    k_at = (pid[:, None], heads, (pos % page)[:, None])
    if T == 2:
        st["k"][k_at] = kn.to(st["k"].dtype)
        v_logical[v_at] = vn.to(st["v"].dtype)
        return {"q": q, "k": st["k"], "v": st["v"], "ks": None, "vs": None}
    # the blocks that each sequence's rows touch, and the first of them
    first = st["pos0"].long() // BLOCK
    part = (st["pos0"].long() % BLOCK)[:, None]              # tokens before the first row
    nblk = (case["rows_hi"] + BLOCK - 1) // BLOCK + 1
    local = pos // BLOCK - first[seq]
    pid0 = st["table"][torch.arange(S, device=DEV), st["pos0"].long() // page].clamp(min=0).long()
    b0 = st["pos0"].long() % page // BLOCK
    at0 = (pid0[:, None], heads, b0[:, None])

    def encode(values, scales):
        amax = values.abs().amax(-1)
        most = torch.zeros(S, nblk, KVH, device=DEV)
        most = most.view(S * nblk, KVH).scatter_reduce(
            0, (seq * nblk + local)[:, None].expand(-1, KVH), amax, "amax").view(S, nblk, KVH)
        e = _need_exp(most)
        old = scales[at0].int() - 127
        e[:, 0] = torch.where(part > 0, torch.maximum(e[:, 0], old), e[:, 0])
        each = e[seq, local]
        codes = torch.ldexp(values, -each[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        scales[pid[:, None], heads, blk[:, None]] = (each + 127).to(torch.uint8)
        return codes, old, e[:, 0]

    def again(block, old, e):
        """The tokens before the first row, [S, KVH, 16, hd] codes, at the new scale."""
        x = block.view(torch.float8_e4m3fn).float()
        y = torch.ldexp(x, (old - e)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        keep = torch.arange(BLOCK, device=DEV)[None, None, :, None] < part[..., None, None]
        return torch.where(keep, y, block)

    k8 = st["k"].view(torch.uint8)
    kb = k8.view(k8.shape[0], KVH, page // BLOCK, BLOCK, hd)
    codes, old, e = encode(kn, st["ks"])
    kb[at0] = again(kb[at0], old, e)
    k8[k_at] = codes
    codes, old, e = encode(vn, st["vs"])
    vb = v_logical[at0].reshape(S, KVH, BLOCK, hd)  # dims in order: c, t, r
    v_logical[at0] = again(vb, old, e).view(S, KVH, 4, 4, hd // (16 * T), T, 16)
    v_logical[v_at] = codes
    return {"q": q, "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _cached(st, case):
    """Keys and values [S, KVH, tokens, hd] f32 of every sequence's pages."""
    at = st["table"].clamp(min=0).long()
    S, cols = at.shape
    KVH, page, hd = st["k"].shape[1:]

    def take(x):
        if x.dtype.itemsize == 1:
            return x.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        return x[at].float()

    k = take(st["k"]).view(S, cols, KVH, page // BLOCK, BLOCK, hd)
    v = take(st["v"]).permute(0, 1, 2, 3, 5, 8, 4, 7, 6).reshape(k.shape)
    if st["ks"] is not None:
        k, v = (torch.ldexp(x, (s[at].int() - 127)[..., None, None])
                for x, s in ((k, st["ks"]), (v, st["vs"])))
    return tuple(x.permute(0, 2, 1, 3, 4, 5).reshape(S, KVH, cols * page, hd) for x in (k, v))


def _attend(st, case):
    q = st["q"]
    rows, H, hd = q.shape
    S, L = st["table"].shape[0], case["rows_hi"]
    k, v = _cached(st, case)
    KVH, T = k.shape[1:3]
    G = H // KVH
    seq, i = _rows(st, rows)
    qp = torch.zeros(S, L, H, hd, device=DEV)
    qp[seq, i] = q.float()
    qp = qp.view(S, L, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(S, KVH, L * G, hd)
    sc = torch.matmul(qp, k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    pos = st["pos0"].long()[:, None] + torch.arange(L, device=DEV)
    hide = torch.arange(T, device=DEV) > pos.repeat_interleave(G, 1)[:, None, :, None]
    sc.masked_fill_(hide, float("-inf"))
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total
    o = o.view(S, KVH, L, G, hd).permute(0, 2, 1, 3, 4).reshape(S, L, H, hd)[seq, i].to(q.dtype)
    if not case["lse"]:
        return o
    lse = (m + total.log()).view(S, KVH, L, G).permute(0, 2, 1, 3).reshape(S, L, H)[seq, i]
    return o, lse


# ---------------------------------------------------- 64-bit definitions --

def exact(case, seed):
    st = prepare(case, seed)
    H, KVH, hd = GEOMETRY[case["geometry"]]
    if case["kind"] == "rope":
        return _turn(st["x"].double(), st["positions"].double(), case["rot"], case["layout"], case["backward"])
    n, c = _lengths(case, seed)
    table = st["table"].cpu().tolist()
    page = case["page"]
    if case["kind"] == "append":
        return _append_exact(st, case, n, c, table)
    # value of (token j, dim d) in a 16-token block of v, by its address
    T = st["v"].shape[6]
    j, d = torch.meshgrid(torch.arange(BLOCK, device=DEV), torch.arange(hd, device=DEV),
                          indexing="ij")
    place = (((d // (16 * T)) * 4 + j // 4) * 16 + d % 16) * 4 * T + d // 16 % T * 4 + j % 4
    outs, lses, row = [], [], 0
    for s in range(case["seqs"]):
        total = n[s] + c[s]
        ids = torch.tensor(table[s][: (total + page - 1) // page], device=DEV)
        out = torch.empty(n[s], H, hd, dtype=torch.float64, device=DEV)
        lse = torch.empty(n[s], H, dtype=torch.float64, device=DEV)
        late = torch.arange(total, device=DEV)[None, :] > \
            torch.arange(c[s], total, device=DEV)[:, None]
        for h in range(KVH):
            k = st["k"][:, h].view(torch.uint8 if T == 4 else st["k"].dtype)[ids]
            v = st["v"][:, h].flatten(2).view(torch.uint8 if T == 4 else st["v"].dtype)[ids]
            if T == 4:
                k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
            k = k.double().view(-1, BLOCK, hd)
            v = v.double().view(-1, BLOCK * hd)[:, place.flatten()].view(-1, BLOCK, hd)
            if T == 4:
                k = k * 2.0 ** (st["ks"][ids, h].double().view(-1, 1, 1) - 127)
                v = v * 2.0 ** (st["vs"][ids, h].double().view(-1, 1, 1) - 127)
            k, v = k.reshape(-1, hd)[:total], v.reshape(-1, hd)[:total]
            for a in range(h * (H // KVH), (h + 1) * (H // KVH)):
                x = st["q"][row:row + n[s], a].double() @ k.t().contiguous() / hd ** 0.5
                x.masked_fill_(late, float("-inf"))
                lse[:, a] = torch.logsumexp(x, -1)
                out[:, a] = torch.exp(x - lse[:, a:a + 1]) @ v
        outs.append(out)
        lses.append(lse)
        row += n[s]
    return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)


def _turn(x, pos, rot, layout, backward=False):
    """Pairs of x [rows, heads, hd] f64 turned by pos * 10000^(-2 p / rot)."""
    y = x.clone()
    for p in range(rot // 2):
        a = pos * 10000.0 ** (-2.0 * p / rot) * (-1 if backward else 1)
        a = a[:, None]
        u, w = (2 * p, 2 * p + 1) if layout == "interleaved" else (p, p + rot // 2)
        y[..., u] = x[..., u] * a.cos() - x[..., w] * a.sin()
        y[..., w] = x[..., w] * a.cos() + x[..., u] * a.sin()
    return y


def _append_exact(st, case, n, c, table):
    """q in 64 bits; the cache with every value that a row brings unrounded, in units of
    its block's scale, and older values of a block whose scale grew divided by that."""
    page, hd = case["page"], GEOMETRY[case["geometry"]][2]
    pos = torch.cat([torch.arange(b, a + b, device=DEV) for a, b in zip(n, c)])
    q = _turn(st["q"].double(), pos.double(), case["rot"], case["layout"])
    kn = _turn(st["kn"].double(), pos.double(), case["rot"], case["layout"])
    vn = st["vn"].double()
    T = st["v"].shape[6]
    k, v = st["k"].double(), st["v"].double()
    kb = k.view(*k.shape[:2], page // BLOCK, BLOCK, hd)
    vb = v.view(*v.shape[:3], -1)
    j, d = torch.meshgrid(torch.arange(BLOCK, device=DEV), torch.arange(hd, device=DEV),
                          indexing="ij")
    place = (((d // (16 * T)) * 4 + j // 4) * 16 + d % 16) * 4 * T + d // 16 % T * 4 + j % 4
    # every touched block: page, block of it, first row, first token, tokens
    touched, row = [], 0
    for s in range(case["seqs"]):
        p = c[s]
        while p < n[s] + c[s]:
            m = min(BLOCK - p % BLOCK, n[s] + c[s] - p)
            touched.append((table[s][p // page], p % page // BLOCK, row, p % BLOCK, m))
            row, p = row + m, p + m
    if len(touched) > 6000:
        return {"q": q, "k": None, "v": None, "ks": None, "vs": None}
    for pid, b, r, t, m in touched:
        for new, blocks, scales, order in ((kn, kb, st["ks"], None), (vn, vb, st["vs"], place)):
            x = new[r:r + m].transpose(0, 1)  # [KVH, tokens, hd]
            if scales is not None:
                most = x.abs().amax((1, 2)).clamp(min=2.0 ** -200)
                e = torch.ceil(torch.log2(most / 448)).clamp(min=MIN_EXP)
                old = scales[pid, :, b].double() - 127
                e = torch.maximum(e, old) if t else e
                x = x * 2.0 ** -e[:, None, None]
                shrink = 2.0 ** (old - e)[:, None, None]
            if order is None:
                if scales is not None and t:
                    blocks[pid, :, b, :t] *= shrink
                blocks[pid, :, b, t:t + m] = x
            else:
                if scales is not None and t:
                    blocks[pid, :, b, order[:t].flatten()] *= shrink[:, 0]
                blocks[pid, :, b, order[t:t + m].flatten()] = x.flatten(1)
    return {"q": q, "k": k, "v": v, "ks": None, "vs": None}
