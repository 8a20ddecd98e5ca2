"""Plain definitions of the tree, page and sampling operators, for the tests: loops on the CPU,
64 bits, nothing of the library."""
import math

import numpy as np
import torch

import _paged as P


def random_tree(n, gen, window=8):
    """Parents of n rows: -1 for the first, of the others one of the `window` rows before."""
    return [-1] + [int(torch.randint(max(0, i - window), i, (1,), generator=gen)) for i in range(1, n)]


def masks(parents):
    """(rows that each row sees, depth) of one tree."""
    sees, depth = [], []
    for i in range(len(parents)):
        at, s = i, set()
        while at >= 0:
            s.add(at)
            p = parents[at]
            at = p if p < at else -1
        sees.append(s)
        depth.append(len(s) - 1)
    return sees, depth


def words(sees, w):
    """int32 words of sets of rows."""
    out = np.zeros((len(sees), w), np.uint32)
    for i, s in enumerate(sees):
        for j in s:
            out[i, j // 32] |= np.uint32(1 << (j % 32))
    return torch.from_numpy(out.view(np.int32))


def attend(q, cached, table, pos0, starts, page, sees):
    """As _paged.attend, row i of sequence s seeing keys < pos0[s] and pos0[s] + j for j of
    sees[row] (those below the sequence's rows and not negative)."""
    K, V, _, evs = cached
    rows, H, hd = q.shape
    KVH = K.shape[1]
    G = H // KVH
    out = torch.full((rows, H, hd), float("nan"), dtype=torch.float64)
    mag, unit = out.clone(), torch.zeros(rows, H, hd, dtype=torch.float64)
    lse, err = torch.full((rows, H), float("nan"), dtype=torch.float64), torch.zeros(rows, H)
    for s in range(len(pos0)):
        n = starts[s + 1] - starts[s]
        for row in range(starts[s], starts[s + 1]):
            keys = list(range(max(0, pos0[s])))
            keys += [pos0[s] + j for j in sorted(sees[row]) if j < n and pos0[s] + j >= 0]
            if not keys:
                out[row], mag[row], lse[row] = 0.0, 0.0, -math.inf
                continue
            ids = [table[s][j // page] if j // page < len(table[s]) else -1 for j in keys]
            if any(i < 0 or i >= K.shape[0] for i in ids):
                continue  # NaN
            at = torch.tensor(ids), torch.tensor(keys) % page
            for h in range(KVH):
                k, v = K[at[0], h, at[1]], V[at[0], h, at[1]]
                vs = torch.ones(len(keys), 1, dtype=torch.float64) if evs is None else \
                    2.0 ** evs[at[0], h, at[1] // P.BLOCK].double()[:, None]
                for a in range(h * G, (h + 1) * G):
                    x = q[row, a].double()
                    sc = k @ x / math.sqrt(hd)
                    w = torch.softmax(sc, 0)
                    out[row, a], mag[row, a] = w @ v, w @ v.abs()
                    lse[row, a] = torch.logsumexp(sc, 0)
                    err[row, a] = float((k.abs() @ x.abs()).max()) / math.sqrt(hd)
                    unit[row, a] = (w[:, None] * vs).max() * (v / vs).abs().sum(0)
    return out, lse, mag, err, unit


def accept(parents, tokens, sampled):
    """(path, emitted) of one tree."""
    path, emitted = [], []
    cur = 0 if parents else None
    while cur is not None:
        path.append(cur)
        emitted.append(sampled[cur])
        cur = next((i for i in range(cur + 1, len(parents))
                    if parents[i] == cur and tokens[i] == sampled[cur]), None)
    return path, emitted


def _scaled(codes, e):
    """uint8 e4m3 codes times 2^e (e <= 0), rounded again; NaN codes stay."""
    x = codes.view(torch.float8_e4m3fn).float()
    y = (x.double() * 2.0 ** e).float().to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where((codes & 0x7f) == 0x7f, codes, y)


def keep(raw, table, pos0, path, page, hd):
    """[k, v] or [k, v, ks, vs] (raw words, as stored) with token pos0 + path[j] at pos0 + j, one
    sequence after the other, one token at a time."""
    k, v = raw[0].clone(), raw[1].clone()
    ks, vs = ([raw[2].clone(), raw[3].clone()] if len(raw) > 2 else [None, None])
    pages, KVH = k.shape[:2]
    T = 4 if ks is not None else 2
    place = P.v_index(hd, T)
    flat = v.view(pages, KVH, page // 16, 16 * hd)
    for s, steps in enumerate(path):
        last, moves = -1, []
        for j, i in enumerate(steps):
            def at(pos):
                ok = 0 <= pos and pos // page < len(table[s])
                return table[s][pos // page] if ok else -1
            a, b = pos0[s] + i, pos0[s] + j
            if pos0[s] < 0 or i <= last or at(a) < 0 or at(a) >= pages or at(b) < 0 or at(b) >= pages:
                break
            last = i
            moves.append((at(a), a % page, at(b), b % page))
        for h in range(KVH):
            if ks is not None:  # scales first, in the order of the blocks written
                for kind, sc in (("k", ks), ("v", vs)):
                    old = sc[:, h].clone()
                    for pa, ta, pb, tb in moves:
                        sc[pb, h, tb // 16] = max(int(sc[pb, h, tb // 16]), int(old[pa, ta // 16]))
                    new = []
                    for pa, ta, pb, tb in moves:
                        src = k[pa, h, ta] if kind == "k" else flat[pa, h, ta // 16][place[ta % 16]]
                        new.append(_scaled(src.clone(), int(old[pa, ta // 16]) - int(sc[pb, h, tb // 16])))
                    for pb, blk in {(m[2], m[3] // 16) for m in moves}:
                        e = int(old[pb, blk]) - int(sc[pb, h, blk])
                        if e:
                            if kind == "k":
                                sl = k[pb, h, 16 * blk:16 * blk + 16]
                                sl.copy_(_scaled(sl.clone().contiguous(), e))
                            else:
                                flat[pb, h, blk] = _scaled(flat[pb, h, blk].clone(), e)
                    for (pa, ta, pb, tb), x in zip(moves, new):
                        if kind == "k":
                            k[pb, h, tb] = x
                        else:
                            flat[pb, h, tb // 16, place[tb % 16]] = x
            else:
                for pa, ta, pb, tb in moves:
                    k[pb, h, tb] = k[pa, h, ta].clone()
                    flat[pb, h, tb // 16, place[tb % 16]] = flat[pa, h, ta // 16][place[ta % 16]].clone()
    return [k, v] + ([ks, vs] if ks is not None else [])


def sample(x, u, T=1.0, k=-1, p=1.0, m=0.0):
    """(token, log-prob) of one row of f64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    d = np.where(x == top, 0.0, -np.inf if top == np.inf else x - top)
    total = np.exp(d).sum()
    if not T > 0:
        tok = int(np.flatnonzero(x == top)[0])
    else:
        kept = np.argsort(-x, kind="stable")
        if 1 <= k < len(x):
            kept = kept[:k]
        w = np.where(d[kept] == 0, 1.0, np.exp(d[kept] / T) if np.isfinite(T) else d[kept] > -np.inf)
        if p < 1:
            kept = kept[: max(1, int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1)]
            w = w[: len(kept)]
        if m > 0:
            kept, w = kept[w >= min(m, 1.0)], w[w >= min(m, 1.0)]
        order = np.argsort(kept)
        kept, w = kept[order], w[order]
        c = np.cumsum(w)
        u = 0.0 if u != u else min(max(float(u), 0.0), 1.0)
        passed = np.flatnonzero(c > u * c[-1])
        tok = int(kept[passed[0]]) if len(passed) else int(kept[np.flatnonzero(w)[-1]])
    return tok, d[tok] - math.log(total)
