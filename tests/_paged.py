"""Plain 64-bit definitions of the rotary and paged-cache operators, for the tests. Loops
over sequences, tokens and heads on the CPU; nothing of the library is used."""
import math

import torch

BLOCK = 16
MIN_EXP = -63


def angles(rot, positions, theta=1e4):
    """[positions, rot / 2, 2] f32 table, angles in 64 bits."""
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def rotate(x, cs, layout, sign=1.0):
    """x [..., hd] in its own precision by the table rows cs [..., rot / 2, 2]."""
    rot = 2 * cs.shape[-2]
    c, s = cs[..., 0].to(x.dtype), cs[..., 1].to(x.dtype) * sign
    y = x.clone()
    at = (slice(0, rot, 2), slice(1, rot, 2)) if layout == "interleaved" else \
        (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]] = a * c - b * s
    y[..., at[1]] = b * c + a * s
    return y


def v_index(hd, T):
    """[16, hd]: place of (token, dim) in a stored 16-token block of values."""
    t, d = torch.meshgrid(torch.arange(16), torch.arange(hd), indexing="ij")
    return (((d // (16 * T) * 4 + t // 4) * 16 + d % 16) * T + d // 16 % T) * 4 + t % 4


def need_exp(amax):
    """Least e >= -63 with amax <= 448 * 2^e."""
    if amax == 0:
        return MIN_EXP
    m, x = math.frexp(amax)
    return max(MIN_EXP, x - 9 if m <= 0.875 else x - 8)


def read(k, v, ks=None, vs=None):
    """(K, V f64 [pages, KVH, page, hd] as they stand for, exponents or None) of storage."""
    k, v = k.detach().cpu(), v.detach().cpu()
    pages, KVH, page, hd = k.shape
    T = 4 if k.dtype.itemsize == 1 else 2
    kk = k.float().double()
    flat = v.float().double().reshape(pages, KVH, page // BLOCK, 16 * hd)
    vv = flat[..., v_index(hd, T)].reshape(pages, KVH, page, hd)
    if ks is None:
        return kk, vv, None, None
    eks, evs = (x.detach().cpu().int() - 127 for x in (ks, vs))
    up = lambda e: (2.0 ** e.double()).repeat_interleave(BLOCK, 2)[..., None]  # noqa: E731
    return kk * up(eks), vv * up(evs), eks, evs


def attend(q, cached, table, pos0, starts, page):
    """f64 (out, lse, sum p |v|, largest |q| . |k| / sqrt(hd), unit) for q [rows, H, hd]
    over ``read``'s cache; rows of no sequence NaN. unit [rows, H, hd]: the largest p_j s_j
    (s_j the scale of v_j's block) times the sum of the codes |v_j / s_j|, which is what an
    absolute error of one in every weight, in the unit of the largest, comes to."""
    K, V, _, evs = cached
    rows, H, hd = q.shape
    KVH = K.shape[1]
    G = H // KVH
    out = torch.full((rows, H, hd), float("nan"), dtype=torch.float64)
    mag, unit = out.clone(), torch.zeros(rows, H, hd, dtype=torch.float64)
    lse, err = torch.full((rows, H), float("nan"), dtype=torch.float64), torch.zeros(rows, H)
    for s in range(len(pos0)):
        for row in range(starts[s], starts[s + 1]):
            p = pos0[s] + row - starts[s]
            if p < 0:
                out[row], mag[row], lse[row] = 0.0, 0.0, -math.inf
                continue
            ids = [table[s][j // page] if j // page < len(table[s]) else -1 for j in range(p + 1)]
            if any(i < 0 or i >= K.shape[0] for i in ids):
                continue  # NaN
            at = torch.tensor(ids), torch.arange(p + 1) % page
            for h in range(KVH):
                k, v = K[at[0], h, at[1]], V[at[0], h, at[1]]
                vs = torch.ones(p + 1, 1, dtype=torch.float64) if evs is None else \
                    2.0 ** evs[at[0], h, at[1] // BLOCK].double()[:, None]
                for a in range(h * G, (h + 1) * G):
                    x = q[row, a].double()
                    sc = k @ x / math.sqrt(hd)
                    w = torch.softmax(sc, 0)
                    out[row, a], mag[row, a] = w @ v, w @ v.abs()
                    lse[row, a] = torch.logsumexp(sc, 0)
                    err[row, a] = float((k.abs() @ x.abs()).max()) / math.sqrt(hd)
                    unit[row, a] = (w[:, None] * vs).max() * (v / vs).abs().sum(0)
    return out, lse, mag, err, unit
