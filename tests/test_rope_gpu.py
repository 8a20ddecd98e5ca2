"""Rotary positions (sm_rope_table, sm_rope) against 64-bit definitions."""
import math

import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def close(got, x, ref, dtype):
    """Products and sum rounded to f32 (three roundings of values up to |a| + |b|), then
    one rounding to the type (f16 below its normal range: half of 2^-24)."""
    big = x.double().abs().amax(-1, keepdim=True) * 2
    tol = 3 * 2.0 ** -24 * big + HALF[dtype] * ref.abs() * 1.001 + 2.0 ** -25
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), (got.double() - ref).abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rows,heads,hd,rot", [(1, 1, 16, 16), (3, 5, 64, 32), (33, 20, 128, 128),
                                               (7, 3, 80, 48), (5, 70, 64, 64), (4, 2, 1024, 96),
                                               (257, 1, 48, 16)])
def test_rope_matches_definition(dev, dtype, layout, rows, heads, hd, rot):
    from summa_amd import ops
    print(f"case rope {dtype} {layout} {rows} {heads} {hd} {rot}", flush=True)
    table = P.angles(rot, 500)
    pos = torch.randint(0, 500, (rows,), dtype=torch.int32)
    qkv = torch.randn(rows, (heads + 2) * hd).to(dtype)
    x = qkv[:, : heads * hd].unflatten(1, (heads, hd))
    xd = qkv.to(dev)[:, : heads * hd].unflatten(1, (heads, hd))
    cs = table[pos.long()][:, None].double()
    for back in (False, True):
        ref = P.rotate(x.double(), cs, layout, -1.0 if back else 1.0)
        got = ops.rope(xd, table.to(dev), pos.to(dev), layout=layout, backward=back)
        assert got.is_contiguous() and got.dtype == dtype
        close(got.cpu(), x, ref, dtype)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rope_in_place_and_strided_out(dev, layout, dtype):
    """In place over the q and k heads of fused rows, v left alone; and into a buffer whose
    other columns are left alone. The same bits as out of place."""
    from summa_amd import ops
    rows, heads, hd = 37, 6, 64
    qkv = torch.randn(rows, 8 * hd, device=dev).to(dtype)
    table, pos = P.angles(32, 64).to(dev), torch.arange(rows, dtype=torch.int32, device=dev)
    x = qkv[:, : heads * hd].unflatten(1, (heads, hd))
    want = ops.rope(x, table, pos, layout=layout)
    wide = torch.full((rows, 1024), 7.0, device=dev, dtype=dtype)
    got = ops.rope(x, table, pos, layout=layout,
                   out=wide[:, 64:64 + heads * hd].unflatten(1, (heads, hd)))
    assert torch.equal(got, want)
    assert bool((wide[:, :64] == 7).all()) and bool((wide[:, 64 + heads * hd:] == 7).all())
    v = qkv[:, heads * hd:].clone()
    got = ops.rope(x, table, pos, layout=layout, out=x)
    assert torch.equal(x, want) and torch.equal(qkv[:, heads * hd:], v)


def test_rope_gradient(dev):
    """backward is the transposed rotation: <rope(x), g> = <x, rope_back(g)>, and it equals
    central differences of that inner product (linear in x, so exact up to rounding)."""
    from summa_amd import ops
    for layout in ("interleaved", "half"):
        x, g = torch.randn(2, 9, 3, 64, dtype=torch.float64)
        table, pos = P.angles(48, 4000), torch.randint(0, 4000, (9,), dtype=torch.int32)
        cs = table[pos.long()][:, None].double()
        gx = ops.rope(g.float().to(dev), table.to(dev), pos.to(dev), layout=layout,
                      backward=True).cpu().double()
        g32 = g.float().double()
        for _ in range(20):
            i = tuple(int(torch.randint(0, n, ())) for n in x.shape)
            d = torch.zeros_like(x)
            d[i] = 0.5
            diff = ((P.rotate(x + d, cs, layout) - P.rotate(x - d, cs, layout)) * g32).sum()
            assert abs(float(diff) - float(gx[i])) < 3 * 2.0 ** -24 * 2 * float(g32.abs().max()) + 1e-12


def test_rope_table_angles_of_far_positions(dev):
    """cos / sin of 64-bit angles, rounded once, up to position 2^21 - 1: sampled against
    an angle reduced in integer-exact f64 (position * frequency has 53 bits, so the angle
    is within 2^-53 * 2^21 = 2^-32 of the product)."""
    from summa_amd import ops
    n, rot = 1 << 21, 32
    t = ops.rope_table(n, rot, 1e4, device=dev)
    assert tuple(t.shape) == (n, rot // 2, 2)
    rows = torch.cat([torch.tensor([0, 1, n - 1]), torch.randint(0, n, (500,))])
    got = t[rows.to(dev)].cpu().double()
    for i, p in enumerate(rows.tolist()):
        for j in range(rot // 2):
            a = p * 1e4 ** (-2.0 * j / rot)
            for x, ref in ((got[i, j, 0], math.cos(a)), (got[i, j, 1], math.sin(a))):
                assert abs(float(x) - ref) <= 2.0 ** -24 * abs(ref) + 2.0 ** -31 + 2.0 ** -31


@pytest.mark.parametrize("scaling", ["linear", "theta", "parts"])
def test_rope_table_scalings(dev, scaling):
    from summa_amd import ops
    rot, n, f, orig = 64, 300, 8.0, 128.0
    t = ops.rope_table(n, rot, 5e5, scaling=scaling, factor=f, original_positions=orig,
                       low_turns=1.0, high_turns=8.0, magnitude=1.25, device=dev).cpu().double()
    for j in range(rot // 2):
        w = 5e5 ** (-2.0 * j / rot)
        if scaling == "linear":
            w = w / f
        elif scaling == "theta":
            w = (5e5 * f ** (rot / (rot - 2))) ** (-2.0 * j / rot)
        else:
            r = orig * w / (2 * math.pi)
            keep = 1.0 if r >= 8 else 0.0 if r <= 1 else (r - 1) / 7
            w = (1 - keep) * w / f + keep * w
        a = torch.arange(n, dtype=torch.float64) * w
        assert float((t[:, j, 0] - 1.25 * a.cos()).abs().max()) <= 1.25 * 2.0 ** -24 * 1.01
        assert float((t[:, j, 1] - 1.25 * a.sin()).abs().max()) <= 1.25 * 2.0 ** -24 * 1.01


def test_rope_outside_the_table_is_nan(dev):
    from summa_amd import ops
    table = P.angles(32, 10).to(dev)
    pos = torch.tensor([9, 10, -1, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    x = torch.ones(4, 2, 64, device=dev)
    for layout in ("interleaved", "half"):
        y = ops.rope(x, table, pos, layout=layout)
        assert bool(torch.isfinite(y[0]).all())
        assert bool(torch.isnan(y[1:, :, :32]).all()) and bool((y[1:, :, 32:] == 1).all())


def test_rope_refusals(dev):
    from summa_amd import SummaError, ops
    t, pos = P.angles(32, 10).to(dev), torch.zeros(4, dtype=torch.int32, device=dev)
    x = torch.zeros(4, 2, 64, device=dev)
    with pytest.raises(SummaError, match="rot_dim must be a multiple of 16"):
        ops.rope(x, P.angles(24, 10).to(dev), pos)
    with pytest.raises(SummaError, match="rot_dim must be a multiple of 16 up to head_dim"):
        ops.rope(x, P.angles(128, 10).to(dev), pos)
    with pytest.raises(SummaError, match="does not overlap"):
        both = torch.zeros(8, 2, 64, device=dev)
        ops.rope(both[:4], t, pos, out=both[1:5])
    with pytest.raises(ValueError, match="layout"):
        ops.rope(x, t, pos, layout="other")
    with pytest.raises(ValueError, match="positions"):
        ops.rope(x, t, pos.long())
    with pytest.raises(ValueError, match="contiguous heads"):
        ops.rope(x.transpose(0, 1), t, pos[:2])
    with pytest.raises(TypeError):
        ops.rope(x.double(), t, pos)
    assert ops.rope(x[:0], t, pos[:0]).shape == (0, 2, 64)
