"""Products whose two scales multiply out of float32's range while the result does not: y = sx sw sum xq wq for every pair of finite scales.

Tolerance: every sum below has one member that is not zero, a power of two or 448 * 448 times one, so what is left are the roundings of the scales'
product, of its product with the sum (one or two) and of the result: 3 * 2^-24 of the value in float32, and half a step of the 16-bit type more
(2^-25 at the lower end of fp16: half its smallest number).  Rows of many products: a float32 sum of K of them, 2 (K + 4) 2^-24 of the sum of their magnitudes,
and 7 * 2^-13 of it where the 8-bit instruction cuts (tests/test_gpu_fp8.py)."""
import pytest
import torch

from dynam3d_amd import fp8_ops as F8

pytestmark = pytest.mark.gpu
E8M0, F32, E4M3 = torch.float8_e8m0fnu, torch.float32, torch.float8_e4m3fn
SIZES = [(1, 264), (20, 264), (40, 264), (8, 4999), (100, 264), (2100, 4104)]          # few rows, tiles, many tiles
K = 272                                                                            # two groups and an eighth
# sx, sw, the one product of every sum (x value, w value); the last value's place differs where the sum is 0
PAIRS = [(2.0 ** 100, 2.0 ** 60, 1.0, 0.0), (2.0 ** 70, 2.0 ** 60, 2.0 ** -9, 2.0 ** -9), (2.0 ** -9, 2.0 ** 115, 448.0, 2.0 ** -6), (2.0 ** -126, 2.0 ** 119, 448.0, 2.0 ** -9),
         (2.0 ** 110, 2.0 ** -126, 2.0 ** -9, 448.0), (2.0 ** -100, 2.0 ** -40, 448.0, 448.0), (1.3 * 2.0 ** -100, 1.7 * 2.0 ** -40, 448.0, 448.0),
         (1.1 * 2.0 ** 90, 1.9 * 2.0 ** 50, 2.0 ** -9, 2.0 ** -9), (2.0 ** -126, 2.0 ** -126, 1.0, 0.0)]


def operand(m, value, where, scale, kind, rows):
    d = torch.zeros(m, K)
    d[:, where] = value
    s = torch.full(((m + rows - 1) // rows, (K + 127) // 128), scale, dtype=F32)
    return F8.Fp8(d.to(E4M3).cuda(), s.to(kind).cuda(), rows)


@pytest.mark.parametrize("kind", [E8M0, F32])
@pytest.mark.parametrize("m,n", SIZES)
def test_any_two_scales(m, n, kind):
    for sx, sw, a, b in PAIRS:
        if kind == E8M0 and (sx != 2.0 ** round(torch.tensor(sx, dtype=torch.float64).log2().item()) or sw != 2.0 ** round(torch.tensor(sw, dtype=torch.float64).log2().item())):
            continue
        for where in (3, 130, 270):
            x, w = operand(m, a, where, sx, kind, 1), operand(n, b if b else 1.0, where if b else where - 1, sw, kind, 128)
            want = a * b * float(x.scale[0, 0].double()) * float(w.scale[0, 0].double())
            for out in (F32, torch.bfloat16, torch.float16):
                y = F8.linear(x, w, out_dtype=out).double()
                if out == torch.float16 and abs(want) > 65520:
                    assert bool((y == float("inf")).all()), (sx, sw, out)
                    continue
                half = 0.0 if out == F32 else torch.finfo(out).eps / 2
                tol = abs(want) * (3 * 2.0 ** -24 + half) + (2.0 ** -25 if out == torch.float16 else 0.0)
                assert bool(((y - want).abs() <= tol).all()), (sx, sw, where, out, y.flatten()[:3], want)


@pytest.mark.parametrize("kind", [E8M0, F32])
@pytest.mark.parametrize("m,i", [(1, 144), (20, 144), (40, 144), (100, 144), (2100, 2064)])
def test_nothing_times_large_scales_is_nothing_behind_swiglu(m, i, kind):
    """Gates and ups that are empty sums between scales whose product overflows."""
    x, w = operand(m, 1.0, 131, 2.0 ** 100, kind, 1), operand(2 * i, 1.0, 130, 2.0 ** 60, kind, 128)
    for out in (torch.bfloat16, torch.float16, F32):
        assert bool((F8.linear_swiglu(x, w, out_dtype=out) == 0).all()), out
    assert bool((F8.dequantize(F8.linear_swiglu(x, w, out_dtype=E4M3), F32) == 0).all())


@pytest.mark.parametrize("kind", [E8M0, F32])
@pytest.mark.parametrize("m,n", SIZES)
def test_a_scale_that_is_nan_stays_in_its_row(m, n, kind):
    x, w = operand(m, 1.0, 130, 1.0, kind, 1), operand(n, 1.0, 130, 1.0, kind, 128)
    s = x.scale.float()
    s[m // 2, 1] = float("nan")
    x = F8.Fp8(x.data, s.to(kind))
    for out in (F32, torch.bfloat16):
        y = F8.linear(x, w, out_dtype=out)
        assert bool(y[m // 2].isnan().all()) and int(y.isnan().any(1).sum()) == 1, out


@pytest.mark.parametrize("out", [F32, torch.bfloat16])
@pytest.mark.parametrize("kind", [E8M0, F32])
@pytest.mark.parametrize("m", [7, 40, 300, 700])
def test_rows_of_zeros_change_nothing_beside_them(m, kind, out):
    """Scales of rows that hold nothing (2^-126) beside those of small weights multiply to denormals, from one K tile on or in all of them: the other rows keep
    their bits, and the zeros give zeros."""
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, 1040, generator=g), torch.randn(520, 1040, generator=g) * 2.0 ** -30
    w = F8.quantize_weight(w.cuda(), kind)
    full = F8.quantize(x.cuda(), kind)
    want, gated = F8.linear(full, w, out_dtype=out), F8.linear_swiglu(full, F8.Fp8(w.data[:512], w.scale[:4], 128), out_dtype=out)
    assert bool((want != 0).any(1).all())
    none = torch.arange(m) % 5 == 2
    for first in (0, 512):
        z = x.clone()
        z[none, first:] = 0.0
        y = F8.linear(F8.quantize(z.cuda(), kind), w, out_dtype=out)
        assert torch.equal(y[~none.cuda()], want[~none.cuda()])
        a = F8.linear_swiglu(F8.quantize(z.cuda(), kind), F8.Fp8(w.data[:512], w.scale[:4], 128), out_dtype=out)
        assert torch.equal(a[~none.cuda()], gated[~none.cuda()])
        if first == 0:
            assert bool((y[none.cuda()] == 0).all()) and bool((a[none.cuda()] == 0).all())
        else:
            d = F8.dequantize(full, F32)[:, :512].double()
            v = F8.dequantize(w, F32)[:, :512].double()
            ref, size = d @ v.t(), d.abs() @ v.abs().t()
            tol = (2 * (512 + 4) * 2.0 ** -24 + (0.0 if out == F32 else 7 * 2.0 ** -13)) * size + torch.finfo(out).eps / 2 * ref.abs()
            assert bool(((y.double() - ref).abs() <= tol)[none.cuda()].all())


@pytest.mark.parametrize("kind", [E8M0, F32])
@pytest.mark.parametrize("k", [16, 1040])
@pytest.mark.parametrize("m", [1, 20, 40, 100, 300])
def test_silu_of_float32_results(m, k, kind):
    """Gates from -80 to 80 and ups of 1, both exact sums: what is left are the exponential (1 ulp: 2^-23), the sum, the quotient and two products behind it (2^-24
    each) -- 2^-21 relative.  Few rows, tiles, and K in slices joined by another kernel (100 rows, K = 1040)."""
    gates = torch.arange(-320, 321).double() / 4
    i = 656
    w = torch.zeros(2 * i, k)
    for n, g in enumerate(gates.tolist()):
        for bit in range(10):                                                       # one power of two per column
            w[n, bit] = (1.0 if g >= 0 else -1.0) * 2.0 ** (bit - 2) if int(abs(g) * 4) >> bit & 1 else 0.0
    w[i:, 12] = 1.0
    one = lambda r, rows: torch.ones((r + rows - 1) // rows, (k + 127) // 128).to(kind).cuda()
    x = F8.Fp8(torch.ones(m, k).to(E4M3).cuda(), one(m, 1))
    y = F8.linear_swiglu(x, F8.Fp8(w.to(E4M3).cuda(), one(2 * i, 128), 128), out_dtype=F32)[:, :641].double().cpu()
    want = gates / (1 + torch.exp(-gates))
    assert bool(((y - want).abs() <= 2.0 ** -21 * want.abs()).all()), float(((y - want).abs() / want.abs().clamp_min(1e-300)).max())
