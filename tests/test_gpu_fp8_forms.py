"""The 8-bit products at the sizes where another form of a kernel takes over: two and three column tiles per workgroup in the kernel for few rows (more than 4096
columns), for one, two and four tiles of 16 rows; the tile kernel in place of the large one where rows do not start on 16 bytes; and the norms of the results behind
the 8-bit instruction."""
import pytest
import torch

from dynam3d_amd import fp8_ops as F8
from tests.test_gpu_fp8 import D, DTYPES, SCALES, check, gen, operands, products64, silu64, sum_tol, values64

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m,n,k", [(1, 9216, 3072), (8, 6001, 528), (16, 9217, 144), (17, 9216, 3072), (32, 5003, 1040), (32, 32064, 272), (31, 12288, 2064), (33, 9217, 400), (48, 5004, 4096),
                                   (64, 16384, 144), (64, 9216, 1024)])
def test_few_rows_by_many_columns(m, n, k, scale, out):
    """Short last workgroups, blocks of 128 weight rows that end inside a workgroup's rows, K that ends inside a group."""
    x, w = operands(m, n, k, scale, m + n + k)
    ref, mag = products64(x, w)
    y = F8.linear(x, w, out_dtype=out)
    check(y, ref, sum_tol(mag, k, out) + torch.finfo(out).eps / 2 * ref.abs())
    assert torch.equal(y, F8.linear(x, w, out_dtype=out))
    b, r = torch.randn(n, generator=gen(4)).to(out).cuda(), torch.randn(m, n, generator=gen(5)).to(out).cuda()
    want, size = ref + b.to(D) + r.to(D), ref.abs() + b.to(D).abs() + r.to(D).abs()
    check(F8.linear(x, w, bias=b, residual=r, out_dtype=out), want, sum_tol(mag, k, out) + 2.0 ** -23 * size + torch.finfo(out).eps / 2 * want.abs())


@pytest.mark.parametrize("out", DTYPES[:2])
def test_large_products_off_16_bytes_keep_their_bits(out):
    """A residual that starts off 16 bytes, a bias that does, and a number of columns that is no multiple of 8 take the tile kernel, which adds in the same order."""
    m, n, k = 2304, 4104, 272
    x, w = operands(m, n, k, SCALES[0], 7)
    r, b = torch.randn(m, n + 9, generator=gen(1)).to(out).cuda(), torch.randn(n + 1, generator=gen(2)).to(out).cuda()
    for off in (1, 2, 4):
        assert torch.equal(F8.linear(x, w, residual=r[:, off:off + n], out_dtype=out), F8.linear(x, w, residual=r[:, off:off + n].contiguous(), out_dtype=out)), off
    assert torch.equal(F8.linear(x, w, bias=b[1:], out_dtype=out), F8.linear(x, w, bias=b[1:].clone(), out_dtype=out))
    full = F8.linear(x, w, out_dtype=out)
    for cols in (4097, 4100, 4102):
        assert torch.equal(F8.linear(x, w[:cols], out_dtype=out), full[:, :cols]), cols
    ref, mag = products64(x, w)
    check(full, ref, sum_tol(mag, k, out) + torch.finfo(out).eps / 2 * ref.abs())


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m,i,k", [(8, 2064, 1040), (40, 2064, 1040), (300, 1040, 1024), (823, 2048, 640), (2100, 4096, 1024)])
def test_swiglu_norms(m, i, k, scale):
    """2-norms.  16-bit results: half a step and 2^-12 (what the instruction cuts: ~2^-14 for each of gate and up).
    Quantised ones, against the 64-bit result on the same scales: a difference d in front of a rounding of step t flips it with probability |d| / t, by t, so the
    expected square is t |d|.  t <= 2^-3 |v|.  d: each of the 7 products beside the largest p of 8 loses between 0 and 2^-13 |p|, rms 2^-13 |p| / sqrt(3), of random
    sign: sqrt(7 / 3) 2^-13 |p|, and the squares of all p are at most the square of a sum of random signs: 2^-12.39 of gate and of up, sqrt(2) times that of v.
    P = 2^-3 2^-11.89 |v|^2 = 2^-14.89 of the squared norm is expected, then.  (The rows differ in size by design of the inputs, up to all of the norm in one row, and the
    products are few: (1) a row's p can be that large; (2) flips are rare, each is one t^2 out of the sum, whose variance is sum t^3 |d| <= t_max^2 P.  A first form of
    this bound, 2^-15 of the squared norm, took |d| for a sum of many equal products and left the variance out.)  P and four deviations are asked for.
    E4M3's own rounding: 2^-4 / sqrt(3) * 0.72 = 2.6 % of the norm, 3 % asked for."""
    x, w = operands(m, 2 * i, k, scale, m + i + 3)
    ref = silu64(products64(x, w)[0], i)
    for out in DTYPES[:2]:
        assert float((F8.linear_swiglu(x, w, out).to(D) - ref).norm()) <= (torch.finfo(out).eps / 2 + 2.0 ** -12) * float(ref.norm())
    q = F8.linear_swiglu(x, w, E4M3)
    s = q.scale.to(D).repeat_interleave(128, 1)[:, :i]
    same = (ref / s).float().clamp(-448.0, 448.0).to(E4M3).to(D) * s
    got = values64(q).cuda()
    expected = 2.0 ** -14.89 * float(ref.norm()) ** 2
    assert float((got - same).norm()) ** 2 <= expected + 4 * 2.0 ** -3 * float(ref.abs().max()) * expected ** 0.5, float((got - same).norm() / ref.norm())
    assert float((got - ref).norm()) <= 0.03 * float(ref.norm())
