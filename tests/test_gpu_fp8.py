"""The 8-bit linear operators (dynam3d_amd/fp8_ops.py) on the GPU against their definitions in 64 bits.

Tolerances.  Quantised values and scales of `quantize` / `quantize_weight` are exact (one correctly rounded division, one rounding): bit for bit
against the CPU expression.  Products: E4M3 products are exact in float32; a float32 sum of K of them in any order is off by at most K 2^-24 times
the sum of the absolute products per rounding, twice that for a matrix core that truncates when it aligns, and the two scales add one rounding each per
group: 2 (K + 4) 2^-24 sum |x w|, and that is what a float32 result is held to; the result is then rounded once (half a step: eps / 2 of the
value).  Results of 8 or 16 bits come from the 8-bit matrix instructions, which align 8 neighbouring products to the largest of them, p, and cut 13
bits below its binade (`test_what_the_8_bit_instructions_cut` shows it with powers of two): each of the 7 others loses less than 2^-13 |p|, so a group
of 8 at most 7 2^-13 |p| <= 7 2^-13 of its own sum |x w|, and the whole sum at most 7 2^-13 sum |x w| more.  The exponential of SwiGLU: 4 ulp of
float32 and the operations around it: 2^-20 relative.  Values behind a quantisation may land on the other neighbour: half a step of E4M3 (2^-4
relative, 2^-10 of the scale near zero) plus the error in front of it."""
import numpy as np
import pytest
import torch

from dynam3d_amd import fp8_ops as F8

pytestmark = pytest.mark.gpu
D = torch.float64
SCALES = [torch.float8_e8m0fnu, torch.float32]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def acts(m, k, dtype, seed):
    g = gen(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))
    x[:, :: max(1, k // 3)] *= 20.0
    return x.to(dtype)


def bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8)


def values64(q):
    s = q.scale.cpu().to(D).repeat_interleave(q.rows, 0)[:q.shape[0]]
    return q.data.cpu().to(D) * s[:, torch.arange(q.shape[1]) // 128]


def operands(m, n, k, scale, seed, x_dtype=torch.bfloat16):
    x = F8.quantize(acts(m, k, x_dtype, seed).cuda(), scale)
    w = F8.quantize_weight((torch.randn(n, k, generator=gen(seed + 1)) / k ** 0.5).cuda(), scale)
    return x, w


def products64(x, w):
    """x w^T in 64 bits, and the sum of the absolute products (on the GPU: float64 matrix product of exactly represented values)."""
    a, b = values64(x).cuda(), values64(w).cuda()
    return a @ b.t(), a.abs() @ b.abs().t()


def sum_tol(mag, k, out):
    return (2.0 * (k + 4) * 2.0 ** -24 + (0.0 if out == torch.float32 else 7 * 2.0 ** -13)) * mag


def check(y, ref, tol):
    y = y.to(D)
    assert torch.isfinite(y).all()
    over = (y - ref).abs() - tol
    assert float(over.max()) <= 0, (float(over.max()), float((y - ref).abs().max()), tuple(y.shape))


# ---- quantisation ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (3, 144), (5, 1040), (257, 3072), (130, 8192)])
def test_quantize_is_exact(m, k, dtype, scale):
    x = acts(m, k, dtype, m * k)
    x[0, 0] = 0.0
    got, want = F8.quantize(x.cuda(), scale), F8.quantize(x, scale)
    assert torch.equal(bits(got.scale), bits(want.scale)) and torch.equal(bits(got.data), bits(want.data))
    got, want = F8.quantize_weight(x.cuda(), scale), F8.quantize_weight(x, scale)
    assert torch.equal(bits(got.scale), bits(want.scale)) and torch.equal(bits(got.data), bits(want.data))


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_borders(dtype, scale):
    """Group maxima at every binade's 448 border and one step beside it, ties, the smallest numbers, zeros, infinities, NaN."""
    rows = []
    top = 15 if dtype == torch.float16 else 127
    for e in range(-14 if dtype == torch.float16 else -126, top + 1, 3):
        for f in (1.0, 1.75, 1.75 * (1 + 2.0 ** -7), 1.75 * (1 - 2.0 ** -7), 1.9921875):
            r = torch.linspace(-1, 1, 128, dtype=D) * f * 2.0 ** e
            r[5] = f * 2.0 ** e
            rows.append(r)
    rows.append(torch.zeros(128, dtype=D))
    rows.append(torch.full((128,), 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133, dtype=D))
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.randn(128, dtype=D, generator=gen(3))
        r[7] = bad
        rows.append(r)
        rows.append(torch.full((128,), bad, dtype=D))
    x = torch.stack(rows).to(dtype)
    got, want = F8.quantize(x.cuda(), scale), F8.quantize(x, scale)
    assert torch.equal(bits(got.scale), bits(want.scale))
    gv, wv = got.data.cpu().float(), want.data.float()
    assert torch.equal(gv.isnan(), wv.isnan()) and torch.equal(gv.isnan(), ~x.float().isfinite())
    assert torch.equal(gv.nan_to_num(0.0), wv.nan_to_num(0.0))
    assert bool(got.scale.float().cpu().isfinite().all()) and float(got.scale.float().min()) >= 2.0 ** -126


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strides_and_offsets(dtype):
    big = acts(40, 3 * 288 + 8, dtype, 1).cuda()
    for v in (big[3:30, 288:576], big[1::2, 8:8 + 272], big[:, 1:1 + 144], big[:, : 2 * 288: 2], big[:32].t()[:16, :32]):
        got, want = F8.quantize(v), F8.quantize(v.cpu().contiguous())
        assert torch.equal(bits(got.scale), bits(want.scale)) and torch.equal(bits(got.data), bits(want.data))


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m,k", [(1, 16), (77, 1040), (300, 3072)])
def test_dequantize(m, k, scale):
    x = acts(m, k, torch.bfloat16, 5)
    for q, c in ((F8.quantize(x.cuda(), scale), F8.quantize(x, scale)), (F8.quantize_weight(x.cuda(), scale), F8.quantize_weight(x, scale))):
        for dt in DTYPES:
            assert torch.equal(F8.dequantize(q, dt).cpu(), F8.dequantize(c, dt)), dt
            if scale == torch.float8_e8m0fnu and dt != torch.float16:
                assert torch.equal(F8.dequantize(q, dt).cpu().to(D), values64(q))


# ---- RMSNorm + residual ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d,res", [(1, 16, True), (1, 3072, True), (7, 144, False), (65, 3072, False), (300, 1040, True), (3, 8192, True), (2, 16384, False),
                                     (1500, 3072, True), (1025, 64, False)])
def test_rms_norm(m, d, res, dtype, scale):
    x, w = acts(m, d, dtype, d + m), 1 + 0.2 * torch.randn(d, generator=gen(2))
    r = acts(m, d, dtype, 9) if res else None
    got = F8.rms_norm(x.cuda(), w.cuda(), 1e-5, residual=None if r is None else r.cuda(), scale_dtype=scale)
    h = x.to(D)
    if res:
        got, total = got
        want_h = (x.float() + r.float()).to(dtype)                       # one float32 addition, one rounding: exact
        assert torch.equal(total.cpu(), want_h)
        h = want_h.to(D)
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * w.to(D)
    err = (d + 8) * 2.0 ** -24 * y.abs()                                   # the sum of squares (positive terms) and four roundings behind it
    s = got.scale.cpu().to(D).repeat_interleave(128, 1)[:, :d]
    tol = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s) + err
    assert float(((values64(got) - y).abs() - tol).max()) <= 0
    groups = torch.nn.functional.pad(y.abs(), (0, -d % 128)).view(m, -1, 128).amax(-1)
    ratio = groups / (got.scale.cpu().to(D) * 448.0)
    slack = (d + 8) * 2.0 ** -24
    assert float(ratio.max()) <= 1 + slack and float(ratio.min()) >= (0.5 if scale == torch.float8_e8m0fnu else 1.0) * (1 - slack)


def test_rms_norm_rows_that_hold_nothing_or_too_much():
    x = torch.zeros(6, 256)
    x[1] = 1.0
    x[2, 3] = float("inf")
    x[3, 200] = float("nan")
    x[4] = 1e-30
    w = torch.ones(256)
    got = F8.dequantize(F8.rms_norm(x.cuda(), w.cuda(), 1e-5), torch.float32).cpu()
    want = F8.dequantize(F8.rms_norm(x, w, 1e-5), torch.float32)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert bool((got[0] == 0).all()) and bool((got[1] == 1).all()) and bool(got[3].isnan().all())


def test_rms_norm_strides():
    big = acts(20, 1000, torch.bfloat16, 3).cuda()
    w = torch.randn(401, generator=gen(1)).cuda()
    for v in (big[2:9, 8:8 + 400], big[::3, 1:401], big[:, 500:900]):
        a, ha = F8.rms_norm(v, w[1:], 1e-6, residual=v)
        b, hb = F8.rms_norm(v.contiguous(), w[1:].clone(), 1e-6, residual=v.contiguous())
        assert torch.equal(bits(a.data), bits(b.data)) and torch.equal(bits(a.scale), bits(b.scale)) and torch.equal(ha, hb)


# ---- products -------------------------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 16), (1, 128, 128), (1, 9216, 3072), (2, 3072, 8192), (5, 1003, 1040), (8, 3072, 8192), (16, 32064, 512), (17, 129, 272), (31, 640, 4096),
          (33, 513, 144), (64, 4096, 1024), (77, 1003, 1040), (127, 255, 384), (128, 256, 128), (129, 257, 2064), (257, 3072, 3072), (577, 4096, 1024), (823, 1024, 4096), (1025, 1, 512), (1100, 2050, 1040),
          (1281, 511, 528), (2049, 1030, 640), (3000, 3072, 512), (1537, 768, 8192)]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(m, n, k, scale):
    x, w = operands(m, n, k, scale, m + n + k)
    ref, mag = products64(x, w)
    out = DTYPES[(m + n + k // 16) % 3]
    y = F8.linear(x, w, out_dtype=out)
    assert y.shape == (m, n) and y.dtype == out
    check(y, ref, sum_tol(mag, k, out) + torch.finfo(out).eps / 2 * ref.abs())
    # 2-norm: one rounding of the result, and what the instructions cut, of random signs: ~2^-14 of it
    assert float((y.to(D) - ref).norm()) <= (torch.finfo(out).eps / 2 + (1e-6 if out == torch.float32 else 2.0 ** -12)) * float(ref.norm())
    assert torch.equal(y, F8.linear(x, w, out_dtype=out))                  # the same bits every time


def test_what_the_8_bit_instructions_cut():
    """2^16 - 2^16 + 2^(16 - s): a float32 result has the small product at every s, wherever it stands; a 16-bit one may have cut it only beside the pair
    (the same 8 neighbours) and only from s = 14 on."""
    one = torch.ones(1, 1, device="cuda")
    for m in (1, 40, 300):
        for j in (2, 7, 8, 15, 16, 31, 64, 127):
            for s in (4, 12, 13, 14, 20, 24):
                x, w = torch.zeros(m, 128), torch.zeros(128, 128)
                x[:, 0], x[:, 1], w[:, 0], w[:, 1] = 256.0, -256.0, 256.0, 256.0
                e = 16 - s
                x[:, j], w[:, j] = 2.0 ** (e // 2), 2.0 ** (e - e // 2)
                xq = F8.Fp8(x.to(torch.float8_e4m3fn).cuda(), one.expand(m, 1))
                wq = F8.Fp8(w.to(torch.float8_e4m3fn).cuda(), one, 128)
                assert bool((F8.linear(xq, wq, out_dtype=torch.float32) == 2.0 ** e).all()), (m, j, s)
                y = F8.linear(xq, wq).float()
                assert bool(((y == 2.0 ** e) | ((y == 0) & (s >= 14 and j < 8 or s >= 24))).all()), (m, j, s, y)


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1003, 1040), (8, 3072, 3072), (77, 129, 272), (300, 1024, 1024), (1100, 2050, 400)])
def test_linear_bias_residual(m, n, k, out):
    for scale in SCALES:
        x, w = operands(m, n, k, scale, 11)
        ref, mag = products64(x, w)
        b, r = torch.randn(n, generator=gen(4)).to(out).cuda(), torch.randn(m, n, generator=gen(5)).to(out).cuda()
        for bias, res in ((b, None), (None, r), (b, r)):
            want = ref.clone()
            size = ref.abs()
            for e in (bias, res):
                if e is not None:
                    want += e.to(D)
                    size = size + e.to(D).abs()
            check(F8.linear(x, w, bias=bias, residual=res, out_dtype=out), want,
                  sum_tol(mag, k, out) + 2.0 ** -23 * size + torch.finfo(out).eps / 2 * want.abs())


def silu64(y, n):
    return y[:, n:] * y[:, :n] * torch.sigmoid(y[:, :n])


def swiglu_tol(x, w, k, n, out):
    ref, mag = products64(x, w)
    a, e = silu64(ref, n), sum_tol(mag, k, out)
    # |d silu| <= 1.1 |d g|
    return a, e[:, n:] * (ref[:, :n] * torch.sigmoid(ref[:, :n])).abs() + 1.1 * e[:, :n] * ref[:, n:].abs() + 1.1 * e[:, :n] * e[:, n:] + 2.0 ** -20 * a.abs()


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m,i,k", [(1, 16, 16), (1, 8192, 3072), (8, 8192, 3072), (3, 144, 272), (16, 1040, 512), (40, 2064, 400), (64, 128, 128), (65, 272, 1040),
                                   (129, 4096, 1024), (823, 2048, 640), (1030, 16, 512), (1100, 272, 528), (1281, 1040, 1024), (2500, 2048, 640)])
def test_linear_swiglu(m, i, k, scale):
    x, w = operands(m, 2 * i, k, scale, m + i)
    out = DTYPES[(m + i // 16) % 3]
    ref, tol = swiglu_tol(x, w, k, i, out)
    y = F8.linear_swiglu(x, w, out_dtype=out)
    check(y, ref, tol + torch.finfo(out).eps / 2 * ref.abs())
    ref, tol = swiglu_tol(x, w, k, i, torch.float8_e4m3fn)
    q = F8.linear_swiglu(x, w, out_dtype=torch.float8_e4m3fn)
    assert q.shape == (m, i) and q.scale.dtype == scale
    s = q.scale.cpu().to(D).repeat_interleave(128, 1)[:, :i].cuda()
    check(values64(q).cuda(), ref, tol + torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * s))
    top = torch.nn.functional.pad(ref.abs(), (0, -i % 128)).view(m, -1, 128).amax(-1)
    slack = torch.nn.functional.pad(tol, (0, -i % 128)).view(m, -1, 128).amax(-1)
    room = q.scale.cpu().to(D).cuda() * 448.0
    assert bool((top <= room + slack).all())
    assert bool((room * (0.5 if scale == torch.float8_e8m0fnu else 1.0) <= top + slack + 1e-6 * room).all())


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m", [3, 40, 300, 1300])
def test_a_bad_row_stays_alone(m, scale):
    """A NaN or an infinity in one row of x, in its ragged last group, makes that row of the product NaN and no other."""
    xf = acts(m, 400, torch.bfloat16, 1)
    bad = m // 2
    xf[bad, 390] = float("inf")
    w = F8.quantize_weight(torch.randn(2 * 1024, 400, generator=gen(2)).cuda(), scale)
    y = F8.linear(F8.quantize(xf.cuda(), scale), w)
    assert bool(y[bad].isnan().all()) and int(y.isnan().any(1).sum()) == 1
    q = F8.linear_swiglu(F8.quantize(xf.cuda(), scale), w, out_dtype=torch.float8_e4m3fn)
    v = F8.dequantize(q)
    assert bool(v[bad].isnan().all()) and int(v.isnan().any(1).sum()) == 1
    z = F8.linear(F8.quantize(torch.zeros(m, 400).cuda(), scale), w)
    assert bool((z == 0).all())


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m", [1, 8, 33, 300])
def test_linear_strides(m, scale):
    """Operands, scales, bias and residual that are views: rows apart, odd offsets, transposed scales."""
    n, k = 264, 528
    x, w = operands(m, n, k, scale, 21)
    y = F8.linear(x, w)
    wide = torch.zeros(m, k + 48, dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + k] = x.data.view(torch.uint8)
    sc = torch.empty(x.scale.shape[1], m, dtype=scale, device="cuda")
    sc.copy_(x.scale.t())
    odd = torch.zeros(m * k + 3, dtype=torch.uint8, device="cuda")
    odd[3:] = x.data.view(torch.uint8).flatten()
    ww = torch.zeros(n, 2 * k, dtype=torch.uint8, device="cuda")
    ww[:, k:] = w.data.view(torch.uint8)
    views = [F8.Fp8(wide.view(torch.float8_e4m3fn)[:, 16:16 + k], x.scale), F8.Fp8(x.data, sc.t()), F8.Fp8(odd[3:].view(torch.float8_e4m3fn).view(m, k), x.scale)]
    for v in views:
        assert torch.equal(F8.linear(v, w), y)
    assert torch.equal(F8.linear(x, F8.Fp8(ww.view(torch.float8_e4m3fn)[:, k:], w.scale, 128)), y)
    r = torch.randn(m, 3 * n + 1, generator=gen(3)).bfloat16().cuda()
    for v in (r[:, :n], r[:, n + 1:2 * n + 1], r[:, : 2 * n: 2]):
        assert torch.equal(F8.linear(x, w, residual=v), F8.linear(x, w, residual=v.contiguous()))
    assert torch.equal(F8.linear(x, w[128:256]), y[:, 128:256])
    assert torch.equal(F8.linear(x[m // 2:], w), F8.linear(F8.Fp8(x.data[m // 2:].clone(), x.scale[m // 2:].clone()), w))


def test_empty():
    x, w = operands(4, 64, 128, torch.float8_e8m0fnu, 1)
    e = x[2:2]
    assert F8.linear(e, w).shape == (0, 64) and F8.linear(x, w[0:0]).shape == (4, 0) and F8.dequantize(e).shape == (0, 128)
    assert F8.linear_swiglu(e, w, out_dtype=torch.float8_e4m3fn).shape == (0, 32) and F8.quantize(torch.zeros(0, 64).cuda()).shape == (0, 64)
    assert F8.rms_norm(torch.zeros(0, 64).cuda(), torch.ones(64).cuda(), 1e-5).shape == (0, 64)


def test_streams_and_graph():
    """Two streams at once, and a captured chain norm -> product -> SwiGLU -> product replayed on new inputs beside eager work."""
    g = gen(1)
    w1 = F8.quantize_weight((torch.randn(2 * 512, 256, generator=g) / 16).cuda())
    w2 = F8.quantize_weight((torch.randn(256, 512, generator=g) / 22).cuda())
    nw = torch.ones(256).cuda()

    def chain(x, r):
        q, h = F8.rms_norm(x, nw, 1e-5, residual=r)
        return F8.linear(F8.linear_swiglu(q, w1, out_dtype=torch.float8_e4m3fn), w2, residual=h)

    for m in (1, 24, 600):
        xs = [acts(m, 256, torch.bfloat16, s).cuda() for s in range(6)]
        want = [chain(x, xs[0]) for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [None] * 6
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[i % 2]):
                got[i] = chain(x, xs[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        sx, sr = xs[0].clone(), xs[0].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            chain(sx, sr)
        torch.cuda.current_stream().wait_stream(s)
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chain(sx, sr)
        with torch.cuda.graph(other):
            out2 = chain(sr, sx)
        for i in range(6):
            sx.copy_(xs[i])
            graph.replay()
            other.replay()
            eager = chain(xs[5 - i], xs[0])
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]) and torch.equal(eager, want[5 - i]) and torch.equal(out2, chain(sr, sx))


# ---- products of many tiles (256 x 256 per workgroup) ---------------------------------------------------------------------------------------------------
LARGE = [(2304, 4104, 272), (8200, 1032, 400), (1281, 7000, 640), (4100, 2048, 256), (2100, 8192, 1024), (4097, 3072, 1152)]


@pytest.mark.parametrize("out", DTYPES[:2])
@pytest.mark.parametrize("m,n,k", LARGE)
def test_linear_of_many_tiles(m, n, k, out):
    x, w = operands(m, n, k, torch.float8_e8m0fnu, m + n)
    ref, mag = products64(x, w)
    y = F8.linear(x, w, out_dtype=out)
    check(y, ref, sum_tol(mag, k, out) + torch.finfo(out).eps / 2 * ref.abs())
    assert torch.equal(y, F8.linear(x, w, out_dtype=out))
    b, r = torch.randn(n, generator=gen(4)).to(out).cuda(), torch.randn(m, n, generator=gen(5)).to(out).cuda()
    want, size = ref + b.to(D) + r.to(D), ref.abs() + b.to(D).abs() + r.to(D).abs()
    check(F8.linear(x, w, bias=b, residual=r, out_dtype=out), want, sum_tol(mag, k, out) + 2.0 ** -23 * size + torch.finfo(out).eps / 2 * want.abs())
    wide = torch.zeros(m, n + 8, dtype=out, device="cuda")
    wide[:, :n] = r
    assert torch.equal(F8.linear(x, w, residual=wide[:, :n]) if out == torch.bfloat16 else F8.linear(x, w, residual=wide[:, :n], out_dtype=out),
                       F8.linear(x, w, residual=r, out_dtype=out))


@pytest.mark.parametrize("m,i,k", [(1100, 4112, 528), (2050, 2048, 384), (2100, 4096, 1024), (4500, 1040, 272)])
def test_linear_swiglu_of_many_tiles(m, i, k):
    test_linear_swiglu(m, i, k, torch.float8_e8m0fnu)


def test_a_bad_row_stays_alone_among_many_tiles():
    m = 4100
    xf = acts(m, 400, torch.bfloat16, 1)
    for bad in (0, 2047, 4099):
        xb = xf.clone()
        xb[bad, 390] = float("nan")
        w = F8.quantize_weight(torch.randn(2 * 1024, 400, generator=gen(2)).cuda())
        y = F8.linear(F8.quantize(xb.cuda()), w)
        assert bool(y[bad].isnan().all()) and int(y.isnan().any(1).sum()) == 1
        v = F8.dequantize(F8.linear_swiglu(F8.quantize(xb.cuda()), w, out_dtype=torch.float8_e4m3fn))
        assert bool(v[bad].isnan().all()) and int(v.isnan().any(1).sum()) == 1


def test_many_tiles_on_two_streams_and_in_a_graph():
    x, w = operands(2100, 8192, 1024, torch.float8_e8m0fnu, 3)
    z = F8.quantize(acts(2100, 1024, torch.bfloat16, 8).cuda())
    want = [F8.linear(x, w), F8.linear(z, w)]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for j in range(6):
        with torch.cuda.stream(streams[j % 2]):
            got.append(F8.linear((x, z)[j % 2], w))
    torch.cuda.synchronize()
    assert all(torch.equal(got[j], want[j % 2]) for j in range(6))
    sx = F8.Fp8(x.data.clone(), x.scale.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F8.linear(sx, w)
    for j in range(4):
        src = (x, z)[j % 2]
        sx.data.view(torch.uint8).copy_(src.data.view(torch.uint8)), sx.scale.view(torch.uint8).copy_(src.scale.view(torch.uint8))
        graph.replay()
        eager = F8.linear(z, w)
        torch.cuda.synchronize()
        assert torch.equal(out, want[j % 2]) and torch.equal(eager, want[1])


@pytest.mark.parametrize("m,n,k", [(65600, 8, 256), (33100, 136, 272), (700, 16392, 640)])
def test_many_tiles_hold_what_few_hold(m, n, k):
    """A large product's rows are, bit for bit, those of products of some of them (K in one piece: both add in the same order)."""
    x, w = operands(m, n, k, torch.float8_e8m0fnu, 2)
    y = F8.linear(x, w)
    for a in (0, 255, m // 2, m - 100):
        assert torch.equal(y[a:a + 100], F8.linear(x[a:a + 100], w)), a
    if n % 32 == 0 or n == 8:
        x, w = operands(m // 2 + 5, 2 * 16, k, torch.float8_e8m0fnu, 2)
        y, q = F8.linear_swiglu(x, w), F8.linear_swiglu(x, w, out_dtype=torch.float8_e4m3fn)
        for a in (0, m // 2 - 95):
            assert torch.equal(y[a:a + 100], F8.linear_swiglu(x[a:a + 100], w))
            part = F8.linear_swiglu(x[a:a + 100], w, out_dtype=torch.float8_e4m3fn)
            assert torch.equal(bits(q.data[a:a + 100]), bits(part.data)) and torch.equal(bits(q.scale[a:a + 100]), bits(part.scale))


def test_operands_past_4_gib():
    """x of 4.9 GB, 9.8 in 16 bits: the last rows."""
    m, k = 600064, 8192
    d = torch.full((m, k), 0x38, dtype=torch.uint8, device="cuda")                # 1.0
    d[-300:] = torch.randint(0, 0x7f, (300, k), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    s = torch.full((m, k // 128), 127, dtype=torch.uint8, device="cuda")
    x = F8.Fp8(d.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu))
    w = F8.quantize_weight(torch.randn(136, k, generator=gen(1)).cuda() / 90)
    y = F8.linear(x, w)
    ref, mag = products64(F8.Fp8(x.data[-300:].clone(), x.scale[-300:].clone()), w)
    check(y[-300:], ref, sum_tol(mag, k, torch.bfloat16) + 2.0 ** -8 * ref.abs())
    assert torch.equal(y[:1].expand(1000, -1), y[m - 1300:m - 300])
    back = F8.dequantize(x[m - 300:])
    assert torch.equal(F8.dequantize(x)[-300:], back)
    q = F8.quantize(torch.ones(1, device="cuda", dtype=torch.bfloat16).expand(m, k))
    assert bool((q.data[-1].float() * q.scale[-1].float().repeat_interleave(128) == 1).all())
