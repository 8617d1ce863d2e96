"""`exact=True`: results of every type from exact products.  A 16-bit result is then the float32 one rounded, a quantised one the float32 one quantised, bit for bit
(float32 results are held to their 64-bit bound in test_gpu_fp8.py), whatever the number of rows."""
import pytest
import torch

from dynam3d_amd import fp8_ops as F8
from tests.test_gpu_fp8 import SCALES, acts, bits, gen, operands

pytestmark = pytest.mark.gpu
F32, E4M3 = torch.float32, torch.float8_e4m3fn
# few rows (one, two and four tiles of 16), tiles with K in slices and without, sizes that the large kernel takes otherwise
SIZES = [(1, 144, 272), (16, 1040, 512), (31, 640, 4096), (40, 2064, 400), (64, 272, 1040), (100, 272, 1040), (300, 1040, 1024), (1100, 4112, 528), (2100, 4096, 272)]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_exact_is_the_float32_result_rounded(m, n, k, scale):
    x, w = operands(m, 2 * n, k, scale, m + n)
    y, a = F8.linear(x, w, out_dtype=F32), F8.linear_swiglu(x, w, out_dtype=F32)
    assert torch.equal(y, F8.linear(x, w, out_dtype=F32, exact=True)) and torch.equal(a, F8.linear_swiglu(x, w, out_dtype=F32, exact=True))
    for out in (torch.bfloat16, torch.float16):
        assert torch.equal(F8.linear(x, w, out_dtype=out, exact=True), y.to(out)), out
        assert torch.equal(F8.linear_swiglu(x, w, out_dtype=out, exact=True), a.to(out)), out
    q, want = F8.linear_swiglu(x, w, out_dtype=E4M3, exact=True), F8.quantize(a, scale)
    assert torch.equal(bits(q.scale), bits(want.scale)) and torch.equal(bits(q.data), bits(want.data))


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("m", [1, 40, 300, 2100])
def test_what_cancels_survives(m, scale):
    """2^16 - 2^16 + 2^(16 - s) beside each other: the small one is there with `exact`, in every type."""
    n = 4104 if m > 2000 else 264
    one = torch.ones(1, 1)
    for s in (13, 14, 20, 24):
        e = 16 - s
        x, w = torch.zeros(m, 256), torch.zeros(n, 256)
        x[:, 130], x[:, 131], w[:, 130], w[:, 131] = 256.0, -256.0, 256.0, 256.0
        x[:, 133], w[:, 133] = 2.0 ** (e // 2), 2.0 ** (e - e // 2)
        xq = F8.Fp8(x.to(E4M3).cuda(), one.expand(m, 2).to(scale).cuda())
        wq = F8.Fp8(w.to(E4M3).cuda(), one.expand((n + 127) // 128, 2).to(scale).cuda(), 128)
        for out in (torch.bfloat16, torch.float16, F32):
            assert bool((F8.linear(xq, wq, out_dtype=out, exact=True) == 2.0 ** e).all()), (s, out)


def test_exact_with_bias_residual_streams_and_graph():
    m, n, k = 300, 1024, 528
    x, w = operands(m, n, k, SCALES[0], 5)
    b, r = torch.randn(n, generator=gen(1)).cuda(), torch.randn(m, n, generator=gen(2)).cuda()
    half = F8.linear(x, w, b.bfloat16(), r.bfloat16(), torch.bfloat16, True)
    assert torch.equal(half, F8.linear(x, w, b.bfloat16().float(), r.bfloat16().float(), F32).bfloat16())
    want, s = F8.linear_swiglu(x, w, E4M3, exact=True), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = F8.linear_swiglu(x, w, E4M3, exact=True)
    torch.cuda.synchronize()
    assert torch.equal(bits(other.data), bits(want.data))
    src = F8.Fp8(x.data.clone(), x.scale.clone())
    z = F8.quantize(acts(m, k, torch.bfloat16, 9).cuda())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F8.linear_swiglu(src, w, E4M3, exact=True)
    for i in range(4):
        new = (x, z)[i % 2]
        src.data.view(torch.uint8).copy_(new.data.view(torch.uint8)), src.scale.view(torch.uint8).copy_(new.scale.view(torch.uint8))
        graph.replay()
        eager = F8.linear_swiglu(new, w, E4M3, exact=True)
        torch.cuda.synchronize()
        assert torch.equal(bits(out.data), bits(eager.data)) and torch.equal(bits(out.scale), bits(eager.scale))
