"""The 8-bit linear operators without a GPU: the CPU expression against its definition in 64 bits, refusals, the C entry points' argument checks."""
import ctypes as C

import pytest
import torch

from dynam3d_amd import _lib
from dynam3d_amd import fp8_ops as F8

E8M0, F32, E4M3 = torch.float8_e8m0fnu, torch.float32, torch.float8_e4m3fn


def _e4m3_values():
    v = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    return v[v.isfinite()].unique()


@pytest.mark.parametrize("scale", [E8M0, F32])
@pytest.mark.parametrize("m,k,rows", [(3, 16, 1), (2, 400, 1), (130, 272, 128)])
def test_cpu_quantize_is_nearest(m, k, rows, scale):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(1)) * 3
    q = F8._cpu_quantize(x, scale, rows)
    s = q.scale.double().repeat_interleave(rows, 0)[:m][:, torch.arange(k) // 128]
    t = x.double() / s
    near = (t[..., None] - _e4m3_values()).abs().amin(-1)
    assert torch.allclose((q.data.double() - t).abs(), near, rtol=0, atol=448 * 2.0 ** -23)      # (the float32 quotient's rounding)
    assert float(t.abs().max()) <= 448 * (1 + 2.0 ** -23)
    if scale == E8M0:
        top = torch.nn.functional.pad(t.abs(), (0, -k % 128)).view(m, -1, 128).amax(-1)
        if rows == 1:
            assert float(top.min()) > 224 and bool((torch.frexp(q.scale.float()).mantissa == 0.5).all())


def test_cpu_linear_and_swiglu():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(5, 272, generator=g), torch.randn(96, 272, generator=g)
    for scale in (E8M0, F32):
        xq, wq = F8.quantize(x, scale), F8.quantize_weight(w, scale)
        ref = F8._cpu_values(xq).double() @ F8._cpu_values(wq).double().t()
        b, r = torch.randn(96, generator=g), torch.randn(5, 96, generator=g)
        assert torch.allclose(F8.linear(xq, wq, b, r, F32).double(), ref + b.double() + r.double(), atol=1e-4)
        a = ref[:, 48:] * ref[:, :48] * torch.sigmoid(ref[:, :48])
        assert torch.allclose(F8.linear_swiglu(xq, wq, F32).double(), a, atol=1e-3)
        q = F8.linear_swiglu(xq, wq, E4M3)
        assert (F8._cpu_values(q).double() - a).norm() < 0.04 * a.norm()
        h, total = F8.rms_norm(x, torch.ones(272), 1e-5, residual=x, scale_dtype=scale)
        assert torch.equal(total, 2 * x) and h.shape == (5, 272)


def test_refusals():
    x, w = F8.quantize(torch.randn(4, 64)), F8.quantize_weight(torch.randn(32, 64))
    wf = F8.quantize_weight(torch.randn(32, 64), F32)
    for exc, f in [
        (ValueError, lambda: F8.quantize(torch.randn(4, 24))), (ValueError, lambda: F8.quantize(torch.randn(4, 0))), (TypeError, lambda: F8.quantize(torch.randn(64))),
        (TypeError, lambda: F8.quantize(torch.randn(4, 64).double())), (TypeError, lambda: F8.quantize(torch.randn(4, 64), torch.bfloat16)),
        (TypeError, lambda: F8.quantize(torch.zeros(4, 64).to(E4M3))),
        (TypeError, lambda: F8.Fp8(torch.zeros(4, 64), x.scale)), (ValueError, lambda: F8.Fp8(x.data, x.scale[:2])), (ValueError, lambda: F8.Fp8(x.data, x.scale, 128)),
        (TypeError, lambda: F8.Fp8(x.data, x.scale, 64)), (ValueError, lambda: w[16:32]), (TypeError, lambda: x[1]),
        (TypeError, lambda: F8.linear(torch.randn(4, 64), w)), (TypeError, lambda: F8.linear(w, w)), (TypeError, lambda: F8.linear(x, x)),
        (TypeError, lambda: F8.linear(x, wf)), (ValueError, lambda: F8.linear(x, F8.quantize_weight(torch.randn(32, 80)))),
        (TypeError, lambda: F8.linear(x, w, out_dtype=E4M3)), (TypeError, lambda: F8.linear(x, w, bias=torch.zeros(32))),
        (TypeError, lambda: F8.linear(x, w, bias=torch.zeros(31).bfloat16())), (TypeError, lambda: F8.linear(x, w, residual=torch.zeros(4, 31).bfloat16())),
        (ValueError, lambda: F8.linear_swiglu(x, F8.quantize_weight(torch.randn(40, 64)))), (TypeError, lambda: F8.linear_swiglu(x, w, torch.int8)),
        (TypeError, lambda: F8.rms_norm(torch.randn(4, 64), torch.ones(63), 1e-5)), (TypeError, lambda: F8.rms_norm(torch.randn(4, 64), torch.ones(64).half(), 1e-5)),
        (TypeError, lambda: F8.rms_norm(torch.randn(4, 64), torch.ones(64), 1e-5, residual=torch.randn(4, 64).half())),
        (TypeError, lambda: F8.dequantize(x, torch.float64)),
    ]:
        with pytest.raises(exc):
            f()
    assert F8.linear(x[1:3], w).shape == (2, 32) and F8.linear(x[2:2], w).shape == (0, 32)


def _args(**kw):
    from dynam3d_amd.fp8_ops import _GemmArgs
    p = 1 << 20                                                           # (never read: every call below is refused before a launch)
    d = dict(x=p, sx=p, w=p, sw=p, out=p, out_scale=p, workspace=p, workspace_bytes=1 << 40, ldx=256, ldsx=2, ldw=256, ldsw=2, ldr=64, ldo=64, ldos=1,
             M=4, N=64, K=256, scale_kind=0, out_type=0, swiglu=0)
    d.update(kw)
    return _GemmArgs(**d)


def test_c_entry_points_refuse():
    lib = _lib.load()
    for kw in (dict(M=-1), dict(K=24), dict(K=0), dict(scale_kind=2), dict(out_type=4), dict(out_type=3), dict(x=None), dict(w=None), dict(sx=None), dict(out=None),
               dict(x=(1 << 20) + 8), dict(ldx=250), dict(ldw=1 << 25), dict(ldsx=1 << 20), dict(ldsw=1 << 29), dict(swiglu=1, N=40), dict(swiglu=1, bias=1 << 20), dict(swiglu=1, residual=1 << 20),
               dict(swiglu=1, out_type=3, out_scale=None), dict(swiglu=1, out_type=3, ldo=40), dict(swiglu=1, N=1 << 12, ldw=1 << 21)):
        a = _args(**kw)
        assert lib.d3d_fp8_gemm(C.byref(a)) == -1, kw
        assert b"d3d_fp8_gemm" in lib.d3d_last_error()
    assert lib.d3d_fp8_gemm(None) == -1
    need = F8._workspace_bytes(4, 64, 4096, 0, 0, 0)
    if need:
        a = _args(K=4096, ldx=4096, ldw=4096, ldsx=32, ldsw=32, workspace_bytes=need - 1)
        assert lib.d3d_fp8_gemm(C.byref(a)) == -1
    a = _args(M=0)
    assert lib.d3d_fp8_gemm(C.byref(a)) == 0
    p = 1 << 20
    assert lib.d3d_fp8_quantize(p, p, p, 4, 24, 24, 24, 1, 0, 0, None) == -1
    assert lib.d3d_fp8_quantize(p + 2, p, p, 4, 32, 32, 32, 1, 0, 0, None) == -1
    assert lib.d3d_fp8_quantize(p, p, p, 4, 32, 32, 32, 1, 3, 0, None) == -1
    assert lib.d3d_fp8_quantize_weight(p, None, p, 4, 32, 32, 32, 1, 0, 0, None) == -1
    assert lib.d3d_fp8_dequantize(p, p, p, 4, 32, 32, 1, 32, 64, 0, 0, None) == -1
    assert lib.d3d_fp8_rms_norm(p, None, p, None, p, p, 4, 16400, 16400, 0, 0, 16400, 1, 1e-5, 0, 0, None) == -1
    assert lib.d3d_fp8_rms_norm(p, p, p, None, p, p, 4, 32, 32, 32, 32, 32, 1, 1e-5, 0, 0, None) == -1


def test_c_entry_points_refuse_more_than_a_launch_holds():
    lib, p, many = _lib.load(), 1 << 20, (1 << 31) - 1
    assert lib.d3d_fp8_quantize(p, p, p, many, 4096, 4096, 4096, 32, 0, 0, None) == -1
    assert lib.d3d_fp8_dequantize(p, p, p, many, 4096, 4096, 32, 4096, 1, 0, 0, None) == -1
    assert lib.d3d_fp8_rms_norm(p, None, p, None, p, p, many, 4096, 4096, 0, 0, 4096, 32, 1e-5, 0, 0, None) == -1
    a = _args(M=many, N=1 << 20, ldo=1 << 20, ldr=0)
    assert lib.d3d_fp8_gemm(C.byref(a)) == -1


def test_decode_token_refusals():
    from dynam3d_amd.hip_dense import Phi3DecodeArgs, Phi3DecodeFp8
    lib = _lib.load()
    good = dict(n_layers=1, rows=2, hidden=192, heads=2, head_dim=96, mlp=256, vocab=64, dtype=0)
    for kw in (dict(head_dim=64), dict(rows=17), dict(mlp=264), dict(dtype=2)):
        a, f = Phi3DecodeArgs(**{**good, **kw}), Phi3DecodeFp8()
        assert lib.d3d_phi3_decode_token_fp8(C.byref(a), C.byref(f)) == -1, kw
    a, f = Phi3DecodeArgs(**{**good, "rows": 0}), Phi3DecodeFp8()
    assert lib.d3d_phi3_decode_token_fp8(C.byref(a), C.byref(f)) == 0
