"""What the 8-bit linear operators refuse because of its size or place: sizes past 32 bits, launches past the grid, workspaces, strides.  No GPU: every call is
refused before a launch."""
import ctypes as C

import pytest
import torch

from dynam3d_amd import _lib
from dynam3d_amd import fp8_ops as F8

E8M0, F32, E4M3 = torch.float8_e8m0fnu, torch.float32, torch.float8_e4m3fn
P = 1 << 20                                                    # an address that is never read


def gemm_args(**kw):
    d = dict(x=P, sx=P, w=P, sw=P, out=P, out_scale=P, workspace=P, workspace_bytes=1 << 40, ldx=256, ldsx=2, ldw=256, ldsw=2, ldr=64, ldo=64, ldos=1,
             M=4, N=64, K=256, scale_kind=0, out_type=0, swiglu=0)
    d.update(kw)
    return F8._GemmArgs(**d)


def refused(message=b"d3d_fp8_gemm", **kw):
    lib = _lib.load()
    a = gemm_args(**kw)
    return lib.d3d_fp8_gemm(C.byref(a)) == -1 and message in lib.d3d_last_error()


@pytest.mark.parametrize("rows", [2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_rows_past_32_bits_are_refused(rows):
    """(one row, repeated: no memory)"""
    x = torch.zeros(1, 16).expand(rows, 16)
    x8 = F8.Fp8(torch.zeros(1, 16).to(E4M3).expand(rows, 16), torch.ones(1, 1).expand(rows, 1))
    w8 = F8.Fp8(torch.zeros(1, 16).to(E4M3).expand(rows, 16), torch.ones(1, 1).expand(rows // 128 + (rows % 128 > 0), 1), 128)
    one, w = F8.quantize(torch.zeros(1, 16), F32), F8.quantize_weight(torch.zeros(32, 16), F32)
    for f in (lambda: F8.quantize(x), lambda: F8.quantize_weight(x), lambda: F8.rms_norm(x, torch.ones(16), 1e-5), lambda: F8.dequantize(x8), lambda: F8.dequantize(w8),
              lambda: F8.linear(x8, w), lambda: F8.linear(one, w8), lambda: F8.linear_swiglu(x8, w), lambda: F8.linear_swiglu(one, w8),
              lambda: F8.workspace_bytes(rows, 64, 256), lambda: F8.workspace_bytes(64, rows, 256)):
        with pytest.raises(ValueError, match="at most 2\\^31 - 1"):
            f()


def test_sizes_near_2_to_the_31():
    lib, most, k = _lib.load(), 2 ** 31 - 1, 2 ** 31 - 16
    assert lib.d3d_fp8_quantize(P, P, P, most, k, k, k, 1 << 24, 0, 0, None) == -1
    assert lib.d3d_fp8_quantize_weight(P, P, P, most, 64, 64, 64, 1, 0, 0, None) == -1
    assert lib.d3d_fp8_quantize_weight(P, P, P, most - 126, 64, 64, 64, 1, 0, 0, None) == -1
    for kw in (dict(M=most, scale_kind=1, N=8, ldo=8), dict(M=most - 126, out_type=2, N=8, ldo=8), dict(M=most, N=most, ldo=most), dict(M=most - 100, N=1 << 20, ldo=1 << 20),
               dict(M=1, N=most, K=4096, ldx=4096, ldw=0, ldsw=0), dict(M=32, N=k - 16, ldw=0, ldsw=0, swiglu=1, out_type=3, ldo=1 << 30, ldos=1 << 23)):
        assert refused(b"d3d_fp8_gemm: too many", **kw), (kw, lib.d3d_last_error())
    for kw in (dict(K=1 << 24), dict(K=k)):
        assert refused(b"d3d_fp8_gemm: K of", ldx=0, ldw=0, ldsx=0, ldsw=0, **kw)
    # 2^31 - 1 rows are whole tiles of 128 and of 256: neither kernel asks for scratch, nor for a number of tiles that wrapped
    for m in (most, most - 120, most - 254):
        for out, kind in ((0, 0), (0, 1), (2, 0)):
            assert F8._workspace_bytes(m, 8, 256, 0, out, kind) == 0
    assert F8._workspace_bytes(32, 2 ** 30, 256, 1, 3, 0) == 32 * 2 ** 30 * 4


def test_strides_that_the_epilogues_do_not_take():
    """Large products address residual and result rows by unsigned 32-bit offsets from a tile's first row."""
    large = dict(M=4096, N=8192, ldo=8192, ldr=8192, residual=P)
    for kw in (dict(ldo=-64), dict(ldo=63), dict(ldo=0), dict(ldr=-64, residual=P), dict(large, ldr=-8192), dict(large, ldo=-8192), dict(large, ldo=8184),
               dict(swiglu=1, out_type=3, ldo=16), dict(swiglu=1, N=512, out_type=3, ldo=256, ldos=1), dict(swiglu=1, N=512, out_type=3, ldo=256, ldos=-2)):
        assert refused(b"rows", **kw), (kw, _lib.load().d3d_last_error())


def test_workspaces_that_are_too_small_missing_or_off_16_bytes():
    lib = _lib.load()
    lds = dict(ldx=4096, ldw=4096, ldsx=32, ldsw=32, K=4096)
    for kw, need in ((dict(lds, M=100), 100 * 64 * 4 * 8), (dict(lds, M=100, out_type=2), 100 * 64 * 4 * 8), (dict(lds, M=100, scale_kind=1), 100 * 64 * 4 * 8),
                     (dict(lds, M=4, swiglu=1, out_type=3, ldo=32), 4 * 64 * 4)):
        assert F8._workspace_bytes(kw["M"], 64, 4096, kw.get("swiglu", 0), kw.get("out_type", 0), kw.get("scale_kind", 0)) == need, kw
        for bad in (dict(workspace_bytes=need - 1), dict(workspace_bytes=0), dict(workspace=None), dict(workspace=P + 8)):
            assert refused(b"d3d_fp8_gemm: workspace", **kw, **bad), (kw, bad, lib.d3d_last_error())
    assert F8.workspace_bytes(4, 64, 4096) == 0 and F8.workspace_bytes(100, 64, 4096) == 100 * 64 * 4 * 8
