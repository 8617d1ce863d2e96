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
