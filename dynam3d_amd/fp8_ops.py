"""8-bit linear layers: E4M3 operands in groups of 128 along K with one scale per group, on the matrix cores of gfx950
(csrc/fp8_quant_kernels.hip, csrc/fp8_gemm_kernels.hip).  `Phi3Decoder(quant="fp8")` runs its four linears per layer through them.

    xq        = quantize(x)                       rows: one scale per row and 128 columns
    wq        = quantize_weight(w)                weights: one scale per 128 x 128 block, once per weight
    xq[, h]   = rms_norm(x, w, eps[, residual])   RMSNorm of h = x + residual with a quantised result
    y         = linear(xq, wq[, bias, residual])  y = xq wq^T
    a         = linear_swiglu(xq, wq)             up * silu(gate) over w = [gate rows; up rows], in 16 / 32 bits or quantised again
    x         = dequantize(xq)

Formats: `scale_dtype` = torch.float8_e8m0fnu (default): s = 2^max(-126, ceil(log2(amax / 448))) -- dividing by it is exact and the matrix core
applies it for free --, or torch.float32: s = max(amax / 448, 2^-126).  amax runs over the finite members of a group; q = E4M3(x / s) to
nearest even, and a member that is not finite becomes E4M3's NaN: it poisons its own row of a product, never its neighbours.  A product takes
two operands of the same scale type.

Products.  gfx950's 8-bit matrix instruction aligns 8 neighbouring products to the largest of them and drops what lies 13 bits below it: a sum is off by at most
7 * 2^-13 sum |x w|, ~2^-14 of a result of random signs, before its one rounding -- inside half a step of bf16 (2^-9) and of fp16 (2^-12) unless most of the
sum cancels; a result that is quantised again lands on the other E4M3 neighbour once in ~650 members.  `exact=True` takes the bf16 instruction instead, whose
products of E4M3 values are exact (float32 sums), for 1 to 3 times the time; float32 results, and `Fp8` results of up to 32 rows, where it costs nothing, are
always made so.

On a CUDA tensor every function is a HIP kernel on the current stream of the tensor's device (captured like any other launch) and raises what it does
not take; on a CPU tensor the same expression runs in PyTorch.  Results have no gradient: inference only, like the 16-bit towers."""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch

from . import _lib
from . import hip_dense  # noqa: F401  (registers the d3d_fp8_* signatures)

GROUP = 128
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
E4M3_MAX = 448.0
_LEAST = 2.0 ** -126
_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, E4M3: 3}
_KIND = {E8M0: 0, torch.float32: 1}
_MOST = 2 ** 31 - 1                                    # rows and columns are 32-bit numbers in the C entry points (ctypes would cut longer ones off without a word)


class _GemmArgs(C.Structure):
    """ctypes mirror of `d3d_fp8_gemm_args` (include/dynam3d_hip.h)."""
    _fields_ = ([(n, C.c_void_p) for n in ("x", "sx", "w", "sw", "bias", "residual", "out", "out_scale", "workspace")]
                + [(n, C.c_int64) for n in ("workspace_bytes", "ldx", "ldsx", "ldw", "ldsw", "ldr", "ldo", "ldos")]
                + [(n, C.c_int32) for n in ("M", "N", "K", "scale_kind", "out_type", "swiglu")] + [("stream", C.c_void_p), ("exact", C.c_int32)])


class Fp8:
    """An E4M3 matrix (rows, K) and its scales: `scale` (rows, ceil(K / 128)) with `rows` = 1, (ceil(rows / 128), ceil(K / 128)) with 128."""
    __slots__ = ("data", "scale", "rows")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, rows: int = 1):
        if data.dtype != E4M3 or data.dim() != 2 or scale.dtype not in _KIND or rows not in (1, GROUP):
            raise TypeError("Fp8: data (rows, K) float8_e4m3fn, scale float8_e8m0fnu or float32, rows 1 or 128")
        m, k = data.shape
        if scale.shape != ((m + rows - 1) // rows, (k + GROUP - 1) // GROUP) or scale.device != data.device:
            raise ValueError(f"Fp8: scale {tuple(scale.shape)} on {scale.device} does not fit data {tuple(data.shape)} on {data.device} with one scale per {rows} rows")
        self.data, self.scale, self.rows = data, scale, rows

    @staticmethod
    def _of(data, scale, rows=1):
        """(unchecked: for results made here)"""
        r = object.__new__(Fp8)
        r.data, r.scale, r.rows = data, scale, rows
        return r

    @property
    def shape(self):
        return self.data.shape

    @property
    def device(self):
        return self.data.device

    def __getitem__(self, rows: slice) -> "Fp8":
        """A block of rows (a view).  Weights: the slice has to start on a block of 128."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("Fp8: only a slice of rows")
        a, b, _ = rows.indices(self.data.shape[0])
        if a % self.rows:
            raise ValueError("Fp8: a slice of a weight starts on a multiple of 128 rows")
        b = max(a, b)
        return Fp8(self.data[a:b], self.scale[a // self.rows:(b + self.rows - 1) // self.rows], self.rows)


def _current_device():
    return torch._C._cuda_getDevice()


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """`t` (2-D) itself if its rows are contiguous and start on 16 bytes, else a copy that is and does."""
    if (t.stride(1) == 1 or t.shape[1] <= 1) and (t.stride(0) * t.element_size()) % 16 == 0 and t.data_ptr() % 16 == 0 and t.stride(0) >= t.shape[1]:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _check_sizes(name, *sizes):
    if max(sizes) > _MOST:
        raise ValueError(f"fp8_ops.{name}: {max(sizes)} rows or columns: at most 2^31 - 1")


def _check_input(name, x, scale_dtype):
    if x.dim() != 2 or x.dtype not in _DT or x.dtype == E4M3:
        raise TypeError(f"fp8_ops.{name}: a matrix (rows, K) of bfloat16, float16 or float32, not {tuple(x.shape)} {x.dtype}")
    if scale_dtype not in _KIND:
        raise TypeError(f"fp8_ops.{name}: scale_dtype is float8_e8m0fnu or float32, not {scale_dtype}")
    if x.shape[1] == 0 or x.shape[1] % 16:
        raise ValueError(f"fp8_ops.{name}: K = {x.shape[1]} has to be a positive multiple of 16 (the operand of the product is read in 16-byte pieces)")
    _check_sizes(name, *x.shape)


def _same_device(name, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"fp8_ops.{name}: operands on {first.device} and {t.device}")


# ---- the expressions in PyTorch (CPU tensors; no gradient, like the kernels) ----------------------------------------------------------------------------------------------
def _cpu_scale(amax, scale_dtype):
    if scale_dtype == torch.float32:
        return torch.clamp(amax / E4M3_MAX, min=_LEAST)
    u = amax.float().contiguous().view(torch.int32)
    code = ((u >> 23) - 8 + ((u & 0x7FFFFF) > 0x600000).int()).clamp(min=1)
    return (code << 23).view(torch.float32)


def _cpu_groups(x):
    pad = -x.shape[1] % GROUP
    return torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], (x.shape[1] + pad) // GROUP, GROUP)


@torch.no_grad()
def _cpu_quantize(x, scale_dtype, rows):
    xg = _cpu_groups(x.float())
    a = torch.where(xg.isfinite(), xg.abs(), torch.zeros_like(xg)).amax(-1)
    if rows > 1:
        a = torch.nn.functional.pad(a, (0, 0, 0, -a.shape[0] % rows)).unflatten(0, (-1, rows)).amax(1)
    s = _cpu_scale(a, scale_dtype)
    t = xg / s.repeat_interleave(rows, 0)[:x.shape[0], :, None]
    t = torch.where(xg.isfinite(), t, torch.full_like(t, float("nan")))
    return Fp8(t.flatten(1)[:, :x.shape[1]].to(E4M3).contiguous(), s.to(scale_dtype), rows)


@torch.no_grad()
def _cpu_values(q: Fp8):
    s = q.scale.float().repeat_interleave(q.rows, 0)[:q.data.shape[0]]
    return (_cpu_groups(q.data.float()) * s[:, :, None]).flatten(1)[:, :q.data.shape[1]]


# ---- quantisation ----------------------------------------------------------------------------------------------------------------------------
def _quantize(name, x, scale_dtype, rows):
    _check_input(name, x, scale_dtype)
    if not x.is_cuda:
        return _cpu_quantize(x, scale_dtype, rows)
    if x.get_device() != _current_device():
        with torch.cuda.device(x.device):
            return _quantize(name, x, scale_dtype, rows)
    m, k = x.shape
    x = _rows16(x)
    q = torch.empty((m, k), dtype=E4M3, device=x.device)
    s = torch.empty(((m + rows - 1) // rows, (k + GROUP - 1) // GROUP), dtype=scale_dtype, device=x.device)
    lib = _lib.load()
    _lib.check((lib.d3d_fp8_quantize if rows == 1 else lib.d3d_fp8_quantize_weight)(x.data_ptr(), q.data_ptr(), s.data_ptr(), m, k, x.stride(0), k, s.shape[1],
                                                                                    _DT[x.dtype], _KIND[scale_dtype], _stream()))
    return Fp8._of(q, s, rows)


def quantize(x: torch.Tensor, scale_dtype: torch.dtype = E8M0) -> Fp8:
    """x (rows, K) bf16 / fp16 / float32, K a multiple of 16 -> E4M3 with one scale per row and group of 128 columns."""
    return _quantize("quantize", x, scale_dtype, 1)


def quantize_weight(w: torch.Tensor, scale_dtype: torch.dtype = E8M0) -> Fp8:
    """w (out, in) -> E4M3 with one scale per 128 x 128 block: what `linear` and `linear_swiglu` take, made once per weight."""
    return _quantize("quantize_weight", w, scale_dtype, GROUP)


def dequantize(q: Fp8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values q.data * q.scale, rounded once to `dtype` (exact in bf16 for power-of-two scales)."""
    if dtype not in _DT or dtype == E4M3:
        raise TypeError(f"fp8_ops.dequantize: to bfloat16, float16 or float32, not {dtype}")
    _check_sizes("dequantize", *q.shape)
    if not q.data.is_cuda:
        return _cpu_values(q).to(dtype)
    if q.shape[1] % 16:
        raise ValueError(f"fp8_ops.dequantize: K = {q.shape[1]} has to be a multiple of 16")
    if q.data.get_device() != _current_device():
        with torch.cuda.device(q.device):
            return dequantize(q, dtype)
    m, k = q.shape
    d, s = _rows16(q.data), _unit_rows(q.scale)
    x = torch.empty((m, k), dtype=dtype, device=d.device)
    _lib.check(_lib.load().d3d_fp8_dequantize(d.data_ptr(), s.data_ptr(), x.data_ptr(), m, k, d.stride(0), s.stride(0), k, q.rows, _DT[dtype],
                                              _KIND[s.dtype], _stream()))
    return x


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None, scale_dtype: torch.dtype = E8M0):
    """quantise(h / sqrt(mean(h^2) + eps) * w) for the rows of h = x, or of h = x + residual rounded to x's type; float32 inside, one rounding,
    to E4M3.  x (rows, D), D a multiple of 16 up to 16384; w (D) float32.  -> Fp8, with a residual (Fp8, h): h is the next residual stream."""
    _check_input("rms_norm", x, scale_dtype)
    m, d = x.shape
    if w.shape != (d,) or w.dtype != torch.float32:
        raise TypeError(f"fp8_ops.rms_norm: w ({d},) float32, not {tuple(w.shape)} {w.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise TypeError(f"fp8_ops.rms_norm: residual {tuple(residual.shape)} {residual.dtype} beside x {tuple(x.shape)} {x.dtype}")
    _same_device("rms_norm", x, w, residual)
    if not x.is_cuda:
        with torch.no_grad():
            h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
            hf = h.float()
            q = _cpu_quantize(hf / torch.sqrt((hf * hf).mean(-1, keepdim=True) + eps) * w, scale_dtype, 1)
        return q if residual is None else (q, h)
    if d > 16384:
        raise ValueError(f"fp8_ops.rms_norm: rows of {d} columns: at most 16384")
    if x.get_device() != _current_device():
        with torch.cuda.device(x.device):
            return rms_norm(x, w, eps, residual, scale_dtype)
    x = _rows16(x)
    w = w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)
    q = torch.empty((m, d), dtype=E4M3, device=x.device)
    s = torch.empty((m, (d + GROUP - 1) // GROUP), dtype=scale_dtype, device=x.device)
    h, hp, rp, ldr = None, None, None, 0
    if residual is not None:
        residual = _rows16(residual)
        h = torch.empty((m, d), dtype=x.dtype, device=x.device)
        hp, rp, ldr = h.data_ptr(), residual.data_ptr(), residual.stride(0)
    _lib.check(_lib.load().d3d_fp8_rms_norm(x.data_ptr(), rp, w.data_ptr(), hp, q.data_ptr(), s.data_ptr(), m, d, x.stride(0), ldr, d, d, s.shape[1],
                                            float(eps), _DT[x.dtype], _KIND[scale_dtype], _stream()))
    q = Fp8._of(q, s)
    return q if residual is None else (q, h)


# ---- products --------------------------------------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(m, n, k, swiglu, out_type, kind):
    """(a function of the sizes and types alone)"""
    fn = _lib.load().d3d_fp8_gemm_workspace
    fn.restype = C.c_int64
    return fn(m, n, k, swiglu, out_type, kind)


def workspace_bytes(m: int, n: int, k: int, swiglu: bool = False, out_dtype: torch.dtype = torch.bfloat16, scale_dtype: torch.dtype = E8M0) -> int:
    """Scratch that a C caller of `d3d_fp8_gemm` has to bring for a product of x (m, k) with w (n, k)."""
    _check_sizes("workspace_bytes", m, n, k)
    return _workspace_bytes(m, n, k, int(swiglu), _DT[out_dtype], _KIND[scale_dtype])


def _gemm(name, x: Fp8, w: Fp8, bias, residual, out_dtype, swiglu, exact):
    m, k = x.data.shape
    n = w.data.shape[0]
    xd, wd, sx, sw = _rows16(x.data), _rows16(w.data), _unit_rows(x.scale), _unit_rows(w.scale)
    dev = xd.device
    cols = n // 2 if swiglu else n
    out = torch.empty((m, cols), dtype=out_dtype, device=dev)
    out_scale, osp, ldos = None, None, 0
    if out_dtype == E4M3:
        ldos = (cols + GROUP - 1) // GROUP
        out_scale = torch.empty((m, ldos), dtype=sx.dtype, device=dev)
        osp = out_scale.data_ptr()
    nbytes = _workspace_bytes(m, n, k, swiglu, _DT[out_dtype], _KIND[sx.dtype])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None      # (stream-ordered: torch's allocator, or the capturing graph's pool)
    bp, rp, ldr = None, None, 0
    if bias is not None:
        bias = bias.contiguous()
        bp = bias.data_ptr()
    if residual is not None:
        residual = _unit_rows(residual)
        rp, ldr = residual.data_ptr(), residual.stride(0)
    a = _GemmArgs(xd.data_ptr(), sx.data_ptr(), wd.data_ptr(), sw.data_ptr(), bp, rp, out.data_ptr(), osp, ws.data_ptr() if nbytes else None, nbytes,
                  xd.stride(0), sx.stride(0), wd.stride(0), sw.stride(0), ldr, cols, ldos, m, n, k, _KIND[sx.dtype], _DT[out_dtype], swiglu, _stream(), exact)
    _lib.check(_lib.load().d3d_fp8_gemm(C.byref(a)))
    return out if out_scale is None else Fp8._of(out, out_scale)


def _check_operands(name, x, w):
    if not isinstance(x, Fp8) or not isinstance(w, Fp8) or x.rows != 1 or w.rows != GROUP:
        raise TypeError(f"fp8_ops.{name}: x from quantize() / rms_norm() (one scale per row), w from quantize_weight() (one per 128 x 128 block)")
    if x.data.shape[1] != w.data.shape[1] or x.data.shape[1] == 0 or x.data.shape[1] % 16:
        raise ValueError(f"fp8_ops.{name}: x {tuple(x.shape)} and w {tuple(w.shape)}: the same K, a positive multiple of 16")
    _check_sizes(name, *x.shape, *w.shape)
    if x.scale.dtype != w.scale.dtype:
        raise TypeError(f"fp8_ops.{name}: scales of x {x.scale.dtype} and of w {w.scale.dtype}: one type for both")
    if x.data.device != w.data.device:
        raise ValueError(f"fp8_ops.{name}: operands on {x.device} and {w.device}")


def linear(x: Fp8, w: Fp8, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           out_dtype: torch.dtype = torch.bfloat16, exact: bool = False) -> torch.Tensor:
    """x w^T [+ bias] [+ residual]: x (M, K), w (N, K), float32 sums, rounded once to `out_dtype` (bf16, fp16, float32 -- the type of bias (N,) and
    residual (M, N) too).  Any M and N, one row included; K a multiple of 16.  A 16-bit result comes from the 8-bit matrix instruction (see the
    module), a float32 one, or any with `exact`, from exact products.  Large products are fastest with N a multiple of 8 and residual rows that start on
    16 bytes (6568 x 9216 x 3072: 194 us, 395 where they do not)."""
    _check_operands("linear", x, w)
    m, n = x.data.shape[0], w.data.shape[0]
    if out_dtype not in _DT or out_dtype == E4M3:
        raise TypeError(f"fp8_ops.linear: out_dtype is bfloat16, float16 or float32, not {out_dtype}")
    if bias is not None and (bias.shape != (n,) or bias.dtype != out_dtype):
        raise TypeError(f"fp8_ops.linear: bias ({n},) {out_dtype}, not {tuple(bias.shape)} {bias.dtype}")
    if residual is not None and (residual.shape != (m, n) or residual.dtype != out_dtype):
        raise TypeError(f"fp8_ops.linear: residual ({m}, {n}) {out_dtype}, not {tuple(residual.shape)} {residual.dtype}")
    _same_device("linear", x.data, bias, residual)
    if not x.data.is_cuda:
        with torch.no_grad():
            y = _cpu_values(x) @ _cpu_values(w).t()
            for e in (bias, residual):
                y = y if e is None else y + e.float()
            return y.to(out_dtype)
    if x.data.get_device() != _current_device():
        with torch.cuda.device(x.device):
            return _gemm("linear", x, w, bias, residual, out_dtype, 0, bool(exact))
    return _gemm("linear", x, w, bias, residual, out_dtype, 0, bool(exact))


def linear_swiglu(x: Fp8, w: Fp8, out_dtype: torch.dtype = torch.bfloat16, exact: bool = False):
    """up * silu(gate) of x w^T, w = [gate (I rows); up (I rows)] as HF's `gate_up_proj` has them, I a multiple of 16; float32 sums, rounded once:
    to bf16 / fp16 / float32, or with out_dtype=torch.float8_e4m3fn to an `Fp8` (scales of the operands' type) for the product that follows.  A float32
    result, an `Fp8` of up to 32 rows, or any with `exact`, comes from exact products, the others from the 8-bit matrix instruction (see the module)."""
    _check_operands("linear_swiglu", x, w)
    n = w.data.shape[0]
    if out_dtype not in _DT:
        raise TypeError(f"fp8_ops.linear_swiglu: out_dtype is bfloat16, float16, float32 or float8_e4m3fn, not {out_dtype}")
    if n % 32:
        raise ValueError(f"fp8_ops.linear_swiglu: {n} rows of w: twice a multiple of 16 are wanted")
    if not x.data.is_cuda:
        g, u = (_cpu_values(x) @ _cpu_values(w).t()).chunk(2, -1)
        y = u * (g / (1.0 + torch.exp(-g)))
        return _cpu_quantize(y, x.scale.dtype, 1) if out_dtype == E4M3 else y.to(out_dtype)
    if x.data.get_device() != _current_device():
        with torch.cuda.device(x.device):
            return _gemm("linear_swiglu", x, w, None, None, out_dtype, 1, bool(exact))
    return _gemm("linear_swiglu", x, w, None, None, out_dtype, 1, bool(exact))
