"""Device time of the 8-bit linear operators (dynam3d_amd/fp8_ops.py): 12 calls captured in a graph over operands in turn (more than the caches hold, for the small
products), median of 10 replays, and the floor: bytes at 5.21 TB/s or operations at 2783 TFLOP/s (a 1 GiB copy and the library's per-tensor 8192^3 product on this card; the matrix pipe
alone runs 4.3 PFLOP/s), 2.5 us for an empty launch in a graph.
usage: bench_fp8.py [substring of the case's name]"""
import os
import statistics
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch

from dynam3d_amd import fp8_ops as F8

E8, F32, BF16, E4M3 = F8.E8M0, torch.float32, torch.bfloat16, F8.E4M3
only = sys.argv[1] if len(sys.argv) > 1 else ""
g = torch.Generator(device="cuda").manual_seed(1)
rand = lambda *s: torch.randn(*s, generator=g, device="cuda")


def timed(name, call, nbytes, flops):
    for i in range(3):
        call(i)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(12):
            call(i)
    times = []
    for _ in range(12):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / 12 * 1e3)
    t, floor = statistics.median(times[2:]), max(nbytes / 5.21e6, flops / 2783e6, 2.5)
    print(f"{name:64s} {t:8.1f} us   floor {floor:7.1f}   x {t / floor:4.2f}   {nbytes / t / 1e6:5.2f} TB/s {flops / t / 1e6:6.0f} TFLOP/s", flush=True)


def kind(s):
    return "E8M0" if s == E8 else "float32 scales"


def short(t):
    return {BF16: "bf16", torch.float16: "fp16", F32: "float32", E4M3: "E4M3"}[t]


def copies(nbytes):                                     # 256 MB of cache
    return max(2, min(12, int(600e6 // max(nbytes, 1)) + 1))


def linear(m, n, k, scale=E8, out=BF16, residual=False, exact=False):
    name = f"linear {m} x {n} x {k} {kind(scale)} -> {short(out)}{' + residual' if residual else ''}{' exact' if exact else ''}"
    if only not in name:
        return
    c = copies(m * k + n * k)
    w = [F8.quantize_weight(rand(n, k) / k ** 0.5, scale) for _ in range(c)]
    x = [F8.quantize(rand(m, k), scale) for _ in range(c)]
    r = rand(m, n).to(out) if residual else None
    o = 4 if out == F32 else 2
    timed(name, lambda i: F8.linear(x[i % c], w[i % c], residual=r, out_dtype=out, exact=exact), m * k + n * k + m * n * o * (2 if residual else 1), 2 * m * n * k)


def swiglu(m, i_, k, scale=E8, out=E4M3, exact=False):
    name = f"linear_swiglu {m} x 2*{i_} x {k} {kind(scale)} -> {short(out)}{' exact' if exact else ''}"
    if only not in name:
        return
    c = copies(m * k + 2 * i_ * k)
    w = [F8.quantize_weight(rand(2 * i_, k) / k ** 0.5, scale) for _ in range(c)]
    x = [F8.quantize(rand(m, k), scale) for _ in range(c)]
    timed(name, lambda i: F8.linear_swiglu(x[i % c], w[i % c], out, exact), m * k + 2 * i_ * k + m * i_ * (1 if out == E4M3 else 4 if out == F32 else 2), 4 * m * i_ * k)


def rows(op, m, k, dtype=BF16, scale=E8, residual=False):
    name = f"{op} {m} x {k} {short(dtype)} {kind(scale)}{' + residual' if residual else ''}"
    if only not in name:
        return
    b = 4 if dtype == F32 else 2
    nbytes = m * k * (b + 1 + (2 * b if residual else 0))
    c = copies(m * k * b)
    x = [rand(m, k).to(dtype) for _ in range(c)]
    gain = torch.ones(k, device="cuda")
    if op == "rms_norm":
        r = rand(m, k).to(dtype) if residual else None
        call = lambda i: F8.rms_norm(x[i % c], gain, 1e-5, r, scale)
    elif op == "quantize":
        call = lambda i: F8.quantize(x[i % c], scale)
    elif op == "quantize_weight":
        call = lambda i: F8.quantize_weight(x[i % c], scale)
    else:
        q = [F8.quantize(t, scale) for t in x]
        call = lambda i: F8.dequantize(q[i % c], dtype)
    timed(name, call, nbytes, 6 * m * k)


rows("rms_norm", 1, 3072)
rows("rms_norm", 6568, 3072)
rows("rms_norm", 6568, 3072, residual=True)
rows("rms_norm", 4617, 4112, torch.float16, F32)
rows("quantize", 8, 3072)
rows("quantize", 6568, 3072)
rows("quantize_weight", 16384, 3072)
rows("dequantize", 6568, 3072)
for m in (1, 8):
    for n, k in ((9216, 3072), (3072, 3072), (3072, 8192)):
        linear(m, n, k, residual=n == 3072)
    swiglu(m, 8192, 3072)
linear(8, 3072, 8192, out=F32)
linear(77, 1003, 1040, F32, torch.float16)
for m, n, k in ((64, 9216, 3072), (128, 3072, 8192), (256, 9216, 3072)):
    linear(m, n, k)
for m in (823, 6568):
    for n, k in ((9216, 3072), (3072, 3072), (3072, 8192)):
        linear(m, n, k, residual=n == 3072)
    swiglu(m, 8192, 3072)
    linear(m, 3072, 8192, scale=F32)
    linear(m, 9216, 3072, out=F32)
    linear(m, 9216, 3072, out=F32, scale=F32)
    linear(m, 9216, 3072, exact=True)
    swiglu(m, 8192, 3072, out=BF16)
    swiglu(m, 8192, 3072, scale=F32)
    swiglu(m, 8192, 3072, out=F32)
    swiglu(m, 8192, 3072, exact=True)
linear(823, 9216, 3072, scale=F32)
linear(1024, 3072, 8192)
linear(8192, 8192, 8192)
