"""The 8-bit operators of the language model's linear layers, as cases that can be timed and compared.

The plain forms below are the operators' definitions in elementary torch operations (float32); with `own` true the same inputs go through
`dynam3d_amd.fp8_ops`.  8-bit results are returned as the values they stand for (bfloat16 holds an e4m3 value times a power of two exactly).

Sizes: Phi-3-mini's linears (hidden 3072, fused qkv 9216, MLP 8192) and the ViT widths (1024, 4096) of this repository's configurations;
rows: 1 and 8 = one decode token of one / eight sequences, 823 = one environment's prompt, 6568 = the packed prompts of eight environments
(all odd or ragged against the 128-wide groups and tiles, as they are in use).
"""
import math

import torch

own = False

G = 128                        # elements per scale along K (weights: 128 x 128)
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -126

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SCALES = {"e8m0": torch.float8_e8m0fnu, "fp32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # RMS norm + residual + quantisation: in front of the qkv and gate_up products of every layer
        dict(name="norm_token", op="rms_norm", m=1, k=3072, dtype="bf16", residual=True, scale="e8m0"),            # one decode token
        dict(name="norm_prompts", op="rms_norm", m=6568, k=3072, dtype="bf16", residual=True, scale="e8m0"),       # eight prompts
        dict(name="norm_fp16_odd", op="rms_norm", m=4617, k=4112, dtype="fp16", residual=False, scale="fp32"),     # ragged last group
        # quantisation of an activation: the attention's output in front of o_proj
        dict(name="quant_token", op="quantize", m=8, k=3072, dtype="bf16", scale="e8m0"),
        dict(name="quant_prompts", op="quantize", m=6568, k=3072, dtype="bf16", scale="e8m0"),
        # the products
        dict(name="qkv_token", op="linear", m=1, n=9216, k=3072, dtype="bf16", bias=False, residual=False, scale="e8m0"),      # decode, one sequence
        dict(name="down_token8", op="linear", m=8, n=3072, k=8192, dtype="bf16", bias=False, residual=True, scale="e8m0"),     # decode, eight
        dict(name="odd_bias_fp16", op="linear", m=77, n=1003, k=1040, dtype="fp16", bias=True, residual=False, scale="fp32"),  # ragged everywhere
        dict(name="qkv_prompt", op="linear", m=823, n=9216, k=3072, dtype="bf16", bias=False, residual=False, scale="fp32"),   # prefill of one
        dict(name="down_prompts", op="linear", m=6568, n=3072, k=8192, dtype="bf16", bias=False, residual=True, scale="e8m0"),  # prefill of eight
        # gate_up product + SwiGLU + re-quantisation for the down product
        dict(name="mlp_token8", op="linear_swiglu", m=8, n=8192, k=3072, scale="e8m0"),
        dict(name="mlp_prompts", op="linear_swiglu", m=6568, n=8192, k=3072, scale="e8m0"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rms_norm", "quantize", "linear", "linear", "linear", "linear_swiglu"])
    scale = rng.choice(["e8m0", "e8m0", "fp32"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    k = 16 * _log(rng, 8, 512)                                       # 128 .. 8192, ragged last groups among them
    if op in ("rms_norm", "quantize"):
        m = _log(rng, 1, min(16384, (6568 * 3072 * 2 // (4 if dtype == "fp32" else 2)) // k))
        c = dict(op=op, m=m, k=k, dtype=dtype, scale=scale)
        if op == "rms_norm":
            c["residual"] = rng.random() < 0.6
        return c
    n = _log(rng, 64, 16384) if op == "linear" else 16 * _log(rng, 8, 512)
    most = 6568 * 8192 * 2 * 3072 // (n * k * (1 if op == "linear" else 2))
    m = _log(rng, 1, max(1, min(8192, most)))
    c = dict(op=op, m=m, n=n, k=k, scale=scale)
    if op == "linear":
        c.update(dtype=dtype, bias=rng.random() < 0.3, residual=rng.random() < 0.4)
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _activation(g, m, k):
    """Rows of different size, a few large channels: what a transformer's residual stream looks like."""
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))
    big = torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")
    x[:, big] *= 20.0
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, m, k = case, case["m"], case["k"]
    if c["op"] in ("rms_norm", "quantize"):
        dt = DTYPES[c["dtype"]]
        s = {"case": c, "x": _activation(g, m, k).to(dt)}
        if c["op"] == "rms_norm":
            s["w"] = 1.0 + 0.2 * torch.randn(k, generator=g, device="cuda")
            if c["residual"]:
                s["residual"] = _activation(g, m, k).to(dt)
        return s
    rows = c["n"] * (2 if c["op"] == "linear_swiglu" else 1)
    xq, xs = _quantize(_activation(g, m, k), c["scale"])
    wq, ws = _quantize_weight(torch.randn(rows, k, generator=g, device="cuda") * (1.5 / math.sqrt(k)), c["scale"])
    s = {"case": c, "xq": xq.to(torch.float8_e4m3fn), "xs": xs.to(SCALES[c["scale"]]), "wq": wq.to(torch.float8_e4m3fn), "ws": ws.to(SCALES[c["scale"]])}
    if c.get("bias"):
        s["bias"] = torch.randn(rows, generator=g, device="cuda").to(DTYPES[c["dtype"]])
    if c.get("residual"):
        s["residual"] = torch.randn(m, rows, generator=g, device="cuda").to(DTYPES[c["dtype"]])
    return s


# ---- the plain forms (float32) -------------------------------------------------------------------------------------------------------
def _scale_of(amax, kind):
    if kind == "fp32":
        return torch.clamp(amax / E4M3_MAX, min=LEAST_SCALE)
    mant, e = torch.frexp(amax)                                       # amax = mant 2^e, mant in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(mant <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    return ((e + 127) << 23).view(torch.float32)                      # (exact: ldexp multiplies by a rounded pow)


def _e4m3(v):
    """Round to the nearest e4m3 value (ties to even); |v| <= 448."""
    return v.to(torch.float8_e4m3fn).to(v.dtype)


def _groups(x):
    pad = -x.shape[-1] % G
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], -1)
    return x.view(*x.shape[:-1], -1, G)


def _quantize(x, kind):
    """x (M, K) -> e4m3 values (M, K) and scales (M, KB), both in x's type."""
    xg = _groups(x)
    s = _scale_of(xg.abs().amax(-1), kind)
    q = _e4m3(xg / s[..., None])
    return q.flatten(-2)[..., :x.shape[-1]], s


def _quantize_weight(w, kind):
    n, k = w.shape
    wg = _groups(w)                                                   # (N, KB, 128)
    pad = -n % G
    a = wg.abs().amax(-1)
    a = torch.cat([a, a.new_zeros(pad, a.shape[1])], 0).view(-1, G, a.shape[1]).amax(1)
    s = _scale_of(a, kind)                                            # (NB, KB)
    q = _e4m3(wg / s.repeat_interleave(G, 0)[:n, :, None])
    return q.flatten(-2)[:, :k], s


def _values(q, s, k):
    return (_groups(q) * s[..., None]).flatten(-2)[..., :k]


def _dequantized_operands(s, dtype):
    k, n = s["xq"].shape[1], s["wq"].shape[0]
    x = _values(s["xq"].to(dtype), s["xs"].to(dtype), k)
    w = _values(s["wq"].to(dtype), s["ws"].to(dtype).repeat_interleave(G, 0)[:n], k)
    return x, w


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        x = s["x"].float()
        return _values(*_quantize(x, c["scale"]), c["k"]).to(torch.bfloat16)
    if c["op"] == "rms_norm":
        h = s["x"].float()
        if c["residual"]:
            total = (h + s["residual"].float()).to(s["x"].dtype)
            h = total.float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5) * s["w"]
        y = _values(*_quantize(y, c["scale"]), c["k"]).to(torch.bfloat16)
        return (y, total) if c["residual"] else y
    x, w = _dequantized_operands(s, torch.float32)
    y = x @ w.t()
    if c["op"] == "linear":
        if c["bias"]:
            y = y + s["bias"].float()
        if c["residual"]:
            y = y + s["residual"].float()
        return y.to(DTYPES[c["dtype"]])
    gate, up = y[:, :c["n"]], y[:, c["n"]:]
    a = up * (gate / (1.0 + torch.exp(-gate)))
    return _values(*_quantize(a, c["scale"]), c["n"]).to(torch.bfloat16)


# ---- the framework's operators --------------------------------------------------------------------------------------------------------
def _own(s):
    from dynam3d_amd import fp8_ops as F8
    c = s["case"]
    if c["op"] == "quantize":
        return F8.dequantize(F8.quantize(s["x"], SCALES[c["scale"]]))
    if c["op"] == "rms_norm":
        if c["residual"]:
            q, total = F8.rms_norm(s["x"], s["w"], 1e-5, residual=s["residual"], scale_dtype=SCALES[c["scale"]])
            return F8.dequantize(q), total
        return F8.dequantize(F8.rms_norm(s["x"], s["w"], 1e-5, scale_dtype=SCALES[c["scale"]]))
    x, w = F8.Fp8(s["xq"], s["xs"]), F8.Fp8(s["wq"], s["ws"], rows=G)
    if c["op"] == "linear":
        return F8.linear(x, w, bias=s.get("bias"), residual=s.get("residual"), out_dtype=DTYPES[c["dtype"]])
    return F8.dequantize(F8.linear_swiglu(x, w, out_dtype=torch.float8_e4m3fn))


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without, and its result in 64 bits ---------------------------------------------------------------------------
def work(case):
    m, k = case["m"], case["k"]
    sb = 1 if case["scale"] == "e8m0" else 4
    kb = -(-k // G)
    if case["op"] == "quantize":
        return {"bytes": m * k * (DTYPES[case["dtype"]].itemsize + 1) + m * kb * sb, "flops": 3.0 * m * k}
    if case["op"] == "rms_norm":
        e = DTYPES[case["dtype"]].itemsize * (3 if case["residual"] else 1)
        return {"bytes": m * k * (e + 1) + m * kb * sb + 4 * k, "flops": 7.0 * m * k}
    n = case["n"]
    if case["op"] == "linear":
        e = DTYPES[case["dtype"]].itemsize
        b = m * k + n * k + (m + -(-n // G)) * kb * sb + m * n * e * (2 if case["residual"] else 1) + (n * e if case["bias"] else 0)
        return {"bytes": b, "flops": 2.0 * m * n * k}
    return {"bytes": m * k + 2 * n * k + (m + -(-2 * n // G)) * kb * sb + m * n + m * -(-n // G) * sb, "flops": 4.0 * m * n * k}


def _two_to(e):
    """2^e in 64 bits, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_quantized(y, kind):
    """The quantiser's definition in 64 bits: nearest multiple of the e4m3 step, group by group."""
    m, k = y.shape
    out = torch.empty_like(y)
    for o in range(0, k, G):
        v = y[:, o:o + G]
        a = v.abs().amax(1, keepdim=True)
        if kind == "fp32":
            s = (a / 448.0).float().double().clamp(min=2.0 ** -126)
        else:
            e = torch.ceil(torch.log2(a.clamp(min=2.0 ** -150) / 448.0))
            e = torch.where(448.0 * _two_to(e - 1) >= a, e - 1, e)                            # (log2 rounds: settle the border exactly)
            e = torch.where(448.0 * _two_to(e) < a, e + 1, e)
            s = _two_to(e.clamp(min=-126.0))
        t = v / s
        step = _two_to(torch.frexp(t.abs().clamp(min=2.0 ** -6)).exponent - 4)                # 8 steps a binade
        out[:, o:o + G] = torch.round(t / step) * step * s
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "quantize":
        return _exact_quantized(s["x"].to(d), case["scale"])
    if case["op"] == "rms_norm":
        h = s["x"].to(d)
        if case["residual"]:
            total = h + s["residual"].to(d)
            h = total.to(s["x"].dtype).to(d)
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["k"] + 1e-5) * s["w"].to(d)
        y = _exact_quantized(y, case["scale"])
        return (y, total) if case["residual"] else y
    k, rows = s["xq"].shape[1], s["wq"].shape[0]
    at_k, at_n = torch.arange(k, device="cuda") // G, torch.arange(rows, device="cuda") // G
    x = s["xq"].to(d) * s["xs"].to(d)[:, at_k]
    w = s["wq"].to(d) * s["ws"].to(d)[at_n][:, at_k]
    y = torch.mm(x, w.t())
    if case["op"] == "linear":
        for extra in ("bias", "residual"):
            if case[extra]:
                y += s[extra].to(d)
        return y
    a = y[:, case["n"]:] * y[:, :case["n"]] * torch.sigmoid(y[:, :case["n"]])
    return _exact_quantized(a, case["scale"])
