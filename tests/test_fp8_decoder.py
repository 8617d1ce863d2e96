"""`Phi3Decoder(quant="fp8")`: RMSNorm, products, SwiGLU and quantisation of `fp8_ops` together, as the language model uses them."""
import numpy as np
import pytest
import torch

from dynam3d_amd import fp8_ops as F8
from dynam3d_amd.towers import LlavaModel, Phi3Config, Phi3Decoder, VitConfig, llava_vision_param_spec, phi3_param_spec
from dynam3d_amd.weights import synth_state_dict
from oracle import towers_ref as TR

CFG = Phi3Config(vocab=512, hidden=384, layers=2, heads=4, kv_heads=4, mlp=528)            # head_dim 96; mlp ends inside a group of 128
LENS = [37, 300, 129, 64]
# 2-norms, relative.  E4M3 keeps 4 bits: errors spread over +- 2^-4 of the power of two below a value, rms 2^-4 / sqrt(3) * 0.72 (mean of 2^e / |x|) = 2.6 % of it.
# A product of two such operands: 3.7 %; eight products in a row that all went into the result unweakened: sqrt(8) * 3.7 % = 10.4 %.
QUANT_ERROR = 8 ** 0.5 * 2 ** 0.5 * 0.026
# Two runs that differ by 16-bit roundings: E (Q(x + d) - Q(x))^2 = step * |d| for d below the step, so a difference of 2^-9 in front of a quantisation is
# sqrt(0.09 * 2^-9) = 1.3 % behind it, 3.4 % behind the next, and grows until both runs round independently: sqrt(2) * 2.6 % per activation operand, of which the
# stack has eight -- the same bound.  (Weights are rounded alike in both.)
RUN_ERROR = QUANT_ERROR


def weights():
    return {k: v.bfloat16().float() for k, v in synth_state_dict(phi3_param_spec(CFG), seed=0).items()}


def prompts(cfg=CFG, lens=LENS):
    g = torch.Generator().manual_seed(7)
    rows = [(torch.randn(n, cfg.hidden, generator=g) * 0.5).bfloat16().float() for n in lens]
    emb = torch.zeros(len(lens), max(lens), cfg.hidden)
    for b, r in enumerate(rows):
        emb[b, :lens[b]] = r
    return rows, emb


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


def test_cpu_decoder_against_the_unquantised_one():
    sd, (rows, emb) = weights(), prompts()
    ref = TR.phi3_prefill_logits(emb, LENS, sd, CFG.layers, CFG.heads, CFG.kv_heads, CFG.rms_eps, CFG.rope_theta).numpy()
    dec = Phi3Decoder(sd, CFG, torch.float32, "cpu", quant="fp8")
    assert all(isinstance(L[k], F8.Fp8) and L[k].rows == 128 for L in dec.layers for k in ("qkv_w", "o_w", "gu_w", "down_w")) and not dec.interleave_gu
    got = dec.prefill_logits(emb, torch.tensor(LENS)).numpy()
    assert 1e-3 < rel(got, ref) < QUANT_ERROR, rel(got, ref)
    assert np.array_equal(got, dec.prefill_logits_rows(rows).numpy())


def test_load_quantises_again_and_refusals():
    sd = weights()
    dec = Phi3Decoder(sd, CFG, torch.float32, "cpu", quant="fp8")
    name = "language_model.model.layers.1.mlp.down_proj.weight"
    before = dec.layers[1]["down_w"].data.view(torch.uint8).clone()
    dec.load({**sd, name: -sd[name]})
    assert not torch.equal(before, dec.layers[1]["down_w"].data.view(torch.uint8))
    with pytest.raises(ValueError, match="quant"):
        Phi3Decoder(sd, CFG, torch.float32, "cpu", quant="int8")
    odd = Phi3Config(vocab=64, hidden=96, layers=1, heads=1, kv_heads=1, mlp=100)
    with pytest.raises(ValueError, match="multiples of 16"):
        Phi3Decoder({}, odd, torch.float32, "cpu", quant="fp8")


def test_the_model_passes_it_on():
    vit = VitConfig(image=28, patch=14, width=64, layers=2, heads=2, mlp=128, proj_dim=128)
    cfg = Phi3Config(vocab=64, hidden=128, layers=1, heads=4, kv_heads=4, mlp=144)
    sd = synth_state_dict(phi3_param_spec(cfg) + llava_vision_param_spec(vit), seed=0)
    net = LlavaModel(sd, vit, cfg, torch.float32, "cpu", llm_quant="fp8")
    assert net.lm.quant == "fp8" and isinstance(net.lm.layers[0]["qkv_w"], F8.Fp8) and LlavaModel(sd, vit, cfg, torch.float32, "cpu").lm.quant is None
    with torch.no_grad():
        net.get_parameter("language_model.model.layers.0.self_attn.o_proj.weight").mul_(2.0)
    old = net.lm.layers[0]["o_w"].scale.float()
    net.refresh()
    assert torch.equal(net.lm.layers[0]["o_w"].scale.float(), 2.0 * old)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_decoder(dtype):
    """Packed and padded prefill against the same decoder on the CPU in float32."""
    from dynam3d_amd import dense_ops as D
    sd, (rows, emb) = weights(), prompts()
    want = Phi3Decoder(sd, CFG, torch.float32, "cpu", quant="fp8").prefill_logits(emb, torch.tensor(LENS)).numpy()
    saved = dict(D.BACKEND)
    try:
        D.enable_hip_kernels(["all"])
        dec = Phi3Decoder(sd, CFG, dtype, "cuda", quant="fp8")
        got = dec.prefill_logits_rows([r.cuda() for r in rows]).cpu().numpy()
        pad = dec.prefill_logits(emb.cuda(), torch.tensor(LENS)).cpu().numpy()
    finally:
        D.BACKEND.update(saved)
    assert rel(got, want) < RUN_ERROR and rel(pad, want) < RUN_ERROR and rel(got, pad) < RUN_ERROR, (rel(got, want), rel(pad, want), rel(got, pad))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[19], LENS, [33] * 9 + [70] * 8])
def test_gpu_generation(lens):
    """KV-cache decode, one token at a time (17 sequences: in two groups): with forced tokens every step's logits are those of the prompt with the tokens behind
    it; free running it takes its own argmax and stops behind `end_id`."""
    from dynam3d_amd import dense_ops as D
    sd, (rows, _) = weights(), prompts(CFG, lens)
    saved = dict(D.BACKEND)
    try:
        D.enable_hip_kernels(["all"])
        dec = Phi3Decoder(sd, CFG, torch.bfloat16, "cuda", quant="fp8")
        n = sum(lens)
        x = torch.zeros(((n + 255) // 256 * 256, CFG.hidden), dtype=torch.bfloat16, device="cuda")
        x[:n] = torch.cat(rows).cuda().bfloat16()
        forced = torch.randint(0, CFG.vocab, (4, len(lens)), generator=torch.Generator().manual_seed(3)).tolist()
        _, logits = dec.generate_packed(x, lens, max_new_tokens=4, forced=forced, return_logits=True)
        assert logits.shape == (4, len(lens), CFG.vocab)
        ids = torch.tensor(forced, device="cuda")
        for i in range(4):
            full = [torch.cat([r.cuda().bfloat16(), dec.embed_tokens(ids[:i, b])]) for b, r in enumerate(rows)]
            again = dec.prefill_logits_rows(full)
            assert rel(logits[i].cpu(), again.cpu()) < RUN_ERROR, (i, rel(logits[i].cpu(), again.cpu()))
        free, logits = dec.generate_packed(x, lens, max_new_tokens=6, return_logits=True)
        assert free == logits.argmax(-1).t().tolist()
        end = free[0][2]
        stopped = dec.generate_packed(x, lens, max_new_tokens=6, end_id=end)
        for a, b in zip(stopped, free):
            assert a == (b[:b.index(end) + 1] if end in b else b)
    finally:
        D.BACKEND.update(saved)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_token_and_layer_are_the_functions_in_turn(dtype):
    """One decode token issued from C++, and one packed layer, against the public functions called one by one: the same bits."""
    from dynam3d_amd import dense_ops as D
    from dynam3d_amd.hip_dense import HipDense
    sd, (rows, _) = weights(), prompts()
    c, hip = CFG, HipDense()
    saved = dict(D.BACKEND)
    try:
        D.enable_hip_kernels(["all"])
        dec = Phi3Decoder(sd, c, dtype, "cuda", quant="fp8")
        n, B = sum(LENS), len(LENS)
        x = torch.zeros(((n + 255) // 256 * 256, c.hidden), dtype=dtype, device="cuda")
        x[:n] = torch.cat(rows).cuda().to(dtype)
        ctx, L = dec.packed_context(LENS, x.shape[0]), dec.layers[0]
        kv = []
        y = dec.layer_packed(0, x, ctx, kv)
        qkv = F8.linear(F8.rms_norm(x, L["n1"], c.rms_eps), L["qkv_w"], out_dtype=dtype)
        assert torch.equal(qkv[:, 2 * c.hidden:], kv[0][:, 2 * c.hidden:])                      # (values: not rotated)
        a = ctx["attn_out"].view(-1, c.hidden)
        h = F8.linear(F8.quantize(a), L["o_w"], residual=x, out_dtype=dtype)
        act = F8.linear_swiglu(F8.rms_norm(h, L["n2"], c.rms_eps), L["gu_w"], out_dtype=torch.float8_e4m3fn)
        assert torch.equal(y, F8.linear(act, L["down_w"], residual=h, out_dtype=dtype))

        kv = []
        dec.prefill_logits_packed(x, LENS, keep_kv=kv)
        side = torch.zeros((c.layers, 2, B, 3, c.heads, c.head_dim), dtype=dtype, device="cuda")
        cos, sin = dec._rope(max(LENS) + 4)
        ids = torch.tensor([5, 77, 401, 12], device="cuda")
        pos = torch.tensor(LENS, dtype=torch.int32, device="cuda")
        run = dec._decode_runner(B, kv, dec._last_cu, side, cos, sin, max(LENS))
        got = run(dec.embed_tokens(ids).to(dtype).contiguous(), pos, 0)
        z, other = dec.embed_tokens(ids).to(dtype).contiguous(), torch.zeros_like(side)
        for li, L in enumerate(dec.layers):
            qkv = F8.linear(F8.rms_norm(z, L["n1"], c.rms_eps), L["qkv_w"], out_dtype=dtype)
            a = hip.decode_attention(qkv, kv[li], dec._last_cu, other[li, 0], other[li, 1], c.heads, 0, max(LENS), rope=(cos, sin, pos))
            z = F8.linear(F8.quantize(a), L["o_w"], residual=z, out_dtype=dtype)
            act = F8.linear_swiglu(F8.rms_norm(z, L["n2"], c.rms_eps), L["gu_w"], out_dtype=torch.float8_e4m3fn)
            z = F8.linear(act, L["down_w"], residual=z, out_dtype=dtype)
        assert torch.equal(side, other) and torch.equal(got, dec.final_logits(z))
    finally:
        D.BACKEND.update(saved)
