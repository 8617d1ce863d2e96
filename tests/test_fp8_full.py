"""`llm_quant="fp8"` from the outside in: the rollout's command line, a whole policy in the closed loop, and the language model at full size against the committed
results of its 16- and 32-bit runs (g16: Phi-3-mini, 32 layers, two prompts)."""
import dataclasses

import numpy as np
import pytest
import torch

from dynam3d_amd import fp8_ops as F8
from dynam3d_amd.policy import ActionGrammarTokenizer, Dynam3D_VLN, PolicyConfig, synth_policy_weights
from tests.test_fp8_decoder import QUANT_ERROR


def test_rollout_command_passes_it_on(monkeypatch):
    from dynam3d_amd import rollout
    seen = []

    class Stop(Exception):
        pass

    def build(cfg, *a, **k):
        seen.append(cfg)
        raise Stop
    monkeypatch.setattr(rollout.torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(rollout.D, "enable_hip_kernels", lambda names: None)
    monkeypatch.setattr(rollout.DD, "init_from_env", lambda: (0, 0, 1))
    monkeypatch.setattr(rollout, "synth_policy_weights", lambda *a, **k: {})
    monkeypatch.setattr(rollout, "Dynam3D_VLN", build)
    for args, want in ((["--llm-quant", "fp8"], "fp8"), ([], None)):
        monkeypatch.setattr(rollout.sys, "argv", ["rollout"] + args)
        with pytest.raises(Stop):
            rollout.main()
        assert seen[-1].llm_quant == want
    monkeypatch.setattr(rollout.sys, "argv", ["rollout", "--llm-quant", "int4"])
    with pytest.raises(SystemExit):
        rollout.main()


def test_policy_in_the_closed_loop_cpu():
    from tests.cpu_ops import CpuOps
    from tests.test_policy_cpu import SMALL
    from tests.test_rollout import _check_loop
    cfg = dataclasses.replace(SMALL, llm_quant="fp8")
    net = Dynam3D_VLN(cfg, synth_policy_weights(cfg, 0), device="cpu", batch_size=2, ops=CpuOps(), max_steps=4, tokenizer=ActionGrammarTokenizer(cfg.llm.vocab, stop_mod=5))
    assert net.llm.quant == "fp8" and isinstance(net.llm.layers[0]["qkv_w"], F8.Fp8)
    _check_loop(net, 2, 3, new_tokens=3, seed=2)
    with pytest.raises(ValueError, match="quant"):
        Dynam3D_VLN(dataclasses.replace(SMALL, llm_quant="int8"), synth_policy_weights(SMALL, 0), device="cpu", batch_size=1, ops=CpuOps())


@pytest.mark.gpu
def test_policy_step_and_closed_loop_gpu():
    """One step's logits beside those of the 16-bit language model (every dense primitive a HIP kernel), then three episodes with generation."""
    from dynam3d_amd import dense_ops as D
    from dynam3d_amd.synthetic import INSTRUCTION_64, SyntheticEpisodes
    from tests.test_policy_cpu import MID
    from tests.test_rollout import _check_loop
    saved, was = dict(D.BACKEND), D.STRICT
    D.enable_hip_kernels(["all"])
    D.strict(True)
    D.reset_counts()
    try:
        out = []
        for cfg in (MID, dataclasses.replace(MID, llm_quant="fp8")):
            net = Dynam3D_VLN(cfg, synth_policy_weights(cfg, 0), device="cuda", batch_size=2, max_steps=4, tokenizer=ActionGrammarTokenizer(cfg.llm.vocab, stop_mod=40))
            assert net.llm.quant == cfg.llm_quant
            net.feature_fields.initialize_camera_setting(90.0, 90.0)
            fr = SyntheticEpisodes(2, seed=3).next()
            obs = dict(rgb=torch.from_numpy(fr.rgb).cuda(), depth=torch.from_numpy(fr.depth).cuda())
            out.append(net.forward_logits(obs, [INSTRUCTION_64] * 2, [p.tolist() for p in fr.positions], list(fr.headings), patch_segm=fr.patch_segm).float().cpu())
        d = float((out[1] - out[0]).norm() / out[0].norm())
        assert 1e-3 < d < QUANT_ERROR, d
        net.feature_fields.reset(2)
        _check_loop(net, 2, 3, new_tokens=4, seed=7)
        assert not D.counts()["fallback"], D.counts()
    finally:
        D.strict(was)
        D.BACKEND.update(saved)


@pytest.mark.gpu
def test_full_depth_against_the_committed_runs():
    """Layers 0, 15, 31 on the reference run's own inputs, all 32 layers free running, and two decode tokens.

    Bounds.  One layer: the update (output - input) passes qkv, o, gate and up, and down, five products' worth of operand roundings at 3.7 % -- 8.3 % in all;
    QUANT_ERROR (eight: 10.4 %) leaves room for what the attention makes of rounded queries and keys.  The whole stack: a layer's rounding error is k times
    that of the 16-bit layer (k: the largest ratio of the update's error to g16's own 16-bit-to-32-bit distance of that layer, over the three layers), errors of this size pass the later
    layers as linear perturbations, so the logits are k times as far from the 32-bit run as the 16-bit ones are; 1.5 for three layers speaking for 32.  A decode token
    against the prefill of the longer prompt: two such runs that share their weights' roundings, half of each square: the same bound."""
    from dynam3d_amd import dense_ops as D
    from dynam3d_amd.towers import Phi3Config, Phi3Decoder, phi3_param_spec
    from dynam3d_amd.weights import synth_state_dict
    from tests.golden_io import load
    from tests.test_gpu_depth_parity import _pack, from_bits, rel
    g, cfg = load("g16_phi3_bf16_fulldepth.npz"), Phi3Config()
    lens = [int(n) for n in g["lengths"]]
    saved, was = dict(D.BACKEND), D.STRICT
    D.enable_hip_kernels(["all"])
    D.strict(True)
    try:
        dec = Phi3Decoder(synth_state_dict(phi3_param_spec(cfg), seed=0), cfg, torch.bfloat16, "cuda", quant="fp8")
        gen = torch.Generator().manual_seed(int(g["input_seed"]))
        rows = [(torch.randn(n, cfg.hidden, generator=gen) * 0.5).to(torch.bfloat16) for n in lens]
        x0, T = _pack(rows)
        ctx = dec.packed_context(lens, x0.shape[0])
        k = 0.0
        for li in [int(v) for v in g["full_layers"]]:
            xin = torch.zeros_like(x0)
            xin[:T] = x0[:T] if li == 0 else from_bits(g[f"in{li}_bits"], torch.bfloat16)
            want = from_bits(g[f"out{li}_bits"], torch.bfloat16)
            d = rel(dec.layer_packed(li, xin, ctx)[:T].float() - xin[:T].float(), want.float() - xin[:T].float())
            print(f"layer {li:2d}: update {d:.2e} from the 16-bit run ({float(g['band_upd'][li]):.2e} from 32 bits)")
            assert 1e-3 < d < QUANT_ERROR, (li, d)
            k = max(k, d / float(g["band_upd"][li]))
        got = dec.prefill_logits_packed(x0, lens).cpu()
        ref16, ref32 = torch.from_numpy(g["bf16_logits"]), torch.from_numpy(g["f32_logits"])
        band = max(rel(ref16[b], ref32[b]) for b in range(len(lens)))
        far = max(rel(got[b], ref32[b]) for b in range(len(lens)))
        print(f"32 layers: logits {far:.2e} from 32 bits, the 16-bit run {band:.2e}, k {k:.1f}")
        assert far < 1.5 * k * band, (far, k, band)
        forced = torch.randint(0, cfg.vocab, (3, len(lens)), generator=torch.Generator().manual_seed(3)).tolist()
        _, logits = dec.generate_packed(x0, lens, max_new_tokens=3, forced=forced, return_logits=True)
        ids = torch.tensor(forced, device="cuda")
        for i in range(3):
            again = dec.prefill_logits_rows([torch.cat([r.cuda(), dec.embed_tokens(ids[:i, b])]) for b, r in enumerate(rows)])
            d = max(rel(logits[i][b].cpu(), again[b].cpu()) for b in range(len(lens)))
            print(f"token {i}: {d:.2e} from the prefill")
            assert d < 1.5 * k * band, (i, d)
        assert not D.counts()["fallback"]
    finally:
        D.strict(was)
        D.BACKEND.update(saved)
