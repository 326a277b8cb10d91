"""The text encoder with 4-bit Linear layers (Qwen2VLTextEncoderHIP(weights="mxfp4")): quantised storage, products and attention run
together over whole layers, against 64-bit implementations of each stage."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from test_mxfp4_gpu import store, values
from test_text_encoder_gpu import CASES, _prompt_batch, _qwen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rounded(x):
    """What the 4-bit storage makes of the rows of x."""
    flat = x.detach().bfloat16().float().reshape(-1, x.shape[-1])
    return values(*store(flat))[:, :flat.shape[1]].float().reshape(x.shape)


STEP = 2.0 ** -8            # half a bf16 step, relative
SLACK = 1.05                # second-order terms and the fp32 sums


def _within(name, got, want, bound):
    err = (got.double().cpu() - want).abs()
    worst = (err / bound.clamp_min(1e-30)).max().item()
    print(f"[parity] {name}: {worst:.2f} of the bound")
    assert worst <= 1.0, (name, worst)


def _rope(x, cos, sin):
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos + turned * sin, x.abs() * cos.abs() + turned.abs() * sin.abs()


# A difference of one bf16 step in a layer's input moves some elements over a boundary between two 4-bit values, a whole step of theirs,
# and every quantised product multiplies that: whole runs cannot be compared closely.  So each stage is computed in 64 bits from what the
# device handed to it, and may differ by the roundings that the device makes inside the stage:
#   norm             x / rms(x)'s, then its product with the gain (the transformers order, ea_rmsnorm_bf16): 2 STEP |y|
#   attention        q, k: the product's and the rotation's (scores off by 4 STEP G, G = scale sum |q||k|, the weights by twice that,
#                    relative), v's, the weights' for the product and for their sum, the output's
#   o, down + input  the output's                                                  STEP |y|
#   SiLU product     gate (|silu'| <= 1.1) and up, the output's
@pytest.mark.parametrize("case", ["hd64", "hd128"])
def test_layers_stage_by_stage(case, monkeypatch):
    from easyanimate_amd import _lib, ops
    from easyanimate_amd.text_encoder import Qwen2VLTextEncoderHIP
    c = CASES[case]
    hf = _qwen(c["hidden"], c["heads"], c["kv_heads"], c["inter"], c["layers"])
    layers = getattr(hf.model, "language_model", hf.model).layers
    weights = [{n: (_rounded(m.weight).double(), m.bias.double() if m.bias is not None else 0.0) for n, m in l.named_modules() if isinstance(m, torch.nn.Linear)}
               for l in layers]
    gains = [(l.input_layernorm.weight.double(), l.post_attention_layernorm.weight.double()) for l in layers]
    hf = hf.to(torch.bfloat16).to(DEV)
    ids, mask = _prompt_batch(c["B"], c["S"], 512, c["lens"])
    tape = {}

    def record(name):
        real = getattr(ops, name)

        def call(*args, **kw):
            y = real(*args, **kw)
            tape.setdefault(name, []).append((args[0].detach().clone(), y.detach().clone()))
            return y
        monkeypatch.setattr(ops, name, call)
    for name in ("rmsnorm", "attention_text", "silu_mul"):
        record(name)
    enc = Qwen2VLTextEncoderHIP(hf, weights="mxfp4")
    run = lambda: enc(input_ids=ids.to(DEV), attention_mask=mask.to(DEV), output_hidden_states=True).hidden_states
    _lib.reset_counters()
    got = run()
    cnt = _lib.counters()
    taken = {k: [(a.cpu(), b.cpu()) for a, b in v] for k, v in tape.items()}
    assert all(torch.equal(a, b) for a, b in zip(got, run()))
    assert sum(v for k, v in cnt.items() if k.startswith("gemm_mxfp4")) == 7 * c["layers"] and not any(k in cnt for k in ("gemm_128", "gemm_256_mi16", "gemm_256_w4a"))
    assert sum(v for k, v in cnt.items() if k.startswith("attention_text")) == c["layers"] and "attention_causal_gqa" not in cnt

    B, S, Hq, Hkv = c["B"], c["S"], c["heads"], c["kv_heads"]
    D = c["hidden"] // Hq
    ang = torch.arange(S, dtype=torch.float32)[:, None] * (1.0 / (1000000.0 ** (torch.arange(0, D, 2, dtype=torch.float32) / D)))
    cos, sin = (torch.cat([t, t], -1).double() for t in (ang.cos(), ang.sin()))
    j, i = torch.arange(S)[None, :], torch.arange(S)[:, None]
    hidden = (j > i)[None, None] | (j >= mask.sum(-1)[:, None])[:, None, :].unsqueeze(1)
    lin = lambda n, name, x: _rounded(x).double() @ weights[n][name][0].t() + weights[n][name][1]
    norm = lambda x, g: x.double() * (x.double().pow(2).mean(-1, keepdim=True) + enc.eps).rsqrt() * g
    for n in range(c["layers"]):
        (h, n1), (h1, n2) = taken["rmsnorm"][2 * n:2 * n + 2]
        a, (_, act), after = taken["attention_text"][n][1].view(B * S, -1), taken["silu_mul"][n], taken["rmsnorm"][2 * n + 2][0]
        for name, x, y, g in (("norm 1", h, n1, gains[n][0]), ("norm 2", h1, n2, gains[n][1])):
            want = norm(x, g)
            _within(f"{case} layer {n} {name}", y, want, SLACK * 2 * STEP * want.abs())
        q, k, v = (lin(n, f"self_attn.{p}_proj", n1).view(B, S, H, D).transpose(1, 2) for p, H in (("q", Hq), ("k", Hkv), ("v", Hkv)))
        (q, qa), (k, ka) = _rope(q, cos, sin), _rope(k, cos, sin)
        k, ka, v = (t.repeat_interleave(Hq // Hkv, 1) for t in (k, ka, v))
        w = (q @ k.transpose(2, 3) * D ** -0.5).masked_fill(hidden, float("-inf")).softmax(-1)
        off = (4 * STEP * D ** -0.5 * (qa @ ka.transpose(2, 3))).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        want = w @ v
        bound = SLACK * ((2 * off + 3 * STEP) * (w @ v.abs()) + STEP * want.abs())
        flat = lambda t: t.transpose(1, 2).reshape(B * S, -1)
        _within(f"{case} layer {n} attention", a, flat(want), flat(bound))
        want = h.double() + lin(n, "self_attn.o_proj", a)
        _within(f"{case} layer {n} o", h1, want, SLACK * STEP * want.abs() + 1e-6)
        g, u = lin(n, "mlp.gate_proj", n2), lin(n, "mlp.up_proj", n2)
        want = torch.nn.functional.silu(g) * u
        _within(f"{case} layer {n} SiLU product", act, want, SLACK * STEP * (1.1 * g.abs() * u.abs() + 2 * want.abs()) + 1e-6)
        want = h1.double() + lin(n, "mlp.down_proj", act)
        _within(f"{case} layer {n} down", after, want, SLACK * STEP * want.abs() + 1e-6)


def test_a_changed_weight_is_laid_out_again():
    from easyanimate_amd._params import weights_frozen
    from easyanimate_amd.text_encoder import Qwen2VLTextEncoderHIP
    c = CASES["hd64"]
    hf = _qwen(c["hidden"], c["heads"], c["kv_heads"], c["inter"], c["layers"]).to(torch.bfloat16).to(DEV)
    ids, mask = (t.to(DEV) for t in _prompt_batch(c["B"], c["S"], 512, c["lens"]))
    enc = Qwen2VLTextEncoderHIP(hf, weights="mxfp4")
    run = lambda e: e(input_ids=ids, attention_mask=mask, output_hidden_states=True).hidden_states[-1]
    before = run(enc)
    with torch.no_grad():
        enc._text[0].layers[0].mlp.down_proj.weight.mul_(-1.0)
    after = run(enc)
    assert not torch.equal(before, after)
    assert torch.equal(after, run(Qwen2VLTextEncoderHIP(hf, weights="mxfp4")))
    enc._text[0].layers[1].mlp.up_proj.weight.data.mul_(-1.0)               # no version counter sees this one
    third = run(enc)
    assert not torch.equal(third, after)
    with weights_frozen():                                                  # laid out once for the region
        assert torch.equal(run(enc), third) and torch.equal(run(enc), third)
    enc._text[0].layers[1].mlp.up_proj.weight.data.mul_(-1.0)
    with weights_frozen():
        assert torch.equal(run(enc), after)


def test_pipeline_slot():
    import types
    from easyanimate_amd.text_encoder import Qwen2VLTextEncoderHIP, use_hip_text_encoder
    hf = _qwen(256, 4, 2, 512, 1, vocab=128).to(torch.bfloat16).to(DEV)
    pipe = types.SimpleNamespace(text_encoder=hf)
    assert use_hip_text_encoder(pipe, weights="mxfp4") is pipe.text_encoder and pipe.text_encoder.weights == "mxfp4"
    assert Qwen2VLTextEncoderHIP(hf).weights == "bf16"
    with pytest.raises(ValueError, match="weights"):
        Qwen2VLTextEncoderHIP(hf, weights="int4")
