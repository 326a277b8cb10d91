"""The text-encoder step on the device library (second half).

Reference call site: easyanimate/pipeline/pipeline_easyanimate.py:438-447 --

    prompt_embeds = text_encoder(input_ids=..., attention_mask=..., output_hidden_states=True).hidden_states[-2]

with `Qwen2VLForConditionalGeneration` (Qwen2-VL-7B) in the slot (predict_t2v.py:205-214): a decoder-only LLM run ONCE per
pipeline call over 256 right-padded prompt tokens (~7e12 FLOP against 50 x 4.5e15 for the loop).  The encoder itself is a
`transformers` dependency of the reference, not code in /root/reference; its decoder layer is restated here from transformers'
Qwen2-VL / Qwen2 modelling code (pinned by tests/test_text_encoder_gpu.py against the installed transformers implementation):

    x -> RMSNorm -> q / k / v Linear (bias) -> rotate-half RoPE (M-RoPE with text-only positions = the 1-D form) -> causal,
    key-padding-masked grouped-query attention -> o Linear -> + x -> RMSNorm -> down(SiLU(gate) * up) -> +

`Qwen2VLTextEncoderHIP(hf_model)` wraps the loaded transformers model WITHOUT copying its weights and answers the one call the
pipelines make: `enc(input_ids=, attention_mask=, output_hidden_states=True).hidden_states[-2]`, plus `.device` / `.dtype`.
Linear layers run on ea_gemm_bf16 (residual adds in its epilogue), norms on ea_rmsnorm_bf16, the rest on ea_text.hip.
Text-only: image / video inputs are refused (the EasyAnimate pipelines never pass any).  There is no CPU fallback.

`weights="mxfp4"` runs the same layers with 4-bit Linear layers (ops.gemm_mxfp4: weights and activations in blocks of 32 e2m1 codes
under one power-of-two scale; a layer's q / k / v and gate / up products share one quantised input) and ops.attention_text, which reads
V as the projection left it.  A coarse approximation: 0.16 relative error (L2) per product on normal inputs, 0.20 where one channel in 256
is 20 times the others.  On random-init weights of the 7B widths, where nothing damps it, `hidden_states[-2]` is 0.75 away from the bf16
path's after 4 layers and 1.2, unrelated, after 28; no checkpoint was at hand to say what trained weights do.  The 4-bit copies stand
beside the model's own weights.  The default is the bf16 path above."""
from __future__ import annotations

import types
from typing import Optional

import torch
import torch.nn as nn

from . import ops
from ._params import derived, f32, gemm_weight, mxfp4_weight


def _find_text_model(hf_model):
    """The decoder stack of a transformers Qwen2-VL / Qwen2 model, whatever the library version calls the path to it
    (4.4x: model; >= 4.52 / 5.x: model.language_model)."""
    cands = [hf_model]
    for path in ("model.language_model", "model", "language_model"):
        m = hf_model
        for a in path.split("."):
            m = getattr(m, a, None)
            if m is None:
                break
        if m is not None:
            cands.append(m)
    for m in cands:
        if hasattr(m, "layers") and hasattr(m, "embed_tokens") and hasattr(m, "norm"):
            return m
    raise TypeError(f"{type(hf_model).__name__}: no decoder stack (layers / embed_tokens / norm) found")


def _check_weights(weights: str) -> None:
    if weights not in ("bf16", "mxfp4"):
        raise ValueError(f"weights must be 'bf16' or 'mxfp4', not {weights!r}")


class Qwen2VLTextEncoderHIP(nn.Module):
    def __init__(self, hf_model, padded_positions: str = "arange", weights: str = "bf16"):
        """padded_positions: the rotary position of the right-PADDED slots (real tokens are 0 .. n-1 either way; the DiT consumes
        the padded rows too, transformer3d.py:1502).  "arange" = transformers 5.x (the installed version: text-only prompts get
        the text model's own arange(S)); "cumsum_fill1" = transformers 4.46 - 4.5x (get_rope_index: cumsum(mask) - 1, padding -> 1).
        weights: "bf16", or "mxfp4" for 4-bit Linear layers (laid out per call, or once inside _params.weights_frozen())."""
        super().__init__()
        if padded_positions not in ("arange", "cumsum_fill1"):
            raise ValueError(f"padded_positions must be 'arange' or 'cumsum_fill1', not {padded_positions!r}")
        _check_weights(weights)
        self.padded_positions = padded_positions
        self.weights = weights
        self.hf = hf_model                                 # (registered: .to() / offload hooks reach the shared parameters)
        text = _find_text_model(hf_model)
        cfg = text.config
        self.hidden = cfg.hidden_size
        self.q_heads = cfg.num_attention_heads
        self.kv_heads = getattr(cfg, "num_key_value_heads", None) or self.q_heads
        self.head_dim = getattr(cfg, "head_dim", None) or self.hidden // self.q_heads
        self.eps = cfg.rms_norm_eps
        rp = getattr(cfg, "rope_parameters", None) or getattr(cfg, "rope_scaling", None) or {}
        self.theta = float(rp.get("rope_theta", None) or getattr(cfg, "rope_theta", None) or 10000.0)
        if self.head_dim not in (64, 128):
            raise NotImplementedError(f"Qwen2VLTextEncoderHIP: head_dim {self.head_dim} (ea_attention_causal_gqa_bf16 is built for 64 and 128)")
        if weights == "mxfp4" and (self.hidden % 8 or cfg.intermediate_size % 8):
            raise NotImplementedError(f"Qwen2VLTextEncoderHIP: weights='mxfp4' needs widths that are multiples of 8 (got {self.hidden}, {cfg.intermediate_size})")
        if getattr(cfg, "use_sliding_window", False):
            raise NotImplementedError("Qwen2VLTextEncoderHIP: sliding-window layers are not implemented (Qwen2-VL-7B does not use them)")
        if getattr(cfg, "hidden_act", "silu") != "silu":
            raise NotImplementedError(f"Qwen2VLTextEncoderHIP: hidden_act {cfg.hidden_act!r}")
        self._text = [text]                                # (a list: not registered a second time)

    # ---- what the pipelines read -------------------------------------------------------------
    @property
    def device(self):
        return next(self.hf.parameters()).device

    @property
    def dtype(self):
        return next(self.hf.parameters()).dtype

    @property
    def config(self):
        return self.hf.config

    def _gate_ones(self) -> torch.Tensor:
        return derived(self._text[0].norm.weight, "ones", lambda t: torch.ones(self.hidden, dtype=torch.float32, device=t.device))

    def _layer_mxfp4(self, layer, h, B, S, cos, sin, valid, ones):
        att, mlp, D, Hq, Hkv = layer.self_attn, layer.mlp, self.head_dim, self.q_heads, self.kv_heads
        fb = lambda lin: f32(lin.bias) if lin.bias is not None else None
        lin = lambda a, l: ops.gemm_mxfp4(a, mxfp4_weight(l.weight), fb(l))
        add = lambda a, l, res: ops.gemm_mxfp4(a, mxfp4_weight(l.weight), fb(l), ops.EPI_BIAS_GATE_RES, res=res, gate=ones)
        n1 = ops.mxfp4_quantize(ops.rmsnorm(h, f32(layer.input_layernorm.weight), self.eps))
        qh = ops.rope_half_scatter(lin(n1, att.q_proj), Hq, D, B, S, cos, sin)
        kh = ops.rope_half_scatter(lin(n1, att.k_proj), Hkv, D, B, S, cos, sin)
        v = lin(n1, att.v_proj).view(B, S, Hkv, D).transpose(1, 2)
        a = ops.attention_text(qh, kh, v, D ** -0.5, causal=True, valid=valid)
        h = add(a.view(B * S, Hq * D), att.o_proj, h)
        n2 = ops.mxfp4_quantize(ops.rmsnorm(h, f32(layer.post_attention_layernorm.weight), self.eps))
        return add(ops.silu_mul(lin(n2, mlp.gate_proj), lin(n2, mlp.up_proj)), mlp.down_proj, h)

    @torch.no_grad()
    def forward(self, input_ids: Optional[torch.Tensor] = None, attention_mask: Optional[torch.Tensor] = None,
                output_hidden_states: bool = False, pixel_values=None, pixel_values_videos=None, inputs_embeds=None, **kwargs):
        if pixel_values is not None or pixel_values_videos is not None:
            raise NotImplementedError("Qwen2VLTextEncoderHIP is text-only (the EasyAnimate pipelines pass prompts only)")
        text = self._text[0]
        if inputs_embeds is None:
            if input_ids is None:
                raise ValueError("input_ids or inputs_embeds")
            inputs_embeds = text.embed_tokens(input_ids)
        x = inputs_embeds
        if not x.is_cuda:
            raise RuntimeError("Qwen2VLTextEncoderHIP: inputs must be on the GPU; there is no CPU fallback")
        if x.dtype != torch.bfloat16:
            raise RuntimeError(f"Qwen2VLTextEncoderHIP: the encoder must be loaded in bfloat16 (got {x.dtype}); the library computes in bf16")
        B, S, d = x.shape
        dev = x.device
        D, Hq, Hkv = self.head_dim, self.q_heads, self.kv_heads
        # ---- positions and key padding (the three M-RoPE axes carry the same ids for text, so the sectioned cos / sin equal the
        # 1-D ones; padded slots: see __init__)
        if attention_mask is not None:
            am = attention_mask.to(device=dev, dtype=torch.long)
            if not bool((am[:, 1:] <= am[:, :-1]).all()):
                raise NotImplementedError("Qwen2VLTextEncoderHIP: only right-padded prompts (padding_side='right', pipeline_easyanimate.py:431)")
            if self.padded_positions == "arange":
                pos = torch.arange(S, device=dev)[None].expand(B, S)
            else:
                pos = (am.cumsum(-1) - 1).masked_fill(am == 0, 1)
            valid = am.sum(-1).to(torch.int32).contiguous()
        else:
            pos = torch.arange(S, device=dev)[None].expand(B, S)
            valid = None
        inv_freq = 1.0 / (self.theta ** (torch.arange(0, D, 2, dtype=torch.float32, device=dev) / D))
        ang = pos.to(torch.float32)[..., None] * inv_freq                     # [B, S, D/2]
        ang = torch.cat([ang, ang], dim=-1).reshape(B * S, D)
        cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
        s_pad = ops.round_up(S, 32)
        four = self.weights == "mxfp4"
        vt = None if four else torch.zeros(B, Hkv, D, s_pad, dtype=torch.bfloat16, device=dev)
        h = x.reshape(B * S, d).contiguous()
        ones = self._gate_ones()
        hidden_states = [x]
        for layer in text.layers:
            if four:
                h = self._layer_mxfp4(layer, h, B, S, cos, sin, valid, ones)
                hidden_states.append(h.view(B, S, d))
                continue
            att, mlp = layer.self_attn, layer.mlp
            n1 = ops.rmsnorm(h, f32(layer.input_layernorm.weight), self.eps)
            q = ops.gemm(n1, gemm_weight(att.q_proj.weight), f32(att.q_proj.bias) if att.q_proj.bias is not None else None)
            k = ops.gemm(n1, gemm_weight(att.k_proj.weight), f32(att.k_proj.bias) if att.k_proj.bias is not None else None)
            v = ops.gemm(n1, gemm_weight(att.v_proj.weight), f32(att.v_proj.bias) if att.v_proj.bias is not None else None)
            qh = ops.rope_half_scatter(q, Hq, D, B, S, cos, sin)
            kh = ops.rope_half_scatter(k, Hkv, D, B, S, cos, sin)
            vt[..., :S] = v.view(B, S, Hkv, D).permute(0, 2, 3, 1)            # V^T (columns >= S stay zero)
            a = ops.attention_causal_gqa(qh, kh, vt, S, D ** -0.5, valid)
            ob = f32(att.o_proj.bias) if att.o_proj.bias is not None else None
            h = ops.gemm(a.view(B * S, Hq * D), gemm_weight(att.o_proj.weight), ob, ops.EPI_BIAS_GATE_RES, res=h, gate=ones)
            n2 = ops.rmsnorm(h, f32(layer.post_attention_layernorm.weight), self.eps)
            g = ops.gemm(n2, gemm_weight(mlp.gate_proj.weight), None)
            u = ops.gemm(n2, gemm_weight(mlp.up_proj.weight), None)
            act = ops.silu_mul(g, u)
            h = ops.gemm(act, gemm_weight(mlp.down_proj.weight), None, ops.EPI_BIAS_GATE_RES, res=h, gate=ones)
            hidden_states.append(h.view(B, S, d))
        last = ops.rmsnorm(h, f32(text.norm.weight), self.eps).view(B, S, d)
        # transformers: hidden_states = (embeddings, layer 1 .. layer L-1 outputs, NORMED layer L output)
        hidden_states[-1] = last
        return types.SimpleNamespace(last_hidden_state=last, hidden_states=tuple(hidden_states) if output_hidden_states else None)


def use_hip_text_encoder(pipeline, index: int = 0, weights: str = "bf16"):
    """Swap the transformers model in a pipeline's text_encoder slot for its device-library forward (weights shared).  A slot that holds
    one already is left as it is, or, where its `weights` differ from what is asked for, gets one with those around the same model."""
    _check_weights(weights)
    name = "text_encoder" if index == 0 else "text_encoder_2"
    enc = getattr(pipeline, name)
    if isinstance(enc, Qwen2VLTextEncoderHIP):
        if enc.weights != weights:
            setattr(pipeline, name, Qwen2VLTextEncoderHIP(enc.hf, enc.padded_positions, weights).train(enc.training))
    elif enc is not None:
        setattr(pipeline, name, Qwen2VLTextEncoderHIP(enc, weights=weights))
    return getattr(pipeline, name)
