"""ops.attention_text (ea_attention_text.hip) against a plain fp64 implementation on the host."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
NINF = float("-inf")


def plain(q, k, v, scale, causal=False, cap=0.0, bias=None, q_docs=None, kv_docs=None, prefix=None, valid=None, q_start=None):
    """fp64 result [B, Sq, Hq, D] and an elementwise bound on the kernel's error.

    Scores: D exact products of bf16 values added in fp32, 2^-23 of their magnitude sum each at most; scale and exponent argument 2^-22
    of the score's log2 value; a cap's tanh to 2^-21 of the cap (its exponential and reciprocal: 1 ulp each) -- together dt, in
    natural units.  The weight then is off by a factor of e^(dt) and one rounding to bf16 (2^-8); the fp32 sums of n weights and n
    products by n 2^-23; the result is rounded to bf16 once (2^-8)."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    qd, kd, vd = q.double(), k.double().repeat_interleave(Hq // Hkv, 1), v.double().repeat_interleave(Hq // Hkv, 1)
    j = torch.arange(Sk)
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64)
    err = torch.zeros_like(out)
    for b in range(B):
        start = int(q_start[b]) if q_start is not None else Sk - Sq
        pos = torch.arange(Sq) + start
        see = torch.ones(Sq, Sk, dtype=torch.bool)
        if causal:
            see = j[None] <= pos[:, None]
            if prefix is not None:
                see = see | (j[None] < int(prefix[b]))
        if valid is not None:
            see = see & (j[None] < int(valid[b]))
        if q_docs is not None:
            see = see & (kv_docs[b][None] == q_docs[b][:, None])
        for h in range(Hq):
            kh = torch.where(see.any(0)[:, None], kd[b, h], torch.zeros(1, dtype=torch.float64))
            t = qd[b, h] @ kh.t() * scale
            dt = (qd[b, h].abs() @ kh.abs().t()) * scale * D * 2.0 ** -23 + t.abs() * 2.0 ** -21
            if cap:
                t = cap * torch.tanh(t / cap)
                dt = dt + min(cap, 300.0) * 2.0 ** -20 + t.abs() * 2.0 ** -19
            if bias is not None:
                R = bias.shape[1] // 2
                bb = bias[h].double()[(j[None] - pos[:, None]).clamp(-R, R) + R]
                t = t + bb
                dt = dt + torch.where(bb.abs() < 1e30, bb.abs(), torch.zeros(1, dtype=torch.float64)) * 2.0 ** -21
            t = torch.where(see, t, NINF)
            top = t.amax(-1, keepdim=True)
            w = torch.exp(t - torch.where(top == NINF, 0.0, top))
            n = w.sum(-1, keepdim=True)
            w = torch.where(n == 0, 0.0, w / n)
            dt = torch.where(see, dt, 0.0).amax(-1, keepdim=True)           # of the numerator and of the sum
            dt = torch.where(torch.isfinite(dt), dt, 0.0)
            vis = (w > 0) & see
            for i0 in range(0, Sq, 64):                                     # per visible pair, so that hidden NaNs stay out
                ww, ok = w[i0:i0 + 64], vis[i0:i0 + 64]
                anyv = torch.isfinite(vd[b, h]).all()
                if anyv:
                    o, mag = ww @ vd[b, h], ww @ vd[b, h].abs()
                else:
                    vv = torch.where(ok[:, :, None], vd[b, h][None], 0.0)
                    o, mag = (ww[:, :, None] * vv).sum(1), (ww[:, :, None] * vv.abs()).sum(1)
                rel = 2.0 ** -8 + 2 * torch.expm1(dt[i0:i0 + 64]) + Sk * 2.0 ** -22
                out[b, i0:i0 + 64, h] = o
                err[b, i0:i0 + 64, h] = (mag * rel) * (1 + 2.0 ** -8) + o.abs() * 2.0 ** -8 + 1e-37
    return out.view(B, Sq, Hq * D), err.view(B, Sq, Hq * D)


def check(q, k, v, scale, kern=None, **kw):
    from easyanimate_amd import _lib, ops
    up = lambda t: t.to(DEV) if torch.is_tensor(t) else t
    _lib.reset_counters()
    got = ops.attention_text(up(q), up(k), up(v), scale, **{n: up(t) for n, t in kw.items()})
    if kern:
        assert _lib.counters().get(kern) == 1, _lib.counters()
    kw.pop("out", None)
    want, err = plain(q, k, v, scale, **kw)
    got = got.cpu().double()
    _inside(got, want, err)
    # the same batch again and again, until there are enough workgroups for the 128-row tiles
    B, Hq, Sq, _ = q.shape
    pack = max(n for n in range(1, 9) if Hq // k.shape[1] % n == 0)
    if Sq * pack > 16:
        reps = 512 // (B * Hq // pack * ((Sq * pack + 127) // 128)) + 1
        rep = lambda t: t.repeat(reps, *[1] * (t.dim() - 1))
        _lib.reset_counters()
        many = ops.attention_text(up(rep(q)), up(rep(k)), up(rep(v)), scale,
                                  **{n: up(rep(t)) if n in ("q_docs", "kv_docs", "prefix", "valid", "q_start") and t is not None else up(t) for n, t in kw.items()})
        assert _lib.counters().get("attention_text") == 1, _lib.counters()
        many = many.view(reps, B, Sq, -1).cpu().double()
        _inside(many[-1], want, err)
        assert torch.equal(many[0].nan_to_num(), many[-1].nan_to_num())
    return got


def _inside(got, want, err):
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    bad = ((got - want).abs() > err) & torch.isfinite(want)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst ratio {torch.nan_to_num((got - want).abs() / err).max().item():.3g}"


def make(B, Hq, Hkv, Sq, Sk, D, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda h, s: torch.randn(B, h, s, D, generator=g)
    return (r(Hq, Sq) * spread).bfloat16(), r(Hkv, Sk).bfloat16(), r(Hkv, Sk).bfloat16(), g


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 2), (7, 1), (4, 4), (17, 1), (34, 2)])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (5, 5), (33, 33), (64, 200), (131, 131)])
def test_causal_sizes_and_heads(Sq, Sk, Hq, Hkv, D):
    q, k, v, _ = make(2, Hq, Hkv, Sq, Sk, D, Sq * 100 + Hq + D)
    check(q, k, v, D ** -0.5, causal=True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk", [(1, 63), (1, 64), (1, 65), (2, 31), (3, 1000), (16, 777), (40, 520), (257, 130), (200, 64), (129, 1)])
def test_both_ways_no_mask(Sq, Sk, D):
    q, k, v, _ = make(2, 2, 1, Sq, Sk, D, Sq + Sk)
    check(q, k, v, D ** -0.5)


FORMS = ["cap", "wide_cap", "bias", "far_bias", "documents", "scattered_documents", "prefix", "valid", "all"]


def form(name, B, Hq, Sq, Sk, g):
    kw = {"causal": name not in ("bias", "far_bias", "valid", "cap")}
    if name in ("cap", "all"):
        kw["cap"] = 5.0
    if name == "wide_cap":
        kw["cap"] = 30000.0
    if name in ("bias", "all"):
        kw["bias"] = torch.randn(Hq, 2 * 20 + 1, generator=g)
    if name == "far_bias":                                  # a slope over every distance there is
        kw["bias"] = -0.02 * torch.arange(-700, 701).abs().float()[None] * (1 + torch.arange(Hq).float())[:, None]
    if name in ("documents", "all"):
        cut = torch.sort(torch.randint(0, Sk, (B, 3), generator=g), -1).values
        kw["kv_docs"] = (torch.arange(Sk)[None, :, None] >= cut[:, None, :]).sum(-1).to(torch.int32) * 1000 - 7
        kw["q_docs"] = kw["kv_docs"][:, Sk - Sq:].contiguous()
    if name == "scattered_documents":
        kw["kv_docs"] = torch.randint(-2, 3, (B, Sk), generator=g).to(torch.int32)
        kw["q_docs"] = torch.randint(-2, 4, (B, Sq), generator=g).to(torch.int32)        # 3: a document without keys
    if name in ("prefix", "all"):
        kw["prefix"] = torch.randint(0, Sk + 1, (B,), generator=g).to(torch.int32)
    if name in ("valid", "all"):
        kw["valid"] = torch.randint(0, Sk + 1, (B,), generator=g).to(torch.int32)
        kw["valid"][0] = Sk
    return kw


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("D,Hq,Hkv,Sq,Sk", [(64, 3, 3, 150, 150), (128, 4, 2, 97, 97), (128, 7, 1, 1, 333), (64, 4, 2, 3, 200), (64, 8, 1, 70, 400)])
def test_forms(name, D, Hq, Hkv, Sq, Sk):
    q, k, v, g = make(3, Hq, Hkv, Sq, Sk, D, len(name) + Sq, spread=2.0)
    check(q, k, v, D ** -0.5, **form(name, 3, Hq, Sq, Sk, g))


@pytest.mark.parametrize("Sq,Sk,kern", [(1, 5000, "attention_text_few"), (40, 3000, "attention_text_64_split"), (40, 9000, "attention_text_64_split"), (600, 600, "attention_text_64")])
@pytest.mark.parametrize("name", ["cap", "all", "far_bias"])
def test_long(Sq, Sk, kern, name):
    q, k, v, g = make(1, 4, 2, Sq, Sk, 128, Sq + Sk)
    check(q, k, v, 128 ** -0.5, kern=kern, **form(name, 1, 4, Sq, Sk, g))


def test_rows_that_see_nothing_are_zero():
    q, k, v, _ = make(4, 2, 1, 70, 70, 64, 3)
    # lengths of zero; queries in front of every key; a document of its own
    got = check(q, k, v, 0.125, causal=True, valid=i32(0, 70, 1, 70), q_start=i32(0, -69, 0, -200))
    assert (got[0] == 0).all() and (got[3] == 0).all() and (got[1, :68] == 0).all() and not (got[1, 69] == 0).all()
    docs = torch.zeros(4, 70, dtype=torch.int32)
    qd = docs.clone()
    qd[2] = 9
    qd[1, 5] = 1
    got = check(q, k, v, 0.125, q_docs=qd, kv_docs=docs)
    assert (got[2] == 0).all() and (got[1, 5] == 0).all() and not (got[1, 6] == 0).any()
    one, kk, vv, _ = make(2, 4, 2, 1, 90, 128, 4)
    got = check(one, kk, vv, 0.1, valid=i32(0, 90))
    assert (got[0] == 0).all()


def test_start_positions():
    q, k, v, g = make(3, 2, 2, 20, 300, 64, 5)
    bias = torch.randn(2, 41, generator=g)
    check(q, k, v, 0.125, causal=True, bias=bias, q_start=i32(0, 140, 290))
    check(q, k, v, 0.125, bias=bias, q_start=i32(-1000000, 2000000000, 17))
    check(q[:, :, :2], k, v, 0.125, causal=True, bias=bias, q_start=i32(2147483647, -2147483648, 5), valid=i32(300, 20, 100))


@pytest.mark.parametrize("Sq", [1, 90])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_hidden_places_may_hold_anything(Sq, what):
    """Keys and values that no query, or not every query, sees."""
    q, k, v, _ = make(2, 4, 2, Sq, 180, 64, 6)
    k[0, :, 150:] = float(what)
    v[0, :, 150:] = float(what)
    check(q, k, v, 0.125, valid=i32(150, 180))
    # one value that the later queries see: theirs is NaN or infinite in that column, the others' is untouched
    q, k, v, _ = make(1, 2, 1, 90, 90, 128, 7)
    v[0, 0, 70, 5] = float(what)
    got = check(q, k, v, 0.1, causal=True)
    assert torch.isfinite(got[0, :70]).all() and not torch.isfinite(got[0, 70:, 5]).any() and torch.isfinite(got[0, 70:, :5]).all()


def test_nan_in_visible_places_stays_in_its_rows():
    q, k, v, _ = make(1, 2, 1, 80, 80, 64, 8)
    q[0, 1, 33] = float("nan")
    got = check(q, k, v, 0.125, causal=True)
    assert torch.isnan(got[0, 33, 64:]).all() and torch.isfinite(got[0, 33, :64]).all()
    k[0, 0, 40, 3] = float("nan")
    q[0, 1, 33] = 0.5
    got = check(q, k, v, 0.125, causal=True)
    assert torch.isfinite(got[0, :40]).all() and torch.isnan(got[0, 40:]).all()


def test_bias_of_the_lowest_float_and_of_minus_infinity():
    q, k, v, _ = make(1, 2, 2, 70, 70, 64, 9)
    low = torch.finfo(torch.float32).min
    bias = torch.zeros(2, 2 * 69 + 1)
    bias[0, :69] = low                                     # head 0: earlier keys are pushed to the floor (an anti-causal mask)
    bias[1] = low                                          # head 1: all of them alike -- they keep their order: plain average here
    got = check(q, k, v, 0.125, bias=bias)
    mean = v[0, 1].double().mean(0)
    assert (got[0, :, 64:] - mean).abs().max() < 2.0 ** -7
    bias[1] = NINF                                         # hidden altogether: zeros
    bias[0, 69:] = NINF
    got = check(q, k, v, 0.125, bias=bias)
    assert (got[0, :, 64:] == 0).all() and (got[0, 0, :64] == 0).all()


def test_scores_far_apart():
    """Scores in the thousands, rising and falling along the keys: the running maximum moves often, or never."""
    q, k, v, _ = make(1, 2, 1, 64, 500, 64, 10)
    ramp = torch.linspace(-30, 30, 500)[None, None, :, None]
    for s in (ramp, -ramp, ramp.abs()):
        check((q * 0 + 4).bfloat16(), (k * 0.05 + s).bfloat16(), v, 0.125)
        check((q[:, :, :1] * 0 + 4).bfloat16(), (k * 0.05 + s).bfloat16(), v, 0.125)


def test_strides():
    """Views: heads of a fused projection, a cache with room behind it, an expanded cache, inner strides that have to be copied."""
    from easyanimate_amd import ops
    g = torch.Generator().manual_seed(11)
    fused = torch.randn(2, 90, (4 + 2 + 2) * 64, generator=g).bfloat16()
    parts = lambda t: (t[..., :256].view(2, 90, 4, 64).transpose(1, 2), t[..., 256:384].view(2, 90, 2, 64).transpose(1, 2),
                       t[..., 384:].view(2, 90, 2, 64).transpose(1, 2))
    up = fused.to(DEV)
    a = ops.attention_text(*parts(up), 0.125, causal=True)
    want, err = plain(*parts(fused), 0.125, causal=True)
    assert ((a.cpu().double() - want).abs() <= err).all()
    q, k, v = (t.contiguous() for t in parts(up))
    assert torch.equal(a, ops.attention_text(q, k, v, 0.125, causal=True))
    room = torch.full((2, 2, 128, 64), float("nan"), device=DEV).bfloat16()
    room[:, :, :90] = k
    assert torch.equal(a, ops.attention_text(q, room[:, :, :90], v, 0.125, causal=True))
    assert torch.equal(a, ops.attention_text(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, 0.125, causal=True))
    odd = torch.zeros(2, 2, 90, 65, device=DEV).bfloat16()
    odd[..., 1:] = v
    assert torch.equal(a, ops.attention_text(q, k, odd[..., 1:], 0.125, causal=True))
    wide = torch.full((2, 92, 304), 7.0, device=DEV).bfloat16()
    ops.attention_text(q, k, v, 0.125, causal=True, out=wide[:, 1:91, 40:296])
    assert torch.equal(wide[:, 1:91, 40:296], a)
    wide[:, 1:91, 40:296] = 7.0
    assert (wide == 7.0).all()
    one = ops.attention_text(q, k[:1, :1].expand(2, 2, 90, 64), v[:1, :1].expand(2, 2, 90, 64), 0.125)
    assert torch.equal(one, ops.attention_text(q, k[:1, :1].expand(2, 2, 90, 64).contiguous(), v[:1, :1].expand(2, 2, 90, 64).contiguous(), 0.125))


def test_empty():
    from easyanimate_amd import ops
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    assert ops.attention_text(z(2, 4, 0, 64), z(2, 2, 5, 64), z(2, 2, 5, 64), 1.0).shape == (2, 0, 256)
    out = ops.attention_text(z(2, 4, 3, 64) + 1, z(2, 2, 0, 64), z(2, 2, 0, 64), 1.0)
    assert out.shape == (2, 3, 256) and (out == 0).all()
    assert ops.attention_text(z(0, 4, 3, 64), z(0, 2, 5, 64), z(0, 2, 5, 64), 1.0).shape == (0, 3, 256)


@pytest.mark.parametrize("Sq,Sk,docs", [(1, 2000, False), (64, 900, True)])
def test_side_stream_and_graph(Sq, Sk, docs):
    from easyanimate_amd import ops
    q, k, v, g = make(2, 4, 2, Sq, Sk, 128, 12)
    kw = {"causal": True, "cap": 20.0, "bias": torch.randn(4, 65, generator=g).to(DEV)}
    if docs:
        kd = (torch.arange(Sk) // 150).to(torch.int32).repeat(2, 1)
        kw["kv_docs"], kw["q_docs"] = kd.to(DEV), kd[:, Sk - Sq:].contiguous().to(DEV)
    qs = [q.to(DEV), (q * 0.3).to(DEV), q.flip(1).contiguous().to(DEV)]
    k, v = k.to(DEV), v.to(DEV)
    eager = [ops.attention_text(t, k, v, 0.09, **kw) for t in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attention_text(qs[0], k, v, 0.09, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, eager[0])
    buf = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_text(buf, k, v, 0.09, **kw)
    for i in (1, 2, 0, 1):
        buf.copy_(qs[i])
        graph.replay()
        assert torch.equal(out, eager[i])
        assert torch.equal(ops.attention_text(qs[i], k, v, 0.09, **kw), eager[i])
        torch.cuda.synchronize()


def test_agrees_with_the_prompt_kernel():
    """The same right-padded causal prompt through ops.attention_causal_gqa: the real tokens' rows within both kernels' roundings."""
    from easyanimate_amd import ops
    q, k, v, _ = make(2, 14, 2, 100, 100, 128, 13)
    valid = i32(100, 41)
    vt = torch.zeros(2, 2, 128, 128, dtype=torch.bfloat16)
    vt[..., :100] = v.transpose(2, 3)
    a = ops.attention_causal_gqa(q.to(DEV), k.to(DEV), vt.to(DEV), 100, 128 ** -0.5, valid.to(DEV)).cpu().double()
    b = ops.attention_text(q.to(DEV), k.to(DEV), v.to(DEV), 128 ** -0.5, causal=True, valid=valid.to(DEV)).cpu().double()
    _, err = plain(q, k, v, 128 ** -0.5, causal=True, valid=valid)
    assert ((a - b).abs() <= 2 * err).all()


def test_a_quantised_encoder_layer():
    """The operators as they are used together: 4-bit projections around attention with a distance bias over packed prompts, residual in
    the last product's epilogue -- each stage against fp64 from the stage before it."""
    from easyanimate_amd import ops
    from test_mxfp4_gpu import _check, _expected, store, values
    g = torch.Generator().manual_seed(14)
    S, H, D, d = 160, 4, 64, 256
    x = torch.randn(S, d, generator=g).bfloat16()
    w = {n: (torch.randn(H * D if n != "o" else d, d if n != "o" else H * D, generator=g) / 16).bfloat16() for n in "qkvo"}
    W = {n: ops.mxfp4_quantize(t.to(DEV)) for n, t in w.items()}
    docs = (torch.arange(S) // 61).to(torch.int32)[None].contiguous()
    bias = torch.randn(H, 2 * 31 + 1, generator=g)
    xa = ops.mxfp4_quantize(x.to(DEV))
    heads = {n: ops.gemm_mxfp4(xa, W[n], None).view(1, S, H, D).transpose(1, 2) for n in "qkv"}
    a = ops.attention_text(heads["q"], heads["k"], heads["v"], 1.0 / 8, bias=bias.to(DEV), q_docs=docs.to(DEV), kv_docs=docs.to(DEV))
    y = ops.gemm_mxfp4(a.view(S, H * D), W["o"], None, ops.EPI_BIAS_GATE_RES, res=x.to(DEV), gate=torch.ones(d, device=DEV))
    for n in "qkv":
        got = heads[n].transpose(1, 2).reshape(S, H * D)
        _check(got, *_expected(values(*store(x)), values(*store(w[n])), None, ops.EPI_BIAS, None, None))
    want, err = plain(*(heads[n].cpu() for n in "qkv"), 1.0 / 8, bias=bias, q_docs=docs, kv_docs=docs)
    assert ((a.cpu().double() - want).abs() <= err).all()
    _check(y, *_expected(values(*store(a.cpu().view(S, -1))), values(*store(w["o"])), None, ops.EPI_BIAS_GATE_RES, x, torch.ones(d)))
