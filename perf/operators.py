"""The text-encoder operators as a measured set: 4-bit microscaled storage (quantise / restore), the product over it, and attention
with capped, distance-biased or masked scores.

`listed()` names the cases, `draw(rng)` makes more of the same ranges, `prepare(case, seed)` builds what a caller holds before the
call, `run(state)` is one pass (the framework's entry points where `own` is true, elementary torch operations in fp32 otherwise),
`exact(case, seed)` the same outputs from the definitions in fp64, `work(case)` the bytes and operations a pass cannot do without.
"""
import math

import torch

own = False
DEV = "cuda"


# ---- cases -----------------------------------------------------------------------------------------------------------------------
def _round(name, rows, k):
    return {"name": name, "kind": "round", "rows": rows, "k": k}


def _linear(name, m, n, k, epi):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "epi": epi}


def _attention(name, b, sq, sk, hq, hkv, d, causal=False, cap=0.0, reach=0, docs=0, prefix=False, ragged=False):
    return {"name": name, "kind": "attention", "b": b, "sq": sq, "sk": sk, "hq": hq, "hkv": hkv, "d": d, "causal": causal, "cap": cap,
            "reach": reach, "docs": docs, "prefix": prefix, "ragged": ragged}


def listed():
    return [
        # the hidden states of one padded 256-token prompt, stored and read back
        _round("round_prompt", 256, 3584),
        # one weight of the encoder's feed-forward, stored and read back: what loading a checkpoint does per layer
        _round("round_weight", 18944, 3584),
        # an odd number of rows whose length is no multiple of the 32-element block
        _round("round_odd", 4099, 1477),
        # one token through an attention projection (latency and the weight's bytes)
        _linear("linear_token", 1, 3584, 3584, "bias"),
        # a padded prompt through the widening half of the feed-forward
        _linear("linear_prompt_up", 256, 18944, 3584, "plain"),
        # a prompt pair through the narrowing half, with the gated residual add
        _linear("linear_prompt_down", 512, 3584, 18944, "residual"),
        # odd rows, a ragged last column tile, a K that is no multiple of the block
        _linear("linear_odd", 777, 1000, 1161, "gelu"),
        # the tokens of a 49-frame 512 x 512 clip through a wide layer with its activation
        _linear("linear_clip", 13312, 8192, 4096, "gelu"),
        # one new token per sequence against long caches of different lengths
        _attention("attention_token", 4, 1, 16384, 28, 4, 128, causal=True, ragged=True),
        # an encoder with a learned bias per distance: no causal order, prompts of different lengths
        _attention("attention_distance", 2, 512, 512, 64, 64, 64, reach=128, ragged=True),
        # prompts packed behind one another in one row, scores capped
        _attention("attention_documents", 1, 8192, 8192, 28, 4, 128, causal=True, cap=50.0, docs=7),
        # an odd length with a prefix that every token sees
        _attention("attention_prefix", 3, 1999, 1999, 16, 8, 64, causal=True, prefix=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["round", "linear", "linear", "attention", "attention"])
    if kind == "round":
        k = _log(rng, 32, 19000)
        return _strip(_round("", _log(rng, 1, max(1, 18944 * 3584 // k)), k))
    if kind == "linear":
        n = 8 * _log(rng, 8, 2368)
        k = _log(rng, 64, 18944)
        if rng.random() < 0.6:
            k = (k + 31) // 32 * 32
        m = _log(rng, 1, max(1, min(13312, 13312 * 8192 * 4096 // (n * k))))
        return _strip(_linear("", m, n, k, rng.choice(["plain", "bias", "gelu", "residual"])))
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 7])
    mode = rng.choice(["token", "encoder", "causal", "documents", "prefix"])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    reach = rng.choice([0, 0, 32, 128, 1000])
    if mode == "token":
        return _strip(_attention("", rng.randint(1, 8), rng.choice([1, 1, 2, 5]), _log(rng, 64, 16384), hq, hkv, d, True, cap, reach,
                                 0, False, rng.random() < 0.5))
    s = _log(rng, 16, 6000)
    b = max(1, min(4, 8192 * 8192 * 14 * 128 // (s * s * hq * d)))
    b = rng.randint(1, b)
    if mode == "encoder":
        return _strip(_attention("", b, s, s, hq, hkv, d, False, cap, reach, 0, False, rng.random() < 0.5))
    if mode == "documents":
        return _strip(_attention("", b, s, s, hq, hkv, d, rng.random() < 0.7, cap, reach, rng.randint(2, 9)))
    return _strip(_attention("", b, s, s, hq, hkv, d, True, cap, reach, 0, mode == "prefix"))


def _strip(case):
    case.pop("name")
    return case


# ---- what the masks of a case are: fixed by the case, so that its work is known ----------------------------------------------------
def _lengths(c):
    """Keys that exist per batch element: the whole cache, or (ragged) a different part of it for each."""
    return [max(1, c["sk"] - (i * c["sk"]) // (2 * c["b"]) - (i % 2)) if c["ragged"] else c["sk"] for i in range(c["b"])]


def _starts(c):
    """Position of the first query: the queries are the last tokens of their sequence (from the padded end where all are computed)."""
    if c["sq"] == c["sk"]:
        return [0] * c["b"]
    return [max(0, n - c["sq"]) for n in _lengths(c)]


def _prefixes(c):
    return [(c["sk"] * (i + 1)) // (2 * c["b"] + 1) for i in range(c["b"])]


def _cuts(c):
    """First token of each packed document, and the end."""
    n = c["docs"]
    return sorted({round(c["sk"] * (i / n) ** 1.3) for i in range(n)} | {0, c["sk"]})


def _pairs(c):
    """Visible (query, key) pairs over the batch, for one head."""
    total = 0
    for n, st, pre in zip(_lengths(c), _starts(c), _prefixes(c)):
        if c["docs"]:
            cut = _cuts(c)
            total += sum((b - a) * (b - a + 1) // 2 if c["causal"] else (b - a) ** 2 for a, b in zip(cut, cut[1:]))
        elif not c["causal"]:
            total += c["sq"] * n
        else:
            total += sum(min(n, max(st + i + 1, pre if c["prefix"] else 0)) for i in range(c["sq"]))
    return total


def work(c):
    if c["kind"] == "round":      # bf16 in, 4-bit + scale bytes out; the same bytes in, bf16 out
        n, blocks = c["rows"] * c["k"], c["rows"] * ((c["k"] + 31) // 32)
        return {"bytes": 4 * n + 2 * ((n + 1) // 2 + blocks), "flops": 4 * n}
    if c["kind"] == "linear":     # bf16 activations in, 4-bit weight + scales in, bf16 out (+ residual in)
        m, n, k = c["m"], c["n"], c["k"]
        by = 2 * m * k + n * ((k + 1) // 2 + (k + 31) // 32) + 2 * m * n
        by += {"plain": 0, "bias": 4 * n, "gelu": 4 * n, "residual": 2 * m * n + 8 * n}[c["epi"]]
        return {"bytes": by, "flops": 2 * m * n * k}
    keys = sum(_lengths(c))
    by = 2 * c["d"] * (2 * c["b"] * c["sq"] * c["hq"] + 2 * keys * c["hkv"]) + (4 * c["hq"] * (2 * c["reach"] + 1) if c["reach"] else 0)
    by += 8 * c["b"] * c["sk"] if c["docs"] else 0
    return {"bytes": by, "flops": 4 * c["d"] * c["hq"] * _pairs(c)}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, rows, k):
    """Hidden states of a decoder: unit rows with a few channels far above the rest, in bf16."""
    x = torch.randn(rows, k, generator=g, device=DEV)
    gain = torch.ones(k, device=DEV)
    gain[torch.randint(0, k, (max(1, k // 256),), generator=g, device=DEV)] = 20.0
    return x.mul_(gain).to(torch.bfloat16)


def _inputs(c, seed):
    """The tensors of a case, from the seed alone."""
    g = _gen(seed)
    if c["kind"] == "round":
        return {"x": _activations(g, c["rows"], c["k"])}
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        s = {"x": _activations(g, m, k), "w": (torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)).to(torch.bfloat16)}
        if c["epi"] != "plain":
            s["bias"] = 0.1 * torch.randn(n, generator=g, device=DEV)
        if c["epi"] == "residual":
            s["res"] = torch.randn(m, n, generator=g, device=DEV).to(torch.bfloat16)
            s["gate"] = torch.randn(n, generator=g, device=DEV)
        return s
    b, sq, sk, hq, hkv, d = (c[x] for x in ("b", "sq", "sk", "hq", "hkv", "d"))

    def heads(s, h):       # a projection's output seen as heads: [b, s, h, d] memory, [b, h, s, d] view
        return torch.randn(b, s, h, d, generator=g, device=DEV).to(torch.bfloat16).transpose(1, 2)
    s = {"q": heads(sq, hq)}
    if sq == sk:
        s["k"], s["v"] = heads(sk, hkv), heads(sk, hkv)
    else:                  # a cache: one run of rows per head
        s["k"], s["v"] = heads(sk, hkv).contiguous(), heads(sk, hkv).contiguous()
    if c["reach"]:
        s["bias"] = torch.randn(hq, 2 * c["reach"] + 1, generator=g, device=DEV)
    i32 = {"dtype": torch.int32, "device": DEV}
    if c["docs"]:
        cut = _cuts(c)
        ids = torch.cat([torch.full((e - a,), i, **i32) for i, (a, e) in enumerate(zip(cut, cut[1:]))])
        s["docs"] = ids.repeat(b, 1).contiguous()
    if c["ragged"]:
        s["valid"] = torch.tensor(_lengths(c), **i32)
    if c["prefix"]:
        s["prefix"] = torch.tensor(_prefixes(c), **i32)
    if sq != sk:
        s["start"] = torch.tensor(_starts(c), **i32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "linear":       # the weight is stored once and kept
        if own:
            from easyanimate_amd import ops
            s["w"] = ops.mxfp4_quantize(s["w"])
        else:
            s["w"] = _microscale(s["w"]).to(torch.bfloat16)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------
def _microscale(x):
    """The fp32 values that 4-bit storage of x's rows stands for: blocks of 32 share 2^(floor(log2 max|x|) - 2), clamped to the range
    of an 8-bit exponent; elements are the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (ties to the even code, 6 at most); a block
    that holds an infinity or a NaN is NaN."""
    rows, k = x.shape
    pad = -k % 32
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    exponent = (((top.view(torch.int32) >> 23) & 255) - 129).clamp(-127, 127)      # subnormal and zero blocks: the least exponent
    scale = ((exponent.long() + 1023) << 52).view(torch.float64)                   # 2^exponent from its bits: exact
    a = v.double().abs() / scale                                                   # exact, borders included
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    a = (torch.round(a / step) * step).clamp(max=6.0)
    out = torch.copysign(a * scale, v.double()).float()
    out = torch.where(torch.isfinite(top), out, torch.full_like(out, float("nan")))
    return out.view(rows, -1)[:, :k]


def _plain_linear(s, epi):
    y = _microscale(s["x"]) @ s["w"].float().t()
    if epi != "plain":
        y = y + s["bias"]
    if epi == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if epi == "residual":
        y = s["res"].float() + s["gate"] * y
    return y.to(torch.bfloat16)


def _visible(c, s, i, lo, hi):
    """Truth table [hi - lo, sk] of batch element i: which keys queries lo .. hi - 1 see."""
    key = torch.arange(c["sk"], device=DEV)
    pos = torch.arange(lo, hi, device=DEV) + (s["start"][i] if "start" in s else 0)
    see = torch.ones(hi - lo, c["sk"], dtype=torch.bool, device=DEV)
    if c["causal"]:
        see = key[None, :] <= pos[:, None]
        if c["prefix"]:
            see = see | (key < s["prefix"][i])[None, :]
    if c["docs"]:
        see = see & (s["docs"][i][None, :] == s["docs"][i, lo:hi][:, None])
    if c["ragged"]:
        see = see & (key < s["valid"][i])[None, :]
    return see, (key[None, :] - pos[:, None]).clamp(-c["reach"], c["reach"]) + c["reach"]


def _plain_attention(s, c):
    group = c["hq"] // c["hkv"]
    out = torch.empty(c["b"], c["sq"], c["hq"], c["d"], dtype=torch.bfloat16, device=DEV)
    rows = max(1, min(c["sq"], (1 << 28) // (group * c["sk"])))
    for i in range(c["b"]):
        for lo in range(0, c["sq"], rows):
            hi = min(c["sq"], lo + rows)
            see, dist = _visible(c, s, i, lo, hi)
            for h in range(c["hkv"]):
                hs = slice(h * group, (h + 1) * group)
                t = s["q"][i, hs, lo:hi].float() @ s["k"][i, h].float().t() * c["d"] ** -0.5
                if c["cap"]:
                    t = c["cap"] * torch.tanh(t / c["cap"])
                if c["reach"]:
                    t = t + s["bias"][hs][:, dist]
                t = torch.where(see, t, float("-inf"))
                top = t.amax(-1, keepdim=True)
                p = torch.exp(t - torch.where(top == float("-inf"), 0.0, top))
                total = p.sum(-1, keepdim=True)
                o = (p @ s["v"][i, h].float()) / torch.where(total == 0, 1.0, total)
                out[i, lo:hi, hs] = o.transpose(0, 1).to(torch.bfloat16)
    return out.view(c["b"], c["sq"], -1)


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        if c["kind"] == "round":
            return _microscale(s["x"]).to(torch.bfloat16)
        return _plain_linear(s, c["epi"]) if c["kind"] == "linear" else _plain_attention(s, c)
    from easyanimate_amd import ops
    if c["kind"] == "round":
        return ops.mxfp4_dequantize(ops.mxfp4_quantize(s["x"]))
    if c["kind"] == "linear":
        epi = {"plain": ops.EPI_BIAS, "bias": ops.EPI_BIAS, "gelu": ops.EPI_BIAS_GELU_TANH, "residual": ops.EPI_BIAS_GATE_RES}[c["epi"]]
        return ops.gemm_mxfp4(s["x"], s["w"], s.get("bias"), epi, res=s.get("res"), gate=s.get("gate"))
    return ops.attention_text(s["q"], s["k"], s["v"], c["d"] ** -0.5, causal=c["causal"], cap=c["cap"], bias=s.get("bias"),
                              q_docs=s.get("docs"), kv_docs=s.get("docs"), prefix=s.get("prefix"), valid=s.get("valid"),
                              q_start=s.get("start"))


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_blocks(x):
    """4-bit storage by search: the eight magnitudes of a 2-bit exponent / 1-bit mantissa number, the nearest one taken."""
    x = x.double()
    rows, k = x.shape
    full = x.new_zeros(rows, (k + 31) // 32 * 32)
    full[:, :k] = x
    full = full.reshape(-1, 32)
    out = torch.empty_like(full)
    powers = torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64, device=x.device)
    mags = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    for lo in range(0, full.shape[0], 1 << 17):
        blk = full[lo:lo + (1 << 17)]
        big = blk.abs().max(1).values
        ok = torch.isfinite(big)
        e = torch.frexp(torch.where(ok & (big > 0), big, torch.ones_like(big))).exponent - 3     # floor(log2 big) - 2
        e = torch.where(big > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
        unit = powers[(e + 127).long()][:, None]
        scaled = blk.abs() / unit
        best = torch.zeros_like(scaled)
        near = torch.full_like(scaled, float("inf"))
        for code in (0, 2, 4, 6, 1, 3, 5, 7):           # even codes first: a tie stays with them
            gap = (scaled - mags[code]).abs()
            take = gap < near
            best = torch.where(take, mags[code], best)
            near = torch.where(take, gap, near)
        val = best * unit * torch.where(torch.signbit(blk), -1.0, 1.0)
        out[lo:lo + (1 << 17)] = torch.where(ok[:, None], val, torch.full_like(val, float("nan")))
    return out.reshape(rows, -1)[:, :k]


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "round":
        return _exact_blocks(s["x"])
    if c["kind"] == "linear":
        y = torch.mm(_exact_blocks(s["x"]), _exact_blocks(s["w"]).t().contiguous())
        if "bias" in s:
            y += s["bias"].double()[None, :]
        if c["epi"] == "gelu":
            inner = (2.0 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)
            y = y * torch.sigmoid(2.0 * inner)
        if c["epi"] == "residual":
            y = s["gate"].double()[None, :] * y + s["res"].double()
        return y
    out = torch.zeros(c["b"], c["sq"], c["hq"] * c["d"], dtype=torch.float64, device=DEV)
    keys = torch.arange(c["sk"], device=DEV)
    for i in range(c["b"]):
        n, st, pre = _lengths(c)[i], _starts(c)[i], _prefixes(c)[i]
        for lo in range(0, c["sq"], 2048):
            hi = min(lo + 2048, c["sq"])
            at = torch.arange(st + lo, st + hi, device=DEV).unsqueeze(1)
            hide = (keys >= n).expand(hi - lo, -1)
            if c["causal"]:
                later = keys > at
                hide = hide | (later & (keys >= pre) if c["prefix"] else later)
            if c["docs"]:
                hide = hide | (s["docs"][i, lo:hi].unsqueeze(1) != s["docs"][i].unsqueeze(0))
            for h in range(c["hq"]):
                kv = h // (c["hq"] // c["hkv"])
                t = torch.mm(s["q"][i, h, lo:hi].double(), s["k"][i, kv].double().t().contiguous()) / math.sqrt(c["d"])
                if c["cap"]:
                    t = torch.tanh(t / c["cap"]) * c["cap"]
                if c["reach"]:
                    far = (keys - at).clamp(min=-c["reach"], max=c["reach"])
                    t += s["bias"][h].double()[far + c["reach"]]
                t.masked_fill_(hide, float("-inf"))
                w = torch.nan_to_num(torch.softmax(t, dim=1), nan=0.0)
                out[i, lo:hi, h * c["d"]:(h + 1) * c["d"]] = torch.mm(w, s["v"][i, kv].double())
    return out
