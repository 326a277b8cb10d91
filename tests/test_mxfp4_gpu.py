"""Microscaled 4-bit storage and its product (ea_mxfp4.hip, ea_gemm_mxfp4.hip) against plain 64-bit implementations on the host:
storage bit for bit, products within the roundings that the kernels make."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
MAGS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def store(x):
    """Codes uint8 [rows, kp], scale bytes uint8 [rows, kp / 32] of x [rows, K] (kp = K padded to whole 256-element tiles)."""
    rows, K = x.shape
    kp = (K + 255) // 256 * 256
    v = torch.zeros(rows, kp, dtype=torch.float64)
    v[:, :K] = x.double()
    blk = v.view(rows, -1, 32)
    top = blk.abs().amax(-1)
    finite = torch.isfinite(top)
    safe = torch.where(finite & (top > 0), top, torch.ones_like(top))
    e = torch.frexp(safe).exponent.long() - 3
    byte = torch.where(top > 0, e + 127, torch.zeros_like(e)).clamp(0, 254)
    byte = torch.where(finite, byte, torch.full_like(byte, 255))
    unit = torch.tensor([2.0 ** (b - 127) for b in range(256)], dtype=torch.float64)[byte][..., None]
    a = (torch.where(finite[..., None], blk, torch.zeros_like(blk)).abs() / unit)
    gap = (a[..., None] - MAGS).abs()
    # the nearest magnitude; a tie goes to the even code
    cand = gap == gap.amin(-1, keepdim=True)
    even = torch.where(cand & (torch.arange(8) % 2 == 0), torch.arange(8), 8).amin(-1)
    code = torch.where(even < 8, even, torch.where(cand, torch.arange(8), 8).amin(-1))
    neg = torch.signbit(blk) & finite[..., None]
    return (code + 8 * neg.long()).to(torch.uint8).view(rows, kp), byte.to(torch.uint8).view(rows, kp // 32)


def values(codes, byte):
    """fp64 values of stored codes [rows, kp] / bytes [rows, kp / 32]."""
    unit = torch.tensor([2.0 ** (b - 127) for b in range(255)] + [float("nan")], dtype=torch.float64)[byte.long()]
    mag = MAGS[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    return (mag.view(*byte.shape, 32) * unit[..., None]).view(codes.shape)


def unpack(q):
    """ops.Mxfp4 -> (codes [rows, kp], bytes [rows, kp / 32]) on the host."""
    c = q.codes.cpu().permute(1, 0, 2).reshape(q.rows, -1)
    kt = q.codes.shape[0]
    s = q.scales.cpu().permute(1, 0, 2).reshape(q.rows, kt, 4, 2).transpose(2, 3)        # block 4 j + g at byte 2 g + j
    return torch.stack([c & 15, c >> 4], -1).view(q.rows, kt * 256), s.reshape(q.rows, kt * 8)


def _same_storage(x):
    from easyanimate_amd import ops
    q = ops.mxfp4_quantize(x if x.is_cuda else x.to(DEV))
    codes, byte = unpack(q)
    want_codes, want_byte = store(x.cpu())
    assert torch.equal(byte, want_byte)
    assert torch.equal(codes, want_codes)
    back = ops.mxfp4_dequantize(q).cpu()
    want = values(want_codes, want_byte)[:, :x.shape[1]]
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(back.double(), nan=7.0), torch.nan_to_num(want, nan=7.0))
    return q


def test_every_bf16_value():
    """All 65 536 bf16 patterns, sorted (blocks of like magnitude: every border of every code) and shuffled (blocks of mixed ones)."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    _same_storage(x.view(256, 256))
    fin = x[torch.isfinite(x)]
    g = torch.Generator().manual_seed(1)
    _same_storage(fin[torch.randperm(fin.numel(), generator=g)][:65024].view(254, 256))
    # one magnitude range at a time: each block holds every mantissa of two neighbouring binades and subnormals among them
    _same_storage(torch.arange(0, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)[:32512].view(127, 256))


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 255), (2, 256), (7, 257), (4, 1477), (130, 3584), (33, 40), (65, 520)])
def test_sizes(rows, K):
    g = torch.Generator().manual_seed(rows * 7919 + K)
    x = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())).bfloat16()
    x[0, 0] = 0.0
    _same_storage(x)


def test_zero_nan_and_infinite_blocks():
    x = torch.randn(4, 96).bfloat16()
    x[0, :32] = 0.0
    x[0, 5] = -0.0
    x[1, 40] = float("nan")
    x[2, 70] = float("inf")
    x[3, 0] = float("-inf")
    x[3, 1] = float("nan")
    x[1, :32] = torch.tensor(1e-40).bfloat16()           # a block of subnormals
    x[2, :32] = torch.finfo(torch.bfloat16).max
    q = _same_storage(x)
    _, byte = unpack(q)
    assert byte[1, 1] == 255 and byte[2, 2] == 255 and byte[3, 0] == 255 and byte[0, 0] == 0


def test_strides_alignment_and_orders():
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(40, 700, generator=g).bfloat16().to(DEV)
    _same_storage(wide[:, 8:328])            # rows 16-byte aligned, stride 700: not a multiple of 8
    _same_storage(wide[:, 3:67])             # an odd element offset
    _same_storage(wide[::3, :256])           # every third row
    _same_storage(wide.t()[:64])             # transposed: inner stride 700
    _same_storage(wide[:1].expand(5, 700))   # one row five times (stride 0)
    odd = torch.randn(3, 7, 512, generator=g).bfloat16().to(DEV)
    _same_storage(odd[:, 2, :])


def test_no_rows():
    from easyanimate_amd import ops
    q = ops.mxfp4_quantize(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV))
    assert q.rows == 0 and ops.mxfp4_dequantize(q).shape == (0, 64)


def test_every_code_and_scale_read_back():
    """All 16 codes under all 256 scale bytes."""
    from easyanimate_amd import ops
    codes = torch.arange(16, dtype=torch.uint8).repeat(256, 16)                     # 256 rows of 256 elements
    byte = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 8)
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).view(1, 256, 128)
    q = ops.Mxfp4(packed.contiguous().to(DEV), byte.view(1, 256, 8).contiguous().to(DEV), 256, 256)
    got = ops.mxfp4_dequantize(q).cpu()
    want = values(codes, byte)
    fits = torch.isnan(want) | (want.abs() <= torch.finfo(torch.bfloat16).max)      # 2^127 * 2 and above are infinities in bf16
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.double(), nan=0.0)[fits], torch.nan_to_num(want, nan=0.0)[fits])
    assert torch.isinf(got[~fits]).all()


# ---- the product -----------------------------------------------------------------------------------------------------------------
def _expected(av, wv, bias, epi, res, gate):
    """fp64 result and an elementwise bound on the kernel's error.  Products of two e2m1 codes and two powers of two are exact; K of
    them are added in fp32 in some order: at most K additions, each off by at most 2^-23 of the running magnitude sum (a half step
    is 2^-24; the matrix unit may cut instead of round).  Then one fp32 operation per epilogue step and one rounding to bf16 (2^-8;
    fp32 out: none).  GELU's slope is below 1.13 and its exponential and reciprocal are good to 2^-20 of its value."""
    from easyanimate_amd import ops
    y = av @ wv.transpose(-1, -2)
    mag = av.abs() @ wv.abs().transpose(-1, -2)
    err = av.shape[-1] * 2.0 ** -23 * mag
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -23 * y.abs()
    if epi == ops.EPI_BIAS_GELU_TANH:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        err = 1.13 * err + 2.0 ** -20 * y.abs()
    if epi == ops.EPI_BIAS_GATE_RES:
        y = res.double() + gate.double()[..., None, :] * y
        err = gate.double().abs()[..., None, :] * err + 2.0 ** -23 * y.abs()
    if epi != ops.EPI_F32_OUT:
        err = err * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs()
    return y, err + 1e-37


def _operands(M, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    x[:, torch.randint(0, K, (max(1, K // 64),), generator=g)] *= 20
    w = torch.randn(N, K, generator=g) / math.sqrt(K)
    return x.bfloat16(), w.bfloat16(), g


def _check(got, y, err):
    bad = ((got.double().cpu() - y).abs() > err)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst ratio {((got.double().cpu() - y).abs() / err).max().item():.3g}"


EPIS = ["plain", "bias", "gelu", "residual", "f32"]


def _run(x, w, N, epi, g, packed=False, kern=None):
    from easyanimate_amd import _lib, ops
    M = x.shape[-2]
    bias = torch.randn(N, generator=g) if epi != "plain" else None
    res = torch.randn(*x.shape[:-1], N, generator=g).bfloat16() if epi == "residual" else None
    gate = torch.randn(*x.shape[:-2], N, generator=g) if epi == "residual" else None
    code = {"plain": ops.EPI_BIAS, "bias": ops.EPI_BIAS, "gelu": ops.EPI_BIAS_GELU_TANH, "residual": ops.EPI_BIAS_GATE_RES, "f32": ops.EPI_F32_OUT}[epi]
    up = lambda t: None if t is None else t.to(DEV)
    W = ops.mxfp4_quantize(w.to(DEV))
    A = ops.mxfp4_quantize(x.to(DEV)) if packed else x.to(DEV)
    _lib.reset_counters()
    got = ops.gemm_mxfp4(A, W, up(bias), code, res=up(res), gate=up(gate))
    if kern:
        assert _lib.counters().get(kern) == 1, _lib.counters()
    K = x.shape[-1]
    av = values(*store(x.reshape(-1, K)))[:, :K].view(x.shape)
    wv = values(*store(w))[:, :K]
    y, err = _expected(av, wv, bias, code, res, gate)
    assert got.shape == y.shape and got.dtype == (torch.float32 if epi == "f32" else torch.bfloat16)
    _check(got, y, err)
    return got


@pytest.mark.parametrize("epi", EPIS)
@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (1, 512, 3584), (3, 24, 1000), (16, 136, 264), (17, 72, 520), (40, 200, 777), (64, 64, 256),
                                   (65, 136, 96), (128, 128, 256), (129, 264, 1161), (200, 1000, 2304), (300, 392, 40)])
def test_product(M, N, K, epi):
    x, w, g = _operands(M, N, K, M * 31 + N + K)
    _run(x, w, N, epi, g)


@pytest.mark.parametrize("M,N,K,kern", [(1, 64, 512, "gemm_mxfp4_skinny_bf16"), (1, 64, 513, "gemm_mxfp4_skinny"), (32, 64, 512, "gemm_mxfp4_skinny"),
                                        (33, 64, 512, "gemm_mxfp4_64x64"), (20, 8200, 300, "gemm_mxfp4_64x64"),
                                        (300, 392, 40, "gemm_mxfp4_64x64"), (70, 136, 13000, "gemm_mxfp4_64x64_split"),
                                        (500, 3200, 1100, "gemm_mxfp4_128x64"), (900, 4000, 700, "gemm_mxfp4_128x128"), (1900, 4072, 264, "gemm_mxfp4_256x128"),
                                        (257, 16000, 520, "gemm_mxfp4_256x128")])
def test_product_variants(M, N, K, kern):
    x, w, g = _operands(M, N, K, M + K)
    _run(x, w, N, "bias", g, kern=kern)


@pytest.mark.parametrize("epi", ["plain", "bias", "gelu", "residual"])
@pytest.mark.parametrize("M,N,K", [(3900, 4000, 96), (3841, 3848, 512), (4096, 4096, 513), (3999, 4088, 1100)])
def test_product_large_tiles(M, N, K, epi):
    """The 256 x 256 kernel: one to five K tiles, ragged rows, columns and K, every epilogue; codes handed over give the same bits."""
    from easyanimate_amd import ops
    x, w, g = _operands(M, N, K, M + K)
    got = _run(x, w, N, epi, g, kern="gemm_mxfp4_256_w4")
    if epi == "plain":
        assert torch.equal(got, ops.gemm_mxfp4(ops.mxfp4_quantize(x.to(DEV)), ops.mxfp4_quantize(w.to(DEV)), None)) or M % 2


def test_product_large_tiles_batched():
    x, w, g = _operands(2 * 1999, 4000, 600, 5)
    _run(x.view(2, 1999, 600), w, 4000, "residual", g, kern="gemm_mxfp4_256_w4")


@pytest.mark.parametrize("M", [1, 16, 30, 90])
def test_product_of_stored_activations_is_the_same(M):
    """Quantising inside the product, in front of it, or by the caller: the same codes, so the same bits."""
    from easyanimate_amd import ops
    x, w, _ = _operands(M, 144, 840, 11)
    W = ops.mxfp4_quantize(w.to(DEV))
    a = ops.gemm_mxfp4(x.to(DEV), W, None)
    b = ops.gemm_mxfp4(ops.mxfp4_quantize(x.to(DEV)), W, None)
    assert torch.equal(a, b)


@pytest.mark.parametrize("B,M,N,K", [(3, 5, 48, 320), (2, 70, 136, 512), (4, 1, 64, 96)])
@pytest.mark.parametrize("epi", ["gelu", "residual"])
def test_product_batched(B, M, N, K, epi):
    x, w, g = _operands(B * M, N, K, B + M)
    _run(x.view(B, M, K), w, N, epi, g)


def test_product_writes_where_it_is_told():
    """A strided output (columns of a wider buffer), the residual read from the output itself, everything beside it left alone."""
    from easyanimate_amd import ops
    x, w, g = _operands(90, 72, 384, 3)
    W = ops.mxfp4_quantize(w.to(DEV))
    gate = torch.randn(72, generator=g)
    wide = torch.randn(94, 96, generator=g).bfloat16()
    buf = wide.to(DEV)
    view = buf[2:92, 8:80]
    ops.gemm_mxfp4(x.to(DEV), W, None, ops.EPI_BIAS_GATE_RES, out=view, res=view, gate=gate.to(DEV))
    av, wv = values(*store(x))[:, :384], values(*store(w))[:, :384]
    _check(buf[2:92, 8:80], *_expected(av, wv, None, ops.EPI_BIAS_GATE_RES, wide[2:92, 8:80], gate))
    after = buf.cpu()
    after[2:92, 8:80] = wide[2:92, 8:80]
    assert torch.equal(after, wide)


@pytest.mark.parametrize("M", [2, 20, 140])
def test_nan_blocks_reach_their_rows_and_columns_only(M):
    from easyanimate_amd import ops
    x, w, _ = _operands(M, 64, 300, 8)
    x[1, 290] = float("inf")
    w[7, 3] = float("nan")
    y = ops.gemm_mxfp4(x.to(DEV), ops.mxfp4_quantize(w.to(DEV)), None).cpu()
    want = torch.zeros(M, 64, dtype=torch.bool)
    want[1], want[:, 7] = True, True
    assert torch.equal(torch.isnan(y), want)


def test_far_apart_scales():
    """Blocks 2^80 apart in one row: the small ones vanish beside the large ones as in the fp64 sum, and alone they are exact."""
    from easyanimate_amd import ops
    x, w, _ = _operands(70, 64, 512, 9)
    x[:35, :256] *= 2.0 ** 40
    x[35:, :] *= 2.0 ** -40
    got = ops.gemm_mxfp4(x.to(DEV), ops.mxfp4_quantize(w.to(DEV)), None, ops.EPI_F32_OUT)
    _check(got, *_expected(values(*store(x)), values(*store(w)), None, ops.EPI_F32_OUT, None, None))


def test_no_rows_no_launch():
    from easyanimate_amd import ops
    W = ops.mxfp4_quantize(torch.randn(16, 64).bfloat16().to(DEV))
    assert ops.gemm_mxfp4(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), W, None).shape == (0, 16)


@pytest.mark.parametrize("M,K", [(1, 512), (100, 13000)])
def test_side_stream_and_graph(M, K):
    """On a stream of its own, and captured: replayed with new inputs between eager calls, every replay equals the eager result."""
    from easyanimate_amd import ops
    x, w, _ = _operands(M, 256, K, 21)
    W = ops.mxfp4_quantize(w.to(DEV))
    xs = [x.to(DEV), (x * 0.5).to(DEV), x.flip(0).to(DEV)]
    eager = [ops.gemm_mxfp4(t, W, None) for t in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gemm_mxfp4(xs[0], W, None)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, eager[0])
    buf = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gemm_mxfp4(buf, W, None)
    for i in (1, 2, 0, 1):
        buf.copy_(xs[i])
        graph.replay()
        assert torch.equal(out, eager[i])
        assert torch.equal(ops.gemm_mxfp4(xs[i], W, None), eager[i])
        torch.cuda.synchronize()


def test_a_decoder_mlp_in_4_bits():
    """The operators as they are used together: down(silu(gate(x)) * up(x)) + x with the three weights in 4-bit storage."""
    from easyanimate_amd import ops
    g = torch.Generator().manual_seed(2)
    d, inter, M = 512, 1536, 96
    x = torch.randn(M, d, generator=g).bfloat16()
    wg, wu = (torch.randn(inter, d, generator=g) / math.sqrt(d)).bfloat16(), (torch.randn(inter, d, generator=g) / math.sqrt(d)).bfloat16()
    wd = (torch.randn(d, inter, generator=g) / math.sqrt(inter)).bfloat16()
    q = {n: ops.mxfp4_quantize(t.to(DEV)) for n, t in (("g", wg), ("u", wu), ("d", wd))}
    xa = ops.mxfp4_quantize(x.to(DEV))
    act = ops.silu_mul(ops.gemm_mxfp4(xa, q["g"], None), ops.gemm_mxfp4(xa, q["u"], None))
    got = ops.gemm_mxfp4(act, q["d"], None, ops.EPI_BIAS_GATE_RES, res=x.to(DEV), gate=torch.ones(d, device=DEV))
    # the last product from the activation the GPU stored: everything up to it is covered above
    _check(got, *_expected(values(*store(act.cpu())), values(*store(wd)), None, ops.EPI_BIAS_GATE_RES, x, torch.ones(d)))
    av = values(*store(x))
    gate, up = av @ values(*store(wg)).t(), av @ values(*store(wu)).t()
    want = torch.nn.functional.silu(gate) * up
    # gate and up carry one bf16 rounding each, silu_mul one more: |d| <= (1.1 |up| 2^-8 |gate| + |silu| 2^-8 |up|) + 2^-8 |want|
    tol = 2.0 ** -8 * (1.1 * (up * gate).abs() + 2 * want.abs()) * 1.02 + 1e-4
    assert ((act.cpu().double() - want).abs() <= tol).all()
