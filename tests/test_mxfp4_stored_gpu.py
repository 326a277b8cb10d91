"""gemm_mxfp4 on activations that the caller has stored (ops.Mxfp4): every kernel and epilogue against the 64-bit product, and bit for bit
what the same activations give in bf16 -- the encoder's q / k / v and gate / up products are such calls."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from test_mxfp4_gpu import DEV, EPIS, _operands, _run

pytestmark = pytest.mark.gpu

# (M, N, K, the kernel that stored activations take; with fp32 results)
SIZES = [(1, 64, 513, "gemm_mxfp4_skinny", None), (16, 136, 512, "gemm_mxfp4_skinny", None), (29, 72, 520, "gemm_mxfp4_skinny", None),
         (257, 512, 700, "gemm_mxfp4_64x64", None), (71, 136, 13000, "gemm_mxfp4_64x64_split", None), (501, 3200, 1100, "gemm_mxfp4_128x64", None),
         (901, 4000, 700, "gemm_mxfp4_128x128", None), (257, 16000, 520, "gemm_mxfp4_256x128", None),
         (3841, 3848, 512, "gemm_mxfp4_256_w4", "gemm_mxfp4_256x128"), (3999, 4088, 1100, "gemm_mxfp4_256_w4", "gemm_mxfp4_256x128"),
         (3900, 4000, 96, "gemm_mxfp4_256_w4", "gemm_mxfp4_256x128")]


@pytest.mark.parametrize("epi", EPIS)
@pytest.mark.parametrize("M,N,K,kern,f32", SIZES)
def test_stored_activations(M, N, K, kern, f32, epi):
    from easyanimate_amd import ops
    x, w, g = _operands(M, N, K, M + 2 * K)
    state = g.get_state()
    got = _run(x, w, N, epi, g, packed=True, kern=f32 if epi == "f32" and f32 else kern)
    g.set_state(state)                                   # the same bias, residual and gate again (_run's order)
    bias = torch.randn(N, generator=g).to(DEV) if epi != "plain" else None
    res = torch.randn(M, N, generator=g).bfloat16().to(DEV) if epi == "residual" else None
    gate = torch.randn(N, generator=g).to(DEV) if epi == "residual" else None
    code = {"gelu": ops.EPI_BIAS_GELU_TANH, "residual": ops.EPI_BIAS_GATE_RES, "f32": ops.EPI_F32_OUT}.get(epi, ops.EPI_BIAS)
    assert torch.equal(got, ops.gemm_mxfp4(x.to(DEV), ops.mxfp4_quantize(w.to(DEV)), bias, code, res=res, gate=gate))


@pytest.mark.parametrize("B,M,kern", [(2, 1999, "gemm_mxfp4_256_w4"), (3, 1279, "gemm_mxfp4_256_w4"), (2, 1998, "gemm_mxfp4_256_w4"), (3, 1411, "gemm_mxfp4_256x128")])
def test_stored_batches(B, M, kern):
    """Elements of an odd number of rows behind one another (the C entry point): their scales begin at odd rows."""
    from easyanimate_amd import _lib, ops
    N, K = 4000, 600
    x, w, _ = _operands(B * M, N, K, B + M)
    X, W = x.to(DEV), ops.mxfp4_quantize(w.to(DEV))
    A = ops.mxfp4_quantize(X)
    want = ops.gemm_mxfp4(X.view(B, M, K), W, None)
    out = torch.full((B, M, N), 7.0, dtype=torch.bfloat16, device=DEV)
    need = _lib.load().ea_gemm_mxfp4_workspace_bytes(B, M, N, K, 0)
    assert (need > 0) == (M % 2 == 1 and kern == "gemm_mxfp4_256_w4")
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    _lib.reset_counters()
    _lib.call("ea_gemm_mxfp4", A.codes.data_ptr(), A.scales.data_ptr(), None, W.codes.data_ptr(), W.scales.data_ptr(), None, out.data_ptr(), None, None,
              B, M, N, K, 0, 0, N, M * N, 0, 0, 0, ops.EPI_BIAS, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert _lib.counters() == {kern: 1}
    assert torch.equal(out, want)


def test_stored_odd_rows_in_a_graph():
    """The copy of the scales is part of the call: replays with other activations, and two graphs, each with a workspace of its own."""
    from easyanimate_amd import ops
    M, N, K = 3841, 3848, 512
    x, w, _ = _operands(M, N, K, 4)
    W = ops.mxfp4_quantize(w.to(DEV))
    xs = [x.to(DEV), (x * 0.25).to(DEV), x.flip(0).to(DEV)]
    stored = [ops.mxfp4_quantize(t) for t in xs]
    want = [ops.gemm_mxfp4(t, W, None) for t in xs]
    buf = [ops.Mxfp4(stored[0].codes.clone(), stored[0].scales.clone(), M, K) for _ in range(2)]
    graphs, outs = [], []
    for b in buf:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.gemm_mxfp4(b, W, None))
        graphs.append(g)
    for i, j in ((1, 2), (2, 0), (0, 1)):
        for b, n in zip(buf, (i, j)):
            b.codes.copy_(stored[n].codes)
            b.scales.copy_(stored[n].scales)
        for g in graphs:
            g.replay()
        assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[j])
        assert torch.equal(ops.gemm_mxfp4(stored[i], W, None), want[i])
