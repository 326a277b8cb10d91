"""What the 4-bit product and the text attention have to survive beside their mathematics: offsets past 32 bits, calls at the same time on
several streams, captured graphs replayed in turn, results written over the residual, outputs whose rows overlap."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from test_attention_text_gpu import check, i32, make, plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture()
def roomy():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("Sq", [1, 12, 100])
def test_a_cache_of_more_than_2_to_the_31_elements(Sq, roomy):
    """Only the last 40 keys belong to the queries' document; everything in front of them is NaN."""
    from easyanimate_amd import ops
    Hq, Hkv, D, Sk, n = 4, 2, 128, 8_500_003, 40
    g = torch.Generator().manual_seed(Sq)
    q = torch.randn(1, Hq, Sq, D, generator=g).bfloat16()
    tail = [torch.randn(1, Hkv, n, D, generator=g).bfloat16() for _ in range(2)]
    cache = []
    for t in tail:
        c = torch.full((1, Sk, Hkv, D), float("nan"), dtype=torch.bfloat16, device=DEV)
        assert c.numel() > 2 ** 31
        c[:, -n:] = t.transpose(1, 2).to(DEV)
        cache.append(c.transpose(1, 2))
    docs = torch.zeros(1, Sk, dtype=torch.int32, device=DEV)
    docs[:, -n:] = 7
    got = ops.attention_text(q.to(DEV), *cache, D ** -0.5, causal=True, q_docs=torch.full((1, Sq), 7, dtype=torch.int32, device=DEV), kv_docs=docs)
    want, err = plain(q, *tail, D ** -0.5, causal=True, q_start=i32(n - Sq))
    # (hidden keys leave no trace, but the row sums of the plain form's bound know 40 keys only: the same weights, summed elsewhere)
    assert ((got.cpu().double() - want).abs() <= err).all()


def test_matrices_of_more_than_2_to_the_31_elements(roomy):
    from easyanimate_amd import ops
    rows, K = 600_008, 3600
    x = torch.empty(rows, K, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(DEV).manual_seed(1))
    q = ops.mxfp4_quantize(x)
    for part in (slice(0, 64), slice(rows - 64, rows)):
        alone = ops.mxfp4_quantize(x[part])
        assert torch.equal(q.codes[:, part], alone.codes) and torch.equal(q.scales[:, part], alone.scales)
    back = ops.mxfp4_dequantize(q)
    assert torch.equal(back[-64:], ops.mxfp4_dequantize(ops.mxfp4_quantize(x[-64:])))
    del back
    w = ops.mxfp4_quantize(x[:64] * 0.5)
    many = ops.gemm_mxfp4(q, w, None)                     # as activations
    assert torch.equal(many[-40:], ops.gemm_mxfp4(x[-40:], w, None))
    del many
    wide = ops.gemm_mxfp4(x[:3], q, None)                 # as weights
    assert torch.equal(wide[:, -64:], ops.gemm_mxfp4(x[:3], ops.mxfp4_quantize(x[-64:]), None))
    wide = ops.gemm_mxfp4(x[:100], q, None)
    assert torch.equal(wide[:, -64:], ops.gemm_mxfp4(x[:100], ops.mxfp4_quantize(x[-64:]), None))


@pytest.mark.parametrize("Sq", [1, 9, 70])
@pytest.mark.parametrize("reach", [0, 3, 1000])
def test_positions_and_lengths_outside_the_cache(Sq, reach):
    far = (2 ** 31 - 1, -2 ** 31, 5, -3, 200)
    q, k, v, g = make(5, 4, 2, Sq, 90, 64, Sq + reach)
    bias = torch.randn(4, 2 * reach + 1, generator=g)
    check(q, k, v, 0.125, causal=True, bias=bias, q_start=i32(*far))
    check(q, k, v, 0.125, causal=True, bias=bias, prefix=i32(*far))
    check(q, k, v, 0.125, bias=bias, valid=i32(*far), q_start=i32(*far[::-1]))
    check(q, k, v, 0.125, causal=True, prefix=i32(*far), valid=i32(*far[::-1]), q_start=i32(*(far[1:] + far[:1])))


def test_documents_of_extreme_numbers():
    q, k, v, g = make(2, 4, 2, 70, 200, 64, 4)
    ids = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, -1], dtype=torch.int32)
    kd, qd = ids[torch.randint(0, 4, (2, 200), generator=g)], ids[torch.randint(0, 4, (2, 70), generator=g)]
    check(q, k, v, 0.125, q_docs=qd, kv_docs=kd)
    check(q, k, v, 0.125, causal=True, q_docs=qd.sort(-1).values, kv_docs=kd.sort(-1).values)
    check(q[:, :, :1], k, v, 0.125, q_docs=qd[:, :1], kv_docs=kd)


def _jobs():
    """Calls that need workspaces: K split, stored activations, key splits of both attention kernels."""
    from easyanimate_amd import ops
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().to(DEV)
    w = ops.mxfp4_quantize(r(256, 13000))
    xs = [r(100, 13000), r(30, 13000)]
    k, v = r(1, 2, 6000, 128), r(1, 2, 6000, 128)
    qs = [r(1, 8, 1, 128), r(1, 8, 40, 128)]
    return [lambda x=x: ops.gemm_mxfp4(x, w, None) for x in xs] + [lambda q=q: ops.attention_text(q, k, v, 0.09, causal=True) for q in qs]


def test_streams_at_the_same_time():
    jobs = _jobs()
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(12):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(((turn + n) % len(jobs), jobs[(turn + n) % len(jobs)]()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[n]) for n, y in got)


def test_graphs_in_turn():
    jobs = _jobs()
    want = [j() for j in jobs]
    graphs = []
    for j in jobs:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = j()
        graphs.append((graph, out))
    for turn in range(4):
        for n, (graph, out) in enumerate(graphs):
            out.zero_()
            graph.replay()
            eager = jobs[(n + turn) % len(jobs)]()
            assert torch.equal(out, want[n]) and torch.equal(eager, want[(n + turn) % len(jobs)])
        torch.cuda.synchronize()


@pytest.mark.parametrize("M,N,K", [(5, 264, 700), (30, 264, 700), (90, 264, 700), (200, 264, 700), (60, 64, 13000), (3900, 4000, 300), (1100, 4096, 300)])
def test_the_residual_may_be_the_output(M, N, K):
    from easyanimate_amd import ops
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, K, generator=g).bfloat16().to(DEV), ops.mxfp4_quantize(torch.randn(N, K, generator=g).bfloat16().to(DEV))
    res, gate = torch.randn(M, N, generator=g).bfloat16().to(DEV), torch.randn(N, generator=g).to(DEV)
    want = ops.gemm_mxfp4(x, w, None, ops.EPI_BIAS_GATE_RES, res=res, gate=gate)
    buf = res.clone()
    assert ops.gemm_mxfp4(x, w, None, ops.EPI_BIAS_GATE_RES, out=buf, res=buf, gate=gate) is buf
    assert torch.equal(buf, want)


def test_outputs_whose_rows_overlap_are_refused():
    from easyanimate_amd import ops
    q = torch.zeros(2, 2, 20, 64, dtype=torch.bfloat16, device=DEV)
    flat = torch.zeros(20 * 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.attention_text(q, q, q, 0.1, out=flat.view(1, 20, 128).expand(2, 20, 128))
    with pytest.raises(ValueError, match="overlap"):
        ops.attention_text(q, q, q, 0.1, out=flat.as_strided((2, 20, 128), (1024, 64, 1)))
    x, w = torch.zeros(20, 64, dtype=torch.bfloat16, device=DEV), ops.mxfp4_quantize(torch.zeros(128, 64, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError, match="overlap"):
        ops.gemm_mxfp4(x, w, None, out=flat.as_strided((20, 128), (64, 1)))
