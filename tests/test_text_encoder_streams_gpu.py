"""The 4-bit text encoder's kept weights (weights_frozen): used from several streams, dropped while another stream still reads, and from
captured graphs."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from test_text_encoder_gpu import CASES, _prompt_batch, _qwen

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture()
def enc():
    from easyanimate_amd.text_encoder import Qwen2VLTextEncoderHIP
    c = CASES["hd64"]
    e = Qwen2VLTextEncoderHIP(_qwen(c["hidden"], c["heads"], c["kv_heads"], c["inter"], c["layers"]).to(torch.bfloat16).to(DEV), weights="mxfp4")
    ids, _ = _prompt_batch(c["B"], c["S"], 512, c["lens"])
    ids = ids.to(DEV)
    return e, lambda: e(input_ids=ids, output_hidden_states=True).hidden_states[-1]


def test_second_stream_waits_for_the_first_ones_weights(enc):
    from easyanimate_amd._params import weights_frozen
    e, run = enc
    want = run()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with weights_frozen():
            with torch.cuda.stream(a):
                torch.cuda._sleep(20_000_000)              # the weights are laid out behind this
                one = run()
            with torch.cuda.stream(b):
                two = run()
        torch.cuda.synchronize()
        assert torch.equal(one, want) and torch.equal(two, want)


def test_first_use_on_two_streams_at_once(enc):
    """Nothing of the encoder's is made before: the gate vector and the weights of the first stream are the second one's too."""
    from easyanimate_amd import _params
    e, run = enc
    want = run()
    for _ in range(3):
        torch.cuda.synchronize()
        _params.invalidate_weight_cache()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with _params.weights_frozen():
            with torch.cuda.stream(a):
                torch.cuda._sleep(20_000_000)
                one = run()
            with torch.cuda.stream(b):
                two = run()
        torch.cuda.synchronize()
        assert torch.equal(one, want) and torch.equal(two, want)


def test_a_graph_outlives_its_region(enc):
    """Captured inside a frozen region after a run that kept the weights; replayed behind the region, with other work and writes between."""
    from easyanimate_amd import _params
    e, run = enc
    first = run()
    with _params.weights_frozen():
        assert torch.equal(run(), first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        assert torch.equal(run(), first)
    weight = e._text[0].layers[0].mlp.up_proj.weight
    want = first
    for i in range(4):
        torch.full((1 << 22,), 0x55, dtype=torch.uint8, device=DEV)         # (what the region held is used for something else)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(run(), want), i
        if i % 2 == 0:
            weight.data.mul_(-1.0)                                          # a replay sees it as a run does
            want = run()
            assert not torch.equal(want, out)


def test_captured_without_a_run_before(enc):
    """The first thing that a fresh encoder does is a capture: what it lays out belongs to the graph, eager calls make their own."""
    from easyanimate_amd import _params
    e, run = enc
    want = run()
    torch.cuda.synchronize()
    _params.invalidate_weight_cache()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    assert torch.equal(run(), want)                                         # before any replay
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(run(), want)


def test_a_graph_outlives_the_cache(enc):
    """The fp32 biases and gains that a graph reads stay when the cache is cleared (every pipeline call does that)."""
    from easyanimate_amd import _params
    e, run = enc
    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        _params.invalidate_weight_cache()
        junk = [torch.full((n,), 7.0, device=DEV) for n in (64, 128, 256, 512, 1024) for _ in range(20)]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(run(), want)
        del junk
