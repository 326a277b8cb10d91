"""The cache of derived weights: streams, graph capture and regions of frozen weights, on the CPU with stand-ins for streams and
events (the order of the calls is what counts)."""
import gc
import types

import pytest
import torch

from easyanimate_amd import _params


class Weight:
    """What _params reads of a parameter."""
    dtype, shape, is_cuda, device, _version = torch.bfloat16, (8, 64), True, torch.device("cuda", 0), 0

    def data_ptr(self):
        return 4096

    def detach(self):
        return self

    def to(self, dtype):
        return self


class Gpu:
    """One device: `now` is the current stream, `log` what was asked of streams and memory."""

    def __init__(self, monkeypatch):
        self.now, self.capture, self.log = 1, False, []
        gpu = self

        class Event:
            def record(self, stream):
                gpu.log.append(("record", stream.id))

        def stream(dev):
            i = gpu.now
            return types.SimpleNamespace(id=i, wait_event=lambda e: gpu.log.append(("wait", i)))
        monkeypatch.setattr(_params, "_raw_stream", lambda index: gpu.now)
        monkeypatch.setattr(_params, "_capturing", lambda index: gpu.capture)
        monkeypatch.setattr(torch.cuda, "Event", Event)
        monkeypatch.setattr(torch.cuda, "current_stream", stream)
        monkeypatch.setattr(_params, "_cache", {})
        monkeypatch.setattr(_params, "_of_graphs", {})

    def make(self, _):
        part = lambda n: types.SimpleNamespace(record_stream=lambda s: self.log.append((n, s.id)))
        self.log.append(("made", self.now))
        return types.SimpleNamespace(codes=part("codes"), scales=part("scales"))


@pytest.fixture()
def gpu(monkeypatch):
    return Gpu(monkeypatch)


def test_another_stream_waits_and_holds_the_memory(gpu):
    w = Weight()
    one = _params.derived(w, "mxfp4", gpu.make)
    assert gpu.log == [("made", 1), ("record", 1)]
    assert _params.derived(w, "mxfp4", gpu.make) is one and len(gpu.log) == 2           # its own stream: nothing to do
    gpu.now = 2
    for _ in range(2):                                                                  # once is enough
        assert _params.derived(w, "mxfp4", gpu.make) is one
    assert gpu.log[2:] == [("wait", 2), ("codes", 2), ("scales", 2)]
    gpu.now = 3
    assert _params.derived(w, "mxfp4", gpu.make) is one and gpu.log[5:] == [("wait", 3), ("codes", 3), ("scales", 3)]


def test_a_copy_made_under_capture_is_not_kept(gpu):
    w = Weight()
    gpu.capture = True
    inside = _params.derived(w, "f32", gpu.make)
    gpu.capture = False
    outside = _params.derived(w, "f32", gpu.make)
    assert outside is not inside and _params.derived(w, "f32", gpu.make) is outside


def test_capture_waits_for_nothing(gpu):
    """An event from outside must not enter a graph; the device was idle when the capture began."""
    w = Weight()
    one = _params.derived(w, "f32", gpu.make)
    n = len(gpu.log)
    gpu.now, gpu.capture = 2, True
    assert _params.derived(w, "f32", gpu.make) is one and len(gpu.log) == n
    gpu.capture = False
    assert _params.derived(w, "f32", gpu.make) is one and gpu.log[n] == ("wait", 2)


@pytest.fixture()
def stored(gpu, monkeypatch):
    from easyanimate_amd import ops
    monkeypatch.setattr(ops, "mxfp4_quantize", gpu.make)
    return lambda: [k for k in _params._cache if k[1] == "mxfp4"]


def test_4_bit_copies_live_in_their_region(gpu, stored):
    w = Weight()
    assert _params.mxfp4_weight(w) is not _params.mxfp4_weight(w) and not stored()
    with _params.weights_frozen():
        one = _params.mxfp4_weight(w)
        with _params.weights_frozen():
            assert _params.mxfp4_weight(w) is one
        assert _params.mxfp4_weight(w) is one and len(stored()) == 1        # the inner region's end drops nothing
    assert not stored()
    with pytest.raises(KeyError):
        with _params.weights_frozen():
            _params.mxfp4_weight(w)
            raise KeyError
    assert not stored() and not _params.frozen()


def test_other_copies_outlive_the_region(gpu, stored):
    w = Weight()
    with _params.weights_frozen():
        one = _params.derived(w, "kblock", gpu.make)
    assert _params.derived(w, "kblock", gpu.make) is one


def test_4_bit_copies_of_a_graph_are_its_own(gpu, stored):
    """A kept copy is dropped with its region, a graph is not."""
    w = Weight()
    with _params.weights_frozen():
        one = _params.mxfp4_weight(w)
        gpu.capture = True
        two = _params.mxfp4_weight(w)
        assert two is not one and _params.mxfp4_weight(w) is not two
        gpu.capture = False
        assert _params.mxfp4_weight(w) is one


def test_what_a_graph_reads_outlives_the_cache(gpu):
    w = Weight()
    one = _params.derived(w, "f32", gpu.make)
    gpu.capture = True
    for _ in range(2):
        assert _params.derived(w, "f32", gpu.make) is one
    gpu.capture = False
    _params.invalidate_weight_cache()
    kept = lambda: [v for d in _params._of_graphs.values() for v in d.values()]
    assert kept() == [one]
    assert _params.derived(w, "f32", gpu.make) is not one                   # eager calls make theirs anew
    del w                                                                   # the parameter goes, and with it what its graphs could read
    gc.collect()
    assert kept() == []
