"""use_hip_text_encoder on a slot that holds a device-library encoder already (no GPU: only the wrapping)."""
import os
import sys
import types

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from test_text_encoder_gpu import _qwen


@pytest.fixture()
def hf():
    return _qwen(256, 4, 2, 512, 1, vocab=128).to(torch.bfloat16)


@pytest.mark.parametrize("first,then", [("bf16", "mxfp4"), ("mxfp4", "bf16")])
def test_other_weights_are_taken(hf, first, then):
    from easyanimate_amd.text_encoder import use_hip_text_encoder
    pipe = types.SimpleNamespace(text_encoder=hf)
    one = use_hip_text_encoder(pipe, weights=first)
    one.padded_positions = "cumsum_fill1"
    assert use_hip_text_encoder(pipe, weights=first) is one                 # the same again: left alone
    two = use_hip_text_encoder(pipe, weights=then)
    assert two is pipe.text_encoder and two is not one
    assert (two.weights, two.padded_positions, two.hf) == (then, "cumsum_fill1", hf) and one.weights == first


def test_bad_weights_are_refused(hf):
    from easyanimate_amd.text_encoder import use_hip_text_encoder
    for slot in (hf, None):
        pipe = types.SimpleNamespace(text_encoder=slot)
        with pytest.raises(ValueError, match="weights"):
            use_hip_text_encoder(pipe, weights="int4")
    pipe = types.SimpleNamespace(text_encoder=hf)
    wrapped = use_hip_text_encoder(pipe)
    with pytest.raises(ValueError, match="weights"):
        use_hip_text_encoder(pipe, weights="int4")
    assert pipe.text_encoder is wrapped


def test_second_slot_and_empty_slot(hf):
    from easyanimate_amd.text_encoder import use_hip_text_encoder
    pipe = types.SimpleNamespace(text_encoder=None, text_encoder_2=hf)
    assert use_hip_text_encoder(pipe, weights="mxfp4") is None
    assert use_hip_text_encoder(pipe, 1) is pipe.text_encoder_2 and pipe.text_encoder_2.weights == "bf16"
    assert use_hip_text_encoder(pipe, 1, "mxfp4").weights == "mxfp4" and pipe.text_encoder is None
