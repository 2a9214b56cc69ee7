"""The example's layer on its way from training to serving."""
import os

import pytest
import torch

from i_amd import rotary


@pytest.fixture
def example(monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(__file__), "..", "examples"))
    import rotary_layer

    return rotary_layer


def test_frequencies_stay_what_they_were(example):
    layer = example.Layer(64, torch.float32)
    kept = rotary.frequencies(example.D // 2, device="cpu")
    assert torch.equal(layer.frequencies, kept) and not torch.equal(kept.bfloat16().float(), kept)
    layer = layer.serving()
    assert layer.frequencies.dtype is torch.float32 and torch.equal(layer.frequencies, kept)
    assert all(p.dtype is torch.bfloat16 for p in layer.parameters())
    assert torch.equal(layer.state_dict()["frequencies"], kept)
