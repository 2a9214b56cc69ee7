"""The example: a layer with norms and rotary positions, trained and served from a cache in few bits."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def example(monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(__file__), "..", "examples"))
    import rotary_layer

    return rotary_layer


@pytest.mark.parametrize("bits", [4, 8])
def test_it_runs(monkeypatch, example, bits):
    monkeypatch.setattr(sys, "argv", ["rotary_layer.py", "--steps", "3", "--prompt", "50", "--tokens", "4", "--bits", str(bits)])
    layer, outputs, off = example.main()
    assert outputs.shape == (2, 4, 128) and bool(outputs.isfinite().all()) and off == off
    assert all(bool(p.isfinite().all()) for p in layer.parameters())


def test_its_gradients(example):
    """Against differences of the loss along a direction, in f32: central, of a step of 1e-3 of the weights.  Either loss is a mean of about
    6000 squares of order 1 in f32, off by some 2^-24 times their spread over the step: 1e-7 / 2e-3 = 5e-5, besides (1e-3)^2 of a third
    derivative."""
    torch.manual_seed(1)
    layer = example.Layer(64, torch.float32).cuda()
    x = torch.randn((2, 49, 64), device="cuda")

    def loss():
        return layer(x).square().mean()

    loss().backward()
    steps = [torch.randn_like(p) * p.detach().norm() / p.numel() ** 0.5 for p in layer.parameters()]
    slope = sum((p.grad * s).sum() for p, s in zip(layer.parameters(), steps)).item()
    h, values = 1e-3, []
    with torch.no_grad():
        for sign in (1, -2):
            for p, s in zip(layer.parameters(), steps):
                p.add_(s, alpha=sign * h)
            values.append(loss().double().item())
    size = sum((p.grad.abs() * s.abs()).sum() for p, s in zip(layer.parameters(), steps)).item()
    assert abs((values[0] - values[1]) / (2 * h) - slope) < 5e-4 + 1e-3 * size
