"""The example's served tokens against attention in 64 bits over what its cache is to hold."""
import os

import pytest
import torch

from attend_oracle import Attention, within
from quantised_oracle import decode, encode

pytestmark = pytest.mark.gpu


@pytest.fixture
def example(monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(__file__), "..", "examples"))
    import rotary_layer

    return rotary_layer


@pytest.mark.parametrize("bits", [4, 8])
def test_served_tokens(example, bits):
    """The rows of a token's keys and values are those of its own position, whichever page they lie in.  The join adds 512 products of bf16
    in f32 to o, which is off by its own bound, and rounds to bf16."""
    from i_amd import rotary

    torch.manual_seed(3)
    layer = example.Layer(128, torch.float32).cuda().serving()
    n, steps = 150, 6
    x = torch.randn((2, n + steps, 128), device="cuda").bfloat16()
    with torch.no_grad():
        served = example.Served(layer, x[:, :n], steps, bits)
        got = torch.cat([served.step(x[:, t:t + 1]) for t in range(n, n + steps)], 1)
        # (projected in the same pieces: the same bits)
        pieces = [layer.project(x[:, :n])] + [layer.project(x[:, t:t + 1]) for t in range(n, n + steps)]
    q, k, v = (torch.cat(parts, 2).detach() for parts in zip(*pieces))
    at = torch.arange(n + steps, dtype=torch.int32, device="cuda")
    q, k = rotary.rotate(q, k, at, rotary.frequencies(example.D // 2), q_weight=layer.q_weight.detach(), k_weight=layer.k_weight.detach())
    kept = [decode(*encode(y.cpu(), bits), example.D, bits).to(torch.bfloat16) for y in (k, v)]
    want = Attention(q[:, :, n:], *kept, causal=True)
    weight = layer.out.weight.detach().cpu().double()
    o, bound = (y.transpose(1, 2).flatten(2) for y in (want.o, want.o_bound))
    joined = o @ weight.T
    within(got, joined, bound @ weight.abs().T + 2.0 ** -8 * joined.abs() + 520 * 2.0 ** -24 * (o.abs() @ weight.abs().T), "served tokens")
