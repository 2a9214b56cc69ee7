"""The example: a layer that learns over packed documents and is served from a cache that was cut."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_a_layer_learns_and_is_served(monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(__file__), "..", "examples"))
    monkeypatch.setattr(sys, "argv", ["attention_layer.py", "--steps", "40", "--prompt", "200", "--keep", "64", "--tokens", "8"])
    import attention_layer

    losses, whole, cut = attention_layer.main()
    # copying the token before is what there is to learn
    assert losses[-1] < 0.8 * losses[0]
    # the same attention in another order of bf16 roundings: a few times 2^-8
    assert whole < 0.02
    # a quarter of the keys, chosen by weight and nearness, is less than no keys at all (an error of 1)
    assert whole <= cut < 0.7
