"""One attention layer with norms and rotary positions, trained, then served from a cache in 4 or 8 bits.

    python examples/rotary_layer.py [--steps 20] [--prompt 200] [--tokens 8] [--bits 4]

The layer learns to copy: the target of a token is the vector of the token before it.  Training runs norm, rotation and attention
with their gradients (`rotary.rotated`, `attention.differentiable`); serving rotates and stores a prompt and then every
token (`rotary.rotate`, `quantised.store`) and attends over what the cache holds (`quantised.tree_attention`).  Prints the loss of the first and
last step, and how far the served outputs are from those of a cache of the layer's own type.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from i_amd import attention, quantised, rotary

HEADS, KEY_HEADS, D, PAGE = 8, 2, 64, 16


class Layer(torch.nn.Module):
    def __init__(self, width, dtype):
        super().__init__()
        self.qkv = torch.nn.Linear(width, (HEADS + 2 * KEY_HEADS) * D, bias=False, dtype=dtype)
        self.out = torch.nn.Linear(HEADS * D, width, bias=False, dtype=dtype)
        self.q_weight, self.k_weight = (torch.nn.Parameter(torch.ones(D, dtype=dtype)) for _ in range(2))
        self.register_buffer("frequencies", rotary.frequencies(D // 2, device="cpu"))

    def project(self, x):
        """q, k, v [b, heads, n, D], views of what the product leaves."""
        q, k, v = self.qkv(x).view(*x.shape[:2], -1, D).split([HEADS, KEY_HEADS, KEY_HEADS], 2)
        return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)

    def norms(self):
        return {"q_weight": self.q_weight, "k_weight": self.k_weight}

    def join(self, o):
        return self.out(o.transpose(1, 2).flatten(2))

    def forward(self, x):
        q, k, v = self.project(x)
        positions = torch.arange(x.shape[1], dtype=torch.int32, device=x.device)
        q, k = rotary.rotated(q, k, positions, self.frequencies, **self.norms())
        return self.join(attention.differentiable(q, k, v, causal=True))

    def serving(self):
        """The layer in bfloat16, but for the frequencies: a position times a rounded one would be another angle than in training."""
        frequencies = self.frequencies
        self.bfloat16()
        self.frequencies = frequencies
        return self


def train(layer, steps, gen, b=4, n=129):
    optimizer = torch.optim.Adam(layer.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        x = torch.randn((b, n, layer.qkv.in_features), generator=gen, device="cuda")
        loss = (layer(x.to(layer.out.weight.dtype)).float()[:, 1:] - x[:, :-1]).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


class Served:
    """A batch of sequences in a cache of pages."""

    def __init__(self, layer, prompt, room, bits):
        self.layer, (b, n, _) = layer, prompt.shape
        pages = -(-(n + room) // PAGE)
        self.cache = quantised.QuantisedCache.empty(b * pages, KEY_HEADS, PAGE, D, bits)
        self.table = torch.randperm(b * pages, device="cuda").int().view(b, pages)
        q, k, v = layer.project(prompt)
        q, k = rotary.rotate(q, k, torch.arange(n, dtype=torch.int32, device="cuda"), layer.frequencies, **layer.norms())
        quantised.store(self.cache, k, v, table=self.table)
        o, _ = attention.attention(q, k, v, causal=True)
        self.prompt_out = layer.join(o)
        self.lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")

    def step(self, x):
        """The outputs of the next token of every sequence, [b, 1, width]."""
        q, k, v = self.layer.project(x)
        q, k = rotary.rotate(q, k, self.lengths[:, None], self.layer.frequencies, **self.layer.norms())
        quantised.store(self.cache, k, v, first=self.lengths, table=self.table)
        o, _ = quantised.tree_attention(q, self.cache, self.lengths, table=self.table)
        self.lengths = self.lengths + 1
        return self.layer.join(o)


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--prompt", type=int, default=200)
    parser.add_argument("--tokens", type=int, default=8)
    parser.add_argument("--bits", type=int, default=4, choices=(4, 8))
    a = parser.parse_args()
    torch.manual_seed(0)
    gen = torch.Generator("cuda").manual_seed(0)
    layer = Layer(128, torch.float32).cuda()
    losses = train(layer, a.steps, gen)
    if losses:
        print(f"training: loss {losses[0]:.3f} -> {losses[-1]:.3f} in {a.steps} steps", flush=True)
    layer = layer.serving()
    with torch.no_grad():
        x = torch.randn((2, a.prompt + a.tokens, 128), generator=gen, device="cuda").bfloat16()
        expected = layer(x)[:, a.prompt:].float()
        served = Served(layer, x[:, :a.prompt], a.tokens, a.bits)
        outputs = torch.cat([served.step(x[:, t:t + 1]) for t in range(a.prompt, a.prompt + a.tokens)], 1).float()
    off = float((outputs - expected).norm() / expected.norm())
    held = sum(t.numel() for t in (served.cache.k, served.cache.k_scales, served.cache.v, served.cache.v_scales))
    print(f"serving {a.tokens} tokens after {a.prompt} from {a.bits} bits: {off:.4f} off, {held} bytes in place of {4 * D * served.cache.pages * KEY_HEADS * PAGE}")
    return layer, outputs, off


if __name__ == "__main__":
    main()
