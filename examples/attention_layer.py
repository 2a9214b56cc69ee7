"""One attention layer trained on packed documents, then served: a prompt, a cache cut to a budget, drafted tokens checked as a tree.

    python examples/attention_layer.py [--steps 30] [--prompt 300] [--keep 96] [--tokens 12]

The layer learns to copy: the target of a token is the vector of the token before it in its document.  Training runs
attention and its gradient (`differentiable`); serving runs the prompt (`attention`), counts what every key received (`key_weights`),
keeps the keys that received most (`evict`) and reads the cache for several drafted tokens a call (`tree_attention`), which goes on
counting.  Prints the loss of the first and last step, and how far the served outputs are from those of a cache with every key.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from i_amd import attention as ops

HEADS, KEY_HEADS, D, CAP, PAGE = 8, 2, 64, 20.0, 16


class Layer(torch.nn.Module):
    def __init__(self, width, dtype):
        super().__init__()
        self.q = torch.nn.Linear(width, HEADS * D, bias=False, dtype=dtype)
        self.kv = torch.nn.Linear(width, 2 * KEY_HEADS * D, bias=False, dtype=dtype)
        self.out = torch.nn.Linear(HEADS * D, width, bias=False, dtype=dtype)
        self.register_buffer("slopes", torch.tensor([2.0 ** (-(h + 1) / 2) for h in range(HEADS)], dtype=torch.float32))

    def project(self, x):
        """q [b, heads, n, D], k and v [b, key heads, n, D], as views of what the products leave."""
        b, n, _ = x.shape
        q = self.q(x).view(b, n, HEADS, D).transpose(1, 2)
        k, v = self.kv(x).view(b, n, 2 * KEY_HEADS, D).transpose(1, 2).chunk(2, 1)
        return q, k, v

    def join(self, o):
        return self.out(o.transpose(1, 2).flatten(2))

    def forward(self, x, first):
        q, k, v = self.project(x)
        return self.join(ops.differentiable(q, k, v, cap=CAP, slopes=self.slopes, causal=True, first=first))


def batch(b, n, width, dtype, gen):
    """Tokens of packed documents, the token before each one in its document, and the bounds of the documents."""
    x = torch.randn((b, n, width), generator=gen, device="cuda")
    first, _ = ops.document_bounds((torch.rand((b, n), generator=gen, device="cuda") < 0.04).int().cumsum(1))
    before = torch.cat([torch.zeros_like(x[:, :1]), x[:, :-1]], 1) * (first < torch.arange(n, device="cuda"))[..., None]
    return x.to(dtype), before, first


def train(layer, steps, gen, b=4, n=257):
    optimizer = torch.optim.Adam(layer.parameters(), lr=3e-3)
    width, dtype = layer.q.in_features, layer.q.weight.dtype
    losses = []
    for _ in range(steps):
        x, target, first = batch(b, n, width, dtype, gen)
        loss = (layer(x, first).float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


class Served:
    """A batch of sequences in a cache of pages."""

    def __init__(self, layer, prompt, room):
        self.layer, (b, n, _) = layer, prompt.shape
        pages = -(-(n + room) // PAGE)
        q, k, v = layer.project(prompt)
        options = dict(cap=CAP, slopes=layer.slopes, causal=True)
        o, lse = ops.attention(q, k, v, **options)
        self.prompt_out = layer.join(o)
        self.table = torch.randperm(b * pages, device="cuda").int().view(b, pages)
        self.k, self.v = (torch.zeros((b * pages, KEY_HEADS, PAGE, D), dtype=k.dtype, device="cuda") for _ in range(2))
        self.weights, self.positions = (torch.zeros((b, KEY_HEADS, pages * PAGE), dtype=t, device="cuda") for t in (torch.float32, torch.int32))
        self.weights[:, :, :n] = ops.key_weights(q, k, lse, **options)
        self.positions[:] = torch.arange(pages * PAGE, device="cuda")
        self.lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
        self.start = self.lengths.clone()  # positions go on where the text does, however many keys leave
        self._store(k, v)

    def _store(self, k, v, at=None):
        """Keys and values [b, key heads, n, D] to slots at .. at + n - 1 (at: [b], none: 0)."""
        slots = torch.arange(k.shape[2], device="cuda") + (0 if at is None else at[:, None].long())
        slots = slots.expand(k.shape[0], -1)
        pages = self.table.gather(1, slots // PAGE).long()
        self.k[pages, :, slots % PAGE], self.v[pages, :, slots % PAGE] = k.transpose(1, 2), v.transpose(1, 2)

    def cut(self, keep, recent):
        b = self.lengths.shape[0]
        new = torch.empty_like(self.k), torch.empty_like(self.v), torch.zeros_like(self.weights), self.positions.clone(), torch.empty_like(self.lengths)
        self.k, self.v, self.weights, self.positions, self.lengths = ops.evict(
            self.k, self.v, self.weights, self.lengths, keep, recent, table=self.table, positions=self.positions, table_out=self.table, out=new)

    def check(self, drafted, visible, accepted):
        """Outputs of drafted tokens [b, nodes, width], a tree; the first `accepted` nodes, a chain, are taken over."""
        q, k, v = self.layer.project(drafted)
        self._store(k, v, self.lengths)
        o, _ = ops.tree_attention(q, self.k, self.v, self.lengths, table=self.table, visible=visible, cap=CAP, slopes=self.layer.slopes,
                                  start=self.start, positions=self.positions, weights=self.weights, counted=(1 << accepted) - 1)
        # what was taken over keeps its slots and gets its positions; the others' slots are written again
        slots = self.lengths[:, None].long() + torch.arange(drafted.shape[1], device="cuda")
        self.weights.scatter_(2, slots[:, None, accepted:].expand(-1, KEY_HEADS, -1), 0.0)
        taken = self.start[:, None] + torch.arange(accepted, device="cuda", dtype=torch.int32)
        self.positions.scatter_(2, slots[:, None, :accepted].expand(-1, KEY_HEADS, -1), taken[:, None].expand(-1, KEY_HEADS, -1).contiguous())
        self.lengths = self.lengths + accepted
        self.start = self.start + accepted
        return self.layer.join(o)


def serve(layer, prompt, text, keep):
    """Outputs of `text` [b, n, width] after the prompt, three drafted tokens a call of which two hold; keep: None or the cache's budget."""
    served = Served(layer, prompt, text.shape[1] + 3)
    if keep is not None:
        served.cut(keep, keep // 4)
    outputs = []
    # node 1 follows node 0, and so does node 2, a guess that fails
    visible = torch.tensor([0b001, 0b011, 0b101], device="cuda")
    for at in range(0, text.shape[1], 2):
        drafted = torch.cat([text[:, at:at + 2], torch.zeros_like(text[:, :1])], 1)
        outputs.append(served.check(drafted, visible, 2)[:, :2])
    return torch.cat(outputs, 1), served


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=30)
    parser.add_argument("--prompt", type=int, default=300)
    parser.add_argument("--keep", type=int, default=96)
    parser.add_argument("--tokens", type=int, default=12)
    a = parser.parse_args()
    torch.manual_seed(0)
    gen = torch.Generator("cuda").manual_seed(0)
    layer = Layer(128, torch.float32).cuda()
    losses = train(layer, a.steps, gen)
    print(f"training: loss {losses[0]:.3f} -> {losses[-1]:.3f} in {a.steps} steps", flush=True)
    layer = layer.bfloat16()
    layer.slopes = layer.slopes.float()
    tokens = a.tokens // 2 * 2
    with torch.no_grad():
        prompt, text = (torch.randn((2, n, 128), generator=gen, device="cuda").bfloat16() for n in (a.prompt, tokens))
        whole, _ = serve(layer, prompt, text, None)
        cut, served = serve(layer, prompt, text, a.keep)
        q, k, v = layer.project(torch.cat([prompt, text], 1))
        o, _ = ops.attention(q, k, v, cap=CAP, slopes=layer.slopes, causal=True)
        expected = layer.join(o)[:, a.prompt:].float()
    far = lambda x: float((x.float() - expected).norm() / expected.norm())
    print(f"serving {tokens} tokens after {a.prompt}: {far(whole):.4f} off with every key, {far(cut):.4f} off with {a.keep} of {a.prompt}, "
          f"{int(served.lengths[0])} entries in the cache")
    return losses, far(whole), far(cut)


if __name__ == "__main__":
    main()
