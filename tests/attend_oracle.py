"""Attention with masks and its gradient in 64 bits, from the definition, with bounds on what a kernel's arithmetic may differ by.

A bound follows the computation: scores carry the rounding of a d-term f32 dot product (and of cap and bias), probabilities
twice that (numerator and sum) and, with bf16 operands, their own rounding to bf16; every product's bound is the product of the
absolute values.  u is the unit roundoff of the operands' type, factor 2 covers what is left out (exponentials, sums of rows).
"""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -9}


def hidden_keys(nq, nk, b, causal=False, first=None, last=None):
    """[b, nq, nk], true where query i does not see key j."""
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
    hidden = torch.zeros((b, nq, nk), dtype=torch.bool)
    if causal:
        hidden |= j > i + nk - nq
    if first is not None:
        hidden |= j < first.cpu().long()[:, :, None]
    if last is not None:
        hidden |= j >= last.cpu().long()[:, :, None]
    return hidden


class Attention:
    """Everything of one call in float64 on the CPU."""

    def __init__(self, q, k, v=None, *, scale=None, cap=0.0, slopes=None, causal=False, first=None, last=None, hidden=None, distance=None):
        dtype = q.dtype
        self.u = UNIT[dtype]
        q, k = q.detach().cpu().double(), k.detach().cpu().double()
        b, hq, nq, d = q.shape
        hkv, nk = k.shape[1], k.shape[2]
        self.shape, self.group = (b, hq, hkv, nq, nk, d), hq // hkv
        self.scale = scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.q, self.k = q, k.repeat_interleave(self.group, 1)
        hidden = hidden_keys(nq, nk, b, causal, first, last) if hidden is None else hidden
        self.hidden = hidden[:, None].expand(b, hq, nq, nk)
        # what nobody sees may be anything
        dead = hidden.all(1)[:, None, :, None]
        self.k = torch.where(dead, 0.0, self.k)
        s = self.q @ self.k.transpose(2, 3) * scale
        error = (d + 16) * 2.0 ** -24 * abs(scale) * (self.q.abs() @ self.k.abs().transpose(2, 3))
        self.bend = torch.ones_like(s)
        if cap:
            t = torch.tanh(s / cap)
            s, self.bend = cap * t, 1 - t * t
            error = error + 2.0 ** -21 * cap
        if slopes is not None:
            if distance is None:
                distance = (torch.arange(nq)[:, None] + nk - nq - torch.arange(nk)[None, :]).abs().double().expand(b, hq, nq, nk)
            bias = slopes.cpu().double().view(1, hq, 1, 1) * distance
            s, error = s - bias, error + 2.0 ** -22 * bias.abs()
        s = s.masked_fill(self.hidden, -math.inf)
        error = (error + 2.0 ** -22 * (1 + s.abs())).masked_fill(self.hidden, 0.0)
        self.lse = torch.logsumexp(s, -1)
        self.p = torch.exp(s - self.lse.masked_fill(self.lse == -math.inf, 0.0)[..., None])
        self.score_error = error.amax(-1, keepdim=True) if nk else error.new_zeros((b, hq, nq, 1))
        self.lse_bound = 2 * self.score_error[..., 0] + 1e-6
        # (a probability of the kernel, before and after its rounding to the operands' type)
        self.relative = 2 * (2 * self.score_error + 2.0 ** -20)
        self.p_bound = (self.relative + self.u) * self.p
        if v is not None:
            self.v = torch.where(dead, 0.0, v.detach().cpu().double().repeat_interleave(self.group, 1))
            self.o = self.p @ self.v
            self.o_bound = 2 * (self.p_bound @ self.v.abs()) + 2 * self.u * self.o.abs() + 1e-30

    def shared(self, x):
        """Sum over the query heads of a key head."""
        b, hq, hkv = self.shape[:3]
        return x.view(b, hkv, self.group, *x.shape[2:]).sum(2)

    def weights(self):
        return self.shared(self.p.sum(2)), self.shared((2 * self.relative * self.p).sum(2)) + 1e-30

    def gradients(self, grad):
        """(dq, dk, dv) and their bounds."""
        g, u, scale = grad.detach().cpu().double(), self.u, abs(self.scale)
        d = self.shape[-1]
        dp = g @ self.v.transpose(2, 3)
        delta = (g * self.o).sum(-1, keepdim=True)
        ds = self.p * (dp - delta) * self.bend
        around = (d + 16) * 2.0 ** -24 * (g.abs() @ self.v.abs().transpose(2, 3) + (g.abs() * self.o.abs()).sum(-1, keepdim=True))
        around = around + (g.abs() * self.o_bound).sum(-1, keepdim=True)
        # (1 - tanh^2) is off by the score's error times its slope, at most 2 / cap < 1 of it
        ds_bound = 2 * self.relative * self.p * (dp - delta).abs() + self.p * around + u * ds.abs() + 2 * self.score_error * self.p * (dp - delta).abs()
        dq, dk, dv = self.scale * (ds @ self.k), self.scale * (ds.transpose(2, 3) @ self.q), self.p.transpose(2, 3) @ g
        dq_bound = 2 * scale * (ds_bound @ self.k.abs()) + 2 * u * dq.abs() + 1e-30
        dk_bound = self.shared(2 * scale * (ds_bound.transpose(2, 3) @ self.q.abs()))
        dv_bound = self.shared(2 * (self.p_bound.transpose(2, 3) @ g.abs()))
        dk, dv = self.shared(dk), self.shared(dv)
        return (dq, dk, dv), (dq_bound, dk_bound + 2 * u * dk.abs() + 1e-30, dv_bound + 2 * u * dv.abs() + 1e-30)


def within(got, want, bound, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} instead of {tuple(want.shape)}"
    same = got == want  # (infinities)
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, the first at {tuple(bad.nonzero()[0].tolist())}: "
                           f"{got[bad][0].item()} instead of {want[bad][0].item()}, bound {bound.expand_as(off)[bad][0].item()}")
