"""Norm and rotary position of heads and its gradient in 64 bits, from the definition, with bounds on what a kernel's arithmetic may differ by.

u is half a step of the operands' type, e of f32.  Of a row of d columns the kernel squares and sums in f32, in an order of its own (its
sum's error is at most (d + 4) e of it, half of that in the root), divides, multiplies twice, turns by a cosine and a sine that are off by at
most 2^-22 (the angle's remainder to 2^-25 of a turn, times 2 pi, and the polynomials) and rounds once.
"""
import torch

E = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TURN = 2.0 ** -21


def turned(x, positions, frequencies, axes, interleaved, back=False):
    """x [b, h, n, d] in 64 bits, its pairs turned.  positions [axes, b, n]."""
    if frequencies is None:
        return x
    pairs = len(frequencies)
    of_pair = torch.zeros(pairs, dtype=torch.long) if axes is None else axes.cpu().long().clamp(0, positions.shape[0] - 1)
    angle = positions.cpu().double()[of_pair].permute(1, 2, 0)[:, None] * frequencies.cpu().double()
    cos, sin = torch.cos(angle), -torch.sin(angle) if back else torch.sin(angle)
    j = torch.arange(pairs)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def spread(x, frequencies, interleaved):
    """What a pair's rounding may move: |a| + |b| for the columns that turn, |x| for the others."""
    x = x.abs()
    if frequencies is None:
        return x
    pairs = len(frequencies)
    j = torch.arange(pairs)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    y = x.clone()
    y[..., a] = y[..., b] = x[..., a] + x[..., b]
    return y


class Rotation:
    """One side (queries or keys) of a call, in float64 on the CPU."""

    def __init__(self, x, positions=None, frequencies=None, axes=None, interleaved=False, weight=None, eps=1e-6):
        self.u, self.x = UNIT[x.dtype], x.detach().cpu().double()
        self.d = x.shape[-1]
        if positions is not None:
            b, n = x.shape[0], x.shape[2]
            count = 1 if axes is None else positions.shape[0]
            positions = positions.cpu()
            shared = positions.dim() == (1 if axes is None else 2)
            positions = positions.reshape(count, 1 if shared else b, n).expand(count, b, n)
        self.turning = (positions, frequencies, axes, interleaved)
        self.weight = None if weight is None else weight.detach().cpu().double()
        self.inverse = 1 / (self.x.square().mean(-1, keepdim=True) + eps).sqrt()
        self.normed = self.x * self.inverse
        before = self.x if weight is None else self.normed * self.weight
        self.relative = 0.0 if weight is None else (self.d + 12) * E
        self.y = turned(before, *self.turning)
        self.y_bound = (self.relative + 4 * E + TURN) * spread(before, frequencies, interleaved) + self.u * self.y.abs() + 1e-37

    def gradients(self, grad, weight_dtype=None):
        """dx, its bound, and the same for the weight (None, None)."""
        frequencies, interleaved = self.turning[1], self.turning[3]
        grad = grad.detach().cpu().double()
        g = turned(grad, *self.turning, back=True)
        off = (4 * E + TURN) * spread(grad, frequencies, interleaved)  # of g
        if self.weight is None:
            return g, off + self.u * g.abs() + 1e-37, None, None
        gw = g * self.weight
        along = (gw * self.normed).mean(-1, keepdim=True)
        dx = (gw - self.normed * along) * self.inverse
        gw_off = off * self.weight.abs() + 4 * E * gw.abs()
        along_off = (gw_off * self.normed.abs() + 2 * (self.relative + self.d * E) * (gw * self.normed).abs()).mean(-1, keepdim=True)
        dx_off = (gw_off + self.normed.abs() * along_off + 2 * self.relative * (gw.abs() + (self.normed * along).abs())) * self.inverse
        rows = (0, 1, 2)
        dw = (g * self.normed).sum(rows)
        # (f32 sums of up to as many terms as there are rows, of which an order by runs leaves far fewer in a row)
        count = self.x[..., 0].numel()
        dw_off = (off * self.normed.abs() + (self.relative + 4 * E) * (g * self.normed).abs()).sum(rows) + min(count, 4096) * E * (g * self.normed).abs().sum(rows)
        return dx, dx_off + self.u * dx.abs() + 1e-37, dw, dw_off + UNIT[weight_dtype] * dw.abs() + 1e-37
