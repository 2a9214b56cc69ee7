"""Norm and rotary position of the heads of queries and keys in one pass, and its gradient.

The kernels of ``include/i_rotate.h`` on ROCm tensors (float32 or bfloat16), on the current stream.  They lie between a model's
projections and ``attention``:

  rotate            every row of q and k normalised (x / sqrt(mean(x^2) + eps) * weight) and turned by its token's position
  rotate_backward   the gradients of q, k and the norms' weights
  rotated           the two as one torch.autograd function
  frequencies, sections   the usual frequencies of the pairs, and the axes of pairs that turn by several positions

The reference has no counterpart (ilang-python/flash-attn.py:45-55 starts from finished heads).
"""
import ctypes
import struct

import torch

from . import _native as nat
from .attention import _check, _dense, _DTYPES, _enqueue, _first_operand, _pointer, _record, _SIZES, _workspace

core = nat.core
_bytes, _vp, _sz = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t

for _name, _args, _result in [
    ("i_rotate", [_bytes] * 5 + [_vp], ctypes.c_int),
    ("i_rotate_backward_workspace", [_bytes], _sz),
    ("i_rotate_backward", [_bytes] * 7 + [_vp, _vp, _vp, _sz, _vp], ctypes.c_int),
]:
    getattr(core, _name).argtypes = _args
    getattr(core, _name).restype = _result

_PROBLEM = struct.Struct("=9qQ2qQQQQqd").pack  # i_rotate_problem


def frequencies(pairs, base=10000.0, device="cuda"):
    """float32 [pairs]: pair j turns by base^(-j / pairs) radians a position."""
    return (float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(device)


def sections(*counts, device="cuda"):
    """int32 axes of the pairs: the first counts[0] pairs turn by the positions on axis 0, the next counts[1] on axis 1, and so on."""
    return torch.tensor([axis for axis, count in enumerate(counts) for _ in range(count)], dtype=torch.int32).to(device)


def _weight(weight, name, d, dtype, index):
    """Its address and type; a float32 one goes with any operands."""
    of_f32 = isinstance(weight, torch.Tensor) and weight.dtype is torch.float32
    _dense(weight, name, (d,), torch.float32 if of_f32 else dtype, index)
    return weight.data_ptr(), weight.dtype


def _problem(q, k, positions, frequencies, axes, interleaved, q_weight, k_weight, eps):
    """The problem's record, its GPU, and the sizes that its workspace depends on."""
    dtype, index = _first_operand(q)
    of_q = q.dtype
    b, hq, n, d = q.shape
    if k is None:
        hkv = 0
        if k_weight is not None:
            raise ValueError("k_weight goes with k")
    else:
        hkv = k.shape[1] if isinstance(k, torch.Tensor) and k.dim() == 4 else None
        _check(k, "k", (b, hkv, n, d), of_q, index)
    pairs = count = along = across = at = turns_at = axes_at = 0
    if frequencies is None:
        if positions is not None or axes is not None:
            raise ValueError("positions and axes go with frequencies")
    else:
        pairs = frequencies.shape[0] if isinstance(frequencies, torch.Tensor) and frequencies.dim() == 1 else None
        _dense(frequencies, "frequencies", (pairs,), torch.float32, index)
        if positions is None:
            raise ValueError("frequencies go with positions")
        dims = positions.dim() if isinstance(positions, torch.Tensor) else 0
        if axes is None:
            count, shared, shape = 1, dims == 1, (n,) if dims == 1 else (b, n)
        else:
            _dense(axes, "axes", (pairs,), torch.int32, index)
            axes_at = axes.data_ptr()
            count, shared = positions.shape[0] if dims > 0 else 1, dims == 2
            shape = (count, n) if shared else (count, b, n)
        strides = _check(positions, "positions", shape, torch.int32, index).stride()
        if n > 1 and strides[-1] != 1:
            raise ValueError("positions have to have unit stride within a sequence")
        if count > 1:
            along = strides[0]
        if not shared and b > 1:
            across = strides[-2]
        at, turns_at = positions.data_ptr(), frequencies.data_ptr()
    q_at = k_at = 0
    weight_type = of_q
    if q_weight is not None:
        q_at, weight_type = _weight(q_weight, "q_weight", d, of_q, index)
    if k_weight is not None:
        k_at, k_type = _weight(k_weight, "k_weight", d, of_q, index)
        if q_weight is not None and k_type is not weight_type:
            raise TypeError(f"q_weight and k_weight have to have one type, got {weight_type} and {k_type}")
        weight_type = k_type
    problem = _PROBLEM(dtype, b, hq, hkv, n, d, pairs, count, 1 if interleaved else 0, at, along, across, turns_at, axes_at, q_at, k_at,
                       _DTYPES[weight_type], float(eps))
    return problem, index, (dtype, b, hq, n, d, hkv, pairs, bool(interleaved), q_weight is None, k_weight is None)


def _laid_out(x):
    """x, or a copy of it where its strides are not those of a kernel's operand (autograd hands over gradients of any layout)."""
    sb, sh, sn, sd = x.stride()
    if sd == 1 and ((sb | sh | sn) * _SIZES[x.dtype] | x.data_ptr()) % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def rotate(q, k=None, positions=None, frequencies=None, *, axes=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6, out=None):
    """``q', k'``: q [b, hq, n, d] and k [b, hkv, n, d] (or None), normalised and turned.

    ``frequencies`` float32 [pairs]: pair j of columns, (j, j + pairs) or with ``interleaved`` (2 j, 2 j + 1), turns by frequencies[j]
    radians a position; columns from 2 pairs on do not turn (None: no column does).  ``positions`` int32 [b, n], or [n] where all
    sequences have the same.  ``axes`` int32 [pairs]: pairs turn by positions on several axes (time, height, width), positions being
    [axes, b, n] or [axes, n] then.  ``q_weight``, ``k_weight`` [d], float32 or of the operands' type: the norm's weight, None: no norm.
    d is a multiple of 8 up to 256; strides are free where they are multiples of 16 bytes and 1 in d.  ``out``: two tensors to write,
    which may be q and k themselves but not share memory with them in any other way."""
    problem, index, _ = _problem(q, k, positions, frequencies, axes, interleaved, q_weight, k_weight, eps)
    if out is None:
        q_out, k_out = torch.empty_like(q), None if k is None else torch.empty_like(k)
    else:
        q_out, k_out = out
        _check(q_out, "the new q", q.shape, q.dtype, index)
        if k is not None:
            _check(k_out, "the new k", k.shape, q.dtype, index)
    of_k = (None, None) if k is None else (_record(k, "k"), _record(k_out, "the new k", True))
    _enqueue(index, core.i_rotate, problem, _record(q, "q"), of_k[0], _record(q_out, "the new q", True), of_k[1])
    return q_out, k_out


def rotate_backward(grad_q, grad_k, q, k=None, positions=None, frequencies=None, *, axes=None, interleaved=False, q_weight=None, k_weight=None,
                    eps=1e-6, grads=None):
    """``dq, dk, dq_weight, dk_weight`` from the gradients of ``rotate``'s results and what it took; None for what was None.
    The weights' gradients are sums over all rows, in a fixed order.  ``grads``: two tensors to write dq and dk to, which may be
    grad_q and grad_k."""
    problem, index, sizes = _problem(q, k, positions, frequencies, axes, interleaved, q_weight, k_weight, eps)
    _check(grad_q, "grad_q", q.shape, q.dtype, index)
    if k is not None:
        _check(grad_k, "grad_k", k.shape, q.dtype, index)
    grad_q, grad_k = _laid_out(grad_q), None if k is None else _laid_out(grad_k)
    if grads is None:
        dq, dk = torch.empty_like(q), None if k is None else torch.empty_like(k)
    else:
        dq, dk = grads
        _check(dq, "dq", q.shape, q.dtype, index)
        if k is not None:
            _check(dk, "dk", k.shape, q.dtype, index)
    dq_weight, dk_weight = (None if w is None else torch.empty_like(w) for w in (q_weight, k_weight))
    workspace, address, size = _workspace(core.i_rotate_backward_workspace, sizes, problem, q.device)
    _enqueue(index, core.i_rotate_backward, problem, _record(grad_q, "grad_q"), None if k is None else _record(grad_k, "grad_k"), _record(q, "q"),
             None if k is None else _record(k, "k"), _record(dq, "dq", True), None if k is None else _record(dk, "dk", True), _pointer(dq_weight),
             _pointer(dk_weight), address, size)
    return dq, dk, dq_weight, dk_weight


class _Gradient(torch.autograd.Function):
    """The gradient where a graph of it is asked for: one that ends in an error."""

    @staticmethod
    def forward(ctx, grad_q, grad_k, q, k, q_weight, k_weight, positions, frequencies, options):
        return rotate_backward(grad_q, grad_k, q, k, positions, frequencies, q_weight=q_weight, k_weight=k_weight, **options)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("rotated has no gradient of its gradient")


class _Rotated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, axes, options):
        # (the constants too, so that one that is changed before the gradient is taken is an error)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies, axes)
        ctx.options = options
        return rotate(q, k, positions, frequencies, axes=axes, q_weight=q_weight, k_weight=k_weight, **options)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, positions, frequencies, axes = ctx.saved_tensors
        options = dict(ctx.options, axes=axes)
        if torch.is_grad_enabled():  # (create_graph)
            grads = _Gradient.apply(grad_q, grad_k, q, k, q_weight, k_weight, positions, frequencies, options)
        else:
            grads = rotate_backward(grad_q, grad_k, q, k, positions, frequencies, q_weight=q_weight, k_weight=k_weight, **options)
        return (*grads, None, None, None, None)


def rotated(q, k=None, positions=None, frequencies=None, *, axes=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6):
    """``rotate`` as a torch.autograd function of q, k and the weights (positions, frequencies and axes are constants, and may not
    change before the gradient is taken).  There is no gradient of its gradient: asking for one is an error."""
    return _Rotated.apply(q, k, q_weight, k_weight, positions, frequencies, axes, {"interleaved": interleaved, "eps": eps})
