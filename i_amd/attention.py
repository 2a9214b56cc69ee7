"""Attention with masks, capped scores and a bias by distance, its gradient, and attention over a cache in pages.

The kernels of ``include/i_attend.h`` on ROCm tensors (float32 or bfloat16), on the current stream:

  attention            o, lse = softmax(scores) v, for prompts and training
  attention_backward   the gradients of q, k and v
  differentiable       the two as one torch.autograd function
  key_weights          the attention weight that every key received
  tree_attention       the nodes of a tree of drafted tokens (or one token) against a cache in pages
  evict                the cache entries of least accumulated weight leave

with  scores(i, j) = cap tanh(scale q_i.k_j / cap) - slope |pos(i) - j|,  pos(i) = i + nk - nq.

What a query sees is an interval of keys: ``first[b, i] <= j < last[b, i]`` (int32 tensors, either may be None), and with ``causal``
only ``j <= pos(i)``.  Documents, prefixes and sliding windows are such intervals: ``document_bounds``, ``prefix_bounds`` and
``window_bounds`` make them.  The reference has no counterpart (ilang-python/flash-attn.py:45-55 is forward only, without a mask).
"""
import ctypes
import math
import struct

import torch

from . import _native as nat

core = nat.core
_bytes, _vp, _sz = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t

for _name, _args, _result in [
    ("i_attend", [_bytes] * 5 + [_vp, _vp], ctypes.c_int),
    ("i_attend_backward_workspace", [_bytes], _sz),
    ("i_attend_backward", [_bytes] * 6 + [_vp] + [_bytes] * 3 + [_vp, _sz, _vp], ctypes.c_int),
    ("i_attend_weights_workspace", [_bytes], _sz),
    ("i_attend_weights", [_bytes] * 3 + [_vp, _vp, _vp, _vp, _sz, _vp], ctypes.c_int),
    ("i_attend_tree_workspace", [_bytes], _sz),
    ("i_attend_tree", [_bytes] * 4 + [_vp, _vp, _sz, _vp], ctypes.c_int),
    ("i_evict_workspace", [_bytes], _sz),
    ("i_evict", [_bytes] * 3 + [_vp, _sz, _vp], ctypes.c_int),
]:
    getattr(core, _name).argtypes = _args
    getattr(core, _name).restype = _result

# the structs of i_attend.h
_TENSOR = struct.Struct("=Qqqq").pack
_PROBLEM = struct.Struct("=7q2dQqQQ").pack
_CACHE = struct.Struct("=QQ6qQ3q").pack
_TREE = struct.Struct("=6q2dQQqQQqQqQQ3q").pack
_EVICT = struct.Struct("=7qQQqQqQQqQ").pack

_DTYPES = {torch.float32: nat.F32, torch.bfloat16: nat.BF16}
_SIZES = {torch.float32: 4, torch.bfloat16: 2}


# ---------------------------------------------------------------- operands
# (a serving loop makes these calls with small operands: what is right is seen in few steps, what is wrong is explained after)
def _check(x, name, shape, dtype, index):
    """A ROCm tensor of this shape, type and GPU (None in the shape: any extent)."""
    if isinstance(x, torch.Tensor) and x.dtype is dtype and x.get_device() == index:
        if x.shape == shape or (len(shape) == x.dim() and all(n is None or n == have for n, have in zip(shape, x.shape))):
            return x
        raise ValueError(f"{name} has to have the shape {tuple('any' if n is None else n for n in shape)}, got {tuple(x.shape)}")
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} has to be a torch tensor, got {type(x).__name__}")
    if x.dtype is not dtype:
        raise TypeError(f"{name} has to be {dtype}, got {x.dtype}")
    raise TypeError(f"{name} has to be on GPU {index}, it is on {x.device}")


def _dense(x, name, shape, dtype, index):
    if not _check(x, name, shape, dtype, index).is_contiguous():
        raise ValueError(f"{name} has to be contiguous")
    return x


def _strides(x, name, out=False):
    """Element strides of a [., ., ., d] tensor, those of extents of one as 0."""
    b, h, n, d = x.shape
    sb, sh, sn, sd = x.stride()
    if sd != 1 and d > 1:
        raise ValueError(f"{name} has to have unit stride in its last dimension")
    if b <= 1:
        sb = 0
    elif out and sb == 0 and h and n and d:
        raise ValueError(f"{name} is written and may not repeat elements")
    if h <= 1:
        sh = 0
    elif out and sh == 0 and b and n and d:
        raise ValueError(f"{name} is written and may not repeat elements")
    if n <= 1:
        sn = 0
    elif out and sn == 0 and b and h and d:
        raise ValueError(f"{name} is written and may not repeat elements")
    return sb, sh, sn


def _record(x, name, out=False):
    return _TENSOR(x.data_ptr(), *_strides(x, name, out))


def _pointer(x):
    return 0 if x is None else x.data_ptr()


def _first_operand(q, name="q"):
    """Element type and GPU of the operand that the others have to match."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"{name} has to be a torch tensor, got {type(q).__name__}")
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise TypeError(f"{name} has to be float32 or bfloat16, got {q.dtype}")
    if not q.is_cuda:
        raise TypeError(f"{name} has to be on a GPU, it is on {q.device}")
    if q.dim() != 4:
        raise ValueError(f"{name} has to be [b, h, n, d], got {tuple(q.shape)}")
    return dtype, q.get_device()


_current_device, _raw_stream = torch.cuda.current_device, getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _enqueue(index, entry, *arguments):
    """entry(*arguments, stream) on the current stream of the GPU, with that GPU current."""
    if index == _current_device():
        code = entry(*arguments, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = entry(*arguments, _raw_stream(index))
    if code != 0:
        nat.check(code)


_sizes = {}  # bytes of workspace by entry and sizes


def _workspace(query, sizes, problem, device):
    """Workspace of a call; ``sizes``: all that its extent depends on."""
    key = query.__name__, sizes
    size = _sizes.get(key)
    if size is None:
        size = query(problem)
        if size == ctypes.c_size_t(-1).value:
            raise RuntimeError(nat.last_error())
        if len(_sizes) >= 256:
            _sizes.clear()
        _sizes[key] = size
    if size == 0:
        return None, 0, 0
    memory = torch.empty(size, dtype=torch.uint8, device=device)
    return memory, memory.data_ptr(), size


def _problem(q, k, scale, cap, slopes, causal, first, last):
    """The problem's record and its GPU."""
    dtype, index = _first_operand(q)
    b, hq, nq, d = q.shape
    _, hkv, nk, _ = _check(k, "k", (b, None, None, d), q.dtype, index).shape
    if slopes is not None:
        _dense(slopes, "slopes", (hq,), torch.float32, index)
    if first is not None:
        _dense(first, "first", (b, nq), torch.int32, index)
    if last is not None:
        _dense(last, "last", (b, nq), torch.int32, index)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    return _PROBLEM(dtype, b, hq, hkv, nq, nk, d, scale, float(cap), _pointer(slopes), 1 if causal else 0, _pointer(first), _pointer(last)), index


# ---------------------------------------------------------------- prompts and training
def attention(q, k, v, *, scale=None, cap=0.0, slopes=None, causal=False, first=None, last=None, out=None, lse=None):
    """``o, lse``: attention of q [b, hq, nq, d] over k, v [b, hkv, nk, d]; lse [b, hq, nq] is the natural logarithm of a row's
    sum of exponentials.  hq is a multiple of hkv, d a multiple of 8 up to 256; strides are free where they are multiples of 16
    bytes and 1 in d.  ``scale`` is 1 / sqrt(d) unless given, ``slopes`` float32 [hq].  A query that sees nothing: 0 and -inf."""
    problem, index = _problem(q, k, scale, cap, slopes, causal, first, last)
    _check(v, "v", k.shape, q.dtype, index)
    o = torch.empty_like(q) if out is None else _check(out, "out", q.shape, q.dtype, index)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if lse is None else _dense(lse, "lse", q.shape[:3], torch.float32, index)
    _enqueue(index, core.i_attend, problem, _record(q, "q"), _record(k, "k"), _record(v, "v"), _record(o, "out", True), lse.data_ptr())
    return o, lse


def attention_backward(grad, q, k, v, o, lse, *, scale=None, cap=0.0, slopes=None, causal=False, first=None, last=None, grads=None):
    """``dq, dk, dv`` from the gradient of o and what ``attention`` took and gave.  Shared key heads get the sum over their query
    heads, in a fixed order.  ``grads``: three tensors to write."""
    problem, index = _problem(q, k, scale, cap, slopes, causal, first, last)
    _check(v, "v", k.shape, q.dtype, index)
    _check(grad, "grad", q.shape, q.dtype, index)
    _check(o, "o", q.shape, q.dtype, index)
    _dense(lse, "lse", q.shape[:3], torch.float32, index)
    if not grad.is_contiguous() and (grad.stride(-1) != 1 or any(s * _SIZES[q.dtype] % 16 for s in grad.stride()[:3]) or grad.data_ptr() % 16):
        grad = grad.contiguous()  # (autograd hands over gradients of any layout, expanded ones too)
    if grads is None:
        grads = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dq, dk, dv = grads
    _check(dq, "dq", q.shape, q.dtype, index)
    _check(dk, "dk", k.shape, q.dtype, index)
    _check(dv, "dv", k.shape, q.dtype, index)
    workspace, address, size = _workspace(core.i_attend_backward_workspace, (q.dtype, q.shape, k.shape, causal, first is None and last is None), problem, q.device)
    _enqueue(index, core.i_attend_backward, problem, _record(grad, "grad"), _record(q, "q"), _record(k, "k"), _record(v, "v"), _record(o, "o"), lse.data_ptr(),
             _record(dq, "dq", True), _record(dk, "dk", True), _record(dv, "dv", True), address, size)
    return dq, dk, dv


class _Gradient(torch.autograd.Function):
    """The gradient where a graph of it is asked for: one that ends in an error.  (torch's once_differentiable gives a constant where
    the gradient of o has no graph itself, and a penalty on the gradients behind it would go on without attention's part.)"""

    @staticmethod
    def forward(ctx, grad, q, k, v, o, lse, options):
        return attention_backward(grad, q, k, v, o, lse, **options)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("attention has no gradient of its gradient")


class _Differentiable(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, first, last, options):
        o, lse = attention(q, k, v, slopes=slopes, first=first, last=last, **options)
        # (the constants too, so that one that is changed before the gradient is taken is an error)
        ctx.save_for_backward(q, k, v, o, lse, slopes, first, last)
        ctx.options = options
        return o

    @staticmethod
    def backward(ctx, grad):
        q, k, v, o, lse, slopes, first, last = ctx.saved_tensors
        options = dict(ctx.options, slopes=slopes, first=first, last=last)
        if torch.is_grad_enabled():  # (create_graph)
            grads = _Gradient.apply(grad, q, k, v, o, lse, options)
        else:
            grads = attention_backward(grad, q, k, v, o, lse, **options)
        return (*grads, None, None, None, None)


def differentiable(q, k, v, *, scale=None, cap=0.0, slopes=None, causal=False, first=None, last=None):
    """``attention`` as a torch.autograd function of q, k and v (the bias and the bounds are constants, and may not change before
    the gradient is taken); returns o.  There is no gradient of its gradient: asking for one is an error."""
    return _Differentiable.apply(q, k, v, slopes, first, last, {"scale": scale, "cap": cap, "causal": causal})


def key_weights(q, k, lse, *, scale=None, cap=0.0, slopes=None, causal=False, first=None, last=None, weights=None, out=None):
    """float32 [b, hkv, nk]: what every key received from all queries of its query heads, sum of exp(score - lse), with the lse of
    ``attention``.  Added to ``weights`` if given; ``out`` may be ``weights``."""
    problem, index = _problem(q, k, scale, cap, slopes, causal, first, last)
    shape = k.shape[:3]
    _dense(lse, "lse", q.shape[:3], torch.float32, index)
    if weights is not None:
        _dense(weights, "weights", shape, torch.float32, index)
    out = torch.empty(shape, dtype=torch.float32, device=q.device) if out is None else _dense(out, "out", shape, torch.float32, index)
    workspace, address, size = _workspace(core.i_attend_weights_workspace, (q.dtype, q.shape, shape, causal, first is None and last is None), problem, q.device)
    _enqueue(index, core.i_attend_weights, problem, _record(q, "q"), _record(k, "k"), lse.data_ptr(), _pointer(weights), out.data_ptr(), address, size)
    return out


# ---------------------------------------------------------------- bounds
def document_bounds(documents):
    """``first, last`` of queries that see their own document: ``documents`` [b, n], any integers, equal within a document and
    different for neighbouring ones (tokens of a document lie together)."""
    b, n = documents.shape
    at = torch.arange(n, device=documents.device).expand(b, n)
    begins = torch.ones((b, n), dtype=torch.bool, device=documents.device)
    begins[:, 1:] = documents[:, 1:] != documents[:, :-1]
    ends = torch.ones_like(begins)
    ends[:, :-1] = begins[:, 1:]
    first = torch.where(begins, at, 0).cummax(1).values
    last = torch.where(ends, at + 1, n).flip(1).cummin(1).values.flip(1)
    return first.int().contiguous(), last.int().contiguous()


def prefix_bounds(prefix, n):
    """``last`` of queries that see the first prefix[b] keys and those up to their own: [b, n] (without ``causal``)."""
    at = torch.arange(1, n + 1, device=prefix.device, dtype=torch.int32)
    return torch.maximum(at[None, :], prefix.int()[:, None]).contiguous()


def window_bounds(b, nq, nk, width, device):
    """``first`` of queries that see the last ``width`` keys up to their own: [b, nq] (with ``causal``)."""
    at = torch.arange(nq, device=device, dtype=torch.int32) + (nk - nq + 1 - width)
    return at.clamp(min=0).expand(b, nq).contiguous()


# ---------------------------------------------------------------- a cache in pages
def _cache(k, v, table, b, name, index, out=False):
    """Record of a cache k, v [pages, hkv, page, d] with the pages of every sequence in ``table`` [b, any]."""
    if table is None:
        listed, stride = 0, 0
    else:
        _check(table, f"{name} table", (b, None), torch.int32, index)
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError(f"{name} table has to have unit stride within a sequence")
        if b > 1 and table.stride(0) < table.shape[1]:
            table = table.contiguous()
        listed, stride = table.data_ptr(), table.shape[1] if b <= 1 else table.stride(0)
    pages, _, page, _ = k.shape
    return _CACHE(k.data_ptr(), v.data_ptr(), *_strides(k, f"{name} k", out), *_strides(v, f"{name} v", out), listed, stride, page, pages), table


def _capacity(k, table):
    return k.shape[2] * (1 if table is None else table.shape[1])


def tree_attention(q, k, v, lengths, *, table=None, visible=None, scale=None, cap=0.0, slopes=None, start=None, positions=None, weights=None,
                   weights_out=None, counted=-1, max_length=None, out=None, lse=None):
    """``o, lse`` of drafted tokens q [b, hq, nodes, d], at most 64 a sequence, over a cache k, v [pages, hkv, page, d].

    ``lengths`` int32 [b]: slots of the cache before the drafted tokens, whose own keys already lie in the slots that follow.
    ``table`` int32 [b, any]: the pages of every sequence in order (None: sequence b is page b).  ``visible`` int64 [b, nodes] or
    [nodes]: bit u set where a node sees node u (itself and its ancestors; None: a chain).  ``max_length``: no sequence is longer,
    drafted tokens included (None: what the pages hold).  With ``slopes``, node t is at position start[b] + bits of its word - 1
    (``start`` None: lengths) and a slot at ``positions`` int32 [b, hkv, any] (None: its index).  ``weights`` float32 [b, hkv, any]:
    what every slot has received so far; ``weights_out`` (None: ``weights`` itself) gets that and the weights of the nodes whose
    bit is set in ``counted`` (-1: all)."""
    dtype, index = _first_operand(q)
    b, hq, nodes, d = q.shape
    hkv = _check(k, "k", (None, None, None, d), q.dtype, index).shape[1]
    _check(v, "v", k.shape, q.dtype, index)
    _dense(lengths, "lengths", (b,), torch.int32, index)
    if visible is not None:
        _dense(visible, "visible", (nodes,) if visible.dim() == 1 else (b, nodes), torch.int64, index)
    if slopes is not None:
        _dense(slopes, "slopes", (hq,), torch.float32, index)
    if start is not None:
        _dense(start, "start", (b,), torch.int32, index)
    if positions is not None:
        _dense(positions, "positions", (b, hkv, None), torch.int32, index)
    if weights is None and weights_out is not None:
        raise ValueError("weights_out goes with weights")
    kept = held = 0
    if weights is not None:
        kept = _dense(weights, "weights", (b, hkv, None), torch.float32, index).shape[2]
        weights_out = weights if weights_out is None else _dense(weights_out, "weights_out", (b, hkv, None), torch.float32, index)
        held = weights_out.shape[2]
    counted = int(counted)
    if counted >> 63 not in (0, 1, -1):
        raise ValueError(f"counted has a bit a node, 64 at most, got {counted}")
    counted -= counted >> 63 << 64 if counted > 0 else 0  # (the 64 bits of a signed number)
    capacity = _capacity(k, table)
    max_length = capacity if max_length is None else min(int(max_length), capacity)
    o = torch.empty_like(q) if out is None else _check(out, "out", q.shape, q.dtype, index)
    lse = torch.empty((b, hq, nodes), dtype=torch.float32, device=q.device) if lse is None else _dense(lse, "lse", (b, hq, nodes), torch.float32, index)
    cache, table = _cache(k, v, table, b, "cache", index)
    problem = _TREE(dtype, b, hq, hkv, nodes, d, 1.0 / math.sqrt(d) if scale is None else float(scale), float(cap), _pointer(slopes),
                    lengths.data_ptr(), max_length, _pointer(start), _pointer(positions), 0 if positions is None else positions.shape[2],
                    _pointer(visible), 0 if visible is None or visible.dim() == 1 else nodes, _pointer(weights), _pointer(weights_out), kept, held,
                    counted)
    workspace, address, size = _workspace(core.i_attend_tree_workspace, (dtype, b, hq, hkv, nodes, d, max_length, weights is None, counted), problem, q.device)
    _enqueue(index, core.i_attend_tree, problem, _record(q, "q"), cache, _record(o, "out", True), lse.data_ptr(), address, size)
    return o, lse


def evict(k, v, weights, lengths, keep, recent, *, table=None, positions=None, table_out=None, out=None, room=0, max_length=None):
    """``k, v, weights, positions, lengths`` of the cache k, v [pages, hkv, page, d] cut to ``keep`` entries a key head: the last
    ``recent`` slots stay, and of the others those of largest ``weights`` (float32 [b, hkv, any]; of equal ones the lowest slots),
    in the order of their slots.  A sequence of at most ``keep`` entries moves whole.  ``out``: the five tensors to write, the
    cache among them in pages listed by ``table_out``, whose columns have to have room for what stays; what lies past a sequence's new length is left as it is.  None: new ones, one
    page of ``keep + room`` slots a sequence, weights and positions past what stays 0.  The keys of the tokens that follow need such slots:
    ``tree_attention`` takes the last slots it is given for the drafted tokens', and cuts a length that leaves none.  ``out`` may not share memory with the cache, its lengths, weights or positions
    (other pages of the same tensors are other memory)."""
    dtype, index = _first_operand(k, "k")
    _check(v, "v", k.shape, k.dtype, index)
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise ValueError("lengths has to be an int32 tensor [b]")
    b, hkv, d, keep, recent, room = lengths.shape[0], k.shape[1], k.shape[3], int(keep), int(recent), int(room)
    _dense(lengths, "lengths", (b,), torch.int32, index)
    kept = _dense(weights, "weights", (b, hkv, None), torch.float32, index).shape[2]
    if positions is not None:
        _dense(positions, "positions", (b, hkv, None), torch.int32, index)
    capacity = _capacity(k, table)
    max_length = capacity if max_length is None else min(int(max_length), capacity)
    if out is None:
        if table_out is not None:
            raise ValueError("table_out goes with out")
        if keep < 1 or room < 0:
            raise ValueError(f"keep has to be at least 1 and room not negative, got {keep} and {room}")
        new = torch.empty((b, hkv, keep + room, d), dtype=k.dtype, device=k.device)
        out = (new, torch.empty_like(new), torch.zeros((b, hkv, keep + room), dtype=torch.float32, device=k.device),
               torch.zeros((b, hkv, keep + room), dtype=torch.int32, device=k.device), torch.empty(b, dtype=torch.int32, device=k.device))
    elif room != 0:
        raise ValueError("room goes without out")
    k_out, v_out, weights_out, positions_out, lengths_out = out
    _check(k_out, "the new k", (None, hkv, None, d), k.dtype, index)
    _check(v_out, "the new v", k_out.shape, k.dtype, index)
    _dense(weights_out, "the new weights", (b, hkv, None), torch.float32, index)
    _dense(positions_out, "the new positions", weights_out.shape, torch.int32, index)
    _dense(lengths_out, "the new lengths", (b,), torch.int32, index)
    old, table = _cache(k, v, table, b, "cache", index)
    new, table_out = _cache(k_out, v_out, table_out, b, "new cache", index, True)
    most = min(keep, max_length)
    if table_out is not None and _capacity(k_out, table_out) < most:  # (a view: its sequences may lie further apart than the pages that it lists)
        raise RuntimeError(f"evict: to: {most} slots do not fit {table_out.shape[1]} pages of {k_out.shape[2]}")
    problem = _EVICT(dtype, b, hkv, d, keep, recent, max_length, lengths.data_ptr(), weights.data_ptr(), kept, _pointer(positions),
                     0 if positions is None else positions.shape[2], weights_out.data_ptr(), positions_out.data_ptr(), weights_out.shape[2],
                     lengths_out.data_ptr())
    workspace, address, size = _workspace(core.i_evict_workspace, (b, hkv, d, keep), problem, k.device)
    _enqueue(index, core.i_evict, problem, old, new, address, size)
    return out
