"""A cache of keys and values in 8 or 4 bits: tokens written to it, read back, and attention over it.

The kernels of ``include/i_quantised.h`` on ROCm tensors, on the current stream:

  QuantisedCache    the cache in pages: codes and scales
  store             keys and values (float32 or bfloat16) of a prompt or of the next tokens to their slots
  load              slots read back
  tree_attention    ``attention.tree_attention`` over such a cache

A row of d columns (a slot of a key head) takes 33/32 d bytes at 8 bits and 17/32 d at 4: blocks of 32 columns share a scale, a power of
two; the numbers at 4 bits are 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives.  An element comes back off by at most 1/5 of the
block's largest magnitude at 4 bits, and at 8 by 1/16 of its own or 2^-17 of the largest, whichever is more.
The reference has no counterpart (ilang-python/flash-attn.py:45-55).
"""
import ctypes
import math
import struct

import torch

from . import _native as nat
from .attention import _check, _dense, _DTYPES, _enqueue, _first_operand, _pointer, _record, _TREE, _workspace

core = nat.core
_bytes, _vp, _sz = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_size_t

for _name, _args, _result in [
    ("i_quantised_store", [_bytes] * 4 + [_vp], ctypes.c_int),
    ("i_quantised_load", [_bytes] * 4 + [_vp], ctypes.c_int),
    ("i_attend_quantised_workspace", [_bytes, ctypes.c_int64], _sz),
    ("i_attend_quantised", [_bytes] * 4 + [_vp, _vp, _sz, _vp], ctypes.c_int),
]:
    getattr(core, _name).argtypes = _args
    getattr(core, _name).restype = _result

# the structs of i_quantised.h
_CACHE_MEMORY, _CACHE_PAGES = struct.Struct("=4Q13q").pack, struct.Struct("=Q4q").pack  # the two halves of i_quantised_cache
_MOVE = struct.Struct("=5qQQ").pack


def _CACHE(*fields, listed=0):
    """i_quantised_cache from all its fields, packed as calls pack it: what it has for good, and what a call adds."""
    return _CACHE_MEMORY(*fields[:17]) + _CACHE_PAGES(*fields[17:], listed)


class QuantisedCache:
    """Codes ``k``, ``v`` uint8 [pages, hkv, page, columns * bits / 8] and their ``k_scales``, ``v_scales`` uint8 [pages, hkv, page,
    columns / 32], columns being d rounded up to a multiple of 32.  Strides are free where they are 1 in a row, and those of codes
    multiples of 16.  The four tensors stay the cache's for as long as it lives."""

    __slots__ = ("_tensors", "_memory", "d", "bits", "pages", "hkv", "page", "device", "index")
    k, k_scales, v, v_scales = (property(lambda self, n=n: self._tensors[n]) for n in range(4))

    def __init__(self, k, k_scales, v, v_scales, d, bits):
        d, bits = int(d), int(bits)
        if bits not in (4, 8):
            raise ValueError(f"bits has to be 4 or 8, got {bits}")
        if d < 8 or d > 256 or d % 8:
            raise ValueError(f"d has to be a multiple of 8 up to 256, got {d}")
        columns = -(-d // 32) * 32
        if not isinstance(k, torch.Tensor):
            raise TypeError(f"k has to be a torch tensor, got {type(k).__name__}")
        if not k.is_cuda:
            raise TypeError(f"k has to be on a GPU, it is on {k.device}")
        index = k.get_device()
        pages, hkv, page, _ = _check(k, "k", (None, None, None, columns * bits // 8), torch.uint8, index).shape
        _check(v, "v", k.shape, torch.uint8, index)
        strides = []
        for name, x in (("k", k), ("k_scales", k_scales), ("v", v), ("v_scales", v_scales)):
            if name.endswith("scales"):
                _check(x, name, (pages, hkv, page, columns // 32), torch.uint8, index)
            if x.stride(3) != 1 and x.shape[3] > 1:
                raise ValueError(f"{name} has to have unit stride in its last dimension")
            if x.numel() and any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
                raise ValueError(f"{name} is written and may not repeat elements")
            strides += [0 if n <= 1 else s for s, n in zip(x.stride()[:3], x.shape[:3])]
        self._tensors = k, k_scales, v, v_scales
        self._memory = _CACHE_MEMORY(*(x.data_ptr() for x in self._tensors), bits, *strides)
        self.d, self.bits, self.pages, self.hkv, self.page = d, bits, pages, hkv, page
        self.device, self.index = k.device, index

    def __reduce__(self):
        # (a copy has its own tensors, and with them its own description)
        return QuantisedCache, (*self._tensors, self.d, self.bits)

    @classmethod
    def empty(cls, pages, hkv, page, d, bits=4, device="cuda"):
        """A cache of zeros."""
        columns = -(-int(d) // 32) * 32
        codes, scales = ((pages, hkv, page, columns * bits // 8), (pages, hkv, page, columns // 32))
        return cls(*(torch.zeros(shape, dtype=torch.uint8, device=device) for shape in (codes, scales, codes, scales)), d, bits)

    def _record(self, table, b, index):
        """The C struct, with the pages of every sequence in ``table`` [b, any], and the table that has to live until the call is enqueued."""
        if self.index != index:
            raise TypeError(f"the cache has to be on GPU {index}, it is on {self.device}")
        if table is None:
            address, stride, per = 0, 0, 0
        else:
            per = table.shape[1] if isinstance(table, torch.Tensor) and table.dim() == 2 else None
            _check(table, "table", (b, per), torch.int32, index)
            if per == 0:
                raise ValueError("table has to list a page for every sequence")
            stride, unit = table.stride()
            if per > 1 and unit != 1:
                raise ValueError("table has to have unit stride within a sequence")
            if b <= 1:
                stride = per
            elif stride < per:
                table, stride = table.contiguous(), per
            address = table.data_ptr()
        return self._memory + _CACHE_PAGES(address, stride, self.page, self.pages, per), table

    def _capacity(self, table):
        return self.page * (1 if table is None else table.shape[1])


def _moved(cache, dtype, b, n, first, counts, index):
    for name, x in (("first", first), ("counts", counts)):
        if x is not None:
            _dense(x, name, (b,), torch.int32, index)
    return _MOVE(_DTYPES[dtype], b, cache.hkv, n, cache.d, _pointer(first), _pointer(counts))


def store(cache, k, v, *, first=None, counts=None, table=None):
    """Writes k, v [b, hkv, n, d] (float32 or bfloat16): token t of sequence s to slot first[s] + t, for t < counts[s] (int32 [b]; None:
    from slot 0, all n).  ``table`` int32 [b, any]: the pages of every sequence in order (None: sequence s is page s); it may be a view of a wider one.  Slots that the
    sequence's pages do not have are not written, and neither are pages that the cache does not have.  No two tokens of a call may
    have the same slot."""
    _, index = _first_operand(k, "k")
    b, _, n, _ = k.shape
    _check(k, "k", (b, cache.hkv, n, cache.d), k.dtype, index)
    _check(v, "v", k.shape, k.dtype, index)
    record, table = cache._record(table, b, index)
    _enqueue(index, core.i_quantised_store, _moved(cache, k.dtype, b, n, first, counts, index), _record(k, "k"), _record(v, "v"), record)


def load(cache, n, *, first=None, counts=None, table=None, b=None, dtype=torch.bfloat16, out=None):
    """``k, v`` [b, hkv, n, d]: slots first[s] .. first[s] + n - 1 of every sequence read back (exact in bfloat16 too), zeros where t >=
    counts[s] or the sequence's pages have no such slot; a page that the cache does not have reads as page 0.  b is that of ``first``, ``counts``, ``table`` or ``out``, else all pages.
    ``out``: two tensors to write."""
    n, index = int(n), cache.index
    if out is not None:
        _first_operand(out[0], "the new k")
        dtype = out[0].dtype
    if dtype not in _DTYPES:
        raise TypeError(f"dtype has to be float32 or bfloat16, got {dtype}")
    if n < 0:
        raise ValueError(f"n may not be negative, got {n}")
    if b is None:
        given = [x for x in (first, counts, table, None if out is None else out[0]) if isinstance(x, torch.Tensor) and x.dim() > 0]
        b = given[0].shape[0] if given else cache.pages
    shape = (b, cache.hkv, n, cache.d)
    if out is None:
        k = torch.empty(shape, dtype=dtype, device=cache.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        _check(k, "the new k", shape, dtype, index)
        _check(v, "the new v", shape, dtype, index)
    record, table = cache._record(table, b, index)
    _enqueue(index, core.i_quantised_load, _moved(cache, dtype, b, n, first, counts, index), record, _record(k, "the new k", True), _record(v, "the new v", True))
    return k, v


def _bits_workspace(bits):
    def query(problem):
        return core.i_attend_quantised_workspace(problem, bits)

    query.__name__ = f"i_attend_quantised_workspace_{bits}"
    return query


_QUERIES = {bits: _bits_workspace(bits) for bits in (4, 8)}


def tree_attention(q, cache, lengths, *, table=None, visible=None, scale=None, cap=0.0, slopes=None, start=None, positions=None, max_length=None,
                   out=None, lse=None):
    """``o, lse`` of drafted tokens q [b, hq, nodes, d] (float32 or bfloat16), at most 64 a sequence, over a quantised cache: the arguments
    of ``attention.tree_attention``, but for weights, which are not kept here.  One node is the step of a single token."""
    dtype, index = _first_operand(q)
    b, hq, nodes, d = q.shape
    if d != cache.d:
        raise ValueError(f"q has to have {cache.d} columns, got {d}")
    _dense(lengths, "lengths", (b,), torch.int32, index)
    if visible is not None:
        _dense(visible, "visible", (nodes,) if visible.dim() == 1 else (b, nodes), torch.int64, index)
    if slopes is not None:
        _dense(slopes, "slopes", (hq,), torch.float32, index)
    if start is not None:
        _dense(start, "start", (b,), torch.int32, index)
    if positions is not None:
        _dense(positions, "positions", (b, cache.hkv, None), torch.int32, index)
    record, table = cache._record(table, b, index)
    capacity = cache._capacity(table)
    max_length = capacity if max_length is None else min(int(max_length), capacity)
    o = torch.empty_like(q) if out is None else _check(out, "out", q.shape, q.dtype, index)
    lse = torch.empty((b, hq, nodes), dtype=torch.float32, device=q.device) if lse is None else _dense(lse, "lse", (b, hq, nodes), torch.float32, index)
    problem = _TREE(dtype, b, hq, cache.hkv, nodes, d, 1.0 / math.sqrt(d) if scale is None else float(scale), float(cap), _pointer(slopes),
                    lengths.data_ptr(), max_length, _pointer(start), _pointer(positions), 0 if positions is None else positions.shape[2],
                    _pointer(visible), 0 if visible is None or visible.dim() == 1 else nodes, 0, 0, 0, 0, -1)
    workspace, address, size = _workspace(_QUERIES[cache.bits], (dtype, b, hq, cache.hkv, nodes, d, max_length), problem, q.device)
    _enqueue(index, core.i_attend_quantised, problem, _record(q, "q"), record, _record(o, "out", True), lse.data_ptr(), address, size)
    return o, lse
