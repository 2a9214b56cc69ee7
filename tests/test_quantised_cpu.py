"""What a cache in 8 or 4 bits refuses before any GPU work, and the oracle of its format."""
import ctypes
import math

import pytest
import torch

from i_amd import attention
from i_amd import quantised as ops
from quantised_oracle import decode, encode, numbers

REFUSED = ctypes.c_size_t(-1).value
BF16 = ops.nat.BF16


def tree(dtype=BF16, b=2, hq=4, hkv=2, nodes=3, d=64, scale=0.125, cap=0.0, lengths=4096, max_length=100, weights=0):
    return ops._TREE(dtype, b, hq, hkv, nodes, d, scale, cap, 0, lengths, max_length, 0, 0, 0, 0, 0, weights, weights, 100, 100, -1)


def cache(k=4096, scales=4096, v=4096, v_scales=4096, bits=4, strides=(1024, 512, 32, 64, 32, 2) * 2, table=0, table_stride=0, page=16, pages=2):
    return ops._CACHE(k, scales, v, v_scales, bits, *strides, table, table_stride, page, pages)


def move(dtype=BF16, b=2, hkv=2, n=4, d=64):
    return ops._MOVE(dtype, b, hkv, n, d, 0, 0)


RECORD = attention._TENSOR(4096, 2048, 512, 64)


@pytest.mark.parametrize("change", [{"dtype": 9}, {"nodes": 0}, {"nodes": 65}, {"max_length": 2}, {"hq": 3}, {"d": 12}, {"cap": -2.0}, {"scale": math.nan},
                                    {"weights": 4096}, {"b": 1 << 20, "hq": 4096, "hkv": 4096}], ids=str)
def test_trees_that_are_refused(change):
    assert ops.core.i_attend_quantised_workspace(tree(), 4) != REFUSED
    assert ops.core.i_attend_quantised_workspace(tree(**change), 4) == REFUSED
    assert "tree_attention" in ops.nat.last_error()
    assert ops.core.i_attend_quantised(tree(**change), RECORD, cache(), RECORD, None, 4096, 1 << 40, None) != 0


@pytest.mark.parametrize("change", [{"b": 1 << 24, "max_length": 16}, {"b": 1 << 20, "hq": 64, "nodes": 32, "max_length": 1 << 12},
                                    {"hq": 65535, "hkv": 1, "nodes": 64, "b": 1 << 6, "max_length": 1 << 20}], ids=str)
def test_trees_of_more_rows_than_a_launch(change):
    assert ops.core.i_attend_quantised_workspace(tree(**change), 8) == REFUSED
    assert " rows" in ops.nat.last_error()


def test_bits_that_there_are_not():
    assert ops.core.i_attend_quantised_workspace(tree(), 6) == REFUSED
    assert ops.core.i_attend_quantised(tree(), RECORD, cache(bits=2), RECORD, None, 4096, 1 << 40, None) != 0
    assert "bits" in ops.nat.last_error()


@pytest.mark.parametrize("change", [{"k": 0}, {"scales": 0}, {"v": 0}, {"v_scales": 0}, {"k": 4104}, {"bits": 16}, {"strides": (1024, 512, 24, 64, 32, 2) * 2},
                                    {"strides": (1024, 512, 32, 64, -32, 2) * 2}, {"page": 0}, {"pages": -1}, {"pages": 1}, {"table": 4096, "table_stride": -1}], ids=str)
def test_caches_that_are_refused(change):
    for code in (ops.core.i_quantised_store(move(), RECORD, RECORD, cache(**change), None), ops.core.i_quantised_load(move(), cache(**change), RECORD, RECORD, None),
                 ops.core.i_attend_quantised(tree(max_length=16), RECORD, cache(**change), RECORD, None, 4096, 1 << 40, None)):
        assert code != 0


@pytest.mark.parametrize("change", [{"dtype": 3}, {"b": -1}, {"hkv": 0}, {"n": -1}, {"d": 20}, {"n": 1 << 30}], ids=str)
def test_moves_that_are_refused(change):
    assert ops.core.i_quantised_store(move(**change), RECORD, RECORD, cache(), None) != 0
    assert ops.nat.last_error().startswith("store: ")
    assert ops.core.i_quantised_load(move(**change), cache(), RECORD, RECORD, None) != 0
    assert ops.nat.last_error().startswith("load: ")


def test_missing_arguments_are_errors():
    assert ops.core.i_quantised_store(None, None, None, None, None) != 0
    assert ops.core.i_quantised_store(move(), RECORD, None, cache(), None) != 0
    assert ops.core.i_quantised_load(move(), None, RECORD, RECORD, None) != 0
    assert ops.core.i_attend_quantised(None, None, None, None, None, None, 0, None) != 0
    assert ops.core.i_attend_quantised(tree(max_length=16), RECORD, cache(), RECORD, None, None, 0, None) != 0 or ops.core.i_attend_quantised_workspace(tree(max_length=16), 4) == 0
    assert ops.core.i_attend_quantised(tree(max_length=16, lengths=0), RECORD, cache(), RECORD, None, 4096, 1 << 40, None) != 0
    # more slots than the pages hold
    assert ops.core.i_attend_quantised(tree(max_length=17), RECORD, cache(), RECORD, None, 4096, 1 << 40, None) != 0


def test_tensors_that_are_not_on_a_gpu():
    x = torch.zeros((1, 1, 4, 64), dtype=torch.uint8)
    for call in (lambda: ops.QuantisedCache(x, x, x, x, 64, 8), lambda: ops.QuantisedCache([1], x, x, x, 64, 8), lambda: ops.QuantisedCache.empty(1, 1, 4, 64, device="cpu")):
        with pytest.raises(TypeError):
            call()
    for d, bits in ((64, 5), (60, 4), (264, 8)):
        with pytest.raises(ValueError):
            ops.QuantisedCache(x, x, x, x, d, bits)


def test_the_oracle():
    assert numbers(4).tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6]
    eight = numbers(8)
    assert eight[126] == 448 and eight[1] == 2.0 ** -9 and eight[8] == 2.0 ** -6 and eight[128 + 56] == -1
    assert torch.equal(eight.nan_to_num(9.0), torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().nan_to_num(9.0))
    row = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.5, -0.3])
    code, scale = encode(row, 4)
    assert scale.tolist() == [127] and decode(code, scale, 10, 4).tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 6, -0.5]
    code, scale = encode(torch.tensor([7.001, 1.0]), 4)
    assert scale.tolist() == [128] and decode(code, scale, 2, 4).tolist() == [8, 1]
    code, scale = encode(torch.tensor([464.0, 465.0]) * 2.0 ** -130, 8)
    assert scale.tolist() == [10] and encode(torch.tensor([0.0, math.inf]), 8)[1].tolist() == [255]
    # the bounds that the module's text gives
    x = torch.randn((2000, 32)) * torch.exp(2 * torch.randn(2000, 1))
    for bits in (4, 8):
        off = (decode(*encode(x, bits), 32, bits) - x).abs()
        top = x.abs().amax(-1, keepdim=True)
        assert bool((off <= (top / 5 if bits == 4 else torch.maximum(x.abs() / 16, top * 2.0 ** -17))).all())
