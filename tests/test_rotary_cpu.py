"""What the norm and rotary position of heads refuses before any GPU work."""
import ctypes
import math

import pytest
import torch

from i_amd import attention
from i_amd import rotary as ops

REFUSED = ctypes.c_size_t(-1).value


def problem(dtype=1, b=2, hq=4, hkv=2, n=8, d=64, pairs=32, axes=1, interleaved=0, positions=4096, stride_axis=0, stride_b=8, frequencies=4096,
            axis_of=0, q_weight=4096, k_weight=4096, weight_dtype=1, eps=1e-6):
    return ops._PROBLEM(dtype, b, hq, hkv, n, d, pairs, axes, interleaved, positions, stride_axis, stride_b, frequencies, axis_of, q_weight, k_weight,
                        weight_dtype, eps)


@pytest.mark.parametrize("change", [{"dtype": 5}, {"b": -1}, {"hq": -1}, {"hq": 0, "hkv": 0}, {"hkv": 70000}, {"n": -1}, {"n": 2 ** 30}, {"d": 60}, {"d": 264},
                                    {"pairs": 33}, {"pairs": -1}, {"axes": 0}, {"interleaved": 2}, {"positions": 0}, {"frequencies": 0}, {"q_weight": 4098},
                                    {"weight_dtype": 7}, {"dtype": 0}, {"eps": math.nan}, {"eps": -1.0}, {"stride_b": -1}], ids=str)
def test_problems_that_are_refused(change):
    assert ops.core.i_rotate_backward_workspace(problem()) != REFUSED
    assert ops.core.i_rotate_backward_workspace(problem(**change)) == REFUSED
    assert "rotate_backward" in ops.nat.last_error()


def record(data=4096, sb=2048, sh=512, sn=64):
    return attention._TENSOR(data, sb, sh, sn)


def test_operands_that_are_refused():
    good = record()
    for bad in (None, record(data=0), record(data=4104), record(sn=63), record(sb=-64)):
        for at in range(4):
            given = [good] * 4
            given[at] = bad
            assert ops.core.i_rotate(problem(), *given, None) != 0
            assert ops.nat.last_error().startswith("rotate: ")
    # over itself with other strides
    assert ops.core.i_rotate(problem(), good, good, record(sh=64, sn=256), record(data=1 << 20), None) != 0
    assert "strides" in ops.nat.last_error()
    # a gradient of a weight that has nowhere to go, and a workspace that is too small
    assert ops.core.i_rotate_backward(problem(), *[good] * 6, None, 4096, 4096, 1 << 20, None) != 0
    assert "weight" in ops.nat.last_error()
    assert ops.core.i_rotate_backward(problem(), *[good] * 6, 4096, 4096, 4096, 1, None) != 0
    assert "workspace" in ops.nat.last_error()
    assert ops.core.i_rotate(None, good, good, good, good, None) != 0


def test_tensors_that_are_not_on_a_gpu():
    x = torch.zeros((1, 2, 4, 64))
    for call in (lambda: ops.rotate(x), lambda: ops.rotate([1.0]), lambda: ops.rotate(x.double()), lambda: ops.rotated(x, x),
                 lambda: ops.rotate_backward(x, x, x, x)):
        with pytest.raises(TypeError):
            call()


def test_frequencies_and_sections():
    f = ops.frequencies(4, 100.0, device="cpu")
    assert f.dtype == torch.float32 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75]))
    assert ops.sections(1, 2, 0, 1, device="cpu").tolist() == [0, 1, 1, 3]
