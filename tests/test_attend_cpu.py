"""What the attention calls with masks refuse before any GPU work, and the check of their compiled code."""
import ctypes
import math

import pytest
import torch

from i_amd import attention as ops
from i_amd import build


def test_tensors_that_are_not_on_a_gpu():
    x = torch.zeros((1, 2, 4, 64))
    lengths = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.attention(x, x, x), lambda: ops.key_weights(x, x, torch.zeros((1, 2, 4))),
                 lambda: ops.tree_attention(x, x, x, lengths), lambda: ops.evict(x, x, torch.zeros((1, 2, 4)), lengths, 2, 1),
                 lambda: ops.attention([1.0], x, x), lambda: ops.attention(x.double(), x, x)):
        with pytest.raises(TypeError):
            call()


def problem(dtype=0, b=1, hq=4, hkv=2, nq=8, nk=8, d=64, scale=0.125, cap=0.0, causal=0):
    return ops._PROBLEM(dtype, b, hq, hkv, nq, nk, d, scale, cap, 0, causal, 0, 0)


def tree(dtype=0, b=1, hq=4, hkv=2, nodes=3, d=64, scale=0.125, cap=0.0, max_length=100):
    return ops._TREE(dtype, b, hq, hkv, nodes, d, scale, cap, 0, 0, max_length, 0, 0, 0, 0, 0, 0, 0, 0, 0, -1)


REFUSED = ctypes.c_size_t(-1).value


@pytest.mark.parametrize("change", [{"dtype": 9}, {"b": -1}, {"hq": 3}, {"hkv": 0}, {"d": 60}, {"d": 264}, {"d": 0}, {"scale": math.nan},
                                    {"cap": -1.0}, {"cap": math.inf}, {"nk": -1}], ids=str)
def test_problems_that_are_refused(change):
    for query, name in ((ops.core.i_attend_backward_workspace, "attention_backward"), (ops.core.i_attend_weights_workspace, "key_weights")):
        assert query(problem()) != REFUSED
        assert query(problem(**change)) == REFUSED
        assert name in ops.nat.last_error()


@pytest.mark.parametrize("change", [{"dtype": 9}, {"nodes": 0}, {"nodes": 65}, {"max_length": 2}, {"hq": 3}, {"d": 12}, {"cap": -2.0}], ids=str)
def test_trees_that_are_refused(change):
    assert ops.core.i_attend_tree_workspace(tree()) != REFUSED
    assert ops.core.i_attend_tree_workspace(tree(**change)) == REFUSED
    assert "tree_attention" in ops.nat.last_error()


def test_missing_arguments_are_errors():
    """Null records and pointers come back as errors; nothing reaches a GPU."""
    assert ops.core.i_attend(None, None, None, None, None, None, None) != 0
    assert ops.core.i_attend(problem(), None, None, None, None, None, None) != 0
    record = ops._TENSOR(0, 2048, 512, 64)
    assert ops.core.i_attend(problem(), record, record, record, record, None, None) != 0
    assert ops.core.i_attend_tree(tree(), record, None, record, None, None, 0, None) != 0


def assembly(body):
    return f"kernel:\n{body}\n.amdhsa_kernel kernel\n.end_amdhsa_kernel\n"


def test_matrix_results_read_too_early_are_found():
    mma = "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], 0\n"
    late = mma + "\ts_nop 7\n\tv_add_f32_e32 v5, v0, v6\n\ts_endpgm"
    assert build.early_mfma_reads(assembly(late)) == []
    early = mma + "\ts_nop 3\n\tv_add_f32_e32 v5, v0, v6\n\ts_endpgm"
    assert len(build.early_mfma_reads(assembly(early))) == 1
    other = mma + "\tv_add_f32_e32 v5, v7, v6\n\ts_endpgm"
    assert build.early_mfma_reads(assembly(other)) == []
    # beyond a branch, on the shorter of two ways
    branch = mma + "\ts_cbranch_scc1 .LBB0_1\n\ts_nop 7\n.LBB0_1:\n\tv_mov_b32_e32 v9, v3\n\ts_endpgm"
    assert len(build.early_mfma_reads(assembly(branch))) == 1
    # a chain: the sum goes on, and its last product counts
    chain = mma + mma.replace(", 0\n", ", v[0:3]\n") + "\ts_nop 7\n\tv_mov_b32_e32 v9, v3\n\ts_endpgm"
    assert build.early_mfma_reads(assembly(chain)) == []
