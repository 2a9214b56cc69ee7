"""What the attention calls with masks refuse before any GPU work, at the edges of what their kernels count and hold."""
import ctypes

import pytest

from i_amd import attention as ops
from i_amd import build

BF16, F32 = ops.nat.BF16, ops.nat.F32
REFUSED = ctypes.c_size_t(-1).value


def problem(dtype, hq, hkv, nq, nk, d, b=1, causal=0):
    return ops._PROBLEM(dtype, b, hq, hkv, nq, nk, d, 0.125, 0.0, 0, causal, 0, 0)


# type, query heads of a key head, queries, keys, head size: (key tile, query head, query tile) triples just past and just below 2^31
PAST = [(BF16, 32, 2 ** 20, 2 ** 19, 128), (BF16, 1, 2 ** 22, 2 ** 22, 64), (F32, 16, 2 ** 19, 2 ** 19, 128), (F32, 32, 2 ** 19, 2 ** 19, 64), (BF16, 1, 2 ** 20, 2 ** 22, 256)]
BELOW = [(BF16, 32, 2 ** 20, 2 ** 19 - 128, 128), (BF16, 1, 2 ** 22 - 64, 2 ** 22, 64), (F32, 16, 2 ** 19 - 32, 2 ** 19, 128)]


@pytest.mark.parametrize("case", PAST, ids=str)
def test_work_on_keys_that_cannot_be_counted_is_refused(case):
    dtype, group, nq, nk, d = case
    assert ops.core.i_attend_backward_workspace(problem(dtype, group, 1, nq, nk, d)) == REFUSED
    assert "2^31" in ops.nat.last_error() and "attention_backward" in ops.nat.last_error()
    # the calls themselves too, before they look at a pointer's memory
    record = ops._TENSOR(4096, nq * d, d, d)
    assert ops.core.i_attend_backward(problem(dtype, group, 1, nq, nk, d), *[record] * 5, 4096, *[record] * 3, 4096, 1 << 40, None) != 0
    assert "2^31" in ops.nat.last_error()


@pytest.mark.parametrize("case", BELOW, ids=str)
def test_work_on_keys_that_can_be_counted_is_not(case):
    dtype, group, nq, nk, d = case
    assert ops.core.i_attend_backward_workspace(problem(dtype, group, 1, nq, nk, d)) != REFUSED


@pytest.mark.parametrize("case", [(BF16, 32, 2 ** 20, 2 ** 20, 128), (F32, 32, 2 ** 19, 2 ** 19, 64), (F32, 16, 2 ** 19, 2 ** 19, 256)], ids=str)
def test_weights_of_keys_that_cannot_be_counted_are_refused(case):
    dtype, group, nq, nk, d = case
    assert ops.core.i_attend_weights_workspace(problem(dtype, group, 1, nq, nk, d)) == REFUSED
    assert "2^31" in ops.nat.last_error() and "key_weights" in ops.nat.last_error()
    record = ops._TENSOR(4096, nq * d, d, d)
    assert ops.core.i_attend_weights(problem(dtype, group, 1, nq, nk, d), record, record, 4096, None, 4096, 4096, 1 << 40, None) != 0
    assert "2^31" in ops.nat.last_error()


def test_trees_with_more_rows_than_can_be_counted_are_refused():
    """Rows (query heads times nodes, of all sequences) are counted in 32 bits by the kernel that joins."""
    def tree(b):
        return ops._TREE(BF16, b, 65535, 1, 64, 8, 0.125, 0.0, 0, 0, 100, 0, 0, 0, 0, 0, 0, 0, 0, 0, -1)

    assert ops.core.i_attend_tree_workspace(tree(1024)) == REFUSED
    assert "rows" in ops.nat.last_error()
    assert ops.core.i_attend_tree_workspace(tree(500)) != REFUSED


def test_more_heads_than_can_be_counted_are_refused():
    """Their number times any other extent stays within 64 bits."""
    b = 2 ** 30
    for query, record in ((ops.core.i_attend_backward_workspace, problem(BF16, 4, 4, 8, 8, 64, b=b)),
                          (ops.core.i_attend_weights_workspace, problem(BF16, 4, 4, 8, 8, 64, b=b)),
                          (ops.core.i_attend_tree_workspace, ops._TREE(BF16, b, 4, 4, 1, 64, 0.125, 0.0, 0, 0, 2 ** 30, 0, 0, 0, 0, 0, 0, 0, 0, 0, -1)),
                          (ops.core.i_evict_workspace, ops._EVICT(BF16, b, 65535, 64, 2 ** 30, 0, 2 ** 30, 0, 0, 0, 0, 0, 0, 0, 0, 0))):
        assert query(record) == REFUSED
        assert "too many heads" in ops.nat.last_error()


# ---------------------------------------------------------------- the check of compiled code
def assembly(body, name="attend_grad_keys_bf16_d128"):
    return f"{name}:\n{body}\n.amdhsa_kernel {name}\n.end_amdhsa_kernel\n"


MMA = "\tv_mfma_f32_16x16x32_bf16 a[0:3], v[8:11], a[12:15], a[0:3]\n\ts_endpgm"


@pytest.mark.parametrize("write", ["v_mov_b32_e32 v9, v1", "v_accvgpr_write_b32 a13, v1", "v_accvgpr_write_b32 a2, v1", "v_permlane16_swap_b32 v1, v8", "v_cvt_pk_bf16_f32 v11, v0, v1"])
def test_matrix_operands_read_too_early_are_found(write):
    """In every kernel, the ones with inline matrix instructions whose names do not end in _w4 among them."""
    for name in ("attend_grad_keys_bf16_d128", "gemm_w4"):
        assert len(build.early_mfma_operands(assembly(f"\t{write}\n{MMA}", name))) == 1
        assert len(build.early_mfma_operands(assembly(f"\t{write}\n\ts_mov_b32 s0, 0\n{MMA}", name))) == 1
        assert len(build.early_mfma_operands(assembly(f"\t{write}\n\ts_cbranch_scc1 .LBB0_1\n\ts_nop 4\n.LBB0_1:\n{MMA}", name))) == 1
        assert build.early_mfma_operands(assembly(f"\t{write}\n\ts_nop 1\n{MMA}", name)) == []
        assert build.early_mfma_operands(assembly(f"\t{write}\n\ts_mov_b32 s0, 0\n\ts_mov_b32 s1, 0\n{MMA}", name)) == []
    with pytest.raises(RuntimeError, match="operands"):
        build.check_assembly(assembly(f"\t{write}\n{MMA}"))


def test_other_writes_before_a_matrix_instruction_are_none():
    for line in ("v_mov_b32_e32 v12, v9", "v_cmp_gt_f32_e64 s[8:9], v8, v9", "v_mfma_f32_16x16x32_bf16 a[0:3], v[16:19], a[16:19], 0", "ds_read_b128 v[8:11], v1"):
        assert build.early_mfma_operands(assembly(f"\t{line}\n{MMA}")) == []


# ---------------------------------------------------------------- eviction over what it reads
def test_eviction_over_its_own_lengths_weights_or_positions_is_refused():
    """Workgroups read them at different times than others write them, so that the result would depend on which comes first."""
    b, hkv, d, keep, n = 2, 2, 64, 10, 30
    cache = ops._CACHE(1 << 20, 2 << 20, hkv * n * d, n * d, d, hkv * n * d, n * d, d, 0, 0, n, b)
    new = ops._CACHE(3 << 20, 4 << 20, hkv * keep * d, keep * d, d, hkv * keep * d, keep * d, d, 0, 0, keep, b)
    places = dict(lengths=1 << 12, weights=2 << 12, positions=4 << 12, weights_out=6 << 12, positions_out=8 << 12, lengths_out=10 << 12)

    def call(**at):
        p = dict(places, **at)
        record = ops._EVICT(BF16, b, hkv, d, keep, 2, n, p["lengths"], p["weights"], n, p["positions"], n, p["weights_out"], p["positions_out"], keep, p["lengths_out"])
        assert ops.core.i_evict(record, cache, new, 1 << 24, 1 << 20, None) != 0
        return ops.nat.last_error()

    floats = 4 * b * hkv
    for name, at in (("lengths", {"lengths_out": places["lengths"]}), ("lengths", {"lengths_out": places["lengths"] + 4}),
                     ("weights", {"weights_out": places["weights"]}), ("weights", {"weights_out": places["weights"] + floats * n - 4}),
                     ("weights", {"weights_out": places["weights"] - floats * keep + 4}), ("positions", {"positions_out": places["positions"]})):
        message = call(**at)
        assert "evict" in message and name in message and "share memory" in message
