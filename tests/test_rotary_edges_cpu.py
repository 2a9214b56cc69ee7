"""What the kept size of the gradient's workspace goes by."""
import pytest
import torch

from i_amd import rotary as ops

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sizes_that_are_kept_name_their_workspace(monkeypatch, dtype):
    """Problems of the same sizes have the same workspace, however their pairs lie and whatever they are given."""
    monkeypatch.setattr(ops, "_first_operand", lambda q: (ops._DTYPES[q.dtype], -1))  # (operands without a GPU, of which only the records are made)
    found, layouts = {}, set()
    for b, hq, hkv, n, d in ((2, 16, 4, 2048, 128), (1, 3, 3, 1500, 40), (2, 4, 0, 800, 256), (1, 2, 1, 3, 64)):
        q, k = (torch.empty(1, dtype=dtype).expand(b, h, n, d) for h in (hq, hkv))
        for pairs in (0, 4, 7, 12, 13, 20, d // 2):
            for interleaved in (False, True, 0, 1):
                for weights in ("", "q", "k", "qk"):
                    for weight_dtype in {dtype, F32}:
                        given = {f"{side}_weight": torch.ones(d, dtype=weight_dtype) if side in weights else None for side in "qk"}
                        if hkv == 0 and "k" in weights:
                            continue
                        turning = (torch.zeros((b, n), dtype=torch.int32), torch.ones(pairs)) if pairs else (None, None)
                        problem, _, sizes = ops._problem(q, k if hkv else None, *turning, None, interleaved, eps=1e-6, **given)
                        size = ops.core.i_rotate_backward_workspace(problem)
                        assert found.setdefault(sizes, size) == size, (b, hq, hkv, n, d, pairs, interleaved, weights)
                        layouts.add((b, hq, hkv, n, d, weights, size))
    assert len(layouts) > len({x[:-1] for x in layouts}) or dtype is F32  # (there are problems that only the pairs tell apart)
