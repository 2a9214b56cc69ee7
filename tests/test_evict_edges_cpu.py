"""Eviction to pages of a table that is a view."""
import pytest
import torch

from i_amd import attention as ops


def test_a_view_lists_the_pages_of_its_columns(monkeypatch):
    """A new cache whose table is cut out of a wider one has no more pages than the table has columns: what does not fit them is
    refused, and not written to pages beside the view."""
    monkeypatch.setattr(ops, "_first_operand", lambda q, name="q": (ops._DTYPES[q.dtype], -1))  # (operands without a GPU, of which only the records are made)
    enqueued = []
    monkeypatch.setattr(ops, "_enqueue", lambda index, entry, *arguments: enqueued.append(entry))
    monkeypatch.setattr(ops, "_workspace", lambda *arguments: (None, 0, 0))
    b, hkv, n, d, page = 2, 2, 90, 64, 16
    k = torch.zeros((b, hkv, n, d))
    new = torch.zeros((b * 8, hkv, page, d))
    wide = torch.arange(b * 8, dtype=torch.int32).view(b, 8)
    weights, lengths = torch.zeros((b, hkv, n)), torch.full((b,), n, dtype=torch.int32)

    def call(keep, table_out, **options):
        out = (new, new.clone(), torch.zeros((b, hkv, 100)), torch.zeros((b, hkv, 100), dtype=torch.int32), torch.zeros(b, dtype=torch.int32))
        ops.evict(k, k, weights, lengths, keep, 2, table_out=table_out, out=out, **options)

    for table in (wide[:, :2], wide[:, 3:5], wide[:, 6:], wide[:, :2].contiguous()):
        call(32, table)
        for keep in (33, 100):
            with pytest.raises(RuntimeError, match="evict.*do not fit 2 pages of 16"):
                call(keep, table)
        call(100, table, max_length=30)  # (no more than 30 slots there are)
    assert enqueued == [ops.core.i_evict] * 8
    call(100, wide)
