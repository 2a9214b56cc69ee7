"""The record of a cache in 8 or 4 bits, as calls pack it and as the C side reads it."""
import struct

import pytest
import torch

from i_amd import quantised as ops


def test_one_description_of_the_struct():
    """What a cache packs when it is made and what a call adds are the halves of what other callers pack whole."""
    fields = list(range(1, 22))
    assert ops._CACHE(*fields, listed=22) == struct.pack("=4Q13qQ4q", *fields, 22)
    assert ops._CACHE(*fields) == ops._CACHE_MEMORY(*fields[:17]) + ops._CACHE_PAGES(*fields[17:], 0)


def record_of(table, b, page=16, pages=9):
    """What a cache on no GPU (index -1) passes of this table."""
    cache = object.__new__(ops.QuantisedCache)
    cache._memory, cache.index, cache.page, cache.pages = b"", -1, page, pages
    record, kept = cache._record(table, b, -1)
    return struct.unpack("=Q4q", record), kept


def test_the_pages_listed_are_those_of_the_view():
    """A table that is a view lists as many pages as it has columns, however far apart its sequences are."""
    wide = torch.arange(24, dtype=torch.int32).view(3, 8)
    for table in (wide, wide[:, :3], wide[:, 3:6], wide[:, 5:], wide[:, 4:5], wide[1:, :7]):
        (address, stride, page, pages, listed), kept = record_of(table, len(table))
        assert (address, stride, page, pages, listed) == (table.data_ptr(), 8, 16, 9, table.shape[1])
    (address, stride, _, _, listed), _ = record_of(wide[1:2, 2:4], 1)
    assert (address, stride, listed) == (wide.data_ptr() + 40, 2, 2)
    # sequences that overlap in memory, or are one: laid out anew
    (address, stride, _, _, listed), kept = record_of(wide[:1].expand(3, 8), 3)
    assert (address, stride, listed) == (kept.data_ptr(), 8, 8) and kept.is_contiguous()
    assert record_of(None, 3)[0] == (0, 0, 16, 9, 0)


@pytest.mark.parametrize("stride, listed, slots", [(8, 2, 32), (8, 0, 128), (2, 2, 32), (8, 8, 128), (0, 3, 48)])
def test_slots_are_those_of_the_pages_listed(stride, listed, slots):
    """More slots than the listed pages hold are refused, whatever lies between two sequences' entries."""
    from i_amd import attention

    operand = attention._TENSOR(4096, 2048, 512, 64)

    def call(max_length):  # (without lengths, which are looked at after the cache: nothing is enqueued)
        problem = ops._TREE(ops.nat.BF16, 2, 4, 2, 3, 64, 0.125, 0.0, 0, 0, max_length, 0, 0, 0, 0, 0, 0, 0, 0, 0, -1)
        cache = ops._CACHE(4096, 4096, 4096, 4096, 4, *(1024, 512, 32, 64, 32, 2) * 2, 4096, stride, 16, 9, listed=listed)
        assert ops.core.i_attend_quantised(problem, operand, cache, operand, None, 4096, 1 << 40, None) != 0
        return ops.nat.last_error()

    assert "slots do not fit" in call(slots + 1)
    assert "lengths" in call(slots)


@pytest.mark.parametrize("listed", [-1, 2 ** 30 + 1])
def test_lists_that_there_are_not(listed):
    from i_amd import attention

    operand = attention._TENSOR(4096, 2048, 512, 64)
    cache = ops._CACHE(4096, 4096, 4096, 4096, 4, *(1024, 512, 32, 64, 32, 2) * 2, 4096, 8, 16, 9, listed=listed)
    move = ops._MOVE(ops.nat.BF16, 2, 2, 4, 64, 0, 0)
    assert ops.core.i_quantised_store(move, operand, operand, cache, None) != 0
    assert "listed" in ops.nat.last_error()
    assert ops.core.i_quantised_load(move, cache, operand, operand, None) != 0
    assert "listed" in ops.nat.last_error()
