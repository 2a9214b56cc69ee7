"""The record of a cache in 8 or 4 bits, as calls pack it and as the C side reads it."""
import struct

import pytest
import torch

from i_amd import quantised as ops


def test_one_description_of_the_struct():
    """What a cache packs when it is made and what a call adds are the halves of what other callers pack whole."""
    fields = list(range(1, 22))
    assert ops._CACHE(*fields) == struct.pack("=4Q13qQ3q", *fields)
    assert ops._CACHE(*fields) == ops._CACHE_MEMORY(*fields[:17]) + ops._CACHE_PAGES(*fields[17:])
