"""Sizes past what the entry points count in are refused by name, not cut: all of it before a launch, on the host."""
import ctypes

import pytest
import torch

from ponderv2_amd import _lib
from ponderv2_amd.embedding import embedding

BADARG = -1


@pytest.mark.parametrize("width", [1 << 30, (1 << 31) + 8, (1 << 32) + 8])
def test_embedding_width(width):
    """(2^32 + 8 columns would be looked up as 8)"""
    weight = torch.zeros(1, 1).expand(2, width)
    with pytest.raises(ValueError, match="channels"):
        embedding(torch.zeros(4, dtype=torch.int64), weight)


def test_embedding_width_of_the_entries():
    L, p, n = _lib.lib(), ctypes.c_void_p(64), None
    assert L.pv2_embedding_forward(p, 1, 4, p, 0, 3, 1 << 30, 1 << 30, 1.0, p, n) == BADARG
    assert L.pv2_embedding_backward(p, 1, 4, p, 0, 3, 1 << 30, 1 << 30, 1.0, p, p, n) == BADARG
