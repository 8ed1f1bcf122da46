"""Sizes past what the entry points count in are refused by name, not cut: all of it before a launch, on the host."""
import ctypes

import pytest
import torch

from ponderv2_amd import _lib
from ponderv2_amd.distillation import topk_distillation
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


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace_of_a_weight_gradient_does_not_grow_with_the_groups(dtype):
    """Only groups that are split leave partial results: 32768 rows have at most 2 * 32767 / 256 of them (16-bit types take
    pieces of 1024 rows or more), however many groups there are."""
    L = _lib.lib()
    slab = 512 * 512 + 512
    floats = [L.pv2_grouped_linear_workspace_floats(dtype, 32768, g, 512, 512) for g in (1, 64, 512, 4096)]
    most = 2 * (32767 // (256 if dtype == 0 else 1024)) * slab
    assert 0 < floats[0] <= most and all(f <= most for f in floats)
    # 20000 rows over 4096 groups: no more than 38 slabs beside a gradient of 4096
    assert L.pv2_grouped_linear_workspace_floats(1, 20000, 4096, 1024, 1024) <= 38 * (1024 * 1024 + 1024)
    for rows in (1, 255, 256):   # none can be split
        assert L.pv2_grouped_linear_workspace_floats(dtype, rows, 8, 64, 64) == 0


def test_gradients_of_nothing():
    """grad_weight may be null (a bias alone), not both; x is needed for the weights."""
    L, p, n = _lib.lib(), ctypes.c_void_p(64), None
    for x, gw, gb in ((p, n, n), (n, n, n), (n, p, p)):
        assert L.pv2_grouped_linear_grad_weight(p, 0, 4, 3, 3, x, 8, 8, 2, n, p, n, gw, gb, n) == BADARG
    # many rows: a bias alone has a workspace of its own size
    assert L.pv2_grouped_linear_grad_weight(p, 0, 1 << 20, 3, 3, n, 8, 8, 2, n, p, n, n, p, n) == BADARG
    assert 0 < L.pv2_grouped_linear_bias_workspace_floats(0, 1 << 20, 2, 3) == (
        L.pv2_grouped_linear_workspace_floats(0, 1 << 20, 2, 3, 8) // (3 * 8 + 3) * 3)


def test_scales_and_temperatures_take_no_gradient():
    """A learnable one is refused: its gradient would be lost."""
    learnable = torch.tensor(2.0, requires_grad=True)
    ids, lists = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 2)
    with pytest.raises(TypeError, match="scale is a number and takes no gradient"):
        embedding(ids, torch.zeros(3, 8), learnable)
    with pytest.raises(TypeError, match="temperature is a number and takes no gradient"):
        topk_distillation(torch.zeros(4, 8), lists.long(), lists, learnable)
    for number in (2, 2.0, torch.tensor(2.0), learnable.detach()):
        for call in (lambda: embedding(ids, torch.zeros(3, 8), number),
                     lambda: topk_distillation(torch.zeros(4, 8), lists.long(), lists, number)):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call()


def test_an_unknown_type_is_refused_before_the_sort():
    L, p, n = _lib.lib(), ctypes.c_void_p(64), None
    for dtype in (-1, 3, 7):
        assert L.pv2_embedding_backward(p, 1, 4, p, dtype, 3, 8, 8, 1.0, p, p, n) == BADARG
