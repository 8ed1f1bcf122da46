"""Refusals of the per-row-id operators (row_groups, embedding, grouped_linear, distillation): what they do not take is
refused by name before anything is launched, so all of this runs on a host without a GPU."""
import ctypes

import pytest
import torch

from ponderv2_amd import _lib
from ponderv2_amd.distillation import topk_distillation
from ponderv2_amd.embedding import embedding
from ponderv2_amd.grouped_linear import grouped_linear
from ponderv2_amd.row_groups import RowGroups, group_rows

BADARG = -1


def ids(*shape, dtype=torch.int64):
    return torch.zeros(shape, dtype=dtype)


def groups_of(n, g):
    return RowGroups._made(torch.arange(n, dtype=torch.int32), torch.zeros(g + 1, dtype=torch.int32), n, g)


def test_host_tensors_are_refused():
    for call in (lambda: group_rows(ids(4), 2), lambda: RowGroups.from_offset(ids(2), 4),
                 lambda: embedding(ids(4), torch.zeros(3, 8)),
                 lambda: grouped_linear(torch.zeros(4, 8), torch.zeros(2, 3, 8), groups_of(4, 2)),
                 lambda: topk_distillation(torch.zeros(4, 8), ids(4, 2), torch.zeros(4, 2))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bool, torch.int16, torch.uint8])
def test_ids_are_int64_or_int32(dtype):
    bad = torch.zeros(4).to(dtype)
    for call in (lambda: group_rows(bad, 2), lambda: RowGroups.from_offset(bad, 4),
                 lambda: embedding(bad, torch.zeros(3, 8)),
                 lambda: topk_distillation(torch.zeros(8), bad, torch.zeros(4))):
        with pytest.raises(TypeError, match="int64 or int32"):
            call()


@pytest.mark.parametrize("count", [0, -1, (1 << 30) + 1])
def test_group_count_range(count):
    with pytest.raises(ValueError, match="groups"):
        group_rows(ids(4), count)


@pytest.mark.parametrize("weight", [torch.zeros(3), torch.zeros(3, 4, 5), torch.zeros(0, 4), torch.zeros(4, 0)])
def test_embedding_weight_shape(weight):
    with pytest.raises(ValueError, match="weight is"):
        embedding(ids(4), weight)


def test_embedding_weight_type():
    with pytest.raises(TypeError, match="float64"):
        embedding(ids(4), torch.zeros(3, 4, dtype=torch.float64))


def test_grouped_linear_shapes_and_types():
    x, w, g = torch.zeros(4, 8), torch.zeros(2, 3, 8), groups_of(4, 2)
    for bad, match in (((x, w, torch.zeros(3)), None), ((x, w, None), None)):
        with pytest.raises(TypeError, match="groups is what"):
            grouped_linear(*bad)
    for bad in ((torch.zeros(4, 7), w, g), (torch.zeros(8), w, g), (x, torch.zeros(3, 8), g)):
        with pytest.raises(ValueError, match="expected, got"):
            grouped_linear(*bad)
    with pytest.raises(ValueError, match="but groups of 5 rows"):
        grouped_linear(x, w, groups_of(5, 2))
    with pytest.raises(ValueError, match="in 3 groups"):
        grouped_linear(x, w, groups_of(4, 3))
    with pytest.raises(ValueError, match="bias is"):
        grouped_linear(x, w, g, torch.zeros(3))
    with pytest.raises(ValueError, match="widths 1 to"):
        grouped_linear(torch.zeros(4, 0), torch.zeros(2, 3, 0), g)
    for bad in ((x.half(), w, g), (x, w.bfloat16(), g), (x.double(), w.double(), g), (x, w, g, torch.zeros(2, 3).half())):
        with pytest.raises(TypeError, match="all float32, all bfloat16 or all float16"):
            grouped_linear(*bad)


def test_row_groups_are_not_made_by_hand():
    """Kernels address memory by their contents."""
    with pytest.raises(TypeError, match="are made by group_rows"):
        RowGroups(torch.arange(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 4, 2)


def test_grouped_linear_group_limit():
    with pytest.raises(ValueError, match="4096 groups"):
        grouped_linear(torch.zeros(4, 1), torch.zeros(4097, 1, 1), groups_of(4, 4097))


def test_topk_distillation_arguments():
    s, i, t = torch.zeros(4, 8), ids(4, 2), torch.zeros(4, 2)
    for bad in ((s, i, torch.zeros(4, 3)), (s, ids(3, 2), torch.zeros(3, 2)), (s, ids(2), torch.zeros(2)),
                (torch.zeros(2, 4, 8), i, t)):
        with pytest.raises(ValueError, match="expected, got"):
            topk_distillation(*bad)
    with pytest.raises(ValueError, match="0 listed"):
        topk_distillation(s, ids(4, 0), torch.zeros(4, 0))
    with pytest.raises(ValueError, match="1025 listed"):
        topk_distillation(s, ids(4, 1025), torch.zeros(4, 1025))
    with pytest.raises(ValueError, match="reduction"):
        topk_distillation(s, i, t, reduction="batchmean")
    for temperature in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            topk_distillation(s, i, t, temperature=temperature)
    for bad in ((s.double(), i, t), (s, i, t.double()), (s.long(), i, t)):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            topk_distillation(*bad)


def test_temperatures_out_of_range():
    s, i, t = torch.zeros(4, 8), ids(4, 2), torch.zeros(4, 2)
    for temperature in (0.99e-4, 1e-30, 1.01e4, 1e30):
        with pytest.raises(ValueError, match="0.0001 to 10000"):
            topk_distillation(s, i, t, temperature=temperature)
    L, p, n = _lib.lib(), ctypes.c_void_p(64), None
    for temperature in (1e-30, 1e30, float("nan")):
        assert L.pv2_topk_distill_forward(p, 0, 4, 8, 8, p, 1, 2, p, 0, 2, 2, temperature, 0, p, p, n, p, p, n) == BADARG
        assert L.pv2_topk_distill_backward(p, 0, 4, 8, 8, p, 1, 2, p, 0, 2, 2, temperature, p, p, 0, n, p, n) == BADARG


def test_c_entries_refuse_before_they_launch():
    """Null pointers, sizes out of range and unknown element types come back as an argument error with a text."""
    L, p, n = _lib.lib(), ctypes.c_void_p(64), None
    calls = [
        (L.pv2_row_groups, (n, 1, 4, 2, p, p, n, p, n)),
        (L.pv2_row_groups, (p, 1, 4, 0, p, p, n, p, n)),
        (L.pv2_row_groups, (p, 1, 5000, 2, p, p, n, n, n)),       # no workspace
        (L.pv2_row_groups, (p, 1, (1 << 31) - 4096, 2, p, p, n, p, n)),
        (L.pv2_row_groups, (p, 1, 4, (1 << 30) + 1, p, p, n, p, n)),
        (L.pv2_row_offsets, (n, 1, 2, 4, p, n)),
        (L.pv2_row_offsets, (p, 1, 0, 4, p, n)),
        (L.pv2_embedding_forward, (p, 1, 4, n, 0, 3, 8, 8, 1.0, p, n)),
        (L.pv2_embedding_forward, (p, 1, 4, p, 3, 3, 8, 8, 1.0, p, n)),
        (L.pv2_embedding_forward, (p, 1, 4, p, 0, 3, 0, 8, 1.0, p, n)),
        (L.pv2_embedding_backward, (p, 1, 4, p, 0, 3, 8, 8, 1.0, ctypes.c_void_p(65), p, n)),
        (L.pv2_embedding_backward, (n, 1, 4, p, 0, 3, 8, 8, 1.0, p, p, n)),
        (L.pv2_grouped_linear_forward, (p, 0, 4, 8, 8, n, 8, 8, 2, 3, n, n, p, p, n)),
        (L.pv2_grouped_linear_forward, (p, 7, 4, 8, 8, p, 8, 8, 2, 3, n, n, p, p, n)),
        (L.pv2_grouped_linear_forward, (p, 0, 0, 8, 8, p, 8, 8, 2, 3, n, n, p, p, n)),
        (L.pv2_grouped_linear_grad_input, (p, 0, 4, 3, 3, p, 8, 8, 0, 8, n, p, p, n)),
        (L.pv2_grouped_linear_grad_input, (p, 0, 4, 3, 3, p, 8, 8, 4097, 8, n, p, p, n)),
        (L.pv2_grouped_linear_grad_weight, (p, 0, 4, 3, 3, p, 0, 8, 2, n, p, n, p, n, n)),
        (L.pv2_grouped_linear_grad_weight, (p, 0, 1 << 20, 3, 3, p, 8, 8, 2, n, p, n, p, n, n)),  # no workspace
        (L.pv2_topk_distill_forward, (p, 0, 4, 8, 8, p, 1, 2, p, 0, 2, 1025, 1.0, 0, p, p, n, p, p, n)),
        (L.pv2_topk_distill_forward, (p, 0, 4, 8, 8, p, 1, 2, p, 0, 2, 2, 0.0, 0, p, p, n, p, p, n)),
        (L.pv2_topk_distill_forward, (p, 5, 4, 8, 8, p, 1, 2, p, 0, 2, 2, 1.0, 0, p, p, n, p, p, n)),
        (L.pv2_topk_distill_backward, (p, 0, 4, 8, 8, p, 1, 2, p, 9, 2, 2, 1.0, p, p, 0, n, p, n)),
        (L.pv2_topk_distill_backward, (p, 0, 4, 8, 8, p, 1, 2, p, 0, 2, 2, 1.0, n, p, 0, n, p, n)),
    ]
    for fn, args in calls:
        assert fn(*args) == BADARG, (fn.__name__, args)
        assert _lib.lib().pv2_last_error(), fn.__name__


def test_workspaces_cover_what_is_asked():
    L = _lib.lib()
    assert L.pv2_row_groups_workspace_ints(0, 5) == 0 == L.pv2_row_groups_workspace_ints(4096, 8192)
    assert L.pv2_row_groups_workspace_ints(4096, 8193) >= 4096
    assert L.pv2_row_groups_workspace_ints(100000, 5) >= 3 * 100000
    assert L.pv2_grouped_linear_workspace_floats(0, 100, 4, 64, 64) == 0          # no group can be split
    # 3 groups of 512 x 96: four 128 x 128 tiles, at most 128 + 3 items
    assert 0 < L.pv2_grouped_linear_workspace_floats(0, 92417, 3, 512, 96) <= (128 + 3) * (512 * 96 + 512)
    assert L.pv2_topk_distill_workspace_floats(1, 131072, 16) > 2
