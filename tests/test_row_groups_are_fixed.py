"""RowGroups hold what kernels address memory by: they are neither assigned to nor used after a write (host tensors: what is
refused is refused before anything is launched)."""
import copy
import pickle

import pytest
import torch

from ponderv2_amd.grouped_linear import grouped_linear
from ponderv2_amd.row_groups import RowGroups


def groups_of(n, g):
    return RowGroups._made(torch.arange(n, dtype=torch.int32), torch.zeros(g + 1, dtype=torch.int32), n, g)


@pytest.mark.parametrize("name", ["order", "offsets", "n_rows", "n_groups"])
def test_no_assignment(name):
    groups = groups_of(4, 2)
    with pytest.raises(AttributeError):
        setattr(groups, name, getattr(groups, name))
    assert groups.n_rows == 4 and groups.n_groups == 2


@pytest.mark.parametrize("write", [lambda g: g.order.add_(7), lambda g: g.offsets.fill_(9),
                                   lambda g: g.order[1:].zero_(), lambda g: torch.add(g.order, 1, out=g.order)])
def test_groups_that_were_written_to_are_refused(write):
    groups, x, w = groups_of(4, 2), torch.zeros(4, 8), torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):   # (as they were made: as far as the host goes)
        grouped_linear(x, w, groups)
    write(groups)
    for call in (lambda: grouped_linear(x, w, groups), lambda: grouped_linear(x, w.requires_grad_(), groups),
                 lambda: copy.copy(groups)):
        with pytest.raises(RuntimeError, match="were written to"):
            call()


def test_reading_and_copies():
    groups = groups_of(5, 3)
    int(groups.order.sum()), groups.offsets.tolist(), groups.order.clone().add_(1)
    for other in (copy.copy(groups), copy.deepcopy(groups), pickle.loads(pickle.dumps(groups))):
        assert torch.equal(other.order, groups.order) and torch.equal(other.offsets, groups.offsets)
        assert (other.n_rows, other.n_groups) == (5, 3)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            grouped_linear(torch.zeros(5, 8), torch.zeros(3, 3, 8), other)
    with torch.inference_mode():
        inside = groups_of(4, 2)
    for made in (inside, groups_of(4, 2)):
        with torch.inference_mode(), pytest.raises(RuntimeError, match="no CPU fallback"):
            grouped_linear(torch.zeros(4, 8), torch.zeros(2, 3, 8), made)
