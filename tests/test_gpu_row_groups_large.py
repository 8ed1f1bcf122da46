"""group_rows at its limits on the device: more than 2^30 rows, ids of 31 bits (four passes of the sort)."""
import numpy as np
import pytest
import torch

from ponderv2_amd.row_groups import group_rows

pytestmark = pytest.mark.gpu


def test_more_than_2_30_rows(device):
    """Two passes, so that the offsets are searched among the sorted ids.  The rows come in strictly increasing (id, row)
    order, n of them: that is a permutation, and the stable one."""
    n, count = (1 << 30) + (1 << 28) + 12345, 50021
    index = torch.arange(n, dtype=torch.int32, device=device).mul_(7919).remainder_(count + 2).sub_(1)   # (wraps; some ids outside)
    got = group_rows(index, count)
    key = torch.where((index < 0) | (index >= count), count, index)
    step = 1 << 28
    for a in range(0, n, step):      # (in pieces: positions are 64-bit)
        order = got.order[a:a + step + 1]
        k = key[order.long()]
        assert int(order.min()) >= 0 and int(order.max()) < n
        assert bool(((k[1:] > k[:-1]) | ((k[1:] == k[:-1]) & (order[1:] > order[:-1]))).all())
        del order, k
    sizes = torch.zeros(count + 1, dtype=torch.int64, device=device)
    for a in range(0, n, step):
        sizes += torch.bincount(key[a:a + step], minlength=count + 1)
    assert torch.equal(got.offsets[1:].long(), sizes[:count].cumsum(0)) and int(got.offsets[0]) == 0


@pytest.mark.parametrize("n", [4096, 9000])
def test_four_passes(n, device):
    """As many groups as there may be: keys of 31 bits."""
    count = 1 << 30
    rng = np.random.RandomState(10)
    index = np.concatenate([rng.randint(0, count, n - 6), [0, count - 1, count - 1, count, -5, (1 << 31) - 1]])
    index[5] = index[7]
    got = group_rows(torch.from_numpy(index).to(device), count)
    key = np.where((index >= 0) & (index < count), index, count)
    assert np.array_equal(got.order.cpu().numpy(), np.argsort(key, kind="stable"))
    for probe in (0, 1, int(index[5]), int(index[5]) + 1, 1 << 29, count - 1, count):
        assert int(got.offsets[probe]) == int(((index >= 0) & (index < probe)).sum()), probe
