"""group_rows / RowGroups.from_offset on the device against numpy's stable argsort: whole numbers, so every value has to
be equal."""
import numpy as np
import pytest
import torch

from ponderv2_amd.row_groups import RowGroups, group_rows
from row_ops_oracle import group_order

pytestmark = pytest.mark.gpu


def check(index, count, device):
    got = group_rows(torch.as_tensor(index).to(device), count)
    order, offsets = group_order(index, count)
    assert got.n_rows == order.size and got.n_groups == count
    assert np.array_equal(got.order.cpu().numpy(), order)
    assert np.array_equal(got.offsets.cpu().numpy(), offsets)


# one workgroup takes up to 4096 rows; more are sorted by many, in one pass (< 1024 groups), two (< 2^20) or three
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1023, 1024, 1025, 4095, 4096, 4097, 8192, 70001])
@pytest.mark.parametrize("count", [1, 2, 7, 255, 256, 1023, 1024, 9001, 1 << 20])
def test_random_ids(n, count, device):
    rng = np.random.RandomState(n * 31 + count)
    index = rng.randint(-2, count + 2, n)          # a few outside on both sides
    check(index, count, device)


@pytest.mark.parametrize("n", [5, 4096, 5000, 300000])
@pytest.mark.parametrize("kind", ["one id", "none", "sorted", "reversed", "extremes", "two ids"])
def test_ordered_ids(n, kind, device):
    index = {"one id": np.full(n, 3), "none": np.full(n, -1), "sorted": np.arange(n) % 997 * 0 + np.sort(
        np.random.RandomState(1).randint(0, 997, n)), "reversed": np.arange(n)[::-1] % 997,
        "extremes": np.where(np.arange(n) % 2, np.iinfo(np.int64).max, np.iinfo(np.int64).min),
        "two ids": np.arange(n) % 2 * 996}[kind]
    check(index, 997, device)


def test_int32_shapes_and_strides(device):
    rng = np.random.RandomState(5)
    index = rng.randint(0, 40, (300, 70))
    t = torch.from_numpy(index).to(device)
    for view, flat in ((t.int(), index), (t[:, ::2], index[:, ::2]), (t.t(), index.T), (t[7], index[7])):
        got = group_rows(view, 40)
        order, offsets = group_order(flat, 40)
        assert np.array_equal(got.order.cpu().numpy(), order) and np.array_equal(got.offsets.cpu().numpy(), offsets)


# where blocks of another size begin, with and without a full last block
@pytest.mark.parametrize("n", [4097, 1 << 18, (1 << 18) + 1, 1 << 21, (1 << 21) + 1])
@pytest.mark.parametrize("count", [36, 50021])
def test_sizes_of_blocks(n, count, device):
    rng = np.random.RandomState(n % 1000 + count)
    check(rng.randint(-1, count, n), count, device)


@pytest.mark.parametrize("count", [1, 5, 2000])
def test_no_rows(count, device):
    got = group_rows(torch.zeros(0, dtype=torch.int64, device=device), count)
    assert got.order.numel() == 0 and got.offsets.tolist() == [0] * (count + 1)


def test_large_group_numbers(device):
    """Four passes of the sort (ids of 30 bits)."""
    rng = np.random.RandomState(9)
    index = np.concatenate([rng.randint(0, 1 << 28, 9000), [0, (1 << 28) - 1, 1 << 28, -5]])
    got = group_rows(torch.from_numpy(index).to(device), 1 << 28)
    order, _ = group_order(index, 1 << 28)
    assert np.array_equal(got.order.cpu().numpy(), order)
    for probe in (0, 1, int(index[3]), int(index[3]) + 1, (1 << 28) - 1, 1 << 28):
        assert int(got.offsets[probe]) == int(((index >= 0) & (index < min(probe, 1 << 28))).sum()), probe


@pytest.mark.parametrize("offset,n,want", [
    ([3, 3, 10], 12, [0, 3, 3, 10]), ([0], 0, [0, 0]), ([5], 3, [0, 3]),
    ([4, 2, 9], 8, [0, 4, 4, 8]), ([-3, 2], 8, [0, 0, 2])])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_from_offset(offset, n, want, dtype, device):
    got = RowGroups.from_offset(torch.tensor(offset, dtype=dtype, device=device), n)
    assert got.order is None and got.offsets.tolist() == want and (got.n_rows, got.n_groups) == (n, len(offset))


def test_from_offset_of_many_groups(device):
    counts = np.random.RandomState(2).randint(0, 5, 1000)
    got = RowGroups.from_offset(torch.from_numpy(np.cumsum(counts)).to(device), int(counts.sum()))
    assert np.array_equal(got.offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(counts)]))


def test_in_a_graph_and_on_another_stream(device):
    index = torch.randint(-1, 300, (20000,), device=device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        group_rows(index, 300)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = group_rows(index, 300)
    for seed in range(3):
        torch.manual_seed(seed)
        index.copy_(torch.randint(-1, 300, (20000,), device=device))
        graph.replay()
        torch.cuda.synchronize()
        order, offsets = group_order(index.cpu().numpy(), 300)
        assert np.array_equal(got.order.cpu().numpy(), order) and np.array_equal(got.offsets.cpu().numpy(), offsets)
