"""grouped_linear() on whole numbers so small that every product and every sum is exact in fp32: results have to equal the
64-bit ones after one rounding, whatever the number of rows, so that a row left out or taken twice shows."""
import pytest
import torch

from ponderv2_amd.grouped_linear import grouped_linear
from ponderv2_amd.row_groups import group_rows
from row_ops_oracle import DTYPES

pytestmark = pytest.mark.gpu


def whole(low, high, *shape, device, dtype):
    return torch.randint(low, high + 1, shape, device=device).to(dtype)


def products(x, w, index, bias, gy):
    """The definition in fp32 where it is exact: sums of whole numbers below 2^24 (by torch, group by group)."""
    x, w, bias, gy = (t.float() for t in (x, w, bias, gy))
    y, d_x, d_w, d_b = x.new_zeros(len(x), w.shape[1]), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    for e in range(len(w)):
        r = torch.nonzero(index == e)[:, 0]
        y[r], d_x[r] = x[r] @ w[e].T + bias[e], gy[r] @ w[e]
        d_w[e], d_b[e] = gy[r].T @ x[r], gy[r].sum(0)
    return y, d_x, d_w, d_b


def check(m, sizes, k, n, dtype, device, most=2):
    """Groups of ``sizes`` rows (the rest of the m rows in no group), in random order."""
    g = len(sizes)
    index = torch.cat([torch.repeat_interleave(torch.arange(g), torch.tensor(sizes)),
                       torch.full((m - sum(sizes),), -1)])[torch.randperm(m)].to(device)
    x, w = whole(-most, most, m, k, device=device, dtype=dtype), whole(-most, most, g, n, k, device=device, dtype=dtype)
    bias, gy = whole(-9, 9, g, n, device=device, dtype=dtype), whole(-1, 1, m, n, device=device, dtype=dtype)
    assert max(most * most * k + 9, most * n, most * max(sizes)) < 2 ** 24
    leaves = [t.detach().requires_grad_() for t in (x, w, bias)]
    y = grouped_linear(leaves[0], leaves[1], group_rows(index, g), leaves[2])
    grads = torch.autograd.grad(y, leaves, gy)
    for name, got, want in zip(("y", "d_x", "d_w", "d_b"), (y.detach(), *grads), products(x, w, index, bias, gy)):
        assert torch.equal(got, want.to(dtype)), f"{name}: {int((got != want.to(dtype)).sum())} values differ"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(40, 24), (33, 17)])
def test_split_groups_among_many(dtype, k, n, device):
    """Groups of no, one, two and many pieces next to each other, in every 64 of more than 200."""
    torch.manual_seed(20)
    sizes = [(0, 1, 5, 256, 257, 1024, 1025, 300, 3000, 513, 0, 2049, 64)[i % 13] for i in range(201)]
    check(sum(sizes) + 77, sizes, k, n, dtype, device)


# Aligned 16-bit operands of so many rows take tiles of 256 x 256 where a width has an even number of 128 columns (1000, 712:
# the last tile is partial and the last step of the reduction short) and of 128 x 128 where it is odd (1032); a group's weight
# gradient is cut into items of 4000 to 8256 rows, whose row numbers are taken in several turns.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(1000, 1000), (712, 1032), (1032, 712), (1032, 1032)])
def test_large_tiles(dtype, k, n, device):
    torch.manual_seed(23)
    check(33000, [1, 0, 20000, 3777, 9000], k, n, dtype, device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1919, 1920, 1921, 1952, 3840, 3841, 8000])
def test_items_about_where_row_numbers_are_taken_anew(dtype, rows, device):
    """A group's rows in one item of a weight gradient, in two at most: 1920 rows' numbers are held at a time (33000 rows and
    72 or 36 tiles of dW make pieces of 8256 or 4160 rows)."""
    torch.manual_seed(rows)
    for k, n in ((1152, 1024), (1024, 1152)):
        check(33000, [rows, 33000 - rows - 40], k, n, dtype, device)


def test_memory_of_a_weight_gradient_with_many_groups(device):
    """4096 groups of 256 x 256: beside the gradient (0.5 GB in bf16) partial results of a few split groups only."""
    torch.manual_seed(21)
    m, g, k = 20000, 4096, 256
    x, gy = (whole(-2, 2, m, k, device=device, dtype=torch.bfloat16) for _ in range(2))
    w = torch.zeros(g, k, k, device=device, dtype=torch.bfloat16, requires_grad=True)
    groups = group_rows(torch.randint(0, g, (m,), device=device), g)
    y = grouped_linear(x, w, groups)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    torch.autograd.grad(y, w, gy)
    assert torch.cuda.max_memory_allocated() - before <= 1.1 * w.numel() * 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(64, 48), (264, 520), (33, 131)])
def test_a_bias_alone(dtype, k, n, device):
    """Frozen weights, a trained bias: the same sums as beside the weight gradient (exact on whole numbers), whose memory is
    not taken."""
    torch.manual_seed(22)
    sizes = torch.tensor([0, 1, 5000, 130, 1024, 1025, 0, 3000])
    index = torch.cat([torch.repeat_interleave(torch.arange(8), sizes), torch.full((60,), -1)])
    index = index[torch.randperm(len(index))].to(device)
    m, groups = len(index), group_rows(index, 8)
    x, gy = torch.randn(m, k, device=device).to(dtype), whole(-9, 9, m, n, device=device, dtype=dtype)
    w, b = torch.randn(8, n, k, device=device).to(dtype), torch.randn(8, n, device=device).to(dtype).requires_grad_()
    sums = torch.zeros(9, n, device=device).index_add_(0, torch.where(index < 0, 8, index), gy.float())[:8]
    trained = w.clone().requires_grad_()
    _, want = torch.autograd.grad(grouped_linear(x, trained, groups, b), (trained, b), gy)
    y = grouped_linear(x, w, groups, b)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got, = torch.autograd.grad(y, b, gy)
    assert torch.equal(got, want) and torch.equal(got, sums.to(dtype))
    # the gradient and at most 2 m / 256 partial rows, fp32; the allocator counts in pieces of 512 bytes
    assert torch.cuda.max_memory_allocated() - before <= 8 * n * 4 + 2 * m // 256 * n * 4 + 4096
