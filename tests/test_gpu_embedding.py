"""embedding() and its gradient on the device against 64-bit sums."""
import numpy as np
import pytest
import torch

from ponderv2_amd.embedding import embedding
from row_ops_oracle import DTYPES, EPS32, assert_within, half_step, least

pytestmark = pytest.mark.gpu


def check(index, weight, scale, gy=None):
    """Forward against scale * W[index] (one product and one rounding); the gradient against the 64-bit sum: a class of n
    tokens takes at most n + 16 fp32 roundings of its sum of absolute terms, then one of the product, one to the type."""
    w = weight.detach().clone().requires_grad_()
    y = embedding(index, w, scale)
    assert y.dtype == weight.dtype and y.shape == (*index.shape, weight.shape[1])
    flat = index.reshape(-1).long()
    rows, c = weight.shape
    ok = (flat >= 0) & (flat < rows)
    table = torch.cat([weight.double(), weight.new_zeros(1, c).double()])
    at = torch.where(ok, flat, torch.full_like(flat, rows))
    scale32 = float(np.float32(scale))
    want = (table[at] * scale32).reshape(y.shape)
    dt = weight.dtype
    assert_within(y.detach(), want, want.abs() * (half_step(dt) + EPS32) * 1.01 + least(dt), "y")
    if gy is None:
        gy = torch.randn(y.shape, device=y.device).to(dt)
    gw, = torch.autograd.grad(y, w, gy)
    assert gw.dtype == dt and gw.shape == weight.shape
    g = gy.reshape(-1, c).double()
    sums = table.new_zeros(rows + 1, c).index_add_(0, at, g)[:rows] * scale32
    sizes = table.new_zeros(rows + 1, c).index_add_(0, at, g.abs())[:rows] * abs(scale32)
    n = torch.bincount(at, minlength=rows + 1)[:rows, None].double()
    assert_within(gw, sums, sizes * (n + 16) * EPS32 + sums.abs() * half_step(dt) + least(dt), "d_weight")
    return y, gw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 257, 5000])
@pytest.mark.parametrize("rows,c", [(1, 8), (5, 1), (36, 512), (300, 203), (9001, 24), (37, 1030)])
def test_sizes(dtype, n, rows, c, device):
    torch.manual_seed(n + rows)
    check(torch.randint(-1, rows + 1, (n,), device=device), torch.randn(rows, c, device=device).to(dtype), 1.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["one", "none", "runs", "blocks", "heavy"])
def test_uneven_classes(dtype, kind, device):
    """A class of all tokens, no class at all, classes of exactly a piece (32 tokens) or a block of them (1024), of
    multiples and around them, one heavy class."""
    torch.manual_seed(3)
    n = 40007
    index = {"one": torch.full((n,), 4), "none": torch.full((n,), -1),
             "runs": torch.repeat_interleave(torch.arange(9), torch.tensor([128, 128, 127, 1, 129, 256, 257, 1, 300])),
             "blocks": torch.repeat_interleave(torch.arange(12), torch.tensor(
                 [32, 31, 1, 33, 31, 64, 832, 1024, 1025, 1023, 1, 3000]))[torch.randperm(7097)],
             "heavy": torch.where(torch.rand(n) < 0.7, torch.tensor(2), torch.randint(0, 5000, (n,)))}[kind]
    check(index.to(device), torch.randn(5000, 40, device=device).to(dtype), -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_types_shapes_and_strides(dtype, device):
    torch.manual_seed(4)
    index = torch.randint(0, 50, (6, 7, 11), device=device)
    base = torch.randn(50, 64, device=device).to(dtype)
    check(index.int(), base, 8.0)
    check(index.transpose(0, 2), base, 1.0)
    check(index[1:, ::2], base[:, 5:40], 1.0)           # rows 64 apart, 10 bytes off
    check(index[0], base[::3].contiguous()[:20, ::2].clone().t().contiguous().t(), 1.0)   # columns apart
    y = embedding(torch.tensor(7, device=device), base)  # a single id: shape (C,)
    assert y.shape == (64,) and torch.equal(y, base[7])
    # gradients that are expanded, transposed and strided views
    n = index.numel()
    flat = index.reshape(-1)
    check(flat, base, 2.0, gy=torch.randn(64, device=device).to(dtype).expand(n, 64))
    check(flat, base, 2.0, gy=torch.randn(64, n, device=device).to(dtype).t())
    check(flat, base, 2.0, gy=torch.randn(n, 100, device=device).to(dtype)[:, 3:67])
    check(flat, base, 2.0, gy=torch.ones((), device=device, dtype=dtype).expand(n, 64))


def test_no_tokens(device):
    w = torch.randn(5, 8, device=device, requires_grad=True)
    y = embedding(torch.zeros((0, 3), dtype=torch.int64, device=device), w)
    gw, = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert y.shape == (0, 3, 8) and torch.equal(gw, torch.zeros_like(w))


def test_not_a_number_and_infinities_stay_in_their_rows(device):
    """A row of the table or of the gradient that holds NaN or an infinity changes its own class only."""
    w = torch.randn(6, 32, device=device)
    w[2, 5], w[3, 0] = float("nan"), float("inf")
    index = torch.tensor([0, 2, 3, -1, 5, 2], device=device)
    y = embedding(index, w, 2.0)
    assert torch.isnan(y[1, 5]) and torch.isinf(y[2, 0]) and torch.isfinite(y[[0, 3, 4]]).all()
    assert torch.equal(y[3], torch.zeros_like(y[3]))
    wr = torch.randn(6, 32, device=device, requires_grad=True)
    gy = torch.randn(6, 32, device=device)
    gy[3] = float("nan")                         # the row without a class
    gy[4, 1] = float("inf")
    gw, = torch.autograd.grad(embedding(index, wr), wr, gy)
    assert torch.isinf(gw[5, 1]) and torch.isfinite(gw[:5]).all()


def test_same_bits_every_time_and_differences(device):
    torch.manual_seed(6)
    index = torch.randint(0, 9, (3000,), device=device)
    w = torch.randn(9, 16, device=device)
    gy = torch.randn(3000, 16, device=device)
    first = check(index, w, 3.0, gy)[1]
    for _ in range(3):
        assert torch.equal(check(index, w, 3.0, gy)[1], first)
    # the map is linear in the weight: <gy, f(w + d) - f(w)> = <gw, d>, in 64 bits on small whole numbers (exact in fp32)
    whole = torch.randint(-8, 9, (9, 16), device=device).float()
    step = torch.randint(-8, 9, (9, 16), device=device).float()
    g = torch.randint(-4, 5, (3000, 16), device=device).float()
    leaf = whole.clone().requires_grad_()
    gw, = torch.autograd.grad(embedding(index, leaf, 2.0), leaf, g)
    diff = (embedding(index, whole + step, 2.0) - embedding(index, whole, 2.0)).double()
    assert float((diff * g.double()).sum()) == float((gw.double() * step.double()).sum())


def test_offsets_past_32_bits(device):
    """A table of 2^31 elements and more, with rows of both ends."""
    rows, c = 1050000, 2048
    w = torch.zeros((rows, c), dtype=torch.bfloat16, device=device)
    w[-1], w[0] = 3.0, 5.0
    y = embedding(torch.tensor([rows - 1, 0, rows], device=device), w)
    assert y[0].eq(3).all() and y[1].eq(5).all() and y[2].eq(0).all()
    w.requires_grad_()
    gw, = torch.autograd.grad(embedding(torch.tensor([rows - 1, 0, rows - 1], device=device), w), w,
                              torch.ones((3, c), dtype=torch.bfloat16, device=device))
    assert gw[-1].eq(2).all() and gw[0].eq(1).all() and int(gw[1:-1].count_nonzero()) == 0


def test_in_a_graph(device):
    index = torch.randint(0, 500, (9000,), device=device)
    w = torch.randn(500, 96, device=device)
    gy = torch.randn(9000, 96, device=device)

    def step():
        leaf = w.detach().requires_grad_()
        y = embedding(index, leaf, 2.0)
        return y.detach(), torch.autograd.grad(y, leaf, gy)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gw = step()
    for seed in range(3):
        torch.manual_seed(seed)
        index.copy_(torch.randint(-1, 500, (9000,), device=device))
        w.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want_y, want_gw = step()
        assert torch.equal(y, want_y) and torch.equal(gw, want_gw)
