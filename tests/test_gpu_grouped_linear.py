"""grouped_linear() and its gradients on the device against 64-bit products."""
import pytest
import torch

from ponderv2_amd.distillation import topk_distillation
from ponderv2_amd.embedding import embedding
from ponderv2_amd.grouped_linear import grouped_linear
from ponderv2_amd.row_groups import RowGroups, group_rows
from row_ops_oracle import (DTYPES, EPS32, assert_within, distill, grouped_linear as exact, half_step, least,
                            product_bound)

pytestmark = pytest.mark.gpu


def ids_of(m, g, device, outside=0.1):
    index = torch.randint(0, g, (m,), device=device)
    return torch.where(torch.rand(m, device=device) < outside, torch.full_like(index, -1), index)


def check(x, w, index, bias=None, gy=None, groups=None):
    """y and, with gy, the gradients of x, w and bias against the oracle."""
    groups = group_rows(index, w.shape[0]) if groups is None else groups
    train = gy is not None
    leaves = [t.detach().requires_grad_(train) for t in (x, w) + (() if bias is None else (bias,))]
    y = grouped_linear(leaves[0], leaves[1], groups, None if bias is None else leaves[2])
    want, size = exact(x, w, index, bias, gy)
    k, n, dt = x.shape[1], w.shape[1], x.dtype
    longest = int(torch.bincount(index[index >= 0].long(), minlength=1).max()) if index.numel() else 0
    assert y.dtype == dt
    assert_within(y.detach(), want["y"], product_bound(want["y"], size["y"], k + 1, dt), "y")
    assert torch.equal(y.detach()[(index < 0) | (index >= w.shape[0])].float(),
                       torch.zeros(int(((index < 0) | (index >= w.shape[0])).sum()), n, device=x.device))
    got = [y.detach()]
    if train:
        grads = torch.autograd.grad(y, leaves, gy)
        got += list(grads)
        for name, t, terms in zip(("d_x", "d_w", "d_b"), grads, (n, longest, longest)):
            assert t.dtype == dt and t.shape == want[name].shape
            assert_within(t, want[name], product_bound(want[name], size[name], terms, dt), name)
    return got


def problem(m, g, k, n, dtype, device, bias=True, train=True):
    x = torch.randn(m, k, device=device).to(dtype)
    w = (torch.randn(g, n, k, device=device) * k ** -0.5).to(dtype)
    b = torch.randn(g, n, device=device).to(dtype) if bias else None
    return x, w, b, torch.randn(m, n, device=device).to(dtype) if train else None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,g,k,n", [
    (1, 1, 1, 1), (1, 5, 16, 24), (7, 3, 33, 5), (17, 4, 64, 64), (128, 1, 64, 128), (129, 1, 65, 127),
    (300, 3, 96, 512), (515, 7, 203, 131), (1000, 40, 40, 8), (2000, 2, 8, 300), (700, 200, 24, 36), (4000, 3, 130, 260)])
def test_sizes(dtype, m, g, k, n, device):
    torch.manual_seed(m + k)
    x, w, b, gy = problem(m, g, k, n, dtype, device)
    index = ids_of(m, g, device)
    check(x, w, index, b, gy)
    check(x, w, index, None, gy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[0, 0, 0], [128, 0, 128], [1, 1, 1], [0, 5000, 0], [127, 129, 256], [3000, 1, 2]])
def test_uneven_groups(dtype, sizes, device):
    """Empty groups (zero weight gradients), whole tiles, one group of all rows (split over many workgroups)."""
    torch.manual_seed(1)
    m = sum(sizes) + 5                               # five rows of no group
    index = torch.cat([torch.full((s,), e) for e, s in enumerate(sizes)] + [torch.full((5,), 3)])
    index = index[torch.randperm(m)].to(device)
    x, w, b, gy = problem(m, 3, 72, 90, dtype, device)
    got = check(x, w, index, b, gy)
    for e, s in enumerate(sizes):
        if s == 0:
            assert int(got[2][e].count_nonzero()) == 0 and int(got[3][e].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,g", [(1, 1), (1, 64), (5, 3), (16, 2), (17, 2), (40, 16), (256, 64), (260, 64)])
@pytest.mark.parametrize("k,n", [(64, 64), (1000, 17), (130, 600)])
def test_serving_rows(dtype, m, g, k, n, device):
    """A handful of rows, on both sides of where the rows' own kernel is taken."""
    torch.manual_seed(m)
    x, w, b, _ = problem(m, g, k, n, dtype, device, train=False)
    check(x, w, ids_of(m, g, device), b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_in_order(dtype, device):
    """Groups by cumulative offset (the points of a batch), rows behind the last one in no group."""
    torch.manual_seed(2)
    offset = torch.tensor([100, 100, 471], device=device)
    x, w, b, gy = problem(500, 3, 48, 56, dtype, device)
    index = torch.cat([torch.full((c,), e) for e, c in enumerate([100, 0, 371, 29])]).to(device)
    check(x, w, index, b, gy, groups=RowGroups.from_offset(offset, 500))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype, device):
    """Row and group strides, bases at odd elements, transposed and expanded operands."""
    torch.manual_seed(3)
    m, g, k, n = 400, 3, 64, 72
    x, w, b, gy = problem(m, g, k, n, dtype, device)
    index = ids_of(m, g, device)
    wide = torch.randn(m, 200, device=device).to(dtype)
    stack = (torch.randn(g, n + 4, k + 9, device=device) * 0.1).to(dtype)
    check(wide[:, 3:3 + k], stack[:, 1:1 + n, 5:5 + k], index, b, torch.randn(m, 90, device=device).to(dtype)[:, 7:7 + n])
    check(wide[:, 8:8 + k], stack[:, :n, :k], index, b, gy)
    check(torch.randn(k, m, device=device).to(dtype).t(), w.transpose(1, 2).contiguous().transpose(1, 2), index, b,
          torch.randn(n, m, device=device).to(dtype).t())
    check(x[:1].expand(m, k), w[:1].expand(g, n, k), index, b, gy[:1].expand(m, n))
    check(x, w, index, torch.randn(n, g, device=device).to(dtype).t(), torch.ones((), device=device, dtype=dtype).expand(m, n))


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_in_no_group_or_another_group_does_not_leak(dtype, device):
    torch.manual_seed(4)
    m, g, k, n = 300, 4, 40, 24
    x, w, b, gy = problem(m, g, k, n, dtype, device)
    index = ids_of(m, g, device, outside=0.2)
    clean = check(x, w, index, b, gy)
    x2, gy2, w2 = x.clone(), gy.clone(), w.clone()
    x2[index < 0], gy2[index < 0] = float("nan"), float("inf")
    groups = group_rows(index, g)
    leaves = [t.detach().requires_grad_() for t in (x2, w2, b)]
    y = grouped_linear(leaves[0], leaves[1], groups, leaves[2])
    got = [y.detach(), *torch.autograd.grad(y, leaves, gy2)]
    for a, c in zip(got, clean):
        assert torch.equal(a, c)
    x2 = x.clone()
    x2[index == 1] = float("nan")                    # a group's rows: its own results and weight gradient only
    leaves = [t.detach().requires_grad_() for t in (x2, w)]
    y = grouped_linear(leaves[0], leaves[1], groups)
    gx, gw = torch.autograd.grad(y, leaves, gy)
    rest = index != 1
    assert torch.isnan(y[index == 1]).all() and torch.isfinite(y[rest]).all() and torch.isfinite(gx).all()
    assert torch.isnan(gw[1]).all() and torch.isfinite(gw[[0, 2, 3]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_every_time(dtype, device):
    torch.manual_seed(5)
    x, w, b, gy = problem(9000, 2, 96, 64, dtype, device)
    index = ids_of(9000, 2, device)
    first = check(x, w, index, b, gy)
    for a, c in zip(check(x, w, index, b, gy), first):
        assert torch.equal(a, c)


def test_differences(device):
    """On whole numbers every product and sum is exact in fp32: <gy, f(. + d) - f(.)> = <grad, d> to the last bit."""
    torch.manual_seed(6)
    m, g, k, n = 700, 3, 24, 40
    whole = lambda *shape: torch.randint(-3, 4, shape, device=device).float()
    x, w, b, gy = whole(m, k), whole(g, n, k), whole(g, n), whole(m, n)
    groups = group_rows(ids_of(m, g, device), g)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(grouped_linear(leaves[0], leaves[1], groups, leaves[2]), leaves, gy)
    base = grouped_linear(x, w, groups, b).double()
    for i, grad in enumerate(grads):
        args = [x, w, b]
        step = whole(*args[i].shape)
        args[i] = args[i] + step
        diff = grouped_linear(args[0], args[1], groups, args[2]).double() - base
        assert float((diff * gy.double()).sum()) == float((grad.double() * step.double()).sum())


def test_gradients_that_are_not_needed(device):
    torch.manual_seed(7)
    x, w, b, gy = problem(300, 3, 32, 16, torch.float32, device)
    groups = group_rows(ids_of(300, 3, device), 3)
    full = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(grouped_linear(full[0], full[1], groups, full[2]), full, gy)
    for i in range(3):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(grouped_linear(args[0], args[1], groups, args[2]), args[i], gy)
        assert torch.equal(got, want[i])


def test_many_groups(device):
    """As many groups as there may be, most of them empty; serving and training."""
    torch.manual_seed(12)
    for m in (300, 20000):
        x, w, b, gy = problem(m, 4096, 24, 16, torch.bfloat16, device)
        check(x, w, ids_of(m, 4096, device), b, gy)


def test_a_second_backward_pass_is_refused(device):
    x = torch.randn(40, 8, device=device, requires_grad=True)
    w = torch.randn(2, 4, 8, device=device, requires_grad=True)
    table = torch.randn(5, 8, device=device, requires_grad=True)
    groups = group_rows(ids_of(40, 2, device), 2)
    logits = torch.randn(6, 9, device=device, requires_grad=True)
    index = torch.randint(0, 9, (6, 2), device=device)
    for out, leaf in ((grouped_linear(x, w, groups).square().sum(), w),
                      (embedding(torch.tensor([1, 4, 1], device=device), table).square().sum(), table),
                      (topk_distillation(logits, index, torch.randn(6, 2, device=device)), logits)):
        first, = torch.autograd.grad(out, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            first.square().sum().backward()


def test_without_a_gradient_the_results_are_the_same(device):
    torch.manual_seed(13)
    x, w, b, _ = problem(500, 3, 40, 24, torch.float16, device)
    groups = group_rows(ids_of(500, 3, device), 3)
    leaf = w.clone().requires_grad_()
    want = grouped_linear(x, leaf, groups, b)
    with torch.no_grad():
        assert torch.equal(grouped_linear(x, leaf, groups, b), want)
    got = grouped_linear(x, w, groups, b)
    assert torch.equal(got, want) and not got.requires_grad and want.requires_grad


def test_no_rows(device):
    x = torch.zeros((0, 8), device=device, requires_grad=True)
    w = torch.randn(3, 4, 8, device=device, requires_grad=True)
    b = torch.randn(3, 4, device=device, requires_grad=True)
    y = grouped_linear(x, w, group_rows(torch.zeros(0, dtype=torch.int64, device=device), 3), b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
    assert y.shape == (0, 4) and gx.shape == (0, 8) and not gw.any() and not gb.any()


def test_offsets_past_32_bits(device):
    """Rows and weights whose element offsets pass 2^31."""
    m, k = 2100000, 1032
    x = torch.zeros((m, k), dtype=torch.bfloat16, device=device)
    index = torch.full((m,), -1, device=device)
    rows = torch.tensor([0, 5, m - 2, m - 1], device=device)
    torch.manual_seed(8)
    x[rows] = torch.randn(4, k, device=device).bfloat16()
    index[rows] = torch.tensor([0, 1, 1, 0], device=device)
    w = (torch.randn(2, 24, k, device=device) * 0.03).bfloat16()
    gy = torch.zeros((m, 24), dtype=torch.bfloat16, device=device)
    gy[rows] = torch.randn(4, 24, device=device).bfloat16()
    groups = group_rows(index, 2)
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    y = grouped_linear(leaves[0], leaves[1], groups)
    gx, gw = torch.autograd.grad(y, leaves, gy)
    want, size = exact(x[rows], w, index[rows], None, gy[rows])
    for name, t, terms in (("y", y.detach()[rows], k), ("d_x", gx[rows], 24), ("d_w", gw, 4)):
        assert_within(t, want[name], product_bound(want[name], size[name], terms, torch.bfloat16), name)
    assert int(y.count_nonzero()) == int(y[rows].count_nonzero())


def test_few_rows_of_a_very_wide_layer(device):
    """More blocks of 16 columns than a grid takes: the larger tiles' work, as for more rows."""
    torch.manual_seed(17)
    m, g, k, n = 256, 56, 8, 3400008
    x = torch.randn(m, k, device=device).bfloat16()
    w = torch.randn(1, n, k, device=device).bfloat16()
    index = ids_of(m, g, device)
    y = grouped_linear(x, w.expand(g, n, k), group_rows(index, g))
    cols = torch.cat((torch.arange(300, device=device), torch.randint(0, n, (300,), device=device),
                      torch.arange(n - 300, n, device=device)))
    want, size = exact(x, w[:, cols], torch.where(index >= 0, torch.zeros_like(index), index), None, None)
    assert_within(y[:, cols], want["y"], product_bound(want["y"], size["y"], k + 1, x.dtype), "y")


def test_in_a_graph_with_eager_work_between(device):
    torch.manual_seed(9)
    x, w, b, gy = problem(3000, 5, 64, 48, torch.bfloat16, device)
    index = ids_of(3000, 5, device)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = grouped_linear(leaves[0], leaves[1], group_rows(index, 5), leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for seed in range(3):
        torch.manual_seed(seed)
        x.normal_()
        index.copy_(ids_of(3000, 5, device))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, got in graphs:
            for a, c in zip(got, want):
                assert torch.equal(a, c)


def test_two_streams_at_once(device):
    torch.manual_seed(10)
    jobs = []
    for m in (2000, 2500):
        x, w, b, gy = problem(m, 3, 64, 80, torch.float32, device)
        jobs.append((x, w, b, gy, ids_of(m, 3, device), torch.cuda.Stream()))

    def step(x, w, b, gy, index):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = grouped_linear(leaves[0], leaves[1], group_rows(index, 3), leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    want = [step(*j[:5]) for j in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for j in jobs:
            with torch.cuda.stream(j[5]):
                got.append(step(*j[:5]))
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, c))


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_operators_together(dtype, device):
    """Class ids -> embedding rows -> products with the weights of each row's dataset -> logits -> loss against a
    teacher's top logits, backward to the table and the weights, against the same chain with every stage's 64-bit oracle
    applied to the stage's own input (so each stage's bound is its own)."""
    torch.manual_seed(11)
    m, classes, width, sets, k = 900, 50, 64, 3, 4
    label = torch.randint(-1, classes, (m,), device=device)
    dataset = ids_of(m, sets, device)
    table = torch.randn(classes, width, device=device).to(dtype).requires_grad_()
    weight = (torch.randn(sets, classes, width, device=device) * width ** -0.5).to(dtype).requires_grad_()
    bias = torch.randn(sets, classes, device=device).to(dtype).requires_grad_()
    top = torch.randint(0, classes, (m, k), device=device)
    teacher = torch.randn(m, k, device=device)
    x = embedding(label, table, 2.0)
    x.retain_grad()
    logits = grouped_linear(x, weight, group_rows(dataset, sets), bias)
    logits.retain_grad()
    loss = topk_distillation(logits, top, teacher, temperature=2.0)
    loss.backward()
    want_loss, want_grad, counts, *_ = distill(logits.detach(), top, teacher, 2.0)
    assert_within(loss.detach(), want_loss.sum() / counts.sum(), 4 * 64 * 8 * EPS32, "loss")
    assert_within(logits.grad, want_grad / counts.sum(),
                  (want_grad.abs() * half_step(dtype) + 2 * 256 * EPS32) / counts.sum() + least(dtype), "d_logits")
    want, size = exact(x.detach(), weight.detach(), dataset, bias.detach(), logits.grad)
    longest = int(torch.bincount(dataset.clamp(min=0)).max())
    for name, got, terms in (("d_x", x.grad, classes), ("d_w", weight.grad, longest), ("d_b", bias.grad, longest)):
        assert_within(got, want[name], product_bound(want[name], size[name], terms, dtype), name)
    at = torch.where(label >= 0, label, torch.full_like(label, classes))
    sums = torch.zeros(classes + 1, width, dtype=torch.float64, device=device).index_add_(0, at, x.grad.double())
    sizes = torch.zeros_like(sums).index_add_(0, at, x.grad.double().abs())
    assert_within(table.grad, 2 * sums[:classes],
                  2 * sizes[:classes] * (m + 16) * EPS32 + 2 * sums[:classes].abs() * half_step(dtype) + least(dtype), "d_table")
