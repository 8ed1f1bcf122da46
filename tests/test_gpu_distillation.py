"""topk_distillation() and its gradient on the device against 64-bit softmaxes."""
import pytest
import torch

from ponderv2_amd.distillation import topk_distillation
from row_ops_oracle import DTYPES, EPS32, assert_within, distill, half_step, least

pytestmark = pytest.mark.gpu


def bounds(logits, big, q, target, temperature):
    """fp32 errors of a row.  log p and log q: an exponent (x - max) log2(e) / T has a relative error of 3 roundings, a
    sum of V terms of at most V / 64 + 16 (no thread adds more than V / 64 in a row), the logarithm and the exponential
    of 2 each; so |error of log| <= (8 |log| + V / 64 + 32) 2^-24, of q and p: q and p times that."""
    v = logits.shape[1]
    unit = (8 * big.amax(1, keepdim=True) + v / 64 + 32) * EPS32
    loss = temperature ** 2 * unit[:, 0] * (2 + 2 * big.amax(1))
    log_q = torch.log(q.clamp(min=1e-45)).abs()
    grad = temperature * (q * (8 * log_q + v / 64 + 32) * EPS32 + target * unit + 2.0 ** -126)
    return loss, grad


def check(logits, index, teacher, temperature=1.0):
    want_loss, want_grad, counts, big, q, target = distill(logits, index, teacher, temperature)
    finite = torch.isfinite(want_loss)
    b_loss, b_grad = bounds(logits, torch.where(torch.isfinite(big), big, torch.zeros_like(big)), q, target, temperature)
    dt, m = logits.dtype, logits.shape[0]
    rounding = want_grad.abs() * half_step(dt) + least(dt) * 4
    n = max(1, int(counts.sum()))

    leaf = logits.detach().requires_grad_()
    rows = topk_distillation(leaf, index, teacher, temperature, "none")
    assert rows.dtype == torch.float32 and rows.shape == (m,)
    assert_within(rows.detach(), want_loss, b_loss, "row losses")
    up = torch.randn(m, device=logits.device)
    grad, = torch.autograd.grad(rows, leaf, up)
    assert grad.dtype == dt
    scale = up.double()[:, None]
    assert_within(grad, want_grad * scale, (b_grad + rounding) * scale.abs() * 1.01 + least(dt) * 4, "gradient, per row")
    assert int(grad[~counts].count_nonzero()) == 0 and int(rows[~counts].count_nonzero()) == 0

    for reduction, div in (("mean", n), ("sum", 1)):
        leaf = logits.detach().requires_grad_()
        loss = topk_distillation(leaf, index, teacher, temperature, reduction)
        assert loss.dtype == torch.float32 and loss.dim() == 0
        if finite.all():
            total = (b_loss.sum() + (m / 16 + 32) * EPS32 * want_loss.abs().sum()) / div
            assert_within(loss.detach(), want_loss.sum() / div, total, reduction)
        grad, = torch.autograd.grad(loss, leaf, torch.tensor(0.75, device=logits.device))
        s = 0.75 / div
        assert_within(grad, want_grad * s, (b_grad + rounding) * s * 1.01 + least(dt) * 4, "gradient, " + reduction)
    return grad


def problem(m, v, k, dtype, device, lists="full"):
    logits = (torch.randn(m, v, device=device) * 2).to(dtype)
    index = torch.randint(0, v, (m, k), device=device)
    teacher = torch.randn(m, k, device=device) * 3
    if lists == "ragged":
        length = torch.randint(0, k + 1, (m, 1), device=device)
        index = torch.where(torch.arange(k, device=device) < length, index, torch.full_like(index, -1))
    return logits, index, teacher


# up to 512 classes: a row per part of a wave; above: a workgroup per row, several where there are few rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 2, 13, 25, 32, 33, 64, 255, 511, 512, 513, 1000, 4097, 20011])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 5), (70, 8)])
def test_sizes(dtype, v, m, k, device):
    torch.manual_seed(v + m)
    check(*problem(m, v, k, dtype, device, "ragged" if m > 3 else "full"), temperature=2.0)


@pytest.mark.parametrize("v,k", [(20, 1024), (400, 300), (512, 65), (3000, 1024), (9000, 257)])
def test_long_lists(v, k, device):
    """Lists as long as they may be, longer than there are classes: most classes are listed more than once."""
    torch.manual_seed(v)
    check(*problem(9, v, k, torch.float32, device, "ragged"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [25, 6001])
def test_the_same_class_twice(dtype, v, device):
    torch.manual_seed(2)
    logits, index, teacher = problem(40, v, 6, dtype, device)
    index[:, 3] = index[:, 0]
    index[:20, 5] = index[:20, 0]
    check(logits, index, teacher, 3.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [25, 700])
@pytest.mark.parametrize("m", [1025, 70001])
def test_many_rows(dtype, v, m, device):
    torch.manual_seed(3)
    if v * m > 3e7:
        m = 6001
    check(*problem(m, v, 5, dtype, device, "ragged"))


@pytest.mark.parametrize("v", [25, 5000])
def test_masked_rows_do_not_read_their_logits(v, device):
    """A row without a list: loss 0 and gradient 0, also where its logits are NaN or infinite; NaN teacher logits at
    entries that do not count do not matter either."""
    torch.manual_seed(4)
    logits, index, teacher = problem(30, v, 4, torch.float32, device)
    want = check(logits, index, teacher)
    index[5], index[6] = -1, v
    teacher[7] = -torch.inf                             # listed, but at -inf: does not count
    clean = check(logits, index, teacher)
    for bad in (torch.nan, torch.inf, -torch.inf):
        dirty, t = logits.clone(), teacher.clone()
        dirty[5:8], t[5:7] = bad, torch.nan
        leaf = dirty.requires_grad_()
        loss = topk_distillation(leaf, index, t, reduction="sum")
        grad, = torch.autograd.grad(loss, leaf, torch.tensor(0.75, device=device))
        assert torch.equal(grad, clean) and not grad[5:8].any()
    assert not torch.equal(want, clean)
    index[:] = -1                                       # no row counts
    leaf = logits.detach().requires_grad_()
    for reduction in ("mean", "sum"):
        loss = topk_distillation(leaf, index, teacher, reduction=reduction)
        grad, = torch.autograd.grad(loss, leaf)
        assert float(loss) == 0.0 and not grad.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [25, 5000])
def test_extreme_values(dtype, v, device):
    """Student classes at -inf and at the type's lowest value, teacher logits at the lowest value, large logits, a teacher
    that puts weight on a class that the student excludes (loss +inf, finite gradient)."""
    torch.manual_seed(5)
    logits, index, teacher = problem(24, v, 4, dtype, device)
    index = torch.stack([torch.randperm(v, device=device)[:4] for _ in range(24)])
    low = torch.finfo(dtype).min
    rest = torch.ones(24, v, dtype=torch.bool, device=device).scatter_(1, index, False)
    mask = rest & (torch.rand(24, v, device=device) < 0.5)
    check(torch.where(mask, torch.full_like(logits, -torch.inf), logits), index, teacher, 2.0)
    check(torch.where(mask, torch.full_like(logits, low), logits), index, teacher, 2.0)
    check(logits + 1000, index, teacher)
    check(logits - 3000, index, teacher, 0.5)
    t = teacher.clone()
    t[:, 2] = torch.finfo(torch.float32).min            # probability 0, also where the student is at -inf
    s = logits.clone()
    s[torch.arange(24), index[:, 2]] = -torch.inf
    check(s, index, t)
    t[:] = torch.finfo(torch.float32).min               # all alike: an even teacher
    check(logits, index, t)
    s = logits.clone()
    s[3, index[3, 0]] = -torch.inf
    check(s, index, teacher)
    assert float(topk_distillation(s, index, teacher, reduction="none")[3]) == float("inf")
    s = logits.clone()
    s[4, 7] = torch.nan                                 # NaN in a row that counts: that row is NaN
    rows = topk_distillation(s, index, teacher, reduction="none")
    assert torch.isnan(rows[4]) and torch.isfinite(rows[[0, 1, 2, 3, 5]]).all()


# (x - max) / T where the maximum itself, over T, is far past 2^24: a few classes share the maximum, the others lie some of
# the type's steps below it.  Temperatures are powers of two, so that the 64-bit side divides exactly.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v,m", [(25, 70), (513, 9), (4097, 600), (20011, 1)])
@pytest.mark.parametrize("base,temperature", [(1e9, 1.0), (1e9, 8192.0), (3e12, 1.0), (-1e20, 2.0), (1e25, 2.0 ** -13),
                                              (4e4, 2.0 ** -13), (-1e10, 64.0)])
def test_large_logits(dtype, v, m, base, temperature, device):
    torch.manual_seed(v)
    step = 2.0 ** (-22 if dtype == torch.float32 else -6)
    near = lambda *shape: base * (1 + torch.randint(-3, 4, shape, device=device) * step)
    check(near(m, v).to(dtype), torch.randint(0, v, (m, 5), device=device), near(m, 5).to(dtype), temperature)


# maxima on both sides of 2^24 ln 2 in one row, in every order: sums relative to one become relative to the other
@pytest.mark.parametrize("v,m", [(25, 70), (512, 70), (513, 70), (4097, 9), (20011, 1), (20011, 600)])
@pytest.mark.parametrize("order", ["random", "up", "down"])
@pytest.mark.parametrize("sign", [1, -1])
def test_logits_about_where_products_are_rounded(v, m, order, sign, device):
    torch.manual_seed(v)
    logits = sign * (11629079 + torch.randint(-6, 7, (m, v), device=device)).float()
    if order != "random":
        logits = logits.sort(1, descending=order == "down").values
    teacher = sign * (11629079 + torch.randint(-6, 7, (m, 5), device=device)).float()
    check(logits, torch.randint(0, v, (m, 5), device=device), teacher)


@pytest.mark.parametrize("v,m", [(25, 70), (4097, 9)])
@pytest.mark.parametrize("temperature", [1e-4, 1e4])
def test_ends_of_the_temperatures(v, m, temperature, device):
    torch.manual_seed(v)
    check(*problem(m, v, 5, torch.float32, device, "ragged"), temperature=temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [25, 1003])
def test_shapes_strides_and_types(dtype, v, device):
    torch.manual_seed(6)
    logits, index, teacher = problem(60, v + 30, 6, dtype, device)
    for first in (0, 3, 8):
        view = logits[:, first:first + v]
        at = index % v
        check(view, at.int(), teacher.to(dtype))
        check(view, at, teacher.bfloat16())
        check(view[::2], at[::2, 1:4], teacher[::2, 1:4])
    check(logits.t().contiguous().t()[:, :v], index % v, teacher)
    base = logits[:, :v].contiguous()
    flat = topk_distillation(base, index % v, teacher, reduction="none")
    deep = topk_distillation(base.view(5, 3, 4, v), (index % v).view(5, 3, 4, 6), teacher.view(5, 3, 4, 6), reduction="none")
    assert deep.shape == (5, 3, 4) and torch.equal(deep.reshape(-1), flat)
    one = topk_distillation(base[0], index[0] % v, teacher[0], reduction="none")
    assert one.shape == () and torch.equal(one, flat[0])


def test_no_rows(device):
    leaf = torch.zeros((0, 9), device=device, requires_grad=True)
    index, teacher = torch.zeros((0, 2), dtype=torch.int64, device=device), torch.zeros((0, 2), device=device)
    for reduction in ("mean", "sum"):
        loss = topk_distillation(leaf, index, teacher, reduction=reduction)
        assert float(loss) == 0.0
        loss.backward()
    assert topk_distillation(leaf, index, teacher, reduction="none").shape == (0,)


@pytest.mark.parametrize("v", [20, 2000])
def test_differences(v, device):
    """The gradient against central differences of the 64-bit oracle along random directions."""
    torch.manual_seed(7)
    logits, index, teacher = problem(50, v, 5, torch.float32, device, "ragged")
    leaf = logits.clone().requires_grad_()
    grad, = torch.autograd.grad(topk_distillation(leaf, index, teacher, 2.0, "sum"), leaf)
    for _ in range(3):
        d = torch.randn(50, v, dtype=torch.float64, device=device)
        h = 1e-4
        up = distill(logits.double() + h * d, index, teacher, 2.0)[0].sum()
        down = distill(logits.double() - h * d, index, teacher, 2.0)[0].sum()
        along = float((grad.double() * d).sum())
        # third derivatives of log-sum-exp are bounded by |d|^3 <= 5^3 per row and step: h^2 * 50 * 125 / 6
        assert abs(float((up - down) / (2 * h)) - along) < 2e-5 + 1e-5 * float(grad.double().norm() * d.norm())


def test_same_bits_every_time(device):
    torch.manual_seed(8)
    for v, m in ((25, 9000), (3001, 40), (30011, 2)):
        logits, index, teacher = problem(m, v, 5, torch.bfloat16, device)
        runs = []
        for _ in range(3):
            leaf = logits.detach().requires_grad_()
            loss = topk_distillation(leaf, index, teacher)
            runs.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
        assert all(torch.equal(a, runs[0][0]) and torch.equal(b, runs[0][1]) for a, b in runs)


def test_offsets_past_32_bits(device):
    m, v = 34000, 65537
    logits = torch.zeros((m, v), dtype=torch.bfloat16, device=device)
    index = torch.full((m, 2), -1, device=device)
    rows = torch.tensor([0, m // 2, m - 1], device=device)
    torch.manual_seed(9)
    logits[rows] = torch.randn(3, v, device=device).bfloat16()
    index[rows] = torch.randint(0, v, (3, 2), device=device)
    teacher = torch.zeros((m, 2), device=device)
    leaf = logits.requires_grad_()
    loss = topk_distillation(leaf, index, teacher)
    grad, = torch.autograd.grad(loss, leaf)
    sub = logits.detach()[rows].requires_grad_()
    few = topk_distillation(sub, index[rows], teacher[rows])
    want, = torch.autograd.grad(few, sub)
    # the same rows by another number of workgroups: only the order of the sums differs
    assert abs(float(loss) - float(few)) <= (v / 64 + 64) * 8 * EPS32 * abs(float(few))
    assert_within(grad[rows], want, want.abs().double() * 2 ** -7 + 2.0 ** -120, "rows")
    assert not grad[1].any() and not grad[m - 2].any()


def test_in_a_graph(device):
    for v, m in ((25, 4000), (3000, 50)):
        torch.manual_seed(10)
        logits, index, teacher = problem(m, v, 5, torch.float32, device, "ragged")

        def step():
            leaf = logits.detach().requires_grad_()
            loss = topk_distillation(leaf, index, teacher, 2.0)
            return loss.detach(), torch.autograd.grad(loss, leaf)[0]

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for seed in range(3):
            torch.manual_seed(seed)
            logits.normal_()
            index.copy_(torch.randint(-1, v, index.shape, device=device))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                assert torch.equal(a, b)
