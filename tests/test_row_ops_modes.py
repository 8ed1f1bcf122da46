"""The operators on rows by id under forward-mode differentiation and tracing: a tangent is refused by name, and a replayed
trace computes, checks and lays out what its own call brings.  On the host the launches are replaced by numpy statements of
them (over the same addresses), on the device the kernels run."""
import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from ponderv2_amd import (_lib, distillation as distillation_module, embedding as embedding_module,
                          grouped_linear as grouped_linear_module, row_groups)
from ponderv2_amd.distillation import topk_distillation
from ponderv2_amd.embedding import embedding
from ponderv2_amd.grouped_linear import grouped_linear
from ponderv2_amd.row_groups import RowGroups, group_rows
from row_ops_oracle import EPS32, distill, group_order


def at(address, n, of):
    return np.ctypeslib.as_array(ctypes.cast(address, ctypes.POINTER(of)), (n,))


def ids_at(address, is64, n):
    return at(address, n, ctypes.c_int64 if is64 else ctypes.c_int32)


def matrix_at(address, rows, cols, stride):
    return np.lib.stride_tricks.as_strided(at(address, (rows - 1) * stride + cols, ctypes.c_float), (rows, cols),
                                           (4 * stride, 4))


def statement(name, device, *args):
    """The entry point ``name`` on host memory, fp32."""
    for of, a in zip(_lib.SIGNATURES[name][1], args):
        of.from_param(a)   # what the entry point itself takes
    args = [int(a) if isinstance(a, torch.Tensor) else a for a in args]   # (sizes while a trace is recorded)
    if name == "pv2_embedding_forward":
        index, is64, n, w, _, rows, c, ldw, scale, y = args
        index = ids_at(index, is64, n)
        inside = ((index >= 0) & (index < rows))[:, None]
        at(y, n * c, ctypes.c_float).reshape(n, c)[:] = np.where(
            inside, matrix_at(w, rows, c, ldw)[index.clip(0, rows - 1)] * np.float32(scale), 0)
    elif name == "pv2_grouped_linear_forward":
        x, _, m, k, ldx, w, w_group, ldw, g, n, bias, order, offsets, y = args
        x, y = matrix_at(x, m, k, ldx), at(y, m * n, ctypes.c_float).reshape(m, n)
        order = np.arange(m) if order is None else at(order, m, ctypes.c_int32)
        offsets = at(offsets, g + 1, ctypes.c_int32)
        y[:] = 0
        for e in range(g):
            rows = order[offsets[e]:offsets[e + 1]]
            y[rows] = x[rows] @ matrix_at(w + 4 * e * w_group, n, k, ldw).T
            if bias is not None:
                y[rows] += at(bias, g * n, ctypes.c_float).reshape(g, n)[e]
    elif name == "pv2_row_groups":
        index, is64, n, count, order, offsets, _, _ = args
        at(order, n, ctypes.c_int32)[:], at(offsets, count + 1, ctypes.c_int32)[:] = group_order(
            ids_at(index, is64, n), count)
    elif name == "pv2_row_offsets":
        cumulative, is64, count, n, offsets = args
        at(offsets, count + 1, ctypes.c_int32)[:] = np.concatenate(
            [[0], np.maximum.accumulate(ids_at(cumulative, is64, count).clip(0, n))])
    elif name == "pv2_topk_distill_forward":
        x, _, m, v, ldx, index, is64, ldi, t, _, ldt, k, temperature, mean, _, _, row_loss, loss, count = args
        ids = np.lib.stride_tricks.as_strided(ids_at(index, is64, (m - 1) * ldi + k), (m, k),
                                              (ldi * (8 if is64 else 4), 8 if is64 else 4))
        rows, _, counts, *_ = distill(*(torch.from_numpy(a.copy()) for a in (
            matrix_at(x, m, v, ldx), ids, matrix_at(t, m, k, ldt))), temperature)
        at(count, 1, ctypes.c_float)[0] = counts.sum()
        at(loss, 1, ctypes.c_float)[0] = rows.sum() / max(1, counts.sum()) if mean else rows.sum()
        if row_loss is not None:
            at(row_loss, m, ctypes.c_float)[:] = rows
    else:
        raise AssertionError(name)


@pytest.fixture(params=["host", pytest.param("device", marks=pytest.mark.gpu)])
def where(request, monkeypatch):
    if request.param == "device":
        return request.getfixturevalue("device")
    for module in (row_groups, embedding_module, grouped_linear_module, distillation_module):
        monkeypatch.setattr(module, "launch", statement)
        monkeypatch.setattr(module, "_require_device", lambda *tensors: None)
    return torch.device("cpu")


def lookup(index, weight):
    inside = (index >= 0) & (index < weight.shape[0])
    return torch.where(inside[..., None], weight[index.long().clamp(0, weight.shape[0] - 1)], 0.0)


def products(x, weight, index, bias):
    y = x.new_zeros(x.shape[0], weight.shape[1])
    for e in range(weight.shape[0]):
        rows = index == e
        y[rows] = x[rows] @ weight[e].T + bias[e]
    return y


def problem(m, g, k, n, device):
    # (whole numbers: every product and sum is exact)
    whole = lambda *shape: torch.randint(-4, 5, shape, device=device).float()
    return whole(m, k), whole(g, n, k), whole(g, n), torch.randint(-1, g, (m,), device=device)


def trace(fn, *example):
    return torch.jit.trace(fn, example, check_trace=False)


def fill_free_memory(device):
    """What the allocator hands out next holds no earlier results."""
    torch.full((1 << 16,), 77.0, device=device)


# ------------------------------------------------------------------------------------------ tangents
@pytest.mark.parametrize("grad_mode", [True, False])
def test_a_tangent_is_refused(where, grad_mode):
    x, w, b, index = problem(20, 3, 8, 4, where)
    groups = group_rows(index, 3)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: embedding(index, dual(w[0])), lambda: grouped_linear(dual(x), w, groups, b),
                     lambda: grouped_linear(x, dual(w), groups, b), lambda: grouped_linear(x, w, groups, dual(b))):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        # an open level without a tangent changes nothing
        assert torch.equal(embedding(index, w[0]), lookup(index, w[0]))
        assert torch.equal(grouped_linear(x, w, groups, b), products(x, w, index, b))


# ------------------------------------------------------------------------------------------ traces
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_traced_lookup_replays(where):
    _, w, _, index = problem(20, 3, 8, 4, where)
    traced = trace(lambda i, w: embedding(i, w, 2.0), index, w[0])
    for rows, shape in ((4, (20,)), (9, (31,)), (6, (3, 5))):
        index = torch.randint(-1, rows + 1, shape, device=where)
        table = torch.randn(rows, 8, device=where)
        for t in (table, table.t().contiguous().t(), torch.randn(rows, 20, device=where)[:, 3:11]):
            fill_free_memory(where)
            assert torch.equal(traced(index, t), 2 * lookup(index, t))
            assert torch.equal(traced(index.int(), t), 2 * lookup(index, t))
        if len(shape) == 2:
            assert torch.equal(traced(index.t(), table), 2 * lookup(index.t(), table))
    for bad in ((index.float(), table), (index, table[0])):
        with pytest.raises(Exception, match="embedding: "):
            traced(*bad)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_products_replay(where):
    x, w, b, index = problem(20, 3, 8, 4, where)
    groups = group_rows(index, 3)
    traced = trace(lambda x, w, b: grouped_linear(x, w, groups, b), x, w, b)
    for _ in range(3):
        x, w, b, _ = problem(20, 3, 8, 4, where)
        fill_free_memory(where)
        assert torch.equal(traced(x, w, b), products(x, w, index, b))
        strided = w.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(traced(x.t().contiguous().t(), strided, b), products(x, w, index, b))
    # the groups are of 20 rows and 3 weights
    for bad in ((x[:19], w, b), (torch.cat([x, x]), w, b), (x, w[:2], b[:2]), (x, w, b.double())):
        with pytest.raises(Exception, match="grouped_linear: "):
            traced(*bad)
    offset = torch.tensor([4, 4, 17], device=where)
    groups = RowGroups.from_offset(offset, 20)
    traced = trace(lambda x, w: grouped_linear(x, w, groups), x, w)
    index = torch.repeat_interleave(torch.tensor([0, 2, -1]), torch.tensor([4, 13, 3])).to(where)
    assert torch.equal(traced(x, w), products(x, w, index, torch.zeros_like(b)))
    with pytest.raises(Exception, match="groups of 20 rows"):
        traced(torch.cat([x, x]), w)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_groups_replay(where):
    """Ids of every replay are sorted anew, for products as well; what is no list of ids is refused."""
    x, w, b, index = problem(20, 3, 8, 4, where)

    def step(x, w, b, index):
        groups = group_rows(index, 3)
        return grouped_linear(x, w, groups, b), groups.order, groups.offsets

    traced = trace(step, x, w, b, index)
    for m in (20, 33, 1):
        x, w, b, index = problem(m, 3, 8, 4, where)
        fill_free_memory(where)
        y, order, offsets = traced(x, w, b, index)
        want = group_order(index.cpu().numpy(), 3)
        assert np.array_equal(order.cpu().numpy(), want[0]) and np.array_equal(offsets.cpu().numpy(), want[1])
        assert torch.equal(y, products(x, w, index, b))
    with pytest.raises(Exception, match="group_rows: integer ids"):
        traced(x, w, b, index.float())
    with pytest.raises(Exception, match="groups of 2 rows"):
        traced(x, w, b, index.repeat(2))

    def in_order(x, w, offset):
        groups = RowGroups.from_offset(offset, x.shape[0])
        return grouped_linear(x, w, groups), groups.offsets

    x, w, b, _ = problem(20, 3, 8, 4, where)
    traced = trace(in_order, x, w, torch.tensor([4, 4, 17], device=where))
    for counts in ([4, 0, 13, 3], [1, 30, 9, 0], [0, 0, 1, 1]):
        x, w, b, _ = problem(sum(counts), 3, 8, 4, where)
        index = torch.repeat_interleave(torch.tensor([0, 1, 2, -1]), torch.tensor(counts)).to(where)
        fill_free_memory(where)
        y, offsets = traced(x, w, torch.tensor(counts[:3], device=where).cumsum(0))
        assert offsets.tolist() == [0, *np.cumsum(counts[:3])]
        assert torch.equal(y, products(x, w, index, torch.zeros_like(b)))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_traced_distillation_replays(where, reduction):
    def lists(shape, v, k):
        return (torch.randn(*shape, v, device=where), torch.randint(-1, v, (*shape, k), device=where),
                torch.randn(*shape, k, device=where))

    def check(logits, index, teacher):
        fill_free_memory(where)
        rows, _, counts, big, *_ = distill(logits.reshape(-1, logits.shape[-1]), index.reshape(-1, index.shape[-1]),
                                           teacher.reshape(-1, teacher.shape[-1]), 2.0)
        want = rows.reshape(logits.shape[:-1]) if reduction == "none" else rows.sum() / counts.sum().clamp(min=1)
        got = traced(logits, index, teacher)
        assert got.shape == want.shape and got.dtype == torch.float32
        # as tests/test_gpu_distillation.py: T^2 (8 |log| + V / 64 + 32) (2 + 2 |log|) roundings of a row; 64 for the mean's sum
        unit = 4 * (8 * big.max() + logits.shape[-1] / 64 + 32) * (2 + 2 * big.max()) * EPS32
        assert float((got.double() - want).abs().max()) <= float(unit + 64 * EPS32 * rows.abs().max())

    args = lists((20,), 9, 3)
    traced = trace(lambda s, i, t: topk_distillation(s, i, t, 2.0, reduction), *args)
    check(*args)
    for shape, v, k in (((31,), 9, 3), ((1,), 600, 5), ((4, 5), 12, 2)):
        logits, index, teacher = lists(shape, v, k)
        check(logits, index, teacher)
        check(logits, index.int(), teacher)
        check(logits.transpose(0, -1).contiguous().transpose(0, -1), index, teacher)
        check(torch.randn(*shape, v + 7, device=where)[..., 3:3 + v], index, teacher)
    for bad in ((logits, index.float(), teacher), (logits, index[:2], teacher[:2]), (logits.double(), index, teacher),
                (logits, index[..., :1], teacher)):
        with pytest.raises(Exception, match="topk_distillation: "):
            traced(*bad)
    empty = traced(torch.zeros(0, 9, device=where), torch.zeros(0, 3, dtype=torch.int64, device=where),
                   torch.zeros(0, 3, device=where))
    assert empty.shape == ((0,) if reduction == "none" else ()) and not empty.any()


# ------------------------------------------------------------------------------------------ torch.compile
@pytest.mark.parametrize("train", [False, True])
def test_compiled_callers(where, train):
    """The operators run as they are inside a function that torch.compile has taken (backend "eager": nothing is generated)."""
    x, w, b, index = problem(20, 3, 8, 4, where)
    groups = group_rows(index, 3)
    teacher = torch.randint(-1, 4, (20, 2), device=where), torch.randn(20, 2, device=where)

    def step(x, w, b, index):
        y = grouped_linear(x, w, group_rows(index, 3), b)
        rows = embedding(index, w[0])
        if where.type == "cuda":
            return y, rows, grouped_linear(x, w, groups, b), topk_distillation(y, *teacher)
        return y, rows, grouped_linear(x, w, groups, b)

    w = w.requires_grad_(train)
    torch._dynamo.reset()
    got = torch.compile(step, backend="eager")(x, w, b, index)
    for a, c in zip(got, step(x, w, b, index)):
        assert torch.equal(a, c) and a.requires_grad == c.requires_grad == train
    assert torch.equal(got[0], products(x, w.detach(), index, b))
