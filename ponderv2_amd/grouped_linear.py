"""Linear layers with weights of their own for each group of rows: experts, datasets, scenes (csrc/grouped_linear.hip).

``grouped_linear(x, weight, groups, bias)`` is ``linear`` (linear.py) with ``weight[g]`` / ``bias[g]`` for the rows of
group g: ``y[r] = x[r] @ weight[g].T + bias[g]``.  ``groups`` comes from ``row_groups.group_rows`` (rows in any order:
they are read and written where they lie) or ``RowGroups.from_offset`` (rows that lie group by group).  Rows of no group
are zeros in the result and take no gradient; groups may be empty (their weight gradient is zero).

fp32, bf16 or fp16, one type for x, weight and bias, accumulated in fp32; the gradients (of x, weight and bias, once
differentiable) are of the same type and summed in a fixed order.  fp32 products are formed from three bf16 pieces per
operand (mfma_split.h): an infinity among them may give NaN where fp32 arithmetic would give an infinity, and operands
below 2^-110 lose low bits.  Up to 4096 groups."""
import torch

from . import _lib
from .embedding import rows_contiguous
from .kernels import DTYPE_CODE, _require_device
from .row_groups import RowGroups, launch, launch_alone, once_differentiable_backward, ptr

MAX_ROWS = (1 << 30) - 1
MAX_GROUPS = 4096   # every workgroup scans the groups' offsets for its own
MAX_WIDTH = (1 << 24) - 1


def _weight_rows(w):
    return w if w.stride(2) == 1 or w.shape[2] == 1 else w.contiguous()


def _products(x, weight, bias, order, offsets, n_rows):
    """(the products, x and weight as the kernels take them).  Checks and layout are part of it, so that a replayed trace
    checks and lays out the tensors of its own call.  n_rows: of groups without an order."""
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2]:
        raise ValueError(f"grouped_linear: x (M, K) and weight (G, N, K) expected, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    (m, k), (g, n, _) = x.shape, weight.shape
    n_rows, n_groups = int(n_rows) if order is None else order.numel(), offsets.numel() - 1
    if n_rows != m or n_groups != g:
        raise ValueError(f"grouped_linear: {m} rows and {g} weights, but groups of {n_rows} rows in "
                         f"{n_groups} groups")
    if bias is not None and tuple(bias.shape) != (g, n):
        raise ValueError(f"grouped_linear: bias is (G, N) = {(g, n)}, got {tuple(bias.shape)}")
    if min(n, k) < 1 or max(n, k) > MAX_WIDTH or m > MAX_ROWS or g > MAX_GROUPS:
        raise ValueError(f"grouped_linear: widths 1 to {MAX_WIDTH}, up to {MAX_ROWS} rows and {MAX_GROUPS} groups")
    dtype, device = x.dtype, x.device
    if dtype not in DTYPE_CODE or weight.dtype != dtype or bias is not None and bias.dtype != dtype:
        raise TypeError("grouped_linear: x, weight and bias are all float32, all bfloat16 or all float16, got "
                        + ", ".join(str(t.dtype) for t in (x, weight, bias) if t is not None))
    _require_device(x, weight, bias)
    if weight.device != device or offsets.device != device or bias is not None and bias.device != device:
        raise ValueError("grouped_linear: x, weight, bias and groups are on different devices")
    x, weight = rows_contiguous(x), _weight_rows(weight)
    bias = None if bias is None else bias.contiguous()
    y = torch.empty((m, n), dtype=dtype, device=device)
    if m:
        launch("pv2_grouped_linear_forward", device, ptr(x), DTYPE_CODE[dtype], m, k, x.stride(0), ptr(weight),
               weight.stride(0), weight.stride(1), g, n, ptr(bias), ptr(order), ptr(offsets), ptr(y))
    return y, x, weight


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, order, offsets, n_rows):
        y, x, weight = _products(x, weight, bias, order, offsets, n_rows)
        ctx.save_for_backward(x, weight, order, offsets)
        return y

    @once_differentiable_backward
    def backward(ctx, gy):
        x, weight, order, offsets = ctx.saved_tensors
        (m, k), (g, n, _) = x.shape, weight.shape
        code, gy = DTYPE_CODE[x.dtype], rows_contiguous(gy)
        new = lambda *shape, dtype=x.dtype: torch.empty(shape, dtype=dtype, device=x.device)
        gx = gw = gb = None
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if m == 0:
            zeros = lambda *shape: torch.zeros(shape, dtype=x.dtype, device=x.device)
            return (zeros(0, k) if need_x else None, zeros(g, n, k) if need_w else None,
                    zeros(g, n) if need_b else None, None, None, None)
        if need_x:
            gx = new(m, k)
            launch("pv2_grouped_linear_grad_input", x.device, ptr(gy), code, m, n, gy.stride(0), ptr(weight),
                   weight.stride(0), weight.stride(1), g, k, ptr(order), ptr(offsets), ptr(gx))
        if need_w or need_b:
            gw = new(g, n, k) if need_w else None
            gb = new(g, n) if need_b else None
            L = _lib.lib()
            floats = (L.pv2_grouped_linear_workspace_floats(code, m, g, n, k) if need_w
                      else L.pv2_grouped_linear_bias_workspace_floats(code, m, g, n))
            workspace = new(floats, dtype=torch.float32) if floats else None
            launch("pv2_grouped_linear_grad_weight", x.device, ptr(gy), code, m, n, gy.stride(0), ptr(x), k,
                   x.stride(0), g, ptr(order), ptr(offsets), ptr(workspace), ptr(gw), ptr(gb))
        return gx, gw, gb, None, None, None


def grouped_linear(x, weight, groups, bias=None):
    """x (M, K), weight (G, N, K), groups: RowGroups of M rows in G groups, bias (G, N) or None.  -> (M, N)."""
    if not isinstance(groups, RowGroups):
        raise TypeError("grouped_linear: groups is what row_groups.group_rows or RowGroups.from_offset returns")
    order, offsets = groups.checked("grouped_linear")
    n_rows = groups.n_rows if order is None else None
    if not launch_alone(x, weight, bias):
        return _GroupedLinear.apply(x, weight, bias, order, offsets, n_rows)
    # (products without a gradient - serving - are the launch alone)
    return _products(x, weight, bias, order, offsets, n_rows)[0]
