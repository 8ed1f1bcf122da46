"""Embedding lookup with scaling, its gradient by sorted tokens (csrc/embedding.hip).

``embedding(index, weight, scale)`` is ``torch.nn.functional.embedding(index, weight) * scale`` for fp32 / bf16 / fp16
tables, except that an index outside the table (-1: an unlabelled point, padding) gives a row of zeros and takes no
gradient.  The gradient is dense, of the table's type, summed in fp32 in a fixed order: the same inputs give the same
bits, however often a class repeats."""
import torch

from . import _lib
from .kernels import DTYPE_CODE, _require_device
from .row_groups import (MAX_GROUPS, MAX_ROWS, launch, launch_alone, number, once_differentiable_backward, ptr,
                         require_index)

MAX_WIDTH = (1 << 30) - 1


def _lookup(index, weight, scale):
    """(the rows, the ids as one list).  Checks and layout are part of it, so that a replayed trace checks and lays out the
    tensors of its own call."""
    require_index(index, "embedding")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"embedding: weight is (rows, channels), got {tuple(weight.shape)}")
    n, (rows, c) = index.numel(), weight.shape
    if n > MAX_ROWS or rows > MAX_GROUPS or c > MAX_WIDTH:
        raise ValueError(f"embedding: up to {MAX_ROWS} indices, {MAX_GROUPS} rows and {MAX_WIDTH} channels")
    if weight.dtype not in DTYPE_CODE:
        raise TypeError(f"embedding: float32, bfloat16 or float16 weight expected, got {weight.dtype}")
    _require_device(index, weight)
    if index.device != weight.device:
        raise ValueError(f"embedding: index on {index.device}, weight on {weight.device}")
    flat = index if index.dim() == 1 and index.is_contiguous() else index.reshape(-1).contiguous()
    weight = rows_contiguous(weight)
    y = torch.empty((*index.shape, c), dtype=weight.dtype, device=weight.device)
    if n:
        launch("pv2_embedding_forward", weight.device, ptr(flat), flat.dtype == torch.int64, n, ptr(weight),
               DTYPE_CODE[weight.dtype], rows, c, weight.stride(0), scale, ptr(y))
    return y, flat


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, index, weight, scale):
        y, flat = _lookup(index, weight, scale)
        ctx.save_for_backward(flat)
        ctx.table = (*weight.shape, scale)
        return y

    @once_differentiable_backward
    def backward(ctx, gy):
        index, = ctx.saved_tensors
        rows, c, scale = ctx.table
        n = index.numel()
        gy = rows_contiguous(gy.reshape(-1, c))
        workspace = torch.empty(_lib.lib().pv2_embedding_backward_workspace_ints(n, rows, c), dtype=torch.int32,
                                device=gy.device)
        gw = torch.empty((rows, c), dtype=gy.dtype, device=gy.device)
        launch("pv2_embedding_backward", gy.device, ptr(index), index.dtype == torch.int64, n, ptr(gy),
               DTYPE_CODE[gy.dtype], rows, c, gy.stride(0), scale, ptr(workspace), ptr(gw))
        return None, gw, None


def rows_contiguous(t):
    """A matrix whose rows are contiguous; any (non-negative) distance between rows is kept."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def embedding(index, weight, scale=1.0):
    """index: int64 / int32 ids of any shape; weight (rows, C).  -> (*index.shape, C) = scale * weight[index]."""
    scale = scale if type(scale) is float else number(scale, "embedding: scale")
    if not launch_alone(weight):
        return _Embedding.apply(index, weight, scale)
    # (a lookup without a gradient - serving - is the launch alone)
    return _lookup(index, weight, scale)[0]
