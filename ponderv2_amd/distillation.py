"""Distillation from a teacher's top logits: the classes and logits of a large (2-D, open-vocabulary) teacher are stored
for its k best classes per row only (csrc/distillation.hip).

With temperature T, p = softmax(teacher_logits / T) over a row's listed classes and q = softmax(logits / T) over all:
``loss_i = T^2 * sum_e p_e (log p_e - log q_{c_e})``, the Kullback-Leibler divergence scaled so that its gradient keeps its
size when T changes (1e-4 <= T <= 1e4; the divergence is summed in fp32, so T^2 scales its rounding too).  An entry counts
if its class is one of the logits' (-1: none) and its logit is above -inf; a row without one has loss 0 and gradient 0,
whatever its logits hold.  A class may be listed twice."""
import torch

from . import _lib
from .embedding import rows_contiguous
from .kernels import DTYPE_CODE, _require_device
from .row_groups import launch, number, once_differentiable_backward, ptr, require_index

MAX_TOP = 1024
MAX_CLASSES = (1 << 30) - 1
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-4, 1e4   # 1 / T and T^2 leave fp32 room for the logits
REDUCTIONS = ("mean", "sum", "none")


def _rows(t, width):
    return rows_contiguous(t if t.dim() == 2 else t.reshape(-1, width))


def check_lists(logits, teacher_index, teacher_logits):
    """What every form of the loss takes as lists."""
    require_index(teacher_index, "topk_distillation: teacher_index")
    if teacher_logits.dtype not in DTYPE_CODE:
        raise TypeError(f"topk_distillation: float32, bfloat16 or float16 teacher_logits expected, got {teacher_logits.dtype}")
    shape, lists = logits.shape, teacher_index.shape
    if len(shape) < 1 or teacher_logits.shape != lists or len(lists) != len(shape) or lists[:-1] != shape[:-1]:
        raise ValueError(f"topk_distillation: logits (..., V), teacher_index and teacher_logits (..., k) expected, got "
                         f"{tuple(shape)}, {tuple(lists)}, {tuple(teacher_logits.shape)}")
    v, k = shape[-1], lists[-1]
    if not 1 <= k <= MAX_TOP or not 1 <= v <= MAX_CLASSES:
        raise ValueError(f"topk_distillation: {v} classes (1 to {MAX_CLASSES}), {k} listed (1 to {MAX_TOP})")
    return v, k


def _checked(logits, teacher_index, teacher_logits):
    """The three as matrices with contiguous rows.  Part of every pass through the operator, so that a replayed trace checks
    and lays out the tensors of its own call."""
    if logits.dtype not in DTYPE_CODE:
        raise TypeError(f"topk_distillation: float32, bfloat16 or float16 logits expected, got {logits.dtype}")
    v, k = check_lists(logits, teacher_index, teacher_logits)
    _require_device(logits, teacher_index, teacher_logits)
    if not logits.device == teacher_index.device == teacher_logits.device:
        raise ValueError("topk_distillation: logits, teacher_index and teacher_logits are on different devices")
    return _rows(logits, v), _rows(teacher_index, k), _rows(teacher_logits, k)


class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, temperature, reduction):
        shape = logits.shape
        logits, index, teacher = _checked(logits, index, teacher)
        (m, v), k = logits.shape, index.shape[1]
        device = logits.device
        ctx.how = (temperature, reduction, None if len(shape) == 2 else shape)
        if m == 0:   # nothing to launch: an exact zero
            ctx.save_for_backward(logits, index, teacher, None)
            return torch.zeros(shape[:-1] if reduction == "none" else (), dtype=torch.float32, device=device)
        # the rows' statistics, their number, and scratch
        saved = torch.empty(2 * m + 1 + _lib.lib().pv2_topk_distill_workspace_floats(m, v, k), dtype=torch.float32,
                            device=device)
        loss = torch.empty((), dtype=torch.float32, device=device)
        row_loss = torch.empty(shape[:-1], dtype=torch.float32, device=device) if reduction == "none" else None
        stats = ptr(saved)
        count = stats + 8 * int(m)   # (sizes are tensors while a trace is recorded)
        launch("pv2_topk_distill_forward", device, ptr(logits), DTYPE_CODE[logits.dtype], m, v, logits.stride(0),
               ptr(index), index.dtype == torch.int64, index.stride(0), ptr(teacher), DTYPE_CODE[teacher.dtype],
               teacher.stride(0), k, temperature, reduction == "mean", count + 4, stats, ptr(row_loss), ptr(loss), count)
        ctx.save_for_backward(logits, index, teacher, saved)
        return loss if row_loss is None else row_loss

    @once_differentiable_backward
    def backward(ctx, up):
        logits, index, teacher, saved = ctx.saved_tensors
        temperature, reduction, shape = ctx.how
        (m, v), k = logits.shape, index.shape[1]
        up = up.contiguous()
        grad = torch.empty((m, v), dtype=logits.dtype, device=logits.device)
        if m:
            stats = ptr(saved)
            launch("pv2_topk_distill_backward", logits.device, ptr(logits), DTYPE_CODE[logits.dtype], m, v,
                   logits.stride(0), ptr(index), index.dtype == torch.int64, index.stride(0), ptr(teacher),
                   DTYPE_CODE[teacher.dtype], teacher.stride(0), k, temperature, stats, ptr(up), reduction == "none",
                   stats + 8 * m if reduction == "mean" else None, ptr(grad))
        return grad if shape is None else grad.view(shape), None, None, None, None


def topk_distillation(logits, teacher_index, teacher_logits, temperature=1.0, reduction="mean"):
    """logits (..., V) fp32 / bf16 / fp16; teacher_index (..., k) int64 / int32 and teacher_logits (..., k) fp32 / bf16 /
    fp16, with the same leading axes.  -> fp32: the mean over the rows that count ("mean", 0 if none does), the sum, or
    every row's loss ("none").  The gradient, of the logits only, has their type."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"topk_distillation: reduction is one of {REDUCTIONS}, got {reduction!r}")
    temperature = number(temperature, "topk_distillation: temperature")
    if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
        raise ValueError(f"topk_distillation: temperature {temperature} ({MIN_TEMPERATURE:g} to {MAX_TEMPERATURE:g})")
    return _TopkDistillation.apply(logits, teacher_index, teacher_logits.detach(), temperature, reduction)
