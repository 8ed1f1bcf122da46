"""Rows by id: which rows belong to which group (expert, dataset, class, scene), as the grouped linear layers
(grouped_linear.py) take it (csrc/row_groups.hip).

``group_rows(index, num_groups)`` sorts the rows by their id on the device, without a host read;
``RowGroups.from_offset(offset, n_rows)`` takes rows that already lie group by group, as the points of a batch do
(``offset``: cumulative row counts, the ``data_dict["offset"]`` convention).
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels import _raw_stream, _require_device

MAX_ROWS = (1 << 31) - 4097
MAX_GROUPS = 1 << 30

_tracing_state = torch._C._get_tracing_state
_compiling = torch.compiler.is_compiling


def launch(name, device, *args):
    """The entry point ``name`` on the current stream of ``device``, whichever device is current.  Tensors are passed by
    ``data_ptr()``: these calls are made once per layer and step, and next to a kernel of a few microseconds what the
    host spends on a call is what it takes."""
    index = device.index
    fn = getattr(_lib.lib(), name)
    stream = _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream
    if index == torch.cuda.current_device():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            status = fn(*args, stream)
    if status:
        _lib.check(status, name)


def ptr(t):
    return None if t is None else t.data_ptr()


def number(value, what):
    """A Python number; a tensor that asks for a gradient is refused, since none is formed for it."""
    if isinstance(value, torch.Tensor) and value.requires_grad:
        raise TypeError(f"{what} is a number and takes no gradient; multiply by it outside or detach it")
    return float(value)


def launch_alone(*tensors):
    """Whether a call may be its launch alone, past the autograd Function: none of ``tensors`` asks for a gradient, none can
    carry a tangent (the Function refuses those by name) and no trace is recorded (it would keep the empty result and not
    the launch that fills it)."""
    if forward_ad._current_level >= 0 or _tracing_state() is not None:
        return False
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return False
    return True


def once_differentiable_backward(fn):
    """A Function's backward whose results carry no gradient (``once_differentiable``, entered only where grad mode is on:
    in an ordinary backward pass it is off already)."""
    strict = once_differentiable(fn)

    def backward(ctx, *grads):
        return strict(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return staticmethod(backward)


def require_index(index, what):
    if index.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: integer ids (int64 or int32) expected, got {index.dtype}")


class RowGroups:
    """``order`` int32 (n_rows,), or None where the rows already lie in order: the rows of group 0, of group 1, ..,
    then the rows of no group; ``offsets`` int32 (n_groups + 1,): where each group's rows begin in it.  Kernels address
    memory by both without a check, so they are made here only, by ``group_rows`` and ``from_offset``, are not assigned to,
    and are refused once they were written to in place."""

    __slots__ = ("_order", "_offsets", "_n_rows", "_n_groups")

    def __init__(self, *args, **kwargs):
        raise TypeError("RowGroups are made by group_rows(index, num_groups) or RowGroups.from_offset(offset, n_rows)")

    @classmethod
    def _made(cls, order, offsets, n_rows, n_groups):
        self = object.__new__(cls)
        self._order, self._offsets, self._n_rows, self._n_groups = order, offsets, n_rows, n_groups
        return self

    @classmethod
    def _copied(cls, order, offsets, n_rows, n_groups):
        return cls._made(None if order is None else order.clone(), offsets.clone(), n_rows, n_groups)

    order = property(lambda self: self._order)
    offsets = property(lambda self: self._offsets)
    n_rows = property(lambda self: self._n_rows)
    n_groups = property(lambda self: self._n_groups)

    def checked(self, what):
        """(order, offsets), which nothing has written to since they were made."""
        order, offsets = self._order, self._offsets
        try:   # (while torch.compile looks at it the counts are symbols: nothing to decide by)
            written = not _compiling() and (offsets._version or order is not None and order._version)
        except RuntimeError:   # (tensors of inference mode do not count their writes)
            written = False
        if written:
            raise RuntimeError(f"{what}: the groups' order or offsets were written to; make new ones with group_rows")
        return order, offsets

    def __reduce__(self):
        return RowGroups._copied, (*self.checked("RowGroups"), self._n_rows, self._n_groups)

    @classmethod
    def from_offset(cls, offset, n_rows):
        """Rows 0 .. offset[0] - 1 are group 0's, offset[0] .. offset[1] - 1 group 1's, ..; rows behind the last
        offset belong to no group."""
        offsets = (_from_offset if _tracing_state() is None else _FromOffset.apply)(offset, n_rows)
        return cls._made(None, offsets, n_rows, offset.numel())


def _from_offset(offset, n_rows):
    require_index(offset, "RowGroups.from_offset")
    if offset.dim() != 1 or offset.numel() < 1:
        raise ValueError("RowGroups.from_offset: offset is (n_groups,), one group at least")
    if not 0 <= n_rows <= MAX_ROWS:
        raise ValueError(f"RowGroups.from_offset: {n_rows} rows (0 to {MAX_ROWS})")
    _require_device(offset)
    offset = offset.contiguous()
    n_groups = offset.numel()
    offsets = torch.empty(n_groups + 1, dtype=torch.int32, device=offset.device)
    launch("pv2_row_offsets", offset.device, ptr(offset), offset.dtype == torch.int64, n_groups, n_rows, ptr(offsets))
    return offsets


def _group_rows(index, num_groups):
    require_index(index, "group_rows")
    n = index.numel()
    if not 1 <= num_groups <= MAX_GROUPS:
        raise ValueError(f"group_rows: {num_groups} groups (1 to {MAX_GROUPS})")
    if n > MAX_ROWS:
        raise ValueError(f"group_rows: {n} rows (up to {MAX_ROWS})")
    _require_device(index)
    index = index.contiguous()
    device = index.device
    order = torch.empty(n, dtype=torch.int32, device=device)
    offsets = torch.empty(num_groups + 1, dtype=torch.int32, device=device)
    ints = _lib.lib().pv2_row_groups_workspace_ints(n, num_groups)
    workspace = torch.empty(ints, dtype=torch.int32, device=device) if ints else None
    launch("pv2_row_groups", device, ptr(index), index.dtype == torch.int64, n, num_groups, ptr(order), ptr(offsets),
           None, ptr(workspace))
    return order, offsets


# (ids have no gradient: these are what a recorded trace keeps of a call)
class _FromOffset(torch.autograd.Function):
    @staticmethod
    def forward(ctx, offset, n_rows):
        return _from_offset(offset, int(n_rows))


class _GroupRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, index, num_groups):
        return _group_rows(index, int(num_groups))


def group_rows(index, num_groups):
    """index: integer ids of the rows (any shape, read as one list).  -> RowGroups with the stable order by id; rows
    whose id is outside 0 .. num_groups - 1 (padding, unlabelled points at -1) belong to no group."""
    order, offsets = (_group_rows if _tracing_state() is None else _GroupRows.apply)(index, num_groups)
    return RowGroups._made(order, offsets, index.numel(), num_groups)
