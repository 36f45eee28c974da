"""Rows of a per-site table at given site ids, with the table's gradient.

Site ids come out of this package as uint32 with UINT32_MAX for "none"
(``nn``, ``farthest_neighbor``, the walk's ``depth_indices`` and site
records), which torch cannot index with on a GPU.  ``lookup_rows`` takes them
as they are: per-site attributes or learned codes at the sites of a query or
a walk, differentiable with respect to the table in reverse and forward mode.
The gradient is summed over the sorted ids in a fixed order, so a training
step gives the same bits every run, where an index_add on the GPU does not.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwad

from . import _lib

_DTYPES = {torch.float32: _lib.SDFOAM_F32, torch.float16: _lib.SDFOAM_F16, torch.bfloat16: _lib.SDFOAM_BF16}
_ID_TYPES = {torch.uint32: _lib.SDFOAM_U32, torch.int32: _lib.SDFOAM_I32, torch.int64: _lib.SDFOAM_I64}
_MAX_COLUMNS = 1 << 20


def _check(what: str, rows: torch.Tensor, ids: torch.Tensor):
    if rows.dtype not in _DTYPES:
        raise RuntimeError(f"{what} must have float32, float16 or bfloat16 dtype")
    if ids.dtype not in _ID_TYPES:
        raise RuntimeError("ids must have uint32, int32 or int64 dtype")
    if rows.shape[-1] > _MAX_COLUMNS:
        raise RuntimeError(f"{what} must have at most {_MAX_COLUMNS} columns")
    if rows.device.type != "cuda":
        raise RuntimeError(f"{what} must be on CUDA device")
    if ids.device != rows.device:
        raise RuntimeError(f"ids must be on the device of {what}")


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x itself when its rows are contiguous (any distance apart), else a copy.
    A view that negates as it is read (the imaginary part of a conjugate) is
    written out: the kernels read memory."""
    if x.is_neg():
        x = x.resolve_neg()
    ld = x.stride(0)
    return x if x.stride(1) == 1 and ld >= x.shape[1] else x.contiguous()


def _lookup(table, ids, scale):
    t, i = _matrix(table), ids.contiguous()
    rows, columns = t.shape
    out = torch.empty((*ids.shape, columns), dtype=t.dtype, device=t.device)
    lib = _lib.load()
    with _lib.on(t.device):
        _lib.check(lib.sdfoam_lookup_rows(t.data_ptr(), rows, columns, max(t.stride(0), columns), _DTYPES[t.dtype],
                                          i.data_ptr(), i.numel(), _ID_TYPES[i.dtype], scale, out.data_ptr(),
                                          _lib.stream(t.device)))
    return out


def _lookup_backward(grad, ids, num_rows, scale):
    columns = grad.shape[-1]
    g, i = _matrix(grad.reshape(ids.numel(), columns)), ids.contiguous()
    n = i.numel()
    out = torch.empty((num_rows, columns), dtype=g.dtype, device=g.device)
    lib = _lib.load()
    nbytes = lib.sdfoam_lookup_rows_workspace_bytes(n, num_rows, columns)
    with _lib.on(g.device):
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=g.device)
        _lib.check(lib.sdfoam_lookup_rows_backward(g.data_ptr(), columns, max(g.stride(0), columns), _DTYPES[g.dtype],
                                                   i.data_ptr(), n, _ID_TYPES[i.dtype], scale, out.data_ptr(),
                                                   num_rows, ws.data_ptr(), nbytes,
                                                   _lib.stream(g.device)))
    return out


class _Lookup(torch.autograd.Function):
    """Linear in table: the tangent of the rows is the lookup of the table's."""

    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.num_rows, ctx.scale = table.shape[0], scale
        return _lookup(table, ids, scale)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return _LookupBackward.apply(grad, ids, ctx.num_rows, ctx.scale), None, None

    @staticmethod
    def jvp(ctx, table, ids, scale):
        return lookup_rows(table, ctx.saved_tensors[0], ctx.scale)


class _LookupBackward(torch.autograd.Function):
    """Linear in grad, so its own gradient is the lookup again, and its tangent
    the gradient of grad's."""

    @staticmethod
    def forward(ctx, grad, ids, num_rows, scale):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.num_rows, ctx.scale = num_rows, scale
        return _lookup_backward(grad, ids, num_rows, scale)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return _Lookup.apply(grad, ids, ctx.scale), None, None, None

    @staticmethod
    def jvp(ctx, grad, ids, num_rows, scale):
        return lookup_rows_backward(grad, ctx.saved_tensors[0], ctx.num_rows, ctx.scale)


def _differentiated(x: torch.Tensor) -> bool:
    """Whether the result must carry a graph or a tangent."""
    return (x.requires_grad and torch.is_grad_enabled()) or fwad.unpack_dual(x).tangent is not None


def lookup_rows(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]``: shape ``ids.shape + (columns,)``, the table's type.

    table: [rows, columns] float32, float16 or bfloat16 on a CUDA device, rows
    any distance apart.  ids: any shape, uint32, int32 or int64.  An id outside
    [0, rows) -- UINT32_MAX, -1 -- names no row: its output row is zero and it
    adds to no gradient.  The product is fp32, rounded once."""
    if table.dim() != 2:
        raise RuntimeError("table must have 2 dimensions")
    if table.shape[0] >= 2 ** 32:
        raise RuntimeError("table must have fewer than 2^32 rows")
    _check("table", table, ids)
    if not _differentiated(table):
        return _lookup(table, ids, float(scale))
    return _Lookup.apply(table, ids, float(scale))


def lookup_rows_backward(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, scale: float = 1.0) -> torch.Tensor:
    """The gradient of :func:`lookup_rows` with respect to its table: row v is
    ``scale`` times the sum of the rows ``grad[i]`` with ``ids[i] == v``, zeros
    where no id names the row; [num_rows, columns] of grad's type.  Sums are
    fp32 in an order that the ids alone fix."""
    if grad.dim() == 0 or tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise RuntimeError("grad must have the shape of ids with one more dimension, the columns")
    if not 0 <= num_rows < 2 ** 32:
        raise RuntimeError("num_rows must be at least 0 and below 2^32")
    if ids.numel() >= 2 ** 31:
        raise RuntimeError("the gradient takes fewer than 2^31 ids")
    _check("grad", grad, ids)
    if not _differentiated(grad):
        return _lookup_backward(grad, ids, int(num_rows), float(scale))
    return _LookupBackward.apply(grad, ids, int(num_rows), float(scale))
