"""Rows of a trained table by id, times a scale, with the gradient of the table: what the reference leaves to PyTorch when it trains
on rows of its memory or history (modules/memory.py:30, modules/history.py:35)."""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .packed import _host_ids


def _device_ids(ids, device, rows):
    """(ids, 0 or 1 for int32 or int64); a host list is refused where an id lies outside the table."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
        ids = _host_ids(ids, rows, "ids")
    elif ids.dtype is not torch.int32 and ids.dtype is not torch.int64:
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.device != device or not ids.is_contiguous():
        ids = ids.to(device).contiguous()
    return ids, int(ids.dtype is torch.int64)


def _status_of(status, device):
    if not (isinstance(status, torch.Tensor) and status.device == device and status.dtype == torch.int32 and status.numel() == 4
            and status.is_contiguous()):
        raise ValueError(f"status is a contiguous int32 tensor of 4 on {device}")
    return status.data_ptr()


def lookup_grad(grad_out, ids, num_rows, scale=1.0, padding=None, status=None):
    """The gradient of a table of ``num_rows`` rows from that of looked-up rows: row v is scale times the sum of grad_out[i] over the
    ids[i] that are v, added up in fp32 in an order that depends on the ids alone, rounded once to grad_out's type; the row ``padding`` and rows that no id
    names are zero.  What ``lookup_rows`` calls in a backward pass; callable in a captured graph."""
    if grad_out.dtype not in _lib.TYPES or not grad_out.is_cuda:
        raise TypeError(f"gradients in fp32, bf16 or fp16 on a CUDA device, not {grad_out.dtype} on {grad_out.device}")
    if padding is not None and not 0 <= int(padding) < num_rows:
        raise ValueError(f"padding {padding} is no row of the table")
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale}")
    d = grad_out.device
    ids, wide = _device_ids(ids, d, num_rows)
    if grad_out.shape[:-1] != ids.shape:
        raise ValueError(f"gradients {tuple(grad_out.shape)} for ids {tuple(ids.shape)}")
    width, n = grad_out.shape[-1], ids.numel()
    g = grad_out if grad_out.dim() == 2 else grad_out.reshape(n, width)
    stride = g.stride(0) if n > 1 else width
    if n and (g.stride(1) != 1 and width > 1 or 0 < stride < width):
        g, stride = g.contiguous(), width
    grad = torch.empty((num_rows, width), dtype=grad_out.dtype, device=d)
    if width == 0:
        return grad
    L = _lib.lib()
    with _lib.launch(d) as stream:
        need = L.orca_rows_grad_workspace_bytes(n, num_rows, width)
        ws = torch.empty((need,), dtype=torch.uint8, device=d) if need else None
        _lib.check(L.orca_rows_grad(g.data_ptr(), stride, width, _lib.TYPES[g.dtype], ids.data_ptr(), wide, n, num_rows, scale,
                                    -1 if padding is None else int(padding), grad.data_ptr(), None if status is None else _status_of(status, d), ws.data_ptr() if need else None,
                                    need, stream))
    return grad


def _lookup(table, ids, wide, scale, status):
    width, d = table.shape[1], table.device
    t = table if table.stride(1) == 1 and table.stride(0) >= width else table.detach().contiguous()
    out = torch.empty((*ids.shape, width), dtype=table.dtype, device=d)
    with _lib.launch(d) as stream:
        _lib.check(_lib.lib().orca_rows_lookup(t.data_ptr(), t.shape[0], max(t.stride(0), width), width, _lib.TYPES[t.dtype], ids.data_ptr(),
                                               wide, ids.numel(), scale, out.data_ptr(), None if status is None else _status_of(status, d), stream))
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, wide, scale, padding, status):
        out = _lookup(table, ids, wide, scale, status)
        ctx.save_for_backward(ids)
        ctx.how = (table.shape[0], scale, padding, status)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        # (what refuses second derivatives costs 10 us: only where somebody may want them)
        return _Lookup.once(ctx, grad_out) if torch.is_grad_enabled() else _Lookup.table_grad(ctx, grad_out)

    @staticmethod
    def table_grad(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        return lookup_grad(grad_out, ids, *ctx.how), None, None, None, None, None

    once = staticmethod(once_differentiable(table_grad.__func__))


def lookup_rows(table, ids, scale=1.0, padding=None, status=None):
    """scale * table[ids], rounded once to the table's type, shape ids.shape + [width].

    table    [rows, width] in fp32, bf16 or fp16 on a CUDA device; its gradient (once) is ``lookup_grad``
    ids      int32 or int64 of any shape; the same id any number of times
    padding  an id whose row is returned but gets no gradient
    status   int32 [4] on the device, zero: set to ORCA_E_BOUNDS by ids outside the table, whose rows are zero (ids from the host
             are refused instead)"""
    if not (isinstance(table, torch.Tensor) and table.is_cuda and table.dim() == 2 and table.dtype in _lib.TYPES):
        raise ValueError("a table is a CUDA tensor [rows, width] in fp32, bf16 or fp16")
    if table.shape[1] == 0:
        raise ValueError("rows of width 0")
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale}")
    if padding is not None and not 0 <= int(padding) < table.shape[0]:
        raise ValueError(f"padding {padding} is no row of the table")
    ids, wide = _device_ids(ids, table.device, table.shape[0])
    if not (table.requires_grad and torch.is_grad_enabled()):
        return _lookup(table, ids, wide, scale, status)
    return _Lookup.apply(table, ids, wide, scale, padding, status)
