"""Rows of a trained table by id, times a scale, with the gradient of the table: what the reference leaves to PyTorch when it trains
on rows of its memory or history (modules/memory.py:30, modules/history.py:35)."""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from .packed import _host_ids

MOST_WIDTH = 1 << 24      # of a row (include/orca_b200.h)


def _scale_of(scale):
    scale = float(scale)
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"scale {scale}: a finite fp32 value")
    return scale


def _device_ids(ids, device, rows):
    """Ids as the kernels take them; a host list is refused where an id lies outside the table."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
        shape = np.shape(ids)
        ids = _host_ids(ids, rows, "ids").reshape(shape)
    elif ids.dtype is not torch.int32 and ids.dtype is not torch.int64:
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.device != device or not ids.is_contiguous():
        ids = ids.to(device).contiguous()
    return ids


def _check_status(status, device):
    if status is not None and not (isinstance(status, torch.Tensor) and status.device == device and status.dtype == torch.int32
                                   and status.numel() == 4 and status.is_contiguous()):
        raise ValueError(f"status is a contiguous int32 tensor of 4 on {device}")


def lookup_grad(grad_out, ids, num_rows, scale=1.0, padding=None, status=None):
    """The gradient of a table of ``num_rows`` rows from that of looked-up rows: row v is scale times the sum of grad_out[i] over the
    ids[i] that are v, added up in fp32 in an order that depends on the ids alone, rounded to grad_out's type; the row ``padding``
    and rows that no id names are zero.  What a backward pass of ``lookup_rows`` calls.  In a captured graph this is the call to make: a
    captured backward pass is refused while an older graph of the table lives, for its accumulator is on that graph's stream.  It has no
    derivative: a tangent of grad_out is refused, a backward pass to grad_out raises."""
    if grad_out.dtype not in _lib.TYPES or not grad_out.is_cuda:
        raise TypeError(f"gradients in fp32, bf16 or fp16 on a CUDA device, not {grad_out.dtype} on {grad_out.device}")
    if grad_out.dim() == 0 or grad_out.shape[-1] > MOST_WIDTH:
        raise ValueError(f"gradients of rows, not {tuple(grad_out.shape)}")
    num_rows, scale = int(num_rows), _scale_of(scale)
    if padding is not None and not 0 <= int(padding) < num_rows:
        raise ValueError(f"padding {padding} is no row of the table")
    d = grad_out.device
    ids = _device_ids(ids, d, num_rows)
    if grad_out.shape[:-1] != ids.shape:
        raise ValueError(f"gradients {tuple(grad_out.shape)} for ids {tuple(ids.shape)}")
    _check_status(status, d)
    return _lib.rows().grad(grad_out, ids, num_rows, scale, -1 if padding is None else int(padding), status)


def lookup_rows(table, ids, scale=1.0, padding=None, status=None):
    """scale * table[ids], a product in fp32 rounded to the table's type, shape ids.shape + [width].

    table    [rows, width] in fp32, bf16 or fp16 on a CUDA device; its gradient (once) is ``lookup_grad``; no forward derivatives, neither
             of the rows nor, in a backward pass, of the gradient
    ids      int32 or int64 of any shape; the same id any number of times
    padding  an id whose row is returned but gets no gradient
    status   int32 [4] on the device, zero: set to ORCA_E_BOUNDS by ids outside the table, whose rows are zero (ids from the host
             are refused instead)"""
    if not (isinstance(table, torch.Tensor) and table.is_cuda and table.dim() == 2 and table.dtype in _lib.TYPES):
        raise ValueError("a table is a CUDA tensor [rows, width] in fp32, bf16 or fp16")
    if not 0 < table.shape[1] <= MOST_WIDTH:
        raise ValueError(f"rows of width {table.shape[1]}")
    scale = _scale_of(scale)
    if padding is not None and not 0 <= int(padding) < table.shape[0]:
        raise ValueError(f"padding {padding} is no row of the table")
    _check_status(status, table.device)
    return _lib.rows().lookup(table, _device_ids(ids, table.device, table.shape[0]), scale, -1 if padding is None else int(padding), status)
