"""Layer norm over the last dimension with its gradients: what the reference leaves to PyTorch behind its attention layers
(model/temporal_attention.py:55), for rows that are trained (orca_b200.lookup)."""
from __future__ import annotations

from . import _lib


def _eps_of(eps):
    eps = float(eps)
    if not 0 <= eps <= 3.4e38:
        raise ValueError(f"eps {eps}: a finite value of 0 or more")
    return eps


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension, computed in fp32 and rounded once to x's type; a row whose squares of (x - mean)
    add up to more than fp32 holds (values of 1.8e19 and more) is NaN, as one with a value that is not finite.

    x             fp32, bf16 or fp16 on a CUDA device, [..., width] with width from 1 to 2^24, of any strides
    weight, bias  [width], of x's type or both fp32; None: one and zero

    Its gradients (once) are ``layer_norm_grad``; nothing but x and weight is kept for them.  No forward derivatives, no traces, no vmap."""
    return _lib.rows().norm(x, weight, bias, _eps_of(eps))


def layer_norm_grad(grad_out, x, weight=None, eps=1e-5):
    """The gradients of x, weight and bias from that of ``layer_norm``'s result: what its backward pass calls.  Those of weight and bias are of
    weight's type (x's where there is none), their sums over rows in fp32; the same rows, strides and alignment give the same bits.  In a captured graph
    this is the call to make: a captured backward pass is refused while an older graph of its inputs lives, for their accumulators are on
    that graph's stream.  Results have no derivative: a tangent is refused, a backward pass raises."""
    return _lib.rows().norm_grad(grad_out, x, weight, _eps_of(eps))
