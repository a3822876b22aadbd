"""Group norm with an activation on channels-last tensors::

    y = act((x - mean) * rstd * weight + bias)

with mean and variance over all positions of a sample and the channels of a group.  ``(samples, *positions, channels)``:
a ``channels_last`` feature map, or tokens ``(samples, channels)`` with one position each.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib, _seq

__all__ = ["GroupNormCL", "group_norm"]


def _forward(x, num_groups, weight, bias, eps, activation):
    """Launches the forward pass: y, and what the backward pass reads."""
    R, S, C = x.shape
    weight, bias = _seq.dense(weight), _seq.dense(bias)
    y = x.new_empty((R, S, C))
    stats = torch.empty((2, R, num_groups), dtype=torch.float32, device=x.device)      # mean, 1 / deviation
    if R * S * C:
        _lib.group_norm_forward(y, stats, x, weight, bias, eps, activation, R, S, C, num_groups)
    return y, (x, weight, bias, stats)


class GroupNormCL(torch.autograd.Function):
    """``apply(x, num_groups, weight, bias, eps, activation) -> y`` on (samples, positions, channels); see
    :func:`group_norm`, which checks the arguments."""

    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, eps, activation):
        y, used = _forward(x, num_groups, weight, bias, eps, activation)
        ctx.num_groups, ctx.activation = num_groups, activation
        ctx.save_for_backward(*used)
        return y

    @staticmethod
    def backward(ctx, dy):
        _seq.refuse_second_order("group_norm", dy)
        x, weight, bias, stats = ctx.saved_tensors
        R, S, C = x.shape
        dx = x.new_empty((R, S, C))
        dweight = torch.empty_like(weight) if weight is not None else None
        dbias = torch.empty_like(bias) if bias is not None else None
        if R * S * C:
            _lib.group_norm_backward(dx, dweight, dbias, dy, x, stats, weight, bias, ctx.activation, R, S,
                                     C, ctx.num_groups)
        else:
            for t in (dweight, dbias):
                if t is not None:
                    t.zero_()
        return dx, None, dweight, dbias, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, activation: Optional[str] = None) -> torch.Tensor:
    """Group norm of a channels-last tensor; differentiable, in reverse mode and once.

    Parameters
    ----------
    x: (samples, *positions, channels), float32, bfloat16 or float16; at most 16384 channels per group.
    num_groups: divides the channels.
    weight, bias: (channels,) float32 or the type of ``x``, both of one type; each may be absent.
    eps: added to the variance.
    activation: None, "silu" or "relu".

    Returns the normalised tensor, contiguous, of the shape and type of ``x``.
    """
    _seq.require_data("x", x)
    if x.ndim < 2:
        raise ValueError("'x' must have at least 2 dimensions, (samples, ..., channels)")
    C = x.shape[-1]
    if not isinstance(num_groups, int) or num_groups < 1 or C % num_groups:
        raise ValueError(f"'num_groups' must divide the {C} channels, got {num_groups!r}")
    if C // num_groups > _lib.NORM_MAX_GROUP:
        raise ValueError(f"at most {_lib.NORM_MAX_GROUP} channels in a group are supported, got {C // num_groups}")
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"'activation' must be None, 'silu' or 'relu', got {activation!r}")
    if not eps >= 0.0:
        raise ValueError(f"'eps' must not be negative, got {eps}")
    kind, dev = getattr(weight if weight is not None else x if bias is None else bias, "dtype", None), x.get_device()
    if dev < 0 or (kind != torch.float32 and kind != x.dtype) or not (_seq.alike(weight, (C,), kind, dev) and _seq.alike(bias, (C,), kind, dev)):
        _seq.require_like("weight", weight, (C,), (torch.float32, x.dtype), x.device)
        _seq.require_like("bias", bias, (C,), (torch.float32, x.dtype), x.device)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"'weight' and 'bias' must have one type, got {weight.dtype} and {bias.dtype}")
    _seq.require_cuda("x", x)
    _seq.refuse_tangents("group_norm", x, weight, bias)
    if x.ndim == 3:
        flat = x
    elif x.ndim == 2:
        flat = x.unsqueeze(1)
    else:
        flat = x.reshape(x.shape[0], math.prod(x.shape[1:-1]), C)
    if _seq.wants_grad(x, weight, bias):
        y = GroupNormCL.apply(flat, num_groups, weight, bias, float(eps), activation)
    else:
        y = _forward(flat, num_groups, weight, bias, float(eps), activation)[0]
    return y if x.ndim == 3 else y.reshape(x.shape)
