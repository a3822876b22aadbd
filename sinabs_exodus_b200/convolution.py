"""Short causal convolution along time, one filter per channel, with an optional silu::

    y_t[m] = act(bias[m] + sum_k weight[m, k] x_{t-W+1+k}[m])

The rows in front of the first step are the ``state`` that the previous call returned (or zeros), so a sequence may come
in chunks or token by token, like the states of the neuron layers.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, _seq

__all__ = ["CausalConvTM", "causal_conv", "causal_conv_step"]


class CausalConvTM(torch.autograd.Function):
    """``apply(x, weight, bias, state, lengths, activation) -> (y, last)``; see :func:`causal_conv`, which checks the
    arguments."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, activation):
        nb, T, M = x.shape
        W = weight.shape[1]
        x = _seq.channels_contiguous(x)
        weight, bias, state = (_seq.dense(t) for t in (weight, bias, state))
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        ctx.set_materialize_grads(False)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, bias, state, lengths)
        if nb * T * M == 0:      # no rows: the state passes through unchanged
            return y, state.clone() if state is not None else torch.zeros(nb, W - 1, M, dtype=x.dtype, device=x.device)
        last = torch.empty(nb, W - 1, M, dtype=x.dtype, device=x.device)
        _lib.causal_conv_forward(y, last, x, weight, bias, state, lengths, activation, nb, T, M, W)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        nb, T, M = x.shape
        W = weight.shape[1]
        empty = nb * T * M == 0
        new = torch.zeros_like if empty else torch.empty_like
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dweight = new(weight)
        dbias = new(bias) if bias is not None else None
        dstate = new(state) if state is not None else None
        dlast = _seq.dense(dlast)
        if empty:
            if dstate is not None and dlast is not None:
                dstate.copy_(dlast)
        else:
            dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else _seq.channels_contiguous(dy)
            _lib.causal_conv_backward(dx, dweight, dbias, dstate, dy, dlast, x, weight, bias, state, lengths, ctx.activation, nb, T, M, W)
        return dx, dweight, dbias, dstate, None, None


def _check(x, weight, bias, activation) -> int:
    """Checks what prompts and single tokens share; returns the filter's width."""
    _seq.require_data("x", x)
    M = x.shape[-1]
    if not isinstance(weight, torch.Tensor):
        raise TypeError(f"'weight' must be a tensor, got {type(weight).__name__}")
    if weight.ndim != 2 or weight.shape[0] != M:
        raise ValueError(f"'weight' must have shape ({M}, width), got {tuple(weight.shape)}")
    W = weight.shape[1]
    if not 1 <= W <= _lib.CONV_MAX_WIDTH:
        raise ValueError(f"filters of 1 to {_lib.CONV_MAX_WIDTH} steps are supported, got {W}")
    if activation not in (None, "silu"):
        raise ValueError(f"'activation' must be None or 'silu', got {activation!r}")
    _seq.require_like("weight", weight, (M, W), (torch.float32, x.dtype), x.device)
    _seq.require_like("bias", bias, (M,), (weight.dtype,), x.device)
    return W


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution over a whole prompt; differentiable.

    Parameters
    ----------
    x: (batch, time, channels), float32, bfloat16 or float16.
    weight: (channels, width), width 1 to 8, float32 or the type of ``x``; ``weight[:, -1]`` meets the current step.
    bias: (channels,), of the type of ``weight``.
    state: (batch, width - 1, channels) rows in front of ``x``, of its type (zeros if absent).
    lengths: (batch,) int32 or int64 numbers of valid steps of a padded batch; outputs and gradients of the rows behind
        them are 0, and what these rows hold does not enter anything.
    activation: None or "silu".

    Returns
    -------
    ``(y, last)``: the output and the ``width - 1`` last valid rows, the ``state`` of the next call; both with gradients.
    """
    if isinstance(x, torch.Tensor) and x.ndim != 3:
        raise ValueError("'x' must be 3D, (batch, time, channels)")
    W = _check(x, weight, bias, activation)
    _seq.require_like("state", state, (x.shape[0], W - 1, x.shape[2]), (x.dtype,), x.device)
    lengths = _seq.check_lengths(lengths, x.shape[0], x.device)
    _seq.require_cuda("x", x)
    return CausalConvTM.apply(x, weight, bias, state, lengths, activation)


def causal_conv_step(state: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     activation: Optional[str] = None) -> torch.Tensor:
    """One step of :func:`causal_conv` for single tokens: appends ``x`` (batch, channels) to ``state`` (batch, width - 1,
    channels) in place, dropping its oldest row, and returns the output (batch, channels).  Not differentiable.

    ``state`` has contiguous (width - 1, channels); its batch items may lie apart (rows of a pool).
    """
    if isinstance(x, torch.Tensor) and x.ndim != 2:
        raise ValueError("'x' must be 2D, (batch, channels)")
    W = _check(x, weight, bias, activation)
    nb, M = x.shape
    _seq.require_like("state", state, (nb, W - 1, M), (x.dtype,), x.device)
    if nb * M and _seq.channels_contiguous(state, 2) is not state:
        raise ValueError("'state' must be contiguous in its rows and channels: it is updated in place")
    if nb > 1 and state.stride(0) < (W - 1) * M:
        raise ValueError("the batch items of 'state' overlap")
    _seq.require_cuda("x", x)
    _seq.refuse_grad("causal_conv_step", state, x, weight, bias)
    y = torch.empty(nb, M, dtype=x.dtype, device=x.device)
    if nb * M == 0:
        return y
    _lib.causal_conv_step(y, state, _seq.channels_contiguous(x), _seq.dense(weight), _seq.dense(bias), activation, nb, M, W)
    _seq.mark_changed(state)
    return y
