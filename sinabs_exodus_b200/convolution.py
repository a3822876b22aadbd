"""Short causal convolution along time, one filter per channel, with an optional silu::

    y_t[m] = act(bias[m] + sum_k weight[m, k] x_{t-W+1+k}[m])

The rows in front of the first step are the ``state`` that the previous call returned (or zeros), so a sequence may come
in chunks or token by token, like the states of the neuron layers.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, _seq

__all__ = ["CausalConvTM", "causal_conv", "causal_conv_step"]


def _forward(x, weight, bias, state, lengths, activation):
    """Launches the forward pass: (y, last), and the tensors as the kernels read them."""
    nb, T, M = x.shape
    W = weight.shape[1]
    weight, bias, state = _seq.dense(weight), _seq.dense(bias), _seq.dense(state)
    y, last = x.new_empty((nb, T, M)), x.new_empty((nb, W - 1, M))
    if nb * T * M:
        _lib.causal_conv_forward(y, last, x, weight, bias, state, lengths, activation, nb, T, M, W)
    elif state is not None:      # no rows: the state passes through unchanged
        last.copy_(state)
    else:
        last.zero_()
    return y, last, (x, weight, bias, state)


class CausalConvTM(torch.autograd.Function):
    """``apply(x, weight, bias, state, lengths, activation) -> (y, last)``; see :func:`causal_conv`, which checks the
    arguments."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, activation):
        y, last, used = _forward(x, weight, bias, state, lengths, activation)
        ctx.set_materialize_grads(False)
        ctx.activation = activation
        ctx.save_for_backward(*used, lengths)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        _seq.refuse_second_order("causal_conv", dy, dlast)
        x, weight, bias, state, lengths = ctx.saved_tensors
        nb, T, M = x.shape
        W = weight.shape[1]
        dx = x.new_empty((nb, T, M))
        dweight = torch.empty_like(weight)
        dbias = torch.empty_like(bias) if bias is not None else None
        dstate = torch.empty_like(state) if state is not None else None
        dlast = _seq.dense(dlast)
        if nb * T * M == 0:
            for t in (dweight, dbias, dstate):
                if t is not None:
                    t.zero_()
            if dstate is not None and dlast is not None:
                dstate.copy_(dlast)
        else:
            if dy is None:
                dy = x.new_zeros((nb, T, M))
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
    kind, dev = weight.dtype, x.get_device()
    if dev < 0 or weight.get_device() != dev or (kind != torch.float32 and kind != x.dtype) or not _seq.alike(bias, (M,), kind, dev):
        _seq.require_like("weight", weight, (M, W), (torch.float32, x.dtype), x.device)
        _seq.require_like("bias", bias, (M,), (weight.dtype,), x.device)
    return W


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution over a whole prompt; differentiable, in reverse mode and once.

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
    if state is not None:
        _seq.require_like("state", state, (x.shape[0], W - 1, x.shape[2]), (x.dtype,), x.device)
    if lengths is not None:
        lengths = _seq.check_lengths(lengths, x.shape[0], x.shape[1], x.device)
    _seq.require_cuda("x", x)
    _seq.refuse_tangents("causal_conv", x, weight, bias, state)
    if not _seq.wants_grad(x, weight, bias, state):
        return _forward(x, weight, bias, state, lengths, activation)[:2]
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
    if state is None:
        raise TypeError("'state' must be a tensor, got None")
    if not _seq.alike(state, (nb, W - 1, M), x.dtype, x.get_device()):
        _seq.require_like("state", state, (nb, W - 1, M), (x.dtype,), x.device)
    if not state.is_contiguous():
        if nb * M and _seq.channels_contiguous(state, 2) is not state:
            raise ValueError("'state' must be contiguous in its rows and channels: it is updated in place")
        if nb > 1 and state.stride(0) < (W - 1) * M:
            raise ValueError("the batch items of 'state' overlap")
    _seq.require_cuda("x", x)
    _seq.refuse_grad("causal_conv_step", state, x, weight, bias)
    y = x.new_empty((nb, M))
    if nb * M == 0:
        return y
    _lib.causal_conv_step(y, state, x, _seq.dense(weight), _seq.dense(bias), activation, nb, M, W)
    _seq.mark_changed(state)
    return y
