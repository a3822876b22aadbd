"""Selective scan: a leaky integrator whose decay, input weight and readout depend on the input.

``LeakyIntegratorTM`` has one state per channel and a decay that is fixed in time.  Here every channel has ``N`` states
with rates ``A``, the step size ``dt`` comes with the input, and ``B`` / ``C`` weigh what goes into and what is read from
the states::

    s_t = softplus(dt_t + dt_bias)
    h_t[m, n] = exp(s_t[m] A[m, n]) h_{t-1}[m, n] + s_t[m] x_t[m] B_t[g, n]
    y_t[m] = (sum_n C_t[g, n] h_t[m, n] + D[m] x_t[m]) * silu(z_t[m])

The layout is the layers' time-major ``(batch, time, channels)``.  Tensors whose channels are contiguous are used where
they lie, so slices of one projection need no copies.  States, parameters and all sums are float32.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, _seq

__all__ = ["SelectiveScanTM", "selective_scan", "selective_step"]


class SelectiveScanTM(torch.autograd.Function):
    """``apply(x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus) -> (y, h_last)``; see :func:`selective_scan`,
    which checks the arguments."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus):
        nb, T, M = x.shape
        G, N = B.shape[2], B.shape[3]
        x, dt, z = (_seq.channels_contiguous(t) for t in (x, dt, z))
        B, C = (_seq.channels_contiguous(t, 2) for t in (B, C))
        A, D, dt_bias, h0 = (_seq.dense(t) for t in (A, D, dt_bias, h0))
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        ctx.set_materialize_grads(False)
        ctx.sizes = (nb, T, M, N, G)
        ctx.softplus = dt_softplus
        ctx.had_h0 = h0 is not None
        if nb * T * M == 0:      # nothing to integrate: the state passes through unchanged
            h_last = h0.clone() if h0 is not None else torch.zeros(nb, M, N, dtype=torch.float32, device=x.device)
            ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, lengths, None)
            return y, h_last
        h_last = torch.empty(nb, M, N, dtype=torch.float32, device=x.device)
        ckpt = _lib.selective_checkpoint(nb, T, M, N, x.device) if any(ctx.needs_input_grad) else None
        _lib.selective_forward(y, h_last, ckpt, x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus, nb, T, M, N, G)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, lengths, ckpt)
        return y, h_last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh_last):
        x, dt, A, B, C, D, z, dt_bias, lengths, ckpt = ctx.saved_tensors
        nb, T, M, N, G = ctx.sizes
        dev = x.device
        new = torch.zeros if ckpt is None else torch.empty
        f32 = dict(dtype=torch.float32, device=dev)
        dx, ddt = (new(nb, T, M, dtype=x.dtype, device=dev) for _ in range(2))
        dz = new(nb, T, M, dtype=x.dtype, device=dev) if z is not None else None
        dB, dC = (new(nb, T, G, N, dtype=x.dtype, device=dev) for _ in range(2))
        dA = new(M, N, **f32)
        dD = new(M, **f32) if D is not None else None
        ddt_bias = new(M, **f32) if dt_bias is not None else None
        dh0 = new(nb, M, N, **f32) if ctx.had_h0 else None
        dh_last = _seq.dense(dh_last)
        if ckpt is None:
            if dh0 is not None and dh_last is not None:
                dh0.copy_(dh_last)
        else:
            dy = torch.zeros(nb, T, M, dtype=x.dtype, device=dev) if dy is None else _seq.channels_contiguous(dy)
            _lib.selective_backward(dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dh0, dy, dh_last, ckpt, x, dt, A, B, C, D, z, dt_bias,
                                    lengths, ctx.softplus, nb, T, M, N, G)
        return dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dh0, None, None


def _grouped(name: str, t: torch.Tensor, lead: Tuple[int, ...]) -> torch.Tensor:
    """``B`` or ``C`` with its group dimension: (..., N) is one group."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"'{name}' must be a tensor, got {type(t).__name__}")
    if t.ndim == len(lead) + 1:
        t = t.unsqueeze(-2)
    if t.ndim != len(lead) + 2 or tuple(t.shape[:-2]) != lead:
        raise ValueError(f"'{name}' must have shape {lead + ('states',)} or {lead + ('groups', 'states')}, got {tuple(t.shape)}")
    return t


def _check(x, dt, A, B, C, D, z, dt_bias):
    """Checks what prompts and single tokens share; returns B and C with their group dimension."""
    _seq.require_data("x", x)
    lead, M = tuple(x.shape[:-1]), x.shape[-1]
    B, C = _grouped("B", B, lead), _grouped("C", C, lead)
    G, N = B.shape[-2], B.shape[-1]
    if not 1 <= N <= _lib.SELECTIVE_MAX_STATES:
        raise ValueError(f"1 to {_lib.SELECTIVE_MAX_STATES} states per channel are supported, got {N}")
    if G < 1 or M % G:
        raise ValueError(f"the {G} groups of 'B' must divide the {M} channels")
    same, f32 = (x.dtype,), (torch.float32,)
    _seq.require_like("dt", dt, x.shape, same, x.device)
    _seq.require_like("z", z, x.shape, same, x.device)
    _seq.require_like("B", B, lead + (G, N), same, x.device)
    _seq.require_like("C", C, lead + (G, N), same, x.device)
    _seq.require_like("A", A, (M, N), f32, x.device)
    _seq.require_like("D", D, (M,), f32, x.device)
    _seq.require_like("dt_bias", dt_bias, (M,), f32, x.device)
    return B, C


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   h0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   dt_softplus: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective scan over a whole prompt; differentiable.

    Parameters
    ----------
    x, dt: (batch, time, channels), float32, bfloat16 or float16 (all data tensors of one type).
    A: (channels, states) float32 rates, negative for states that decay.
    B, C: (batch, time, states), or (batch, time, groups, states) with the channels split evenly over the groups.
    D: (channels,) float32 weight of the input in the output.
    z: (batch, time, channels) gate: the output is multiplied by ``silu(z)``.
    dt_bias: (channels,) float32, added to ``dt``.
    h0: (batch, channels, states) float32 state in front of the first step (zeros if absent).
    lengths: (batch,) int32 or int64 numbers of valid steps of a padded batch.  Rows behind them do not enter anything,
        whatever they hold; their outputs and gradients are 0, and ``h_last`` is the state after the last valid row.
    dt_softplus: pass ``dt + dt_bias`` through softplus.

    Returns
    -------
    ``(y, h_last)``: the output, of the type of ``x``, and the float32 state after the last step, both with gradients.
    """
    if isinstance(x, torch.Tensor) and x.ndim != 3:
        raise ValueError("'x' must be 3D, (batch, time, channels)")
    B, C = _check(x, dt, A, B, C, D, z, dt_bias)
    _seq.require_like("h0", h0, (x.shape[0], x.shape[2], B.shape[3]), (torch.float32,), x.device)
    lengths = _seq.check_lengths(lengths, x.shape[0], x.device)
    _seq.require_cuda("x", x)
    return SelectiveScanTM.apply(x, dt, A, B, C, D, z, dt_bias, h0, lengths, bool(dt_softplus))


def selective_step(h: torch.Tensor, x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   dt_softplus: bool = True) -> torch.Tensor:
    """One step of :func:`selective_scan` for single tokens: updates the state ``h`` (batch, channels, states) in place
    and returns the output (batch, channels).  Arguments as there, without the time dimension.  Not differentiable.

    ``h`` is float32 with contiguous (channels, states); its batch items may lie apart (rows of a pool).
    """
    if isinstance(x, torch.Tensor) and x.ndim != 2:
        raise ValueError("'x' must be 2D, (batch, channels)")
    B, C = _check(x, dt, A, B, C, D, z, dt_bias)
    nb, M = x.shape
    G, N = B.shape[1], B.shape[2]
    _seq.require_like("h", h, (nb, M, N), (torch.float32,), x.device)
    if nb * M and _seq.channels_contiguous(h, 2) is not h:
        raise ValueError("'h' must be contiguous in its channels and states: it is updated in place")
    if nb > 1 and h.stride(0) < M * N:
        raise ValueError("the batch items of 'h' overlap")
    _seq.require_cuda("x", x)
    _seq.refuse_grad("selective_step", h, x, dt, A, B, C, D, z, dt_bias)
    y = torch.empty(nb, M, dtype=x.dtype, device=x.device)
    if nb * M == 0:
        return y
    _lib.selective_step(y, h, _seq.channels_contiguous(x), _seq.channels_contiguous(dt), _seq.dense(A), _seq.channels_contiguous(B, 2),
                        _seq.channels_contiguous(C, 2), _seq.dense(D), _seq.channels_contiguous(z), _seq.dense(dt_bias),
                        bool(dt_softplus), nb, M, N, G)
    _seq.mark_changed(h)
    return y
