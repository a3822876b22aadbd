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

from . import _lib, _seq

__all__ = ["SelectiveScanTM", "selective_scan", "selective_step"]


def _forward(x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus, keep):
    """Launches the forward pass: (y, h_last, checkpoints or None), and the tensors as the kernels read them."""
    nb, T, M = x.shape
    G, N = B.shape[2:]
    A, D, dt_bias, h0 = _seq.dense(A), _seq.dense(D), _seq.dense(dt_bias), _seq.dense(h0)
    y = x.new_empty((nb, T, M))
    h_last = A.new_empty((nb, M, N))
    ckpt = None
    if nb * T * M:
        if keep:
            ckpt = _lib.selective_checkpoint(nb, T, M, N, x)
        _lib.selective_forward(y, h_last, ckpt, x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus, nb, T, M, N, G)
    elif h0 is not None:      # nothing to integrate: the state passes through unchanged
        h_last.copy_(h0)
    else:
        h_last.zero_()
    return y, h_last, ckpt, (x, dt, A, B, C, D, z, dt_bias)


class SelectiveScanTM(torch.autograd.Function):
    """``apply(x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus) -> (y, h_last)``; see :func:`selective_scan`,
    which checks the arguments."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus):
        y, h_last, ckpt, used = _forward(x, dt, A, B, C, D, z, dt_bias, h0, lengths, dt_softplus, True)
        ctx.set_materialize_grads(False)
        ctx.softplus = dt_softplus
        ctx.had_h0 = h0 is not None
        ctx.save_for_backward(*used, lengths, ckpt)
        return y, h_last

    @staticmethod
    def backward(ctx, dy, dh_last):
        _seq.refuse_second_order("selective_scan", dy, dh_last)
        x, dt, A, B, C, D, z, dt_bias, lengths, ckpt = ctx.saved_tensors
        nb, T, M = x.shape
        G, N = B.shape[2:]
        dx, ddt = x.new_empty((nb, T, M)), x.new_empty((nb, T, M))
        dz = x.new_empty((nb, T, M)) if z is not None else None
        dB, dC = x.new_empty((nb, T, G, N)), x.new_empty((nb, T, G, N))
        dA = A.new_empty((M, N))
        dD = A.new_empty((M,)) if D is not None else None
        ddt_bias = A.new_empty((M,)) if dt_bias is not None else None
        dh0 = A.new_empty((nb, M, N)) if ctx.had_h0 else None
        dh_last = _seq.dense(dh_last)
        if ckpt is None:      # an empty problem
            for t in (dx, ddt, dz, dB, dC, dA, dD, ddt_bias, dh0):
                if t is not None:
                    t.zero_()
            if dh0 is not None and dh_last is not None:
                dh0.copy_(dh_last)
        else:
            if dy is None:
                dy = x.new_zeros((nb, T, M))
            _lib.selective_backward(dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dh0, dy, dh_last, ckpt, x, dt, A, B, C, D, z, dt_bias,
                                    lengths, ctx.softplus, nb, T, M, N, G)
        return dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dh0, None, None


def _grouped(name: str, t: torch.Tensor, lead: Tuple[int, ...]) -> torch.Tensor:
    """``B`` or ``C`` with its group dimension: (..., N) is one group."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"'{name}' must be a tensor, got {type(t).__name__}")
    if t.ndim == len(lead) + 1:
        t = t.unsqueeze(-2)
    if t.ndim != len(lead) + 2 or t.shape[:-2] != lead:
        lead = tuple(lead)
        raise ValueError(f"'{name}' must have shape {lead + ('states',)} or {lead + ('groups', 'states')}, got {tuple(t.shape)}")
    return t


def _check(x, dt, A, B, C, D, z, dt_bias):
    """Checks what prompts and single tokens share; returns B and C with their group dimension."""
    _seq.require_data("x", x)
    shape, kind, dev, f = x.shape, x.dtype, x.get_device(), torch.float32
    lead, M = shape[:-1], shape[-1]
    B, C = _grouped("B", B, lead), _grouped("C", C, lead)
    grouped = B.shape
    G, N = grouped[-2], grouped[-1]
    if not 1 <= N <= _lib.SELECTIVE_MAX_STATES:
        raise ValueError(f"1 to {_lib.SELECTIVE_MAX_STATES} states per channel are supported, got {N}")
    if G < 1 or M % G:
        raise ValueError(f"the {G} groups of 'B' must divide the {M} channels")
    # the quick form of what follows
    if (dev >= 0 and dt is not None and A is not None and _seq.alike(dt, shape, kind, dev) and B.dtype == kind and B.get_device() == dev
            and _seq.alike(C, grouped, kind, dev) and _seq.alike(A, (M, N), f, dev) and _seq.alike(D, (M,), f, dev)
            and _seq.alike(z, shape, kind, dev) and _seq.alike(dt_bias, (M,), f, dev)):
        return B, C
    for name, t in (("dt", dt), ("A", A)):
        if t is None:
            raise TypeError(f"'{name}' must be a tensor, got None")
    same, f32 = (kind,), (f,)
    _seq.require_like("dt", dt, shape, same, x.device)
    _seq.require_like("z", z, shape, same, x.device)
    _seq.require_like("B", B, grouped, same, x.device)
    _seq.require_like("C", C, grouped, same, x.device)
    _seq.require_like("A", A, (M, N), f32, x.device)
    _seq.require_like("D", D, (M,), f32, x.device)
    _seq.require_like("dt_bias", dt_bias, (M,), f32, x.device)
    return B, C


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   h0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   dt_softplus: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective scan over a whole prompt; differentiable, in reverse mode and once.

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
    if h0 is not None:
        _seq.require_like("h0", h0, (x.shape[0], x.shape[2], B.shape[3]), (torch.float32,), x.device)
    if lengths is not None:
        lengths = _seq.check_lengths(lengths, x.shape[0], x.shape[1], x.device)
    _seq.require_cuda("x", x)
    _seq.refuse_tangents("selective_scan", x, dt, A, B, C, D, z, dt_bias, h0)
    if _seq.wants_grad(x, dt, A, B, C, D, z, dt_bias, h0):
        return SelectiveScanTM.apply(x, dt, A, B, C, D, z, dt_bias, h0, lengths, bool(dt_softplus))
    return _forward(x, dt, A, B, C, D, z, dt_bias, h0, lengths, bool(dt_softplus), False)[:2]


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
    if h is None:
        raise TypeError("'h' must be a tensor, got None")
    if not _seq.alike(h, (nb, M, N), torch.float32, x.get_device()):
        _seq.require_like("h", h, (nb, M, N), (torch.float32,), x.device)
    if not h.is_contiguous():
        if nb * M and _seq.channels_contiguous(h, 2) is not h:
            raise ValueError("'h' must be contiguous in its channels and states: it is updated in place")
        if nb > 1 and h.stride(0) < M * N:
            raise ValueError("the batch items of 'h' overlap")
    _seq.require_cuda("x", x)
    _seq.refuse_grad("selective_step", h, x, dt, A, B, C, D, z, dt_bias)
    y = x.new_empty((nb, M))
    if nb * M == 0:
        return y
    _lib.selective_step(y, h, x, dt, _seq.dense(A), B, C, _seq.dense(D), z, _seq.dense(dt_bias), bool(dt_softplus), nb, M, N, G)
    _seq.mark_changed(h)
    return y
