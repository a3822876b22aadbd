"""Layers on the sequence operators: ``GroupNorm`` (channels last, with an activation) and ``SelectiveLeak``.

No counterpart in the reference.  ``SelectiveLeak`` keeps its states between calls like the neuron layers do
(``reset_states``, ``zero_grad`` detaches them), so ``GraphedStep`` takes it as it takes those.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import nn

from ..convolution import causal_conv, causal_conv_step
from ..normalization import group_norm
from ..selective import selective_scan, selective_step

__all__ = ["GroupNorm", "SelectiveLeak"]


class GroupNorm(nn.GroupNorm):
    """``nn.GroupNorm`` with an activation, on the channels-last kernels.

    Input ``(batch*time, channels, height, width)`` or ``(batch, time, channels, height, width)``: every map is
    normalised over its positions.  A map in ``channels_last`` memory is used where it lies, any other is brought into
    it; the output has the input's shape in ``channels_last`` memory, which the ``*Squeeze`` layers take without a copy.
    Input ``(batch, time, channels)`` or ``(tokens, channels)``: every token is normalised on its own.
    """

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: Optional[str] = None, device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine, device=device, dtype=dtype)
        if activation not in (None, "silu", "relu"):
            raise ValueError(f"'activation' must be None, 'silu' or 'relu', got {activation!r}")
        self.activation = activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        args = (self.num_groups, self.weight, self.bias, self.eps, self.activation)
        if x.ndim in (2, 3):
            self._check_channels(x.shape[-1], x)
            return group_norm(x.reshape(-1, x.shape[-1]), *args).reshape(x.shape)
        if x.ndim in (4, 5):
            self._check_channels(x.shape[-3], x)
            maps = x.reshape(math.prod(x.shape[:-3]), *x.shape[-3:]).permute(0, 2, 3, 1)      # maps may be empty: not -1
            return group_norm(maps, *args).permute(0, 3, 1, 2).reshape(x.shape)
        raise ValueError(f"GroupNorm takes 2 to 5 dimensions, got {tuple(x.shape)}")

    def _check_channels(self, found: int, x: torch.Tensor) -> None:
        if found != self.num_channels:
            raise ValueError(f"GroupNorm was made for {self.num_channels} channels, got {tuple(x.shape)}")

    def extra_repr(self) -> str:
        return super().extra_repr() + f", activation={self.activation!r}"


class SelectiveLeak(nn.Module):
    """Leaky integrator block whose decay, input weight and readout depend on the input.

    ``(batch, time, channels) -> (batch, time, channels)``: input projection to a signal and a gate, short causal
    convolution with silu, projections to step size, input weight and readout, selective scan with the gate, group norm
    per token, output projection.

    Parameters
    ----------
    channels: of input and output.
    inner_channels: of the scan; twice ``channels`` by default.
    num_states: states per inner channel.
    step_rank: rank of the step sizes' projection; ``channels / 16`` by default.
    conv_width: steps of the convolution.
    groups: of inner channels that share one input weight and readout.
    norm_groups: groups of the norm behind the scan; 0 leaves it out.
    step_min, step_max: range of the initial step sizes.

    The states (``conv_state``, ``h``) carry over from call to call until ``reset_states``; ``zero_grad`` cuts them from
    the graph.  Single tokens (one time step, no gradients) update them in place.  ``forward(x, lengths)``: see
    ``selective_scan``; the outputs of padding rows are those of a zero scan output.
    """

    def __init__(self, channels: int, inner_channels: Optional[int] = None, num_states: int = 16,
                 step_rank: Optional[int] = None, conv_width: int = 4, groups: int = 1, norm_groups: int = 1,
                 step_min: float = 0.001, step_max: float = 0.1):
        super().__init__()
        inner = 2 * channels if inner_channels is None else inner_channels
        if inner % groups:
            raise ValueError(f"'groups' ({groups}) must divide the {inner} inner channels")
        if norm_groups and inner % norm_groups:
            raise ValueError(f"'norm_groups' ({norm_groups}) must divide the {inner} inner channels")
        if not 0.0 < step_min <= step_max:
            raise ValueError("step sizes need 0 < step_min <= step_max")
        self.channels, self.inner_channels, self.num_states = channels, inner, num_states
        self.step_rank = max(1, math.ceil(channels / 16)) if step_rank is None else step_rank
        self.groups = groups
        self.in_proj = nn.Linear(channels, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, conv_width).uniform_(-1, 1) / math.sqrt(conv_width))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.x_proj = nn.Linear(inner, self.step_rank + 2 * groups * num_states, bias=False)
        self.step_proj = nn.Linear(self.step_rank, inner, bias=False)
        # softplus(step_bias) is spread evenly over the logarithm of the range
        first = torch.exp(torch.empty(inner).uniform_(math.log(step_min), math.log(step_max)))
        self.step_bias = nn.Parameter(first + torch.log(-torch.expm1(-first)))
        self.log_rate = nn.Parameter(torch.log(torch.arange(1, num_states + 1, dtype=torch.float32)).repeat(inner, 1))
        self.skip = nn.Parameter(torch.ones(inner))
        self.norm = GroupNorm(norm_groups, inner) if norm_groups else None
        self.out_proj = nn.Linear(inner, channels, bias=False)
        self.register_buffer("conv_state", None, persistent=False)
        self.register_buffer("h", None, persistent=False)

    def reset_states(self) -> None:
        """The next call starts from zero states."""
        self.conv_state = None
        self.h = None

    def zero_grad(self, set_to_none: bool = True) -> None:
        super().zero_grad(set_to_none)
        if self.h is not None:
            self.conv_state, self.h = self.conv_state.detach(), self.h.detach()

    def _check_states(self, batch: int, like: torch.Tensor) -> None:
        if self.h is not None and (self.h.shape[0] != batch or self.h.device != like.device or self.conv_state.dtype != like.dtype
                                   or self.h.dtype != torch.float32):
            raise ValueError(f"the states are those of a batch of {self.h.shape[0]} on {self.h.device}, in {self.conv_state.dtype} "
                             f"and {self.h.dtype} (here: {batch}, {like.device}, {like.dtype} and {torch.float32}); "
                             "call reset_states() before another one")

    def _projections(self, u: torch.Tensor):
        """Step size, input weight and readout from the convolved signal."""
        r, gn = self.step_rank, self.groups * self.num_states
        p = self.x_proj(u)
        shape = (*u.shape[:-1], self.groups, self.num_states)
        return self.step_proj(p[..., :r]), p[..., r:r + gn].unflatten(-1, shape[-2:]), p[..., r + gn:].unflatten(-1, shape[-2:])

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.ndim != 3 or x.shape[2] != self.channels:
            raise ValueError(f"SelectiveLeak takes (batch, time, {self.channels}), got {tuple(x.shape)}")
        signal, gate = self.in_proj(x).split(self.inner_channels, dim=-1)
        self._check_states(x.shape[0], signal)
        rate, skip, bias = -torch.exp(self.log_rate.float()), self.skip.float(), self.step_bias.float()
        weight, conv_bias = self.conv_weight, self.conv_bias
        if weight.dtype not in (torch.float32, signal.dtype):
            weight, conv_bias = weight.to(signal.dtype), conv_bias.to(signal.dtype)
        if x.shape[1] == 1 and lengths is None and not torch.is_grad_enabled():
            y = self._token(signal[:, 0], gate[:, 0], weight, conv_bias, rate, skip, bias).unsqueeze(1)
        else:
            u, conv_state = causal_conv(signal, weight, conv_bias, state=self.conv_state, lengths=lengths, activation="silu")
            step, B, C = self._projections(u)
            y, h = selective_scan(u, step, rate, B, C, D=skip, z=gate, dt_bias=bias, h0=self.h, lengths=lengths)
            self.conv_state, self.h = conv_state, h      # both or, where a call fails, neither
        if self.norm is not None:
            y = self.norm(y)
        return self.out_proj(y)

    def _token(self, signal, gate, weight, conv_bias, rate, skip, bias) -> torch.Tensor:
        if self.h is None:
            self.conv_state = signal.new_zeros(signal.shape[0], weight.shape[1] - 1, self.inner_channels)
            self.h = torch.zeros(signal.shape[0], self.inner_channels, self.num_states, device=signal.device)
        elif self.h.requires_grad or self.conv_state.requires_grad:      # a graph may still need these values
            self.conv_state, self.h = self.conv_state.detach().clone(), self.h.detach().clone()
        u = causal_conv_step(self.conv_state, signal, weight, conv_bias, activation="silu")
        step, B, C = self._projections(u)
        return selective_step(self.h, u, step, rate, B, C, D=skip, z=gate, dt_bias=bias)

    def extra_repr(self) -> str:
        return (f"channels={self.channels}, inner_channels={self.inner_channels}, num_states={self.num_states}, "
                f"groups={self.groups}, conv_width={self.conv_weight.shape[1]}")
