"""Argument checks shared by the sequence operators (``selective``, ``convolution``, ``normalization``)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib


def require_data(name: str, x: torch.Tensor) -> None:
    """The main input of an operator: a tensor of a type that the kernels take."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"'{name}' must be a tensor, got {type(x).__name__}")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"'{name}' must be float32, bfloat16 or float16, got {x.dtype}")


def require_cuda(name: str, x: torch.Tensor) -> None:
    """Comes last: shapes and types are checked wherever the tensors are."""
    if not x.is_cuda:
        raise _lib.ExodusLibraryError(
            f"exodus_b200 kernels only run on CUDA tensors; '{name}' is on {x.device}. There is no CPU implementation in this package.")


def require_like(name: str, t: Optional[torch.Tensor], shape: Tuple[int, ...], dtypes: Tuple[torch.dtype, ...],
                 device: torch.device) -> None:
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"'{name}' must be a tensor, got {type(t).__name__}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"'{name}' must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"'{name}' must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    if t.device != device:
        raise _lib.ExodusLibraryError(f"tensors on different devices: {device} and {t.device} ('{name}')")


def alike(t: Optional[torch.Tensor], shape, dtype: torch.dtype, device: int) -> bool:
    """Whether ``t`` is absent or what it should be: the quick form of :func:`require_like`, which says what is wrong."""
    return t is None or (type(t) in _TENSORS and t.shape == shape and t.dtype == dtype and t.get_device() == device)


_TENSORS = (torch.Tensor, torch.nn.Parameter)


def check_lengths(lengths: torch.Tensor, batch: int, steps: int, device: torch.device) -> torch.Tensor:
    """``lengths`` as the kernels take them; 64-bit values are clamped before they lose their upper half."""
    require_like("lengths", lengths, (batch,), (torch.int32, torch.int64), device)
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, steps).to(torch.int32)
    return lengths.contiguous()


def channels_contiguous(t: Optional[torch.Tensor], trailing: int = 1) -> Optional[torch.Tensor]:
    """``t`` with its last ``trailing`` dimensions contiguous: itself where they are, else a copy."""
    if t is None:
        return None
    step = 1
    shape, stride = t.shape, t.stride()
    for d in range(len(shape) - 1, len(shape) - 1 - trailing, -1):
        if shape[d] > 1 and stride[d] != step:
            return t.contiguous()
        step *= shape[d]
    return t


def dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd has to record a call on these tensors."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether forward-mode differentiation follows one of these tensors (which says nothing in ``requires_grad``)."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # no dual_level() around this call: quicker than asking every tensor
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def refuse_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The kernels know nothing of tangents: a call would drop them, which stands for a derivative of zero."""
    if has_tangent(*tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative (torch.autograd.forward_ad)")


def refuse_grad(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The in-place single-token forms are not differentiable."""
    if wants_grad(*tensors):
        raise RuntimeError(f"{what} updates its state in place and is not differentiable: call it under torch.no_grad()")
    refuse_tangents(what, *tensors)


def refuse_second_order(what: str, *upstream: Optional[torch.Tensor]) -> None:
    """Called in a backward pass, where autograd only records with ``create_graph=True``, and where gradients from above
    have tangents in forward-over-reverse differentiation."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} is differentiable once: its backward pass cannot be recorded (create_graph=True)")
    refuse_tangents(f"the backward pass of {what}", *upstream)


def mark_changed(t: torch.Tensor) -> None:
    """Tells autograd that a kernel wrote to ``t``."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)
