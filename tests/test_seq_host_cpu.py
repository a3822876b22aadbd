"""The sequence operators' host side where autograd or a layer's states could go wrong unseen (no GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

import sinabs_exodus_b200 as ex
from sinabs_exodus_b200 import _lib, _seq


@pytest.fixture
def launched(monkeypatch):
    """Lets CPU tensors through to the launching calls, which are noted and leave their outputs as they are."""
    calls = []
    monkeypatch.setattr(_seq, "require_cuda", lambda name, x: None)
    for name in ("selective_forward", "selective_backward", "selective_step", "causal_conv_forward", "causal_conv_backward",
                 "causal_conv_step", "group_norm_forward", "group_norm_backward"):
        monkeypatch.setattr(_lib, name, lambda *a, _n=name: calls.append(_n))
    monkeypatch.setattr(_lib, "selective_checkpoint", lambda *a: torch.zeros(1))
    return calls


SCAN = dict(x=(2, 5, 8), dt=(2, 5, 8), A=(8, 4), B=(2, 5, 2, 4), C=(2, 5, 2, 4), D=(8,), z=(2, 5, 8), dt_bias=(8,), h0=(2, 8, 4))
STEP = {**{k: (v[0],) + v[2:] if len(v) > 2 else v for k, v in SCAN.items() if k != "h0"}, "h": (2, 8, 4)}
CALLS = {
    "selective_scan": (lambda t: ex.selective_scan(**t)[0], SCAN),
    "selective_step": (lambda t: ex.selective_step(**t), STEP),
    "causal_conv": (lambda t: ex.causal_conv(**t)[0], dict(x=(2, 5, 8), weight=(8, 4), bias=(8,), state=(2, 3, 8))),
    "causal_conv_step": (lambda t: ex.causal_conv_step(**t), dict(state=(2, 3, 8), x=(2, 8), weight=(8, 4), bias=(8,))),
    "group_norm": (lambda t: ex.group_norm(num_groups=2, **t), dict(x=(2, 3, 8), weight=(8,), bias=(8,))),
}


@pytest.mark.parametrize("name,leaf", [(n, k) for n, (_, shapes) in CALLS.items() for k in shapes])
def test_forward_mode_is_refused_and_not_dropped(launched, name, leaf):
    call, shapes = CALLS[name]
    t = {k: torch.zeros(*s) for k, s in shapes.items()}
    with forward_ad.dual_level():
        with torch.no_grad():
            call(t)                 # a level without a dual tensor among the arguments is none of the call's business
        launched.clear()
        t[leaf] = forward_ad.make_dual(t[leaf], torch.ones(*shapes[leaf]))
        for graph in (False, True):
            with torch.set_grad_enabled(graph), pytest.raises(NotImplementedError, match=f"{name} has no forward-mode"):
                call(t)
    assert not launched             # nothing ran, so no state was changed either


@pytest.mark.parametrize("name", ["selective_scan", "causal_conv", "group_norm"])
def test_tangents_from_above_are_refused_in_the_backward_pass(launched, name):
    call, shapes = CALLS[name]
    t = {k: torch.zeros(*s, requires_grad=True) for k, s in shapes.items()}
    y = call(t)
    with forward_ad.dual_level():
        up = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match=f"backward pass of {name}"):
            torch.autograd.grad(y, t["x"], up)


def test_reverse_mode_under_a_dual_level_runs(launched):
    t = {k: torch.zeros(*s, requires_grad=True) for k, s in SCAN.items()}
    with forward_ad.dual_level():
        y, _ = ex.selective_scan(**t)
        torch.autograd.grad(y, t["x"], torch.ones_like(y))
    assert launched == ["selective_forward", "selective_backward"]
