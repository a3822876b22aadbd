"""The sequence operators' host side where autograd or a layer's states could go wrong unseen (no GPU needed)."""
import ctypes
import os

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


@pytest.fixture(scope="module")
def library():
    from sinabs_exodus_b200 import build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


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


def test_empty_problems_write_nothing(library):
    """What the header says of sizes of zero: success, and no output is touched (none of these addresses exists)."""
    lib, p, r, null = library, ctypes.c_void_p(64), ctypes.byref(_lib.Rows(64, 64, 16)), None
    for B, T, M in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        assert lib.exb_selective_forward(p, p, p, r, r, p, r, r, p, r, p, p, p, 1, p, 0, 0, B, T, M, 4, 1, 0, null) == 0
        assert lib.exb_selective_backward(p, p, p, p, p, p, p, p, p, r, p, p, r, r, p, r, r, p, r, p, p, 1, p, 0, 0, B, T, M, 4, 1, 0, null) == 0
        assert lib.exb_causal_conv_forward(p, p, r, p, p, p, p, 0, 1, 0, B, T, M, 4, 0, null) == 0
        assert lib.exb_causal_conv_backward(p, p, p, p, r, p, r, p, p, p, p, 0, 1, p, 0, 0, B, T, M, 4, 0, null) == 0
        assert lib.exb_group_norm_forward(p, p, p, r, p, p, 1e-5, 0, 1, p, 0, 0, B, T, M, 1, 0, null) == 0
        assert lib.exb_group_norm_backward(p, p, p, r, r, p, p, p, p, 0, 1, p, 0, 0, B, T, M, 1, 0, null) == 0
        if T:
            assert lib.exb_selective_step(p, p, 32, r, r, p, r, r, p, r, p, 1, 0, B, M, 4, 1, 0, null) == 0
            assert lib.exb_causal_conv_step(p, p, 24, r, p, p, 0, 1, 0, B, M, 4, 0, null) == 0


@pytest.mark.parametrize("nb,T,M", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_the_package_fills_the_outputs_of_empty_problems(launched, nb, T, M):
    G, N, W = 1, 4, 4

    def leaf(*shape):
        return torch.randn(*shape).requires_grad_(True)

    t = dict(x=leaf(nb, T, M), dt=leaf(nb, T, M), A=leaf(M, N), B=leaf(nb, T, G, N), C=leaf(nb, T, G, N), D=leaf(M), h0=leaf(nb, M, N))
    y, h = ex.selective_scan(**t)
    up = torch.randn(nb, M, N)
    g = dict(zip(t, torch.autograd.grad([y, h], list(t.values()), [torch.randn(nb, T, M), up])))
    assert torch.equal(h, t["h0"]) and torch.equal(g["h0"], up) and all((g[k] == 0).all() for k in g if k != "h0")
    t = dict(x=leaf(nb, T, M), weight=leaf(M, W), bias=leaf(M), state=leaf(nb, W - 1, M))
    y, last = ex.causal_conv(**t)
    up = torch.randn(nb, W - 1, M)
    g = dict(zip(t, torch.autograd.grad([y, last], list(t.values()), [torch.randn(nb, T, M), up])))
    assert torch.equal(last, t["state"]) and torch.equal(g["state"], up) and all((g[k] == 0).all() for k in g if k != "state")
    t = dict(x=leaf(nb, T, M), weight=leaf(M), bias=leaf(M))
    g = torch.autograd.grad(ex.group_norm(num_groups=1, **t), list(t.values()), torch.randn(nb, T, M))
    assert all((v == 0).all() for v in g)
    assert not launched


def test_states_of_another_type_are_refused_before_anything_changes(launched):
    """``half()`` also converts the states that a layer holds; the scan's are float32."""
    layer = ex.layers.SelectiveLeak(8, num_states=4)
    x = torch.randn(2, 3, 8)
    with torch.no_grad():
        layer(x)
        layer.half()
        before = layer.conv_state, layer.h
        for steps in (3, 1):
            with pytest.raises(ValueError, match="reset_states"):
                layer(x[:, :steps].half())
            assert layer.conv_state is before[0] and layer.h is before[1]
        layer.reset_states()
        layer(x.half())
        assert layer.h.dtype == torch.float32 and layer.conv_state.dtype == torch.float16


def test_a_call_that_fails_leaves_both_states(launched, monkeypatch):
    layer = ex.layers.SelectiveLeak(8, num_states=4)
    x = torch.randn(2, 3, 8)
    with torch.no_grad():
        layer(x)
        before = layer.conv_state, layer.h

        def out_of_memory(*a):
            raise torch.cuda.OutOfMemoryError("no room")

        monkeypatch.setattr(_lib, "selective_forward", out_of_memory)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            layer(x)
    assert layer.conv_state is before[0] and layer.h is before[1]


@pytest.mark.parametrize("shape", [(2, 8, 0, 4), (2, 8, 3, 0), (0, 8, 3, 4), (2, 0, 8, 3, 4), (2, 3, 8, 0, 4), (2, 0, 8), (0, 8)])
@pytest.mark.parametrize("channels_last", [False, True])
def test_norm_layer_on_empty_maps(launched, shape, channels_last):
    layer = ex.layers.GroupNorm(2, 8)
    x = torch.zeros(shape)
    if channels_last and len(shape) == 4:
        x = x.to(memory_format=torch.channels_last)
    x.requires_grad_(True)
    y = layer(x)
    assert y.shape == shape and y.dtype == x.dtype
    y.sum().backward()
    assert x.grad.shape == shape and (layer.weight.grad == 0).all()
    assert not launched


@pytest.mark.parametrize("name", list(CALLS))
def test_function_transforms_are_refused(monkeypatch, name):
    """``torch.func`` hands in tensors without memory of their own."""
    monkeypatch.setattr(_seq, "require_cuda", lambda name, x: None)
    call, shapes = CALLS[name]
    t = {k: torch.zeros(*s) for k, s in shapes.items()}
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: call(dict(t, x=x)))(torch.zeros(3, *shapes["x"]))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.grad(lambda x: call(dict(t, x=x)).sum())(t["x"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: call(dict(t, x=x)), (t["x"],), (t["x"],))
