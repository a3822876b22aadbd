"""Sequence operators at the edges of what their arguments may be.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref
from tests.test_gpu_selective import DEV, F32, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nb,M,N", [(3, 24, 5), (20, 4096, 16)])      # one batch item per thread, and several
def test_infinite_rates_in_a_step(nb, M, N):
    """A rate of minus infinity forgets everything in a step of any size, and nothing in a step of size 0, as in the scan."""
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(1, nb, 1, M, N, 1, F32, bias=False, softplus=False)
    p["A"][::2] = float("-inf")
    p["dt"][:, :, ::4] = 0.0
    h = p["h0"].clone()
    y = ex.selective_step(h, A=p["A"], D=p["D"], dt_softplus=False, **{k: p[k][:, 0] for k in ("x", "dt", "B", "C", "z")})
    whole, last = ex.selective_scan(**p)
    assert torch.equal(h[:, ::4], p["h0"][:, ::4]) and torch.equal(last[:, ::4], p["h0"][:, ::4])
    x, dt, B, C, z = (p[k][:, 0].double() for k in ("x", "dt", "B", "C", "z"))
    A = torch.where(torch.isinf(p["A"]), torch.zeros_like(p["A"]), p["A"]).double()
    keep = torch.where((torch.isinf(p["A"]) & (dt[..., None] > 0)), torch.zeros_like(A), torch.exp(dt[..., None] * A))
    want = keep * p["h0"].double() + (dt * x)[..., None] * B
    raw, gate = (want * C).sum(-1) + p["D"].double() * x, ref.silu(z)
    # a handful of roundings of each term, the exponent's at most 20 of them
    size = keep * p["h0"].double().abs() + (dt * x).abs()[..., None] * B.abs()
    ref.assert_close(h, want, 30 * 2.0 ** -24 * size, F32, "h")
    ref.assert_close(y, raw * gate, 40 * 2.0 ** -24 * ((size * C.abs()).sum(-1) + (p["D"].double() * x).abs()) * (gate.abs() + 0.1), F32, "y")
    torch.testing.assert_close(h, last, rtol=1e-6, atol=1e-6)


def test_backward_twice():
    """A kept graph gives the same gradients again: nothing that it saved is used up."""
    import sinabs_exodus_b200 as ex
    g = torch.Generator(device=DEV).manual_seed(2)

    def leaf(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).requires_grad_(True)

    scan = dict(x=leaf(2, 300, 24), dt=leaf(2, 300, 24), A=(-torch.rand(24, 8, generator=g, device=DEV)).requires_grad_(True), B=leaf(2, 300, 1, 8),
                C=leaf(2, 300, 1, 8), h0=leaf(2, 24, 8))
    conv = dict(x=leaf(2, 70, 24), weight=leaf(24, 4), bias=leaf(24), state=leaf(2, 3, 24))
    norm = dict(x=leaf(3, 50, 24), weight=leaf(24), bias=leaf(24))
    for y, t in ((ex.selective_scan(**scan)[0], scan), (ex.causal_conv(**conv, activation="silu")[0], conv),
                 (ex.group_norm(num_groups=4, activation="silu", **norm), norm)):
        up = torch.randn(y.shape, generator=g, device=DEV)
        first = torch.autograd.grad(y, list(t.values()), up, retain_graph=True)
        for a, b in zip(first, torch.autograd.grad(y, list(t.values()), up)):
            assert torch.equal(a, b)


def test_prompts_and_tokens_in_and_out_of_inference_mode():
    import sinabs_exodus_b200 as ex
    torch.manual_seed(0)
    layer = ex.layers.SelectiveLeak(24, num_states=8).to(DEV)
    x = torch.randn(2, 9, 24, device=DEV)
    with torch.no_grad():
        want = torch.cat([layer(x[:, :6])] + [layer(x[:, t:t + 1]) for t in range(6, 9)], 1)
    for modes in ((torch.no_grad, torch.inference_mode), (torch.inference_mode, torch.no_grad)):
        layer.reset_states()
        parts = []
        with modes[0]():
            parts.append(layer(x[:, :6]))
        for t in range(6, 9):
            with modes[t % 2]():
                parts.append(layer(x[:, t:t + 1]))
        assert torch.equal(torch.cat(parts, 1), want)


def test_truncated_training_in_a_graph():
    """``GraphedStep`` with carried states, trained: chunk after chunk, as eager steps with ``zero_grad`` between them."""
    import sinabs_exodus_b200 as ex
    torch.manual_seed(0)
    layer = ex.layers.SelectiveLeak(24, num_states=8, norm_groups=2).to(DEV)
    x, g = torch.randn(4, 2, 40, 24, device=DEV), torch.randn(4, 2, 40, 24, device=DEV)
    want = []
    for c in range(4):
        layer.zero_grad()
        y = layer(x[c])
        y.backward(g[c])
        want.append((y.detach(), {k: p.grad.clone() for k, p in layer.named_parameters()}))
    del y
    layer.reset_states()
    step = ex.GraphedStep(layer, x[0], g[0], carry_state=True)
    for name in ("h", "conv_state"):
        getattr(layer, name).zero_()
    for c in range(4):
        out = step(x[c], g[c])
        torch.testing.assert_close(out, want[c][0], rtol=1e-5, atol=1e-6)
        for k, p in layer.named_parameters():
            torch.testing.assert_close(p.grad, want[c][1][k], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("kind", [F32, torch.bfloat16])
@pytest.mark.parametrize("M", [8, 7])      # packs of channels, and single ones
def test_an_infinity_reaches_only_the_taps_that_meet_it(kind, M):
    """The last row meets the current tap alone: the gradients of the others stay finite, and the infinite one is not NaN.  One in
    the middle, next to the end of a thread's run, meets all of them."""
    import sinabs_exodus_b200 as ex
    x = torch.ones(2, 70, M, device=DEV).to(kind)
    x[0, 69, 2] = x[1, 15, 3] = x[1, 16, 4] = float("inf")
    w = torch.ones(M, 4, device=DEV, requires_grad=True)
    y, _ = ex.causal_conv(x, w, lengths=torch.tensor([70, 60], device=DEV))
    dw, = torch.autograd.grad(y, w, torch.ones_like(y))
    want = torch.tensor([67.0 + 57, 68 + 58, 69 + 59, 70 + 60], device=DEV).repeat(M, 1)      # rows that each tap meets
    want[2, 3] = want[3] = want[4] = float("inf")
    assert torch.equal(dw, want)


def test_no_graph_of_the_warm_up_lives_while_a_step_is_captured(monkeypatch):
    """The leaves' accumulators of an older graph belong to another stream than the one that captures."""
    import weakref

    import sinabs_exodus_b200 as ex
    torch.manual_seed(0)
    layer = ex.layers.SelectiveLeak(24, num_states=8).to(DEV)
    states, alive = [], []
    layer.register_forward_hook(lambda module, args, out: states.extend(weakref.ref(t) for t in (module.h, module.conv_state)))
    capture = torch.cuda.graph

    def watched(graph):
        alive.append(sum(r() is not None for r in states))
        return capture(graph)

    monkeypatch.setattr(torch.cuda, "graph", watched)
    x, g = torch.randn(2, 40, 24, device=DEV), torch.randn(2, 40, 24, device=DEV)
    ex.GraphedStep(layer, x, g, carry_state=True)
    assert alive == [0] and len(states) == 8
