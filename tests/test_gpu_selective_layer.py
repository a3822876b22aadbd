"""The sequence operators together, as ``layers.SelectiveLeak`` calls them.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(channels=24, **kw):
    import sinabs_exodus_b200 as ex
    torch.manual_seed(0)
    return ex.layers.SelectiveLeak(channels, num_states=8, step_rank=4, **kw).to(DEV)


def plain(layer, x):
    """The layer in float64, in plain operations."""
    p = {k: v.detach().double().requires_grad_(True) for k, v in layer.named_parameters()}
    x = x.detach().double().requires_grad_(True)
    inner, G, N, r = layer.inner_channels, layer.groups, layer.num_states, layer.step_rank
    signal, gate = (x @ p["in_proj.weight"].t()).split(inner, -1)
    u, _ = ref.conv(signal, p["conv_weight"], p["conv_bias"], activation="silu")
    q = u @ p["x_proj.weight"].t()
    s = torch.nn.functional.softplus(q[..., :r] @ p["step_proj.weight"].t() + p["step_bias"])
    B = q[..., r:r + G * N].unflatten(-1, (G, N)).repeat_interleave(inner // G, 2)
    C = q[..., r + G * N:].unflatten(-1, (G, N)).repeat_interleave(inner // G, 2)
    A = -torch.exp(p["log_rate"])
    h, ys = torch.zeros(x.shape[0], inner, N, device=DEV, dtype=torch.float64), []
    for t in range(x.shape[1]):
        h = torch.exp(s[:, t, :, None] * A) * h + (s[:, t] * u[:, t])[..., None] * B[:, t]
        ys.append((h * C[:, t]).sum(-1) + p["skip"] * u[:, t])
    y = torch.stack(ys, 1) * ref.silu(gate)
    if layer.norm is not None:
        y = ref.norm(y.reshape(-1, 1, inner), layer.norm.num_groups, p["norm.weight"], p["norm.bias"], layer.norm.eps).view(y.shape)
    return y @ p["out_proj.weight"].t(), x, p


@pytest.mark.parametrize("kw", [{}, dict(groups=2, norm_groups=4), dict(norm_groups=0, inner_channels=40, conv_width=3)])
def test_layer_is_its_definition(kw):
    layer = make(**kw)
    x = torch.randn(3, 70, 24, device=DEV, requires_grad=True)
    up = torch.randn(3, 70, 24, device=DEV)
    y = layer(x)
    y.backward(up)
    want, xr, p = plain(layer, x)
    grads = torch.autograd.grad(want, [xr] + list(p.values()), up.double())
    # the chain is some hundred roundings deep; norms of the difference against 1e-4 of the value's leave a factor of
    # ten over 2^-24 * 200
    def near(a, b, name):
        assert float((a.double() - b).norm()) <= 1e-4 * float(b.norm()) + 1e-9, name
    near(y, want, "output")
    near(x.grad, grads[0], "input")
    for (k, v), g in zip(layer.named_parameters(), grads[1:]):
        near(v.grad, g, k)


def test_prompt_then_tokens_is_the_whole_sequence():
    layer = make(groups=2, norm_groups=3)
    x = torch.randn(2, 20, 24, device=DEV)
    with torch.no_grad():
        whole = layer(x)
        layer.reset_states()
        assert layer.h is None
        parts = [layer(x[:, :11])] + [layer(x[:, t:t + 1]) for t in range(11, 16)] + [layer(x[:, 16:])]
        got = torch.cat(parts, 1)
        layer.reset_states()
        tokens = torch.cat([layer(x[:, t:t + 1]) for t in range(20)], 1)
    assert float((got - whole).abs().max()) <= 1e-4 * float(whole.abs().max())
    assert float((tokens - whole).abs().max()) <= 1e-4 * float(whole.abs().max())


def test_tokens_leave_a_graph_alone():
    """States that a graph still needs are not overwritten by the in-place form."""
    layer = make()
    x = torch.randn(2, 6, 24, device=DEV)
    y = layer(x)
    z = layer(x)          # uses the states of the first call
    with torch.no_grad():
        layer(x[:, :1])
    a = torch.autograd.grad((y.sum() + z.sum()), layer.conv_weight)[0]
    layer.reset_states()
    b = torch.autograd.grad((layer(x).sum() + layer(x).sum()), layer.conv_weight)[0]
    assert torch.equal(a, b)
    layer.zero_grad()
    assert not layer.h.requires_grad


def test_padded_batch_of_prompts():
    layer = make()
    x = torch.randn(3, 30, 24, device=DEV)
    n = torch.tensor([30, 7, 0], device=DEV)
    with torch.no_grad():
        y = layer(x, lengths=n)
        h, c = layer.h.clone(), layer.conv_state.clone()
        layer.reset_states()
        alone = layer(x[1:2, :7].contiguous())
    assert float((y[1, :7] - alone[0]).abs().max()) <= 1e-5 * float(alone.abs().max())
    assert torch.allclose(h[1], layer.h[0], rtol=1e-5, atol=1e-6) and torch.allclose(c[1], layer.conv_state[0], rtol=1e-5, atol=1e-6)
    assert (h[2] == 0).all() and (c[2] == 0).all()


def test_bfloat16_layer_runs():
    layer = make().to(torch.bfloat16)
    x = torch.randn(2, 40, 24, device=DEV).to(torch.bfloat16)
    layer(x).float().sum().backward()
    assert all(torch.isfinite(p.grad.float()).all() for p in layer.parameters())
    with torch.no_grad():
        layer.reset_states()
        layer(x[:, :1])


def test_states_of_another_batch_are_refused():
    layer = make()
    with torch.no_grad():
        layer(torch.randn(2, 4, 24, device=DEV))
        with pytest.raises(ValueError, match="reset_states"):
            layer(torch.randn(3, 4, 24, device=DEV))


def test_in_a_network_with_spiking_layers_and_graphs():
    """Next to the neuron layers, trained and streamed through ``GraphedStep``."""
    import sinabs_exodus_b200 as ex
    net = torch.nn.Sequential(make(), ex.layers.LIF(tau_mem=10.0, norm_input=False), torch.nn.Linear(24, 4)).to(DEV)
    x, g = torch.randn(2, 50, 24, device=DEV), torch.randn(2, 50, 4, device=DEV)
    step = ex.GraphedStep(net, x, g, input_grad=True)
    out = step(x, g).clone()
    got = {k: p.grad.clone() for k, p in net.named_parameters()}
    for m in net.modules():
        if hasattr(m, "reset_states"):
            m.reset_states()
    net.zero_grad()
    want = net(x)
    want.backward(g)
    assert torch.equal(out, want)
    for k, p in net.named_parameters():
        torch.testing.assert_close(got[k], p.grad, rtol=1e-5, atol=1e-6)


def test_streaming_tokens_in_a_graph():
    import sinabs_exodus_b200 as ex
    layer = make()
    x = torch.randn(2, 12, 24, device=DEV)
    with torch.no_grad():
        want = torch.cat([layer(x[:, t:t + 1]) for t in range(12)], 1)
    layer.reset_states()
    stream = ex.GraphedStep(layer, x[:, :1], carry_state=True)
    for name in ("h", "conv_state"):
        getattr(layer, name).zero_()
    got = torch.cat([stream(x[:, t:t + 1]).clone() for t in range(12)], 1)
    assert torch.equal(got, want)
