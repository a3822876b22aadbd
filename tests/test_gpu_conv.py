"""Short causal convolution and its single-token form against their definition in float64.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LEAVES = ("x", "weight", "bias", "state")


def problem(seed, nb, T, M, W, kind, act="silu", bias=True, carry=True, lengths=None, params=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    params = kind if params is None else params

    def normal(*shape, dtype=kind):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    p = dict(x=normal(nb, T, M), weight=normal(M, W, dtype=params), bias=normal(M, dtype=params) if bias else None,
             state=normal(nb, W - 1, M) if carry else None,
             lengths=None if lengths is None else torch.tensor(lengths, device=DEV), activation=act)
    return p, normal(nb, T, M), normal(nb, W - 1, M)


def run(p, dy, dlast):
    import sinabs_exodus_b200 as ex
    q = {k: (v.detach().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}
    y, last = ex.causal_conv(**q)
    names = [k for k in LEAVES if q[k] is not None]
    grads = torch.autograd.grad([y, last], [q[k] for k in names], [dy, dlast])
    return {"y": y.detach(), "last": last.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def check(got, p, dy, dlast):
    """The slack: a sum of n products in float32 is off by at most (n + 1) 2^-24 of the products' absolute sum, the
    activation and its slope (of size 1.1 at most, second derivative 0.5) by 8 roundings more; the filter's gradients
    sum batch * time of those, in one chain per thread of at most 64 steps and a tree behind it."""
    def ev(absolute):
        q = {k: (v.double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in p.items()}
        if absolute:
            q = {k: (v.abs() if k in LEAVES and v is not None else v) for k, v in q.items()}
            if q["lengths"] is not None:
                keep = (torch.arange(q["x"].shape[1], device=DEV)[None] < q["lengths"].clamp(min=0)[:, None])[..., None]
                q["x"] = torch.where(keep, q["x"], torch.zeros_like(q["x"]))
            q["activation"] = None
        names = [k for k in LEAVES if q[k] is not None]
        for k in names:
            q[k] = q[k].clone().requires_grad_(True)
        y, last = ref.conv(**q)
        up = [dy.double(), dlast.double()]
        if absolute:
            up = [1.1 * torch.nan_to_num(dy.double().abs()) * (1 + y.detach()), dlast.double().abs()]
        grads = torch.autograd.grad([y, last], [q[k] for k in names], up)
        return {"y": y.detach(), "last": last.detach(), **{"d" + k: v for k, v in zip(names, grads)}}

    want, bound = ev(False), ev(True)
    n = p["weight"].shape[1] + 10
    for k, v in got.items():
        kind = p[{"dweight": "weight", "dbias": "bias"}.get(k, "x")].dtype
        terms = n + (70 if k in ("dweight", "dbias") else 0)
        ref.assert_close(v, want[k], 0.0 if k == "last" else terms * 2.0 ** -24 * bound[k], kind, k)


# batch, time, channels, width: single steps, fewer steps than the filter, channels that leave a pack or a block
# incomplete, several blocks along time, every width
SIZES = [(1, 1, 1, 1), (1, 1, 8, 4), (2, 2, 24, 4), (3, 5, 7, 3), (2, 130, 264, 4), (1, 257, 40, 2), (2, 33, 1023, 3), (1, 600, 16, 8),
         (2, 20, 12, 5), (1, 19, 9, 6), (2, 12, 16, 7)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_gradients(size, kind):
    p, dy, dl = problem(1, *size, kind)
    check(run(p, dy, dl), p, dy, dl)


@pytest.mark.parametrize("act,bias,carry,params", [(None, True, True, None), ("silu", False, False, None), (None, False, True, F32),
                                                   ("silu", True, False, F32)])
def test_options(act, bias, carry, params):
    p, dy, dl = problem(2, 2, 45, 72, 4, BF16, act, bias, carry, params=params)
    check(run(p, dy, dl), p, dy, dl)


def test_padded_batch():
    T, n = 70, [0, 1, 2, 70, 66]
    p, dy, dl = problem(3, 5, T, 48, 4, F32, lengths=n)
    for b, k in enumerate(n):
        p["x"][b, k:] = float("nan")
    got = run(p, dy, dl)
    for b, k in enumerate(n):
        assert (got["y"][b, k:] == 0).all() and (got["dx"][b, k:] == 0).all()
    assert torch.equal(got["last"][0], p["state"][0]) and torch.equal(got["dstate"][0], dl[0])
    check(got, p, dy, dl)
    for b, k in enumerate(n):
        dy[b, k:] = float("inf")      # of rows that have no output
    again = run(p, dy, dl)
    for k in got:
        assert torch.equal(got[k], again[k]), k


def test_views_and_odd_addresses():
    import sinabs_exodus_b200 as ex
    p, dy, dl = problem(4, 2, 50, 64, 4, BF16)
    wide = torch.randn(2, 50, 200, device=DEV).to(BF16)
    for lo in (8, 9):
        a, b = run(dict(p, x=wide[..., lo:lo + 64]), dy, dl), run(dict(p, x=wide[..., lo:lo + 64].contiguous()), dy, dl)
        for k in ("y", "last", "dx", "dstate"):
            assert torch.equal(a[k], b[k]), (lo, k)
        # one channel per thread or four: the blocks of the filter's gradient are others, its sum may round differently
        for k in ("dweight", "dbias"):
            torch.testing.assert_close(a[k], b[k], rtol=2 ** -7, atol=1e-2)
    turned = p["x"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ex.causal_conv(turned, p["weight"])[0], ex.causal_conv(p["x"], p["weight"])[0])


@pytest.mark.parametrize("cut", [1, 2, 17])
def test_chunks_of_a_sequence_are_the_sequence(cut):
    import sinabs_exodus_b200 as ex
    p, dy, dl = problem(5, 2, 30, 24, 4, F32)
    q = {k: (v.detach().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}
    y1, s = ex.causal_conv(**dict(q, x=q["x"][:, :cut]))
    y2, s = ex.causal_conv(**dict(q, x=q["x"][:, cut:], state=s))
    y = torch.cat([y1, y2], 1)
    grads = torch.autograd.grad([y, s], [q[k] for k in LEAVES], [dy, dl])
    check({"y": y.detach(), "last": s.detach(), **{"d" + k: v for k, v in zip(LEAVES, grads)}}, p, dy, dl)


@pytest.mark.parametrize("nb,T,M", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_empty(nb, T, M):
    p, dy, dl = problem(6, nb, T, M, 4, F32)
    got = run(p, dy, dl)
    assert torch.equal(got["last"], p["state"]) and torch.equal(got["dstate"], dl)
    assert (got["dweight"] == 0).all() and (got["dbias"] == 0).all()


@pytest.mark.parametrize("nb,M,W", [(1, 1, 1), (3, 66, 4), (2, 128, 4), (64, 24, 2), (5, 7, 8)])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_step(nb, M, W, kind):
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(7, nb, 1, M, W, kind)
    pool = torch.full((nb, 3, W - 1, M), 7.0, device=DEV).to(kind)
    state = pool[:, 1]
    state.copy_(p["state"])
    want, want_state = ex.causal_conv(**p)
    version = state._version
    y = ex.causal_conv_step(state, p["x"][:, 0], p["weight"], p["bias"], activation="silu")
    assert state._version > version and (pool[:, 0] == 7).all() and (pool[:, 2] == 7).all()
    assert torch.equal(state, want_state)
    # the same products; the order of the bias and the taps may differ
    torch.testing.assert_close(y, want[:, 0], rtol=4 * ref.HALF_STEP[kind], atol=1e-5 if kind == F32 else 2e-3)


def test_determinism_graph_and_stream():
    import sinabs_exodus_b200 as ex
    p, dy, dl = problem(8, 2, 300, 128, 4, BF16)
    a, b = run(p, dy, dl), run(p, dy, dl)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    q = {k: (v.detach().clone().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}

    def step():
        y, last = ex.causal_conv(**q)
        grads = torch.autograd.grad([y, last], [q[k] for k in LEAVES], [dy, dl])
        return [y.detach(), last.detach(), *grads]      # no graph of the leaves stays behind when the next one is captured

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for x, y in zip(eager, held):
        assert torch.equal(x, y)


def test_step_refuses_gradients():
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(9, 2, 1, 8, 4, F32)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ex.causal_conv_step(p["state"], p["x"][:, 0], p["weight"].requires_grad_(True))


def test_step_of_many():
    """Several batch items per thread."""
    import sinabs_exodus_b200 as ex
    for nb, M in ((515, 1024), (33, 4098)):
        p, _, _ = problem(10, nb, 1, M, 4, BF16)
        want, want_state = ex.causal_conv(**p)
        state = p["state"].clone()
        y = ex.causal_conv_step(state, p["x"][:, 0], p["weight"], p["bias"], activation="silu")
        assert torch.equal(state, want_state)
        torch.testing.assert_close(y, want[:, 0], rtol=4 * ref.HALF_STEP[BF16], atol=2e-3)


def test_long_runs():
    """Rows enough that a thread walks its longest run, several times round the ring of rows on their way."""
    p, dy, dl = problem(11, 2, 5000, 136, 4, F32, lengths=[5000, 4103])
    check(run(p, dy, dl), p, dy, dl)


def test_second_derivatives_are_refused():
    import sinabs_exodus_b200 as ex
    p, dy, _ = problem(12, 1, 6, 8, 4, F32)
    p["x"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ex.causal_conv(**p)[0], p["x"], dy, create_graph=True)
