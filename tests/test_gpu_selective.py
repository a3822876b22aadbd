"""Selective scan and its single-token form against their definition in float64.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def problem(seed, nb, T, M, N, G, kind, gate=True, skip=True, bias=True, carry=True, lengths=None, softplus=True):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=kind):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    p = dict(x=normal(nb, T, M), dt=normal(nb, T, M, std=0.5), B=normal(nb, T, G, N), C=normal(nb, T, G, N),
             A=-(torch.rand(M, N, generator=g, device=DEV) * 3 + 0.05), dt_softplus=softplus)
    if not softplus:
        p["dt"] = p["dt"].abs()
    p["D"] = normal(M, dtype=F32) if skip else None
    p["z"] = normal(nb, T, M) if gate else None
    p["dt_bias"] = (torch.rand(M, generator=g, device=DEV) * -2 - 0.5 if softplus else torch.rand(M, generator=g, device=DEV)) if bias else None
    p["h0"] = normal(nb, M, N, dtype=F32) if carry else None
    p["lengths"] = None if lengths is None else torch.tensor(lengths, device=DEV, dtype=torch.int32)
    return p, normal(nb, T, M), normal(nb, M, N, dtype=F32)


LEAVES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0")
NAMES = {"x": "dx", "dt": "ddt", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "dt_bias": "ddt_bias", "h0": "dh0"}


def run(p, dy=None, dh=None):
    import sinabs_exodus_b200 as ex
    if dy is None:
        y, h = ex.selective_scan(**p)
        return {"y": y, "h": h}
    q = {k: (v.detach().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}
    y, h = ex.selective_scan(**q)
    names = [k for k in LEAVES if q[k] is not None]
    outs, ups = ([y], [dy]) if dh is None else ([y, h], [dy, dh])
    grads = torch.autograd.grad(outs, [q[k] for k in names], ups)
    return {"y": y.detach(), "h": h.detach(), **{NAMES[k]: v for k, v in zip(names, grads)}}


def check(got, p, dy=None, dh=None):
    want, bound, emax, kinds = ref.scan(**p, dy=dy, dh=dh)
    T = p["x"].shape[1]
    for k, v in got.items():
        if k == "dB" or k == "dC":
            want[k], bound[k] = want[k].view(v.shape), bound[k].view(v.shape)
        ref.assert_close(v, want[k], ref.scan_tolerance(bound[k], emax, T, kinds.get(k, F32)), kinds.get(k, F32), k)


# batch, time, channels, states, groups: one of everything, odd sizes, every number of lanes per channel (states up to
# 4, 8, ... 128), channel tiles that end inside a block, groups narrower than a block, times around the chunk of 8 and
# the stage of 16 steps and long enough to be split
SIZES = [(1, 1, 1, 1, 1), (2, 7, 5, 3, 1), (1, 16, 64, 16, 1), (3, 33, 66, 10, 3), (2, 100, 128, 16, 2), (1, 300, 40, 64, 1),
         (2, 65, 24, 128, 2), (1, 40, 16, 32, 1), (1, 1000, 8, 4, 4), (4, 17, 36, 8, 1), (1, 129, 300, 5, 1), (2, 8, 130, 16, 1),
         (1, 9, 12, 100, 1)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind", [F32, BF16])
def test_forward(size, kind):
    p, _, _ = problem(1, *size, kind)
    check(run(p), p)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind", [F32, F16])
def test_gradients(size, kind):
    p, dy, dh = problem(2, *size, kind)
    check(run(p, dy, dh), p, dy, dh)


@pytest.mark.parametrize("gate,skip,bias,carry,softplus", [(False, False, False, False, False), (True, False, False, True, True),
                                                           (False, True, True, False, True), (False, True, True, True, False)])
def test_absent_arguments(gate, skip, bias, carry, softplus):
    p, dy, dh = problem(3, 2, 70, 36, 6, 2, F32, gate, skip, bias, carry, softplus=softplus)
    check(run(p, dy, dh if carry else None), p, dy, dh if carry else None)


@pytest.mark.parametrize("T", [20, 200])      # whole, and split over time
def test_padded_batch(T):
    """Rows behind a sequence hold NaN and infinities: they reach nothing, and come back as zeros."""
    p, dy, dh = problem(4, 5, T, 40, 16, 2, F32, lengths=[0, 1, T, T - 3, T // 2])
    for b, n in enumerate(p["lengths"].tolist()):
        for k, junk in (("x", float("nan")), ("dt", float("inf")), ("B", float("nan")), ("C", float("-inf")), ("z", float("nan"))):
            p[k][b, n:] = junk
        dy[b, n:] = float("nan")
    got = run(p, dy, dh)
    for k in ("y", "dx", "ddt", "dB", "dC", "dz"):
        for b, n in enumerate(p["lengths"].tolist()):
            assert (got[k][b, n:] == 0).all(), k
    assert torch.equal(got["h"][0], p["h0"][0]) and torch.equal(got["dh0"][0], dh[0])      # a sequence of length 0
    check(got, p, dy, dh)


def test_lengths_beyond_the_ends_are_clamped():
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(5, 2, 12, 8, 4, 1, F32)
    p["lengths"] = torch.tensor([-5, 99], device=DEV)
    a = ex.selective_scan(**p)
    p["lengths"] = torch.tensor([0, 12], device=DEV)
    b = ex.selective_scan(**p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_views_are_used_where_they_lie():
    """Slices of wider tensors, odd offsets, a broadcast input and a transposed one give what their copies give."""
    import sinabs_exodus_b200 as ex
    p, dy, _ = problem(6, 3, 50, 48, 12, 2, BF16)
    g = torch.Generator(device=DEV).manual_seed(7)
    wide = torch.randn(3, 50, 1 + 2 * 48 + 48, generator=g, device=DEV).to(BF16)
    proj = torch.randn(3, 50, 3 + 2 * 24, generator=g, device=DEV).to(BF16)
    q = dict(p, x=wide[..., 1:49], z=wide[..., 49:97], dt=wide[..., 97:145],
             B=proj[..., 3:27].unflatten(-1, (2, 12)), C=proj[..., 27:51].unflatten(-1, (2, 12)))
    assert q["x"].data_ptr() == wide.data_ptr() + 2
    c = {k: v.contiguous() if torch.is_tensor(v) else v for k, v in q.items()}
    a, b = run(q, dy), run(c, dy)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    one = p["x"][:1].expand(3, 50, 48)
    a, b = ex.selective_scan(**dict(p, x=one)), ex.selective_scan(**dict(p, x=one.contiguous()))
    assert torch.equal(a[0], b[0])
    turned = p["dt"].transpose(1, 2).contiguous().transpose(1, 2)
    a, b = ex.selective_scan(**dict(p, dt=turned)), ex.selective_scan(**p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # the upstream gradient may be a view too
    a, b = run(p, wide[..., 1:49]), run(p, wide[..., 1:49].contiguous())
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_one_group_without_its_dimension():
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(8, 2, 20, 16, 8, 1, F32)
    a = ex.selective_scan(**p)
    b = ex.selective_scan(**dict(p, B=p["B"].squeeze(2), C=p["C"].squeeze(2)))
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("cut", [1, 8, 13])
def test_chunks_of_a_sequence_are_the_sequence(cut):
    """Two calls that hand the state on are the one call, gradients through the state included."""
    p, dy, dh = problem(9, 2, 40, 24, 16, 1, F32)
    import sinabs_exodus_b200 as ex
    q = {k: (v.detach().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}
    parts, h = [], q["h0"]
    for sl in (slice(0, cut), slice(cut, 40)):
        r = {k: q[k][:, sl] for k in ("x", "dt", "B", "C", "z")}
        y, h = ex.selective_scan(**dict(q, **r, h0=h))
        parts.append(y)
    y = torch.cat(parts, 1)
    grads = torch.autograd.grad([y, h], [q[k] for k in LEAVES], [dy, dh])
    check({"y": y.detach(), "h": h.detach(), **{NAMES[k]: v for k, v in zip(LEAVES, grads)}}, p, dy, dh)


def test_gradients_against_differences():
    """Central differences of the float64 definition along random directions: an independent check of the formulas."""
    p, dy, dh = problem(10, 2, 24, 12, 6, 2, F32)
    got = run(p, dy, dh)
    g = torch.Generator(device=DEV).manual_seed(11)
    for k in LEAVES:
        u = torch.randn(p[k].shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-5

        def loss(sign):
            q = {n: (v.double() if torch.is_tensor(v) else v) for n, v in p.items()}
            q[k] = q[k] + sign * eps * u
            v = ref.scan(**q)[0]
            return float((v["y"] * dy.double()).sum() + (v["h"] * dh.double()).sum())

        slope = (loss(1) - loss(-1)) / (2 * eps)
        have = float((got[NAMES[k]].double().view(u.shape) * u).sum())
        scale = float((got[NAMES[k]].double().view(u.shape) * u).abs().sum())
        # differences: third derivatives times eps^2 (1e-10) and cancellation (1e-16 / 1e-5 of the loss's terms)
        assert abs(have - slope) <= 2e-5 * scale + 1e-6, (k, have, slope)


def test_results_do_not_change_between_calls():
    p, dy, dh = problem(12, 1, 500, 200, 16, 1, BF16)
    a, b = run(p, dy, dh), run(p, dy, dh)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("nb,T,M", [(0, 5, 8), (2, 0, 8), (2, 5, 0)])
def test_empty(nb, T, M):
    p, dy, dh = problem(13, nb, T, M, 4, 1, F32)
    got = run(p, dy, dh)
    assert torch.equal(got["h"], p["h0"]) and torch.equal(got["dh0"], dh)
    assert got["y"].shape == (nb, T, M) and (got["dA"] == 0).all() and (got["dD"] == 0).all()


def test_rates_at_the_ends():
    """Rates of 0 (an integrator) and of minus infinity (no memory at all)."""
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(14, 1, 30, 8, 4, 1, F32, lengths=[19])
    p["A"][0] = 0.0
    p["A"][1] = float("-inf")
    y, h = ex.selective_scan(**p)
    assert torch.isfinite(y).all() and torch.isfinite(h).all()
    s = torch.nn.functional.softplus(p["dt"].double() + p["dt_bias"])
    b = (s * p["x"].double())[..., None] * p["B"].double()
    torch.testing.assert_close(h[0, 1].double(), b[0, 18, 1], rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(h[0, 0].double(), p["h0"][0, 0].double() + b[0, :19, 0].sum(0), rtol=1e-5, atol=1e-5)


def test_graph_and_side_stream():
    """Captured forward and backward replay on new values; a call on another stream uses that stream."""
    import sinabs_exodus_b200 as ex
    p, dy, dh = problem(15, 1, 200, 64, 16, 1, F32)
    other, dy2, _ = problem(16, 1, 200, 64, 16, 1, F32)
    q = {k: (v.detach().clone().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}

    def step():
        y, h = ex.selective_scan(**q)
        grads = torch.autograd.grad([y, h], [q[k] for k in LEAVES], [dy, dh])
        return [y.detach(), h.detach(), *grads]      # no graph of the leaves stays behind when the next one is captured

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for a, b in zip(eager, held):
        assert torch.equal(a, b)
    with torch.no_grad():
        for k in LEAVES:
            q[k].copy_(other[k])
    graph.replay()
    want = step()
    for a, b in zip(want, held):
        assert torch.equal(a, b)


@pytest.mark.parametrize("nb,M,N,G", [(1, 1, 1, 1), (3, 66, 10, 3), (2, 128, 16, 1), (5, 40, 64, 2), (1, 24, 128, 1), (70, 32, 4, 8)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_step(nb, M, N, G, kind):
    """One token is a prompt of one step; the state is updated where it lies, among the rows of a pool."""
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(17, nb, 1, M, N, G, kind)
    pool = torch.full((nb, 2, M, N), float("nan"), device=DEV)
    h = pool[:, 1]
    h.copy_(p["h0"])
    version = h._version
    args = {k: p[k][:, 0] for k in ("x", "dt", "B", "C", "z")}
    y = ex.selective_step(h, A=p["A"], D=p["D"], dt_bias=p["dt_bias"], **args)
    assert h._version > version and torch.isnan(pool[:, 0]).all()
    check({"y": y[:, None], "h": h}, p)


def test_steps_follow_a_prompt():
    """A prompt and then single tokens are the whole sequence."""
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(18, 2, 30, 48, 16, 1, F32)
    first = {k: p[k][:, :20] for k in ("x", "dt", "B", "C", "z")}
    y, h = ex.selective_scan(**dict(p, **first))
    ys = [y]
    for t in range(20, 30):
        args = {k: p[k][:, t] for k in ("x", "dt", "B", "C", "z")}
        ys.append(ex.selective_step(h, A=p["A"], D=p["D"], dt_bias=p["dt_bias"], **args)[:, None])
    check({"y": torch.cat(ys, 1), "h": h}, p)


def test_step_refuses_gradients():
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(19, 2, 1, 8, 4, 1, F32)
    args = {k: p[k][:, 0] for k in ("x", "dt", "B", "C", "z")}
    args["x"] = args["x"].clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ex.selective_step(p["h0"], A=p["A"], **args)
    with torch.no_grad():
        ex.selective_step(p["h0"], A=p["A"], **args)


# The kernels come in two forms, for problems with one block of channels per SM and for larger ones; the sizes above are
# all of the first.  Many batch items and channels, whole and split over time, every number of lanes.
LARGE = [(20, 24, 512, 16, 1), (20, 11, 1000, 8, 1), (5, 19, 1024, 32, 2), (4, 24, 640, 64, 1), (3, 9, 408, 128, 1), (5, 560, 256, 16, 1),
         (4, 600, 258, 7, 1)]


@pytest.mark.parametrize("size", LARGE)
@pytest.mark.parametrize("kind", [F32, BF16])
def test_many_blocks(size, kind):
    p, dy, dh = problem(20, *size, kind)
    check(run(p, dy, dh), p, dy, dh)


def test_many_blocks_padded():
    T = 560
    p, dy, dh = problem(21, 5, T, 256, 16, 1, F32, lengths=[0, 1, T, 333, 48])
    for b, n in enumerate(p["lengths"].tolist()):
        p["x"][b, n:] = p["B"][b, n:] = p["z"][b, n:] = float("nan")
        dy[b, n:] = float("inf")
    got = run(p, dy, dh)
    for k in ("y", "dx", "ddt", "dB", "dC", "dz"):
        for b, n in enumerate(p["lengths"].tolist()):
            assert (got[k][b, n:] == 0).all(), k
    check(got, p, dy, dh)


def test_lengths_of_64_bits():
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(22, 2, 12, 8, 4, 1, F32)
    a = ex.selective_scan(**dict(p, lengths=torch.tensor([2 ** 40, 5], device=DEV)))
    b = ex.selective_scan(**dict(p, lengths=torch.tensor([12, 5], device=DEV, dtype=torch.int32)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_second_derivatives_are_refused():
    import sinabs_exodus_b200 as ex
    p, dy, _ = problem(23, 1, 6, 8, 4, 1, F32)
    p["x"].requires_grad_(True)
    y, _ = ex.selective_scan(**p)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, p["x"], dy, create_graph=True)


def test_upstream_gradient_of_a_sum():
    """An expanded upstream gradient, as sum() sends it; and one for the state alone."""
    import sinabs_exodus_b200 as ex
    p, _, dh = problem(24, 2, 20, 24, 8, 1, F32)
    a = run(p, torch.ones(2, 20, 24, device=DEV))
    x = p["x"].clone().requires_grad_(True)
    ex.selective_scan(**dict(p, x=x))[0].sum().backward()
    assert torch.equal(x.grad, a["dx"])
    x.grad = None
    ex.selective_scan(**dict(p, x=x))[1].backward(dh)
    b = run(p, torch.zeros(2, 20, 24, device=DEV), dh)
    assert torch.equal(x.grad, b["dx"])


def test_two_graphs_and_two_streams_at_once():
    """Calls that run side by side have scratch memory of their own."""
    import sinabs_exodus_b200 as ex
    ps = [problem(25 + i, 1, 900, 64, 16, 1, F32)[0] for i in range(2)]
    want = [ex.selective_scan(**p) for p in ps]
    graphs, held = [], []
    for p in ps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(ex.selective_scan(**p))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, h in zip(want, held):
        assert torch.equal(w[0], h[0]) and torch.equal(w[1], h[1])
    outs = []
    for s, p in zip(streams, ps):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([ex.selective_scan(**p) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])


@pytest.mark.parametrize("nb", [4, 7, 130])
@pytest.mark.parametrize("N", [3, 8, 16, 40])
def test_step_of_many(nb, N):
    """Several batch items per thread, a number that does not divide them among it."""
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(30, nb, 1, 2048, N, 1, BF16)
    h = p["h0"].clone()
    args = {k: p[k][:, 0] for k in ("x", "dt", "B", "C", "z")}
    y = ex.selective_step(h, A=p["A"], D=p["D"], dt_bias=p["dt_bias"], **args)
    check({"y": y[:, None], "h": h}, p)


def test_step_in_a_graph_and_inference_mode():
    import sinabs_exodus_b200 as ex
    p, _, _ = problem(31, 3, 1, 40, 16, 1, F32)
    args = {k: p[k][:, 0].contiguous() for k in ("x", "dt", "B", "C", "z")}
    rest = dict(A=p["A"], D=p["D"], dt_bias=p["dt_bias"])
    a, b = p["h0"].clone(), p["h0"].clone()
    for _ in range(4):
        want = ex.selective_step(a, **args, **rest)
    ex.selective_step(b.clone(), **args, **rest)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ex.selective_step(b, **args, **rest)
    for _ in range(4):
        g.replay()
    assert torch.equal(a, b) and torch.equal(want, got)
    with torch.inference_mode():
        c = p["h0"].clone()
        ex.selective_step(c, **args, **rest)
