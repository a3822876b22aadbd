"""Channels-last group norm with an activation against its definition in float64.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def problem(seed, R, S, C, kind, mean=0.5, std=1.5, affine=True, params=F32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(R, S, C, generator=g, device=DEV) * std + mean).to(kind)
    w = (torch.randn(C, generator=g, device=DEV) * 0.3 + 1).to(params) if affine else None
    b = (torch.randn(C, generator=g, device=DEV) * 0.3).to(params) if affine else None
    return x, w, b, torch.randn(R, S, C, generator=g, device=DEV).to(kind)


def run(x, G, w, b, dy, act, eps=1e-5):
    import sinabs_exodus_b200 as ex
    x, w, b = (None if t is None else t.detach().requires_grad_(True) for t in (x, w, b))
    y = ex.group_norm(x, G, w, b, eps=eps, activation=act)
    have = [("dx", x), ("dweight", w), ("dbias", b)]
    grads = torch.autograd.grad(y, [t for _, t in have if t is not None], dy)
    return {"y": y.detach(), **{k: v for (k, t), v in zip([h for h in have if h[1] is not None], grads)}}


def check(got, x, G, w, b, dy, act, eps=1e-5, offset=1.0):
    """The slack.  Mean and variance are those of values about their first one, so they are good to about
    log2(values) + 8 roundings of a value's distance from it; ``offset`` is the largest such distance in units of the
    group's deviation.  (x - mean) rstd is then off by 2^-24 times (30 + 8) times max(offset^2, |n|), and the
    gradients' sums by the same factor of their terms' absolute values; near the border of relu the slope is either."""
    q = [None if t is None else t.detach().double().requires_grad_(True) for t in (x, w, b)]
    y = ref.norm(q[0], G, q[1], q[2], eps, act)
    names = [(k, t) for k, t in zip(("dx", "dweight", "dbias"), q) if t is not None]
    want = {"y": y.detach(), **{k: g for (k, _), g in zip(names, torch.autograd.grad(y, [t for _, t in names], dy.double()))}}
    R, S, C = x.shape
    unit = 38 * 2.0 ** -24 * max(1.0, offset ** 2)
    n = ref.norm(x.double(), G, eps=eps)
    rstd = (n.detach() * 0 + 1) / torch.sqrt(((x.double().view(R, S, G, -1) - x.double().view(R, S, G, -1).mean((1, 3), keepdim=True)) ** 2)
                                             .mean((1, 3), keepdim=True) + eps).expand(R, S, G, C // G).reshape(R, S, C)
    wa = torch.ones(C, device=DEV, dtype=torch.float64) if w is None else w.double().abs()
    up = 1.5 * dy.double().abs() * (1 + n.abs())
    group = lambda t: t.view(R, S, G, -1).mean((1, 3), keepdim=True).expand(R, S, G, C // G).reshape(R, S, C)      # noqa: E731
    slack = {"y": unit * (1 + n.abs()) * (wa + 1),
             "dx": unit * rstd * (up * wa + group(up * wa) + n.abs() * group(up * wa * n.abs()) + 1e-30) * 3,
             "dweight": unit * 3 * (up * (n.abs() + 1)).sum((0, 1)), "dbias": unit * 3 * up.sum((0, 1))}
    if act == "relu":      # values that float32 may see on the other side of the border
        pre = ref.norm(x.double(), G, None if w is None else w.double(), None if b is None else b.double(), eps)
        at_border = (pre.abs() <= slack["y"]).double() * dy.double().abs()
        slack["dbias"] += at_border.sum((0, 1))
        slack["dweight"] += (at_border * n.abs()).sum((0, 1))
        slack["dx"] += rstd * (at_border * wa + group(at_border * wa) + n.abs() * group(at_border * wa * n.abs()))
    for k, v in got.items():
        kind = x.dtype if k in ("y", "dx") else w.dtype
        ref.assert_close(v, want[k], slack[k], kind, k)


# samples, positions, channels, groups: tokens with groups of 1 to over 1024 channels (a few lanes, a whole warp with 1
# to 8 packs, a block), maps whose channels leave packs incomplete or let a pack belong to several groups, one block to
# many per sample, one channel, one position short of a block's rows
SIZES = [(1, 1, 1, 1), (5, 1, 6, 3), (7, 1, 64, 8), (33, 1, 1536, 24), (3, 1, 1000, 1), (2, 1, 2400, 2), (9, 1, 40, 5), (300, 1, 96, 2),
         (3, 1, 260, 2), (2, 1, 140, 1), (4, 1, 520, 1),
         (2, 9, 64, 8), (1, 1000, 32, 4), (3, 49, 48, 3), (2, 100, 20, 10), (1, 33, 7, 1), (2, 4096, 16, 2), (1, 70, 1536, 1),
         (2, 31, 1040, 4), (1, 17, 2304, 768), (1, 5, 4098, 2), (40, 4, 24, 3)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind,act", [(F32, "silu"), (BF16, None), (F16, "relu")])
def test_values_and_gradients(size, kind, act):
    R, S, C, G = size
    x, w, b, dy = problem(1, R, S, C, kind)
    if S * C // G == 1:      # a group of one value: the norm is 0 and its gradient too, exactly
        got = run(x, G, w, b, dy, act)
        assert (got["dx"] == 0).all()
        return
    check(run(x, G, w, b, dy, act), x, G, w, b, dy, act, offset=6.0)


@pytest.mark.parametrize("affine,params,act", [(False, F32, "silu"), (True, BF16, "silu"), (True, BF16, None)])
@pytest.mark.parametrize("S", [1, 50])
def test_parameters(affine, params, act, S):
    x, w, b, dy = problem(2, 6, S, 64, BF16, affine=affine, params=params)
    check(run(x, 4, w, b, dy, act), x, 4, w, b, dy, act, offset=6.0)


def test_weight_without_bias_and_bias_without_weight():
    x, w, b, dy = problem(3, 4, 20, 32, F32)
    check(run(x, 4, w, None, dy, "silu"), x, 4, w, None, dy, "silu", offset=6.0)
    got = run(x, 4, None, b, dy, "silu")
    ref.assert_close(got["y"], ref.norm(x.double(), 4, None, b.double(), 1e-5, "silu"), 1e-5, F32, "y")


@pytest.mark.parametrize("S,C,G", [(1, 256, 2), (400, 64, 4)])
def test_large_common_offset(S, C, G):
    """Values around 1000 with a deviation of 1: 2^-24 * 1000 of each value is lost in the input already (they are given
    in float32), none in the sums."""
    x, w, b, dy = problem(4, 3, S, C, F32, mean=1000.0, std=1.0)
    check(run(x, G, w, b, dy, None), x, G, w, b, dy, None, offset=7.0)


def test_constant_groups_and_extremes():
    import sinabs_exodus_b200 as ex
    for S in (1, 40):
        x = torch.full((2, S, 16), 3.0, device=DEV)
        assert (ex.group_norm(x, 2) == 0).all()
        x[1, 0, 3] = float("nan")
        y = ex.group_norm(x, 2)
        assert torch.isnan(y[1, :, :8]).all() and (y[1, :, 8:] == 0).all() and (y[0] == 0).all()
        z = torch.randn(2, S, 16, device=DEV) * 1e-30
        assert torch.isfinite(ex.group_norm(z, 2)).all()


def test_shapes_and_views():
    import sinabs_exodus_b200 as ex
    x, w, b, dy = problem(5, 6, 35, 48, BF16)
    y = ex.group_norm(x, 4, w, b, activation="silu")
    assert torch.equal(ex.group_norm(x.view(6, 5, 7, 48), 4, w, b, activation="silu").view(6, 35, 48), y)
    wide = torch.randn(6, 35, 200, device=DEV).to(BF16)
    for lo in (8, 9, 12):
        part = wide[..., lo:lo + 48]
        a, c = run(part, 4, w, b, dy, "silu"), run(part.contiguous(), 4, w, b, dy, "silu")
        for k in ("y", "dx"):
            d = (a[k].float() - c[k].float()).abs()
            assert (d <= 2.0 ** -7 * c[k].float().abs() + 1e-5).all(), (lo, k)      # blocks of other shape: other orders of sums
    every_other = wide[::2, :, :48]
    assert torch.equal(ex.group_norm(every_other, 4, w, b), ex.group_norm(every_other.contiguous(), 4, w, b))
    tokens = wide[:, 0, :48]
    assert torch.equal(ex.group_norm(tokens, 4, w, b), ex.group_norm(tokens.contiguous(), 4, w, b))


@pytest.mark.parametrize("shape", [(0, 4, 8), (3, 0, 8), (0, 8)])
def test_empty(shape):
    import sinabs_exodus_b200 as ex
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = ex.group_norm(x, 2, w)
    y.sum().backward()
    assert y.shape == shape and (w.grad == 0).all() and x.grad.shape == shape


@pytest.mark.parametrize("S", [1, 300])
def test_determinism_graph_and_stream(S):
    import sinabs_exodus_b200 as ex
    x, w, b, dy = problem(6, 20, S, 64, BF16)
    a, c = run(x, 4, w, b, dy, "silu"), run(x, 4, w, b, dy, "silu")
    for k in a:
        assert torch.equal(a[k], c[k]), k
    xs, ws, bs = (t.clone().requires_grad_(True) for t in (x, w, b))

    def step():
        y = ex.group_norm(xs, 4, ws, bs, activation="silu")
        grads = torch.autograd.grad(y, [xs, ws, bs], dy)
        return [y.detach(), *grads]      # no graph of the leaves stays behind when the next one is captured

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        xs.copy_(x * 2 + 1)
    graph.replay()
    for p, q in zip(step(), held):
        assert torch.equal(p, q)
    assert not torch.equal(eager[1], held[1])


def test_layer():
    """``layers.GroupNorm``: feature maps in either memory format, with and without a time dimension, and tokens."""
    import sinabs_exodus_b200 as ex
    layer = ex.layers.GroupNorm(4, 16, activation="relu").to(DEV)
    with torch.no_grad():
        layer.weight.uniform_(0.5, 1.5)
        layer.bias.normal_()
    x = torch.randn(6, 16, 5, 7, device=DEV)
    want = torch.relu(torch.nn.functional.group_norm(x.double(), 4, layer.weight.double(), layer.bias.double(), layer.eps))
    for v in (x, x.to(memory_format=torch.channels_last)):
        y = layer(v)
        assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
        ref.assert_close(y, want, 1e-5, F32, "maps")
    ref.assert_close(layer(x.view(2, 3, 16, 5, 7)).reshape(x.shape), want, 1e-5, F32, "maps of a sequence")
    t = torch.randn(3, 9, 16, device=DEV)
    want = torch.relu(torch.nn.functional.group_norm(t.double().view(-1, 16), 4, layer.weight.double(), layer.bias.double(), layer.eps))
    ref.assert_close(layer(t), want.view(3, 9, 16), 1e-5, F32, "tokens")
    net = torch.nn.Sequential(torch.nn.Conv2d(2, 16, 3, padding=1), layer,
                              ex.layers.LIFSqueeze(batch_size=2, tau_mem=10.0, norm_input=False)).to(DEV)
    out = net(torch.randn(6, 2, 5, 7, device=DEV).to(memory_format=torch.channels_last))
    out.sum().backward()
    assert out.shape == (6, 16, 5, 7) and torch.isfinite(layer.weight.grad).all() and net[0].weight.grad.abs().sum() > 0


# samples enough that clusters of blocks take one each: of 8, 2, 1 blocks; rows that do not fill a pack; several slabs
CLUSTERS = [(40, 2100, 64, 8), (150, 1100, 44, 4), (300, 70, 32, 4), (40, 1300, 160, 32), (60, 600, 2048, 8), (310, 3, 24, 2)]


@pytest.mark.parametrize("size", CLUSTERS)
@pytest.mark.parametrize("kind,act", [(F32, "silu"), (BF16, "silu"), (F16, None)])
def test_clusters(size, kind, act):
    R, S, C, G = size
    x, w, b, dy = problem(7, R, S, C, kind)
    check(run(x, G, w, b, dy, act), x, G, w, b, dy, act, offset=7.0)


def test_largest_groups():
    """Groups as wide as they may be, where the sums over channels fill a block's shared memory."""
    for S, C, G in ((1, 16384, 1), (5, 16384, 1), (3, 32766, 2)):
        x, w, b, dy = problem(8, 2, S, C, BF16)
        check(run(x, G, w, b, dy, "silu"), x, G, w, b, dy, "silu", offset=6.0)


def test_second_derivatives_are_refused():
    import sinabs_exodus_b200 as ex
    x = torch.randn(2, 5, 8, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ex.group_norm(x, 2).sum(), x, create_graph=True)
