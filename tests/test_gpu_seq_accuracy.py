"""Selective scan on states that grow or hardly decay, whole, split over time and token by token.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref
from tests._seq_err import scan_bounds
from tests.test_gpu_selective import DEV, F16, F32, check, problem, run

pytestmark = pytest.mark.gpu


def growing(nb, T, M=8, N=4):
    """Rate 3 and step size 1 in every other channel: 2^138 over 32 steps."""
    p, dy, _ = problem(1, nb, T, M, N, 1, F32, gate=False, skip=False, bias=False, carry=False, softplus=False)
    p["A"][::2] = 3.0
    p["dt"].fill_(1.0)
    return p, dy


@pytest.mark.parametrize("nb", [1, 100])      # split over time, and whole
def test_growing_states_that_are_still_zero(nb):
    """Inputs only at the end and gradients only at the start: in between, states and their gradients are 0, which any
    growth leaves as it is."""
    p, dy = growing(nb, 1024)
    p["x"][:, :-10] = 0.0
    dy[:, 10:] = 0.0
    check(run(p, dy), p, dy)


@pytest.mark.parametrize("nb", [1, 100])
def test_growth_beyond_float32_of_a_small_state(nb):
    """The factor of 32 steps is 2^138, the state it applies to 1e-32: the product is an ordinary number."""
    p, _ = growing(nb, 1024)
    p["x"].zero_()
    p["lengths"] = torch.full((nb,), 40, device=DEV, dtype=torch.int32)
    p["h0"] = torch.full((nb, 8, 4), 1e-32, device=DEV)
    check(run(p), p)


# Rates and what the errors of one step's decay may have in common (of its value), from the decays' mean errors octave by
# octave: 6.5e-9 where a step decays by more than 2^-8, 2e-9 below.
SLOW = [(1e-2, 6.5e-9), (3e-3, 6.5e-9), (1e-3, 2e-9), (1e-4, 2e-9)]
STEPS = 4096


def slow_problem(nb, M, seed, fed, N=4):
    g = torch.Generator(device=DEV).manual_seed(seed)
    A = -torch.tensor([r for r, _ in SLOW], device=DEV).repeat(M, N // 4)
    dt = torch.rand(nb, STEPS, M, generator=g, device=DEV) + 0.5
    x = (torch.rand(nb, STEPS, M, generator=g, device=DEV) + 0.5) * fed
    ones = torch.ones(nb, STEPS, 1, N, device=DEV)
    h0 = (torch.rand(nb, M, N, generator=g, device=DEV) + 0.5) * (1 - fed)
    return dict(x=x, dt=dt, A=A, B=ones, C=ones, h0=h0, dt_softplus=False)


def slow_exact(p):
    """The last state, by the definition in float64."""
    h, A = p["h0"].double(), p["A"].double()
    for s, u in zip(p["dt"].double().unbind(1), (p["dt"].double() * p["x"].double()).unbind(1)):
        h = torch.exp(s[..., None] * A) * h + u[..., None]
    return h


def relative(got, want, pure):
    """A state of positive terms, each off by its decays: their common error times the number of steps (those in the
    state's memory, or all of them where a single value decays: ``pure``), a random walk of their 1e-7 at most, the
    rounding of A log2(e) and of the sums of step sizes, 1e-7 of the exponent, and a few roundings.  The mean over the
    states is bound by what is common, with an eighth of the walk (64 states or more)."""
    off = (got.double() - want) / want
    for n, (rate, common) in enumerate(SLOW):
        age = STEPS if pure else min(STEPS, 1 / rate)
        rest = 1e-7 * rate * age + 5e-7
        mean, rms = float(off[..., n::4].mean()), float(off[..., n::4].square().mean().sqrt())
        assert abs(mean) <= common * age + rest + 1e-7 * age ** 0.5 / 8, (rate, mean)
        assert rms <= common * age + rest + 1e-7 * age ** 0.5, (rate, rms)


@pytest.mark.parametrize("fed", [0, 1])      # a state that only decays, and one that inputs keep up
@pytest.mark.parametrize("nb,M", [(1, 64), (100, 8)])      # split over time, and whole
def test_slow_decays(nb, M, fed):
    import sinabs_exodus_b200 as ex
    p = slow_problem(nb, M, 2, fed)
    relative(ex.selective_scan(**p)[1], slow_exact(p), not fed)


@pytest.mark.parametrize("nb,M", [(1, 64), (100, 8)])
def test_slow_decays_of_the_gradient(nb, M):
    """The gradient of the first state is that of the last one, decayed."""
    import sinabs_exodus_b200 as ex
    p = slow_problem(nb, M, 3, 0)
    p["h0"].requires_grad_(True)
    up = torch.rand(nb, M, 4, device=DEV) + 0.5
    got, = torch.autograd.grad(ex.selective_scan(**p)[1], p["h0"], up)
    relative(got, up.double() * torch.exp(p["dt"].double().sum(1)[..., None] * p["A"].double()), True)


@pytest.mark.parametrize("fed", [0, 1])
@pytest.mark.parametrize("nb,M,N", [(8, 8, 4), (20, 4096, 16)])      # one batch item per thread, and several
def test_slow_decays_token_by_token(nb, M, N, fed):
    import sinabs_exodus_b200 as ex
    p = slow_problem(nb, M, 4, fed, N)
    h = p["h0"].clone()
    for t in range(STEPS):
        ex.selective_step(h, A=p["A"], dt_softplus=False, **{k: p[k][:, t] for k in ("x", "dt", "B", "C")})
    relative(h, slow_exact(p), not fed)


# batch, time, channels, states, groups: split over time and whole, states in every number of lanes, long beyond any memory
@pytest.mark.parametrize("size", [(1, 1500, 40, 16, 2), (100, 1500, 8, 4, 1), (2, 1100, 24, 64, 1), (1, 2100, 128, 8, 4), (100, 1100, 8, 128, 1),
                                  (4, 1300, 600, 32, 1)])
@pytest.mark.parametrize("kind", [F32, F16])
def test_long_sequences(size, kind):
    p, dy, dh = problem(5, *size, kind)
    got = run(p, dy, dh)
    del p["lengths"]
    want, _, _, kinds = ref.scan(**p, dy=dy, dh=dh)
    bound = scan_bounds(**p, dy=dy, dh=dh)
    for k, v in got.items():
        if k in ("dB", "dC"):
            want[k], bound[k] = want[k].view(v.shape), bound[k].view(v.shape)
        ref.assert_close(v, want[k], bound[k], kinds.get(k, F32), k)
