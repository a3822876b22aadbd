"""Parameter gradients that sum many equal terms: float32 sums of those drift, because every addition rounds the same way.
Needs a GPU."""
import math

import pytest
import torch

from tests import _seq_ref as ref
from tests.test_gpu_selective import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nb", [1, 100])      # split over time, and whole: 2048 chunks of steps in one block
@pytest.mark.parametrize("M,N", [(8, 4), (40, 40)])
def test_scan(nb, M, N):
    """One input everywhere: after some steps, states and gradients stand still, and so do the terms of the sums.  In the
    kernel a term passes through sums of 8, 32 and 64 at most and a few roundings of its own (the one of the step size is
    a difference of a quarter of its terms); the last sums are in float64."""
    import sinabs_exodus_b200 as ex
    T, x = 16384, 0.3
    ones = torch.ones(nb, T, 1, N, device=DEV)
    p = dict(x=torch.full((nb, T, M), x, device=DEV), dt=torch.zeros(nb, T, M, device=DEV), A=-torch.ones(M, N, device=DEV), B=ones, C=ones,
             D=torch.ones(M, device=DEV), dt_bias=torch.ones(M, device=DEV), dt_softplus=False)
    leaves = [p[k].requires_grad_(True) for k in ("A", "D", "dt_bias")]
    y, _ = ex.selective_scan(**p)
    dA, dD, dbias = torch.autograd.grad(y, leaves, torch.ones_like(y))
    x, a, h, g = float(p["x"][0, 0, 0]), math.exp(-1.0), [0.0], 0.0
    for _ in range(T):
        h.append(a * h[-1] + x)
    sum_A = sum_dt = 0.0
    for t in range(T - 1, -1, -1):
        g = 1.0 + a * g
        sum_A += g * a * h[t]
        sum_dt += N * (g * x - g * a * h[t])
    for name, got, want, roundings in (("dA", dA, nb * sum_A, 104 + 20), ("dD", dD, nb * T * x, 104), ("ddt_bias", dbias, nb * sum_dt, 104 + 80)):
        off = float((got.double() / want - 1).abs().max())
        assert off <= roundings * 2.0 ** -24, (name, off)


# tokens: 1351 samples for each group of lanes; maps in clusters of blocks and in two kernels: 1024 positions for each thread
@pytest.mark.parametrize("R,S,C,G,up,roundings", [(50000, 1, 8192, 128, 0.9, 147), (40, 8192, 1024, 4, 0.7, 88), (1, 262144, 1024, 4, 0.7, 88)])
def test_norm(R, S, C, G, up, roundings):
    """The upstream gradient of a mean: every term of the bias's gradient is the same.  It passes through sums of 64 positions (128
    samples) and of their 16 (11) totals, and a few more; the last sums are in float64."""
    import sinabs_exodus_b200 as ex
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(R, S, C, generator=g, device=DEV)
    w, b = torch.ones(C, device=DEV, requires_grad=True), torch.zeros(C, device=DEV, requires_grad=True)
    dy = torch.full_like(x, up)
    dw, db = torch.autograd.grad(ex.group_norm(x, G, w, b), [w, b], dy)
    want = R * S * float(dy.flatten()[0])
    assert float((db.double() / want - 1).abs().max()) <= roundings * 2.0 ** -24
    # the weight's: the norm itself, summed; its terms' absolute sum is below the number of terms
    total = torch.zeros(C, device=DEV, dtype=torch.float64)
    for r in range(0, R, max(1, (1 << 27) // (S * C))):
        n = ref.norm(x[r:r + max(1, (1 << 27) // (S * C))].double(), G)
        total += n.sum((0, 1))
    assert float((dw.double() - up * total).abs().max()) <= (roundings + 50) * 2.0 ** -24 * R * S * up
