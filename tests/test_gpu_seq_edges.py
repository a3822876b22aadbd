"""Sequence operators at the edges of what their arguments may be.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref
from tests.test_gpu_selective import F32, problem

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
