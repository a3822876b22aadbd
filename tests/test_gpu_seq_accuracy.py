"""Selective scan on states that grow or hardly decay, whole, split over time and token by token.  Needs a GPU."""
import pytest
import torch

from tests.test_gpu_selective import DEV, F32, check, problem, run

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
