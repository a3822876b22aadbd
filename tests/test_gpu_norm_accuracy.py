"""Group norm of values whose mean or whose first one lies far from the others.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref
from tests.test_gpu_norm import BF16, DEV, F16, F32, problem, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,S,C,G", [(3, 1, 7, 1), (5, 1, 100, 1), (9, 1, 1000, 1), (4, 1, 1536, 24), (3, 1, 2400, 2), (2, 1, 520, 1),
                                     (2, 40, 48, 3), (300, 50, 100, 4)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_equal_values_of_any_size(R, S, C, G, kind):
    """Values that are all the same are their mean, exactly: what is left is the bias, and nothing comes back."""
    x, w, b, dy = problem(1, R, S, C, kind)
    for value in (1000.3, -0.1, 29999.0):
        got = run(torch.full_like(x, value), G, w, b, dy, None)
        assert torch.equal(got["y"], b.to(kind).expand_as(x)), value
        assert (got["dweight"] == 0).all()


@pytest.mark.parametrize("R,C,G", [(5, 300, 1), (40, 1536, 24), (3, 1000, 1), (7, 96, 32)])
def test_tokens_with_a_very_large_offset(R, C, G):
    """Values around 1e5 with a deviation of 1.  About their first one, which is at most 8 deviations off, they are as good
    as any: the sums of at most 1000 of them round 10 + 28 times."""
    import sinabs_exodus_b200 as ex
    x, w, b, _ = problem(2, R, 1, C, F32, mean=1e5, std=1.0)
    n = ref.norm(x.double(), G)
    want = n * w.double() + b.double()
    ref.assert_close(ex.group_norm(x, G, w, b), want, 38 * 2.0 ** -24 * 64 * (1 + n.abs()) * (w.double().abs() + 1) , F32, "y")


@pytest.mark.parametrize("R,S", [(40, 8192), (1, 262144)])      # clusters of blocks, and two kernels: 1024 positions per thread
def test_maps_whose_first_values_lie_far_off(R, S):
    """Every thread begins on a value of 1e4 and has a thousand of deviation 1 behind it.  About the means of the first 8, 64 and
    512 of its values, the sums of their squares round like sums of 64 equal terms."""
    import sinabs_exodus_b200 as ex
    x, w, b, _ = problem(3, R, S, 1024, F32, mean=0.0, std=1.0)
    x[:, ::1024] = 1e4
    y = ex.group_norm(x, 4, w, b)
    for r in range(0, R, 13):
        n = ref.norm(x[r:r + 1].double(), 4)
        ref.assert_close(y[r:r + 1], n * w.double() + b.double(), 120 * 2.0 ** -24 * (1 + n.abs()) * (w.double().abs() + 1), F32, "y")
