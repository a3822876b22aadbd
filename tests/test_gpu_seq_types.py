"""Types and sizes of the sequence operators that the other tests leave out.  Needs a GPU."""
import pytest
import torch

from tests import _seq_ref as ref
from tests import test_gpu_conv as conv
from tests import test_gpu_selective as scan

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("size", scan.LARGE)
def test_scan_of_many_blocks_in_float16(size):
    p, dy, dh = scan.problem(20, *size, F16)
    scan.check(scan.run(p, dy, dh), p, dy, dh)


@pytest.mark.parametrize("nb,M,W", [(1, 1, 1), (3, 66, 4), (2, 128, 4), (64, 24, 2), (5, 7, 8), (515, 1024, 4), (33, 4098, 3)])
@pytest.mark.parametrize("act", ["silu", None])
def test_conv_step_in_float16(nb, M, W, act):
    import sinabs_exodus_b200 as ex
    p, _, _ = conv.problem(7, nb, 1, M, W, F16, act)
    state = p["state"].clone()
    y = ex.causal_conv_step(state, p["x"][:, 0], p["weight"], p["bias"], activation=act)
    assert torch.equal(state, torch.cat([p["state"], p["x"]], 1)[:, 1:])
    q = {k: p[k].double() for k in ("x", "weight", "bias", "state")}
    want, _ = ref.conv(**q, activation=act)
    size, _ = ref.conv(**{k: v.abs() for k, v in q.items()})
    # a sum of W products and the bias, and the activation's 8 roundings with a slope of 1.1
    ref.assert_close(y, want[:, 0], (W + 10) * 1.1 * 2.0 ** -24 * size[:, 0], F16, "y")
