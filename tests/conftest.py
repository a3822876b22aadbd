import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200)")


@pytest.fixture(scope="session", autouse=True)
def _built_checker():
    """The CPU checker library is needed by almost every test; build it once."""
    from oracle import build as oracle_build

    oracle_build.build_oracle()


@pytest.fixture(autouse=True)
def _queues_by_value(request, monkeypatch):
    """Results of worker processes that end right after they have put them."""
    if request.module.__name__.split(".")[-1] == "test_dist_cpu":
        import copy

        import torch.multiprocessing as mp

        from tests import _by_value
        get_context = mp.get_context
        monkeypatch.setattr(mp, "get_context", lambda method=None: _by_value.context_with(copy.copy(get_context(method))))
