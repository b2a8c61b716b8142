import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


@pytest.fixture(scope="session")
def golden_dir():
    return os.path.join(ROOT, "tests", "golden")


@pytest.fixture(autouse=True)
def _restore_torch_threads():
    """VolOpt pins torch to one intra-op thread like the reference (train.py:24); keep that from leaking into later tests."""
    import torch

    n = torch.get_num_threads()
    yield
    if torch.get_num_threads() != n:
        torch.set_num_threads(n)


@pytest.fixture(autouse=True)
def _restore_arithmetic():
    """The kernels' arithmetic is process state (ops.set_geo_mode and its like): a test leaves it as it found it, whatever its own fixtures set."""
    from spurfies_amd import ops

    arith, h2 = dict(ops._ARITH), dict(ops._H2)
    yield
    ops._ARITH.update(arith)
    ops._H2.update(h2)
