import os
import sys
import threading

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200)")


@pytest.fixture(scope="session")
def golden_dir():
    return GOLDEN


@pytest.fixture(scope="session")
def cuda_lib():
    """Build (if stale) and load libgnnagg.so; GPU tests call the kernels only through it."""
    from gnn_benchmark_b200 import _lib, build

    build.build()
    return _lib.lib()


@pytest.fixture(scope="session", autouse=True)
def npz_arrays_are_read_one_at_a_time():
    """Ranks that run as threads read their arrays from one open .npz archive, whose zip file has a single position: two
    reads at a time fail now and then.  So an array is read under a lock."""
    archive, lock = type(np.load(os.path.join(GOLDEN, "quant_v1.npz"))), threading.Lock()
    read = archive.__getitem__

    def read_alone(self, key):
        with lock:
            return read(self, key)

    archive.__getitem__ = read_alone
    yield
    archive.__getitem__ = read
