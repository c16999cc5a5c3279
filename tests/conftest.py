import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


@pytest.fixture(scope="session")
def golden():
    return np.load(os.path.join(ROOT, "tests", "golden", "reference_golden.npz"))


# Their arguments are made-up addresses, and some calls pass all checks: they must fail for want of a device.
MADE_UP_ADDRESSES = ("test_paged_cpu", "test_paged_refusals_cpu")


def pytest_runtest_setup(item):
    if item.module.__name__ in MADE_UP_ADDRESSES:
        import torch
        if torch.cuda.is_available():
            pytest.skip("made-up addresses: only where there is no GPU")
