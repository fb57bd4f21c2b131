import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


@pytest.fixture(scope="session")
def dev():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


# A test that asks for 2 round(g) where the gradient is round(2 g), which differ where g lies below fp16's normal numbers.  One of the case's 140,000 numbers
# does: g = -0x1.6dc59ep-15.  Steps of fp16 there are 2^-24 for both g and 2 g: 2 g = -0x1.6dc59ep-14 rounds to -0x1.6dcp-14, 0.09 steps away;
# g rounds to -0x1.6ep-15, and its double, -0x1.6ep-14, is 0.91 steps from 2 g, where a rounding is off by half a step at most.  The test stands as it was;
# tests/test_gpu_preference_grad.py holds the same numbers to half a step.
ROUNDED_TWICE = "test_gpu_preference.py::test_loss_margins_and_gradient[700-300-200-most10-dtype10-False]"


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.endswith(ROUNDED_TWICE):
            item.add_marker(pytest.mark.xfail(reason="asks for a gradient that is rounded twice", raises=AssertionError, strict=True))
