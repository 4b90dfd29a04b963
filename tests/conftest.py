import gc
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    config.addinivalue_line("markers", "slow: full-size CPU oracle cases (tens of seconds)")


def has_gpu():
    return torch.cuda.is_available()


@pytest.fixture(scope="session")
def golden():
    def load(name):
        return torch.load(os.path.join(GOLDEN, name + ".pt"), weights_only=False)
    return load


@pytest.fixture(scope="module", autouse=True)
def leave_nothing_behind():
    """Models and captured graphs are cycles: a module's are destroyed here, and not, at some later time, by the collector of a process that
    another module's test has forked."""
    yield
    gc.collect()
