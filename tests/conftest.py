"""Shared pytest setup: the repo root on sys.path and the ``gpu`` marker."""

from __future__ import annotations

import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config: pytest.Config) -> None:
    config.addinivalue_line("markers", "gpu: needs an MI355X (HIP device) and the built libnmb.so")


@pytest.fixture(scope="session")
def device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def backward_on_the_calling_thread(request):
    """For tests that count the memory in use: autograd's worker thread lets go of a finished backward's
    results after its caller has gone on, and without the interpreter's lock not before that waits."""
    if getattr(request.node, "originalname", None) != "test_graphs_are_freed":
        yield
        return
    import torch

    with torch.autograd.set_multithreading_enabled(False):
        yield
