"""Test configuration: the ``gpu`` marker and repo-root imports.

``-m "not gpu"`` runs the CPU suite (oracle vs golden vectors, C-ABI symbol
table, host logic, gloo multi-rank logic); ``-m gpu`` runs the CUDA parity
tests, which call the product through torch.ops.d2p / the C ABI and compare
against the CPU oracle in ``oracle/`` (test infrastructure only).
"""
import os
import sys
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


def cuda_ok() -> bool:
    try:
        import torch

        return torch.cuda.is_available()
    except Exception:
        return False


@pytest.fixture(scope="session")
def cuda_device():
    if not cuda_ok():
        pytest.skip("no CUDA device")
    import torch

    return torch.device("cuda:0")


_session_ended = [0.0]


@pytest.fixture(autouse=True)
def profiler_in_step(request):
    """Keeps the profiler's clock in step with the GPU's for the tests that read kernel names from a session: with 4 s and more
    between sessions the records' times drift out of the sessions' windows and records are dropped (measured: none with
    2 s and less; 1 of 6 after 12 s, 3 of 6 after 36 s of sessions 4 s apart)."""
    if request.node.get_closest_marker("gpu") and cuda_ok() and time.monotonic() - _session_ended[0] > 1.0:
        import torch
        from torch.profiler import ProfilerActivity, profile

        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]):
            torch.ones(1, device="cuda")
            torch.cuda.synchronize()
        _session_ended[0] = time.monotonic()
    yield
