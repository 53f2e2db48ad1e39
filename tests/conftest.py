"""Shared pytest setup: repository root on sys.path and the `gpu` marker."""
import inspect
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
GOLDEN = os.path.join(ROOT, "tests", "golden")
if GOLDEN not in sys.path:
    sys.path.insert(0, GOLDEN)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a); run with -m gpu")


def _uses_reference(fn, seen):
    """Whether a test calls the reference's kernels (oracle.refgpu), itself or through functions of its module."""
    if fn in seen:
        return False
    seen.add(fn)
    codes = [fn.__code__]
    for code in codes:
        if "refgpu" in code.co_names:
            return True
        codes += [c for c in code.co_consts if inspect.iscode(c)]
    called = (fn.__globals__.get(name) for code in codes for name in code.co_names)
    return any(inspect.isfunction(f) and f.__module__ == fn.__module__ and _uses_reference(f, seen) for f in called)


def pytest_collection_modifyitems(items):
    """Where the reference's kernels are not built (no checkout of it), the tests that compare with them fail: they run
    last, so that a run that stops at the first failure has run all the others."""
    from oracle import refgpu

    if not refgpu.available():
        items.sort(key=lambda item: _uses_reference(item.function, set()))


@pytest.fixture(scope="session")
def cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("CUDA GPU required for -m gpu tests")
    return torch.device("cuda:0")
