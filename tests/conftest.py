import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "tensor-inference_b200")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200); run with -m gpu")


def pytest_collection_modifyitems(items):
    """The drop-in tests need a library built from the reference's sources.  Where it is not there they fail, after all the
    others, so that a run that stops at the first failure (-x) has run those."""
    lib = os.path.join(ROOT, "tensor-inference_b200", "backend", "_build", "libref_models_on_b200.so")
    if not os.path.exists(lib):
        items.sort(key=lambda item: os.path.basename(str(item.fspath)) == "test_gpu_dropin.py")


@pytest.fixture(scope="session")
def orc():
    import oracle

    oracle.build()
    return oracle


@pytest.fixture(scope="session")
def ti():
    import ti_b200

    ti_b200.lib()
    return ti_b200
