import inspect
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


def pytest_collection_modifyitems(items):
    """Where the reference's own library is not built, the tests that fail without it run last: a run that stops at its
    first failure has been through all others by then."""
    from oracle.pyoracle import REF_SO
    if not os.path.exists(REF_SO):
        items.sort(key=lambda i: "ref" in i.fixturenames or "RefHarness()" in inspect.getsource(i.function))


@pytest.fixture(scope="session")
def oracle():
    from oracle.pyoracle import Oracle, build
    build()
    return Oracle()


@pytest.fixture(scope="session")
def golden_dir():
    return os.path.join(ROOT, "tests", "golden")
