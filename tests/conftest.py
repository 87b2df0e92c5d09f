import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) and runs the CUDA path")


@pytest.fixture(autouse=True)
def _no_wait_ran_out(request):
    """After a GPU test, no kernel of this process's contexts has given up a bounded wait."""
    yield
    if request.node.get_closest_marker("gpu"):
        import pyxis_b200 as px

        for ctx in list(px._CUDA.values()):
            if ctx is not None and ctx.handle:
                ctx.check_device_error()


@pytest.fixture(scope="session", autouse=True)
def _built():
    """Both native libraries, built once per session (no-op when up to date)."""
    from oracle import build as ob
    from pyxis_b200 import build as pb

    ob.build()
    pb.build()
    yield
