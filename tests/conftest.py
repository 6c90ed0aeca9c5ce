import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "test-model-thing-cuda_b200")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


@pytest.fixture(autouse=True)
def _gpu_idle_after(request):
    """A GPU test's work is done before the next test takes its memory, and a fault or a wait that ran out names the test it belongs to."""
    yield
    if request.node.get_closest_marker("gpu"):
        import torch
        if torch.cuda.is_available():
            torch.cuda.synchronize()
            import tmt_moe_b200 as M
            if M._lib is not None:
                assert M.mxfp4_status() == 0           # no product gave up waiting


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as o
    o.build()
    return o
