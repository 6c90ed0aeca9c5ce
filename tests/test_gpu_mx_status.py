"""A wait that runs out in a product is not lost when the caller hands in no status word."""
import os
import subprocess
import sys

import pytest
import torch

import test_gpu_mx_use as U
import tmt_moe_b200 as M

pytestmark = pytest.mark.gpu


def test_the_shared_status_word_reports_once():
    lib = M.load()
    assert M.mxfp4_status() == 0
    for stream in (None, torch.cuda.Stream().cuda_stream):
        assert lib.tmt_moe_mxfp4_selftest_bounded_wait(2_000_000, stream) == 0          # about 1 ms
        assert M.mxfp4_status() == 2
        assert M.mxfp4_status() == 0
    for limit in (0, 1 << 40):
        assert lib.tmt_moe_mxfp4_selftest_bounded_wait(limit, None) == -1
    for f in U.FORMS:
        assert U.Layer(*f, 1).run().isfinite().all()
    assert M.mxfp4_status() == 0


def test_a_status_word_of_the_caller_is_the_one_that_is_used():
    """The library's word holds a code meanwhile: the caller's stays as it was, and products go on."""
    lib = M.load()
    layer, status = U.Layer(300, 264, 448, 1), torch.full((1,), 7, dtype=torch.int32, device="cuda")
    want = layer.value()
    assert lib.tmt_moe_mxfp4_selftest_bounded_wait(1000, None) == 0
    M.linear_mxfp4(layer.X, layer.W, layer.Y, layer.work, status=status)
    assert torch.equal(layer.Y, want) and status.item() == 7 and M.mxfp4_status() == 2


FIRST_CALL = """
import sys
sys.path[:0] = sys.argv[1:]
import torch
import tmt_moe_b200 as M
rows, n, k = 300, 264, 448
raw = lambda n: torch.full((n,), 127, dtype=torch.uint8, device="cuda")
X, Y, work = torch.randn(rows, k, device="cuda").bfloat16(), torch.zeros(rows, n, device="cuda"), raw(M.linear_mxfp4_work_bytes(rows, k))
W = M.Mxfp4Weights([(raw(n * k // 2), raw(M.mxfp4_scale_bytes(n, k)), n, k)])
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    M.linear_mxfp4(X, W, Y, work, stream=s.cuda_stream)
g.replay()
torch.cuda.synchronize()
a = Y.clone()
M.linear_mxfp4(X, W, Y, work)
assert torch.equal(a, Y) and a.abs().sum() > 0 and M.mxfp4_status() == 0
"""


def test_the_first_call_of_a_process_may_be_a_recorded_one():
    paths = [os.path.dirname(os.path.dirname(os.path.abspath(M.__file__)))]
    subprocess.run([sys.executable, "-c", FIRST_CALL, *paths], check=True, timeout=300)
