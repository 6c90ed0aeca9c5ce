"""Host side of the microscaled operators without a GPU: sizes at the end of the integer range, and the front end's bookkeeping."""
import pytest
import torch


@pytest.fixture(scope="module")
def M():
    import tmt_moe_b200 as m
    from tmt_moe_b200 import build
    build.build()
    m.load()
    return m


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 100, 2 ** 31 - 256])
def test_layernorm_scratch_at_the_end_of_the_row_range(M, rows):
    """Both backward passes count rows up to 2^31 - 1: rounding up to whole blocks must not pass the range."""
    for dim in (32, 64, 128, 256, 1024, 8192):
        assert M.ln_backward_act8_scratch_bytes(rows, dim) == M.ln_backward_act8_scratch_bytes(1 << 30, dim) > 0        # as many teams as the GPU holds
    for dim in (8, 2048):
        assert M.ln_backward_scratch_bytes(rows, dim) == -(-rows // 128) * 2 * dim * 4
