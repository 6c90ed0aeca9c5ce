"""The microscaled products at the end of the row range."""
import pytest
import torch

import tmt_moe_b200 as M

pytestmark = pytest.mark.gpu


def test_a_product_of_as_many_rows_as_an_int_counts():
    rows, n, k = 2 ** 31 - 1, 8, 64
    torch.cuda.empty_cache()
    need = rows * (k // 2 + n * 2) + M.mxfp4_scale_bytes(rows, k)
    if torch.cuda.mem_get_info()[0] < need + (4 << 30):
        pytest.skip("needs %d GB" % (need >> 30))
    c, s = torch.randint(0, 256, (n * k // 2,), dtype=torch.uint8, device="cuda"), torch.full((M.mxfp4_scale_bytes(n, k),), 127, dtype=torch.uint8, device="cuda")
    codes = torch.zeros(rows * k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((M.mxfp4_scale_bytes(rows, k),), 127, dtype=torch.uint8, device="cuda")
    Y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    # the first rows, some around 2^30 and the last ones (the last tile is not full) hold something
    spots = [0, (1 << 30) - 300, rows - 700]
    few = [torch.randint(0, 256, (700, k // 2), dtype=torch.uint8, device="cuda") for _ in spots]
    for r, f in zip(spots, few):
        codes.view(rows, -1)[r:r + 700] = f
        Y[r:r + 700] = float("nan")
    M.matmul_mxfp4(codes, scales, (c, s, n, k), Y)
    for r, f in zip(spots, few):
        want = torch.empty(700, n, dtype=torch.bfloat16, device="cuda")
        M.matmul_mxfp4(f.view(-1), torch.full((M.mxfp4_scale_bytes(700, k),), 127, dtype=torch.uint8, device="cuda"), (c, s, n, k), want)
        assert torch.equal(Y[r:r + 700], want)
    del codes, scales, Y
    torch.cuda.empty_cache()
