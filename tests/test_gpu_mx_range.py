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


def needs(gb):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip("needs %d GB" % gb)


def test_a_layer_of_as_many_inputs_as_are_taken():
    rows, n, k = 2, 8, 2 ** 28
    needs(8)
    X = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    wc = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    ws = torch.full((M.mxfp4_scale_bytes(n, k),), 127, dtype=torch.uint8, device="cuda")
    # blocks at the front, in the middle and at the end hold small whole numbers, which 4 bits keep
    want = torch.zeros(rows, n, device="cuda")
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    for i, at in enumerate((0, (1 << 27) - 64, k - 128, k - 64)):
        g = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randint(-2, 3, (rows, 64), device="cuda", generator=g).float()
        x[:, ::32] = 6                                   # each block's largest: a scale of 1
        c = torch.randint(0, 256, (n, 32), device="cuda", generator=g, dtype=torch.uint8)
        X[:, at:at + 64], wc[:, at // 2:at // 2 + 32] = x.bfloat16(), c
        want += x @ torch.stack([grid[(c & 15).long()], grid[(c >> 4).long()]], -1).reshape(n, 64).T
    Y = torch.full((rows, n), float("nan"), device="cuda")
    M.linear_mxfp4(X, (wc.view(-1), ws, n, k), Y, torch.empty(M.linear_mxfp4_work_bytes(rows, k), dtype=torch.uint8, device="cuda"))
    assert torch.equal(Y, want)
    del X, wc, ws
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 200])
def test_a_layer_of_as_many_outputs_as_an_int_counts(rows):
    n, k = (2 ** 31 - 8, 64) if rows == 1 else (2 ** 27 - 8, 64)          # 200 rows of outputs take 400 bytes for each
    needs(100)
    wc = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    ws = torch.full((M.mxfp4_scale_bytes(n, k),), 127, dtype=torch.uint8, device="cuda")
    X = torch.randint(-2, 3, (rows, k), device="cuda").bfloat16()
    Y = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    spots, some = [0, n // 2 - 100, n - 504], []
    for r in spots:
        some.append(torch.randint(0, 256, (504, k // 2), dtype=torch.uint8, device="cuda"))
        wc[r:r + 504] = some[-1]
        Y[:, r:r + 504] = float("nan")
    work = torch.empty(M.linear_mxfp4_work_bytes(rows, k), dtype=torch.uint8, device="cuda")
    M.linear_mxfp4(X, (wc.view(-1), ws, n, k), Y, work)
    for r, c in zip(spots, some):
        want = torch.empty(rows, 504, device="cuda", dtype=torch.bfloat16)
        M.linear_mxfp4(X, (c.view(-1), torch.full((M.mxfp4_scale_bytes(504, k),), 127, dtype=torch.uint8, device="cuda"), 504, k), want, work)
        assert torch.equal(Y[:, r:r + 504], want)
    del wc, ws, Y
    torch.cuda.empty_cache()
