"""Microscaled operators without a GPU: refused arguments (checked before anything is queued), sizes, and the plain statement the
GPU tests compare with (known answers)."""
import ctypes

import numpy as np
import pytest
import torch

import mx_ref as R


@pytest.fixture(scope="module")
def M():
    import tmt_moe_b200 as m
    from tmt_moe_b200 import build
    build.build()
    m.load()
    return m


def refused(M, rc, *words):
    assert rc == -1
    msg = M.load().tmt_moe_last_error().decode()
    assert all(w in msg for w in words), msg


P = 1 << 20        # an aligned address that nothing may read: every call below is refused before


@pytest.mark.parametrize("rows,cols,dtype,word", [(-1, 64, 0, "rows"), (4, 0, 0, "cols"), (4, 100, 0, "cols"), (4, -64, 0, "cols"), (4, 64, 2, "dtype")])
def test_casts_refuse_bad_shapes_and_types(M, rows, cols, dtype, word):
    lib = M.load()
    refused(M, lib.tmt_moe_quantize_mxfp4(P, dtype, rows, cols, P, P, None), word)
    refused(M, lib.tmt_moe_dequantize_mxfp4(P, P, rows, cols, P, dtype, None), word)
    refused(M, lib.tmt_moe_act8_save(P, dtype, rows, cols, 1, P, P, None), word)
    refused(M, lib.tmt_moe_act8_restore(P, P, rows, cols, 1, P, dtype, None), word)


def test_a_4_bit_matrix_has_whole_pairs_of_blocks(M):
    lib = M.load()
    for cols in (32, 96):
        refused(M, lib.tmt_moe_quantize_mxfp4(P, 0, 4, cols, P, P, None), "64")
        refused(M, lib.tmt_moe_dequantize_mxfp4(P, P, 4, cols, P, 0, None), "64")


def test_casts_refuse_other_formats(M):
    lib = M.load()
    for fmt in (0, 3, -1):
        refused(M, lib.tmt_moe_act8_save(P, 0, 4, 64, fmt, P, P, None), "format")
        refused(M, lib.tmt_moe_act8_restore(P, P, 4, 64, fmt, P, 0, None), "format")


def test_zero_rows_do_nothing(M):
    lib = M.load()
    assert lib.tmt_moe_quantize_mxfp4(None, 0, 0, 64, None, None, None) == 0
    assert lib.tmt_moe_dequantize_mxfp4(None, None, 0, 64, None, 0, None) == 0
    assert lib.tmt_moe_act8_save(None, 0, 0, 32, 1, None, None, None) == 0
    assert lib.tmt_moe_act8_restore(None, None, 0, 32, 2, None, 1, None) == 0
    assert lib.tmt_ln_forward_act8(*[None] * 8, 1, 0, 64, None) == 0
    W = M._Mxfp4WeightDesc(P, P, 8, 64)
    assert lib.tmt_moe_matmul_mxfp4(None, None, 0, ctypes.byref(W), None, 0, None, None) == 0
    assert lib.tmt_moe_linear_mxfp4(None, 0, 0, ctypes.byref(W), None, 0, None, 0, None, None) == 0


@pytest.mark.parametrize("n,k", [(0, 64), (7, 64), (12, 64), (8, 0), (8, 32), (8, 96), (-8, 64)])
def test_products_refuse_bad_weights(M, n, k):
    lib = M.load()
    W = M._Mxfp4WeightDesc(P, P, n, k)
    refused(M, lib.tmt_moe_matmul_mxfp4(P, P, 4, ctypes.byref(W), P, 0, None, None), "multiple of 8")
    refused(M, lib.tmt_moe_linear_mxfp4(P, 0, 4, ctypes.byref(W), P, 0, P, 1 << 30, None, None), "multiple of 8")


def test_products_refuse_bad_arguments(M):
    lib = M.load()
    W = M._Mxfp4WeightDesc(P, P, 8, 64)
    refused(M, lib.tmt_moe_matmul_mxfp4(P, P, -1, ctypes.byref(W), P, 0, None, None), "rows")
    refused(M, lib.tmt_moe_matmul_mxfp4(P, P, 4, None, P, 0, None, None), "null")
    refused(M, lib.tmt_moe_matmul_mxfp4(P, P, 4, ctypes.byref(W), P, 5, None, None), "dtype")
    refused(M, lib.tmt_moe_linear_mxfp4(P, 0, 4, ctypes.byref(W), P, 0, P, 4 * 32 + 511, None, None), "work")
    refused(M, lib.tmt_moe_forward_mxfp4(None, P, P, ctypes.byref(W), ctypes.byref(W), P, 0.0, 1), "null handle")


@pytest.mark.parametrize("rows,dim,fmt,word", [(-1, 64, 1, "rows"), (4, 48, 1, "32"), (4, 0, 1, "rows"), (4, 8224, 1, "8192")])
def test_layernorm_checkpoints_refuse_bad_shapes(M, rows, dim, fmt, word):
    lib = M.load()
    refused(M, lib.tmt_ln_forward_act8(*[P] * 8, fmt, rows, dim, None), word)
    refused(M, lib.tmt_ln_backward_act8(P, P, fmt, *[P] * 7, rows, dim, P, None), "32")
    assert lib.tmt_ln_backward_act8_scratch_bytes(rows, dim) == 0


def test_layernorm_backward_refuses_other_formats(M):
    lib = M.load()
    for fmt in (0, 3):
        refused(M, lib.tmt_ln_backward_act8(P, P, fmt, *[P] * 7, 4, 64, P, None), "format")


def test_sizes(M):
    assert M.mxfp4_scale_bytes(1, 64) == 512 and M.mxfp4_scale_bytes(128, 128) == 512 and M.mxfp4_scale_bytes(129, 192) == 2048
    assert M.mxfp4_scale_bytes(0, 64) == 0 and M.mxfp4_scale_bytes(4, 96) == 0 and M.mxfp4_scale_bytes(-1, 64) == 0
    assert M.mxfp4_scale_bytes(1 << 31, 4096) == (1 << 31) // 128 * 32 * 512         # past 32 bits
    assert M.linear_mxfp4_work_bytes(3, 192) == 3 * 96 + 1024
    assert M.ln_backward_act8_scratch_bytes(1, 32) >= 2 * 32 * 4


def test_the_front_end_refuses_what_the_library_cannot_see(M):
    X = torch.zeros(8, 128, dtype=torch.bfloat16)
    codes, scales = torch.zeros(8 * 64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    W = (torch.zeros(16 * 64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 16, 128)
    work = torch.zeros(M.linear_mxfp4_work_bytes(8, 128), dtype=torch.uint8)
    Y = torch.zeros(8, 16)
    bad = [
        lambda: M.quantize_mxfp4(X.t(), codes, scales),
        lambda: M.quantize_mxfp4(X[:, ::2], codes, scales),
        lambda: M.quantize_mxfp4(X.half(), codes, scales),
        lambda: M.quantize_mxfp4(X[0], codes, scales),
        lambda: M.quantize_mxfp4(X, codes[:-1], scales),
        lambda: M.quantize_mxfp4(X, codes, scales[:-1]),
        lambda: M.quantize_mxfp4(X, codes.int(), scales),
        lambda: M.dequantize_mxfp4(codes[:-1], scales, X),
        lambda: M.act8_save(X, codes, scales),
        lambda: M.act8_restore(codes, scales, X),
        lambda: M.linear_mxfp4(X, W, Y[:, :8], work),
        lambda: M.linear_mxfp4(X, W, Y[:4], work),
        lambda: M.linear_mxfp4(X[:, :64].contiguous(), W, Y, work),
        lambda: M.linear_mxfp4(X, (W[0][:-1], *W[1:]), Y, work),
        lambda: M.linear_mxfp4(X, (W[0], W[1][:-1], 16, 128), Y, work),
        lambda: M.linear_mxfp4(X, M.Mxfp4Weights([W, W]), Y, work),
        lambda: M.matmul_mxfp4(codes[:-1], scales, W, Y),
        lambda: M.ln_forward_act8(X, Y.view(-1)[:127], Y.view(-1), X, Y.view(-1), Y.view(-1), codes, scales),
        lambda: M.ln_forward_act8(X, Y.view(-1), Y.view(-1), X[:4], Y.view(-1), Y.view(-1), codes, scales),
    ]
    for call in bad:
        with pytest.raises(M.MoeError):
            call()


def test_plain_statement_known_answers():
    # the midpoints of e2m1 go to the even code; the block's largest value picks the scale
    x = np.zeros((1, 32))
    x[0, :12] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -5, 0.2500001, 0.74]
    c, s = R.quantize(x, "e2m1")
    assert s[0, 0] == 127
    assert R.values(c, s, "e2m1")[0, :12].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -4, 0.5, 0.5]
    assert c[0, 8] == 8 and c[0, 20] == 0
    x[0, 0] = 6.0000001
    assert R.quantize(x, "e2m1")[1][0, 0] == 128
    for fmt, v in R.MAXV.items():
        for e, byte in ((0, 127), (-126, 1), (-127, 0), (-140, 0), (100, 227)):
            y = np.zeros((1, 32))
            y[0, 3] = v * 2.0 ** e
            assert R.quantize(y, fmt)[1][0, 0] == byte, (fmt, e)
    z = np.zeros((1, 64))
    z[0, 5] = np.inf
    c, s = R.quantize(z, "e4m3")
    assert s.tolist() == [[255, 0]] and (c == 0).all() and np.isnan(R.values(c, s, "e4m3")[0, :32]).all()
    # e4m3 and e5m2 grids as torch has them
    for fmt, t, top in (("e4m3", torch.float8_e4m3fn, 0x7e), ("e5m2", torch.float8_e5m2, 0x7b)):
        want = torch.arange(top + 1, dtype=torch.uint8).view(t).double().numpy()
        np.testing.assert_array_equal(R.grid(fmt), want)


def test_scale_tiles_cover_every_byte_once():
    at = R.tile_index(256, 8)
    assert sorted(at.reshape(-1).tolist()) == list(range(2 * 2 * 512))
    assert at[33, 5] == 512 + 16 + 4 + 1 and at[128, 0] == 1024
