"""Microscaled operators on the GPU (include/tmt_mx.h) against plain float64 statements (mx_ref.py)."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tmt_moe_b200 as M
from oracle import oracle as O

pytestmark = pytest.mark.gpu

FMT8 = {"e4m3": M.ACT8_E4M3, "e5m2": M.ACT8_E5M2}
SENTINEL = 0xA5


def values_with_edges(rows, cols, seed):
    """Activations over many magnitudes, with the values where a block can go wrong: midpoints between two elements, the largest
    element and its neighbours, zeros of both signs, blocks of zeros, subnormals, the smallest and largest numbers."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-6, 7, (rows, cols // 32)).repeat(32, 1)
    b = x.reshape(rows, cols // 32, 32)
    n = b.shape[0] * b.shape[1]
    flat = b.reshape(n, 32)
    kinds = rng.integers(0, 12, n)
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 4.0, 0.5, 1.0, -0.25, -0.75, -1.25, -2.5, -5.0] * 2)
    flat[kinds == 1] = mids
    flat[kinds == 2] = mids * 2.0 ** -20
    flat[kinds == 3] = 0.0
    flat[kinds == 4] = -0.0
    flat[kinds == 5] = mids * 2.0 ** -130                 # subnormal in bf16 and fp32
    flat[kinds == 6] = mids * 2.0 ** 124
    flat[kinds == 7, 1:] = 0.0                            # a single element
    flat[kinds == 8, 0] = 6.03125                         # just past the largest element of e2m1
    return x


def to_device(x, dtype):
    t = torch.from_numpy(np.asarray(x, np.float32)).cuda()
    return t.bfloat16() if dtype == "bf16" else t


def exact64(t):
    return t.float().cpu().numpy().astype(np.float64)


def poisoned(n):
    return torch.full((n + 256,), SENTINEL, dtype=torch.uint8, device="cuda")


SHAPES = [(1, 64), (1, 8192), (3, 192), (37, 320), (128, 256), (129, 64), (300, 1088), (2049, 128), (5, 4160)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_mxfp4_is_exact(rows, cols, dtype):
    X = to_device(values_with_edges(rows, cols, rows * 7 + cols), dtype)
    codes, scales = poisoned(rows * cols // 2), poisoned(M.mxfp4_scale_bytes(rows, cols))
    M.quantize_mxfp4(X, codes, scales)
    wc, ws = R.quantize(exact64(X), "e2m1")
    got = codes.cpu().numpy()
    np.testing.assert_array_equal(got[:rows * cols // 2].reshape(rows, -1), R.pack4(wc))
    assert (got[rows * cols // 2:] == SENTINEL).all()
    at = R.tile_index(rows, cols // 32)
    gs = scales.cpu().numpy()
    np.testing.assert_array_equal(gs[at], ws)
    assert (gs[M.mxfp4_scale_bytes(rows, cols):] == SENTINEL).all()
    if cols // 32 % 4:                                    # blocks past the last column: a scale that is no NaN
        assert (gs[R.tile_index(rows, (cols // 32 + 3) // 4 * 4)][:, cols // 32:] == 0).all()
    for out in ("bf16", "f32"):
        Y = torch.full((rows, cols), 7.0, dtype=torch.bfloat16 if out == "bf16" else torch.float32, device="cuda")
        M.dequantize_mxfp4(codes, scales, Y)
        want = R.values(wc, ws, "e2m1")
        if out == "bf16":
            want = torch.from_numpy(want).to(torch.bfloat16).double().numpy()
        np.testing.assert_array_equal(Y.double().cpu().numpy(), want)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (7, 96)] + SHAPES)
def test_act8_is_exact(rows, cols, dtype, fmt):
    X = to_device(values_with_edges(rows, cols, rows * 3 + cols), dtype)
    codes, scales = poisoned(rows * cols), poisoned(rows * cols // 32)
    M.act8_save(X, codes, scales, FMT8[fmt])
    wc, ws = R.quantize(exact64(X), fmt)
    np.testing.assert_array_equal(codes.cpu().numpy()[:rows * cols].reshape(rows, cols), wc)
    np.testing.assert_array_equal(scales.cpu().numpy()[:rows * cols // 32].reshape(rows, -1), ws)
    assert (codes[rows * cols:] == SENTINEL).all() and (scales[rows * cols // 32:] == SENTINEL).all()
    Y = torch.full((rows, cols), 7.0, device="cuda")
    M.act8_restore(codes, scales, Y, FMT8[fmt])
    np.testing.assert_array_equal(Y.double().cpu().numpy(), R.values(wc, ws, fmt).astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_block_with_an_infinity_or_nan_stands_for_nan_and_its_neighbours_stay(fmt, dtype, bad):
    x = np.random.default_rng(5).standard_normal((5, 256))
    x[1, 40] = bad
    x[4, 255] = bad
    X = to_device(x, dtype)
    Y = torch.zeros(5, 256, device="cuda")
    if fmt == "e2m1":
        codes, scales = poisoned(5 * 128), poisoned(M.mxfp4_scale_bytes(5, 256))
        M.quantize_mxfp4(X, codes, scales)
        M.dequantize_mxfp4(codes, scales, Y)
    else:
        codes, scales = poisoned(5 * 256), poisoned(5 * 8)
        M.act8_save(X, codes, scales, FMT8[fmt])
        M.act8_restore(codes, scales, Y, FMT8[fmt])
    want = R.q(exact64(X), fmt)
    assert np.isnan(want[1, 32:64]).all() and np.isnan(want[4, 224:]).all() and np.isnan(want).sum() == 64
    np.testing.assert_array_equal(Y.double().cpu().numpy(), want)


def random_blocks(rows, cols, rng, lo=125, hi=130):
    """(device codes, device scale tiles, float64 values): every code, scales 2^-2 .. 2^2, so that sums of a few thousand products are
    multiples of 2^-6 below 2^18 and fit the 24 bits of fp32: any order of summation gives the same result, exactly."""
    c = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    s = rng.integers(lo, hi, (rows, cols // 32)).astype(np.uint8)
    t = R.tile(s, fill=255)                               # padding rows and blocks: NaN scales that must not reach a result
    if cols // 32 % 4:
        pad = R.tile_index((rows + 127) // 128 * 128, (cols // 32 + 3) // 4 * 4)
        t[pad[:, cols // 32:]] = 255
    return torch.from_numpy(R.pack4(c)).cuda(), torch.from_numpy(t).cuda(), R.values(c, s, "e2m1")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n,k", [(1, 8, 64), (1, 128, 256), (2, 136, 128), (31, 64, 192), (32, 256, 512), (33, 264, 320), (64, 128, 1024),
                                      (65, 2504, 448), (127, 72, 256), (128, 128, 256), (129, 384, 1344), (257, 512, 576), (500, 1000, 2048),
                                      (1000, 136, 64), (1, 2048, 4096), (20, 4096, 64), (2300, 2056, 320),
                                      (4096, 1288, 64), (3000, 2504, 448), (5000, 1160, 1344), (2049, 4096, 2048), (9000, 128, 256),
                                      (5, 136, 8192), (32, 264, 5120), (3, 64, 8256), (24, 1000, 1088)])
def test_matmul_is_exact_where_fp32_is(rows, n, k, dtype):
    rng = np.random.default_rng(rows * 31 + n + k)
    ac, asc, a = random_blocks(rows, k, rng)
    wc, wsc, w = random_blocks(n, k, rng)
    Y = torch.full((rows + 1, n), 77.0, dtype=torch.bfloat16 if dtype == "bf16" else torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    M.matmul_mxfp4(ac, asc, (wc, wsc, n, k), Y[:rows], status)
    want = a @ w.T
    assert (want == want.astype(np.float32)).all()
    if dtype == "bf16":
        want = torch.from_numpy(want).to(torch.bfloat16).double().numpy()
    np.testing.assert_array_equal(Y[:rows].double().cpu().numpy(), want)
    assert (Y[rows:] == 77).all() and status.item() == 0


@pytest.mark.parametrize("x_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n,k", [(1, 2048, 1024), (17, 72, 192), (777, 2504, 1344), (300, 128, 4096)])
def test_linear_against_float64(rows, n, k, x_dtype):
    rng = np.random.default_rng(rows + n)
    X = to_device(rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, k // 32))).repeat(32, 1), x_dtype)
    W = to_device(rng.standard_normal((n, k)) * 0.02, "bf16")
    wc, wsc = poisoned(n * k // 2), poisoned(M.mxfp4_scale_bytes(n, k))
    M.quantize_mxfp4(W, wc, wsc)
    work = poisoned(M.linear_mxfp4_work_bytes(rows, k))
    Y = torch.empty(rows, n, device="cuda")
    M.linear_mxfp4(X, M.Mxfp4Weights([(wc, wsc, n, k)]), Y, work)
    a, w = R.q(exact64(X), "e2m1"), R.q(exact64(W), "e2m1")
    # products are exact; k additions, each off by at most one step (2^-23) of a partial sum that the magnitudes bound
    tol = k * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)
    assert (np.abs(Y.double().cpu().numpy() - a @ w.T) <= tol).all()
    Yb = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    M.linear_mxfp4(X, (wc, wsc, n, k), Yb, work)
    assert torch.equal(Yb, Y.bfloat16())                  # one rounding of the same sums


def experts_case(T, D, H, E, K, seed, skew=False):
    """Rows and router on grids on which every partial sum of a logit fits fp32."""
    rng = np.random.default_rng(seed)
    x = np.round(np.clip(rng.standard_normal((T, D)), -4, 4) * 16) / 16
    wr = np.clip(np.round(rng.standard_normal((E, D)) * 0.05 * 512), -31, 31) / 512
    if skew:
        wr[E // 2:] = wr[0]                               # ties: the lower index wins, the upper half stays without tokens but for E // 2
    up, down = rng.standard_normal((E, H, D)) * 0.05, rng.standard_normal((E, D, H)) * 0.05
    return x, wr, up, down


def quantized(ws):
    out = []
    for w in ws:
        W = to_device(w, "bf16")
        n, k = W.shape
        c, s = torch.empty(n * k // 2, dtype=torch.uint8, device="cuda"), torch.empty(M.mxfp4_scale_bytes(n, k), dtype=torch.uint8, device="cuda")
        M.quantize_mxfp4(W, c, s)
        out.append((c, s, n, k))
    return out


def experts_ref(x, up, down, idx, w):
    """float64 forward for the routing the handle chose, and the sum of the magnitudes that a rounding can be relative to."""
    xq = R.q(x, "e2m1")
    y, mag = np.zeros(x.shape), np.zeros(x.shape)
    for e in range(len(up)):
        uq, dq = R.q(O.bf16_to_f32(O.f32_to_bf16(up[e].astype(np.float32))).astype(np.float64), "e2m1"), \
            R.q(O.bf16_to_f32(O.f32_to_bf16(down[e].astype(np.float32))).astype(np.float64), "e2m1")
        t, j = np.where(idx == e)
        if not len(t):
            continue
        p = xq[t] @ uq.T
        g = w[t, j][:, None] * (R.q(p / (1 + np.exp(-p)), "e2m1") @ dq.T)
        np.add.at(y, t, g)
        np.add.at(mag, t, np.abs(g))
    return y, mag


@pytest.mark.parametrize("T,D,H,E,K,f32,skew", [(1, 64, 64, 1, 1, False, False), (1, 128, 256, 4, 2, True, False), (64, 256, 512, 16, 2, False, False),
                                               (63, 192, 320, 8, 4, True, True), (300, 128, 64, 3, 2, True, False), (1000, 512, 192, 5, 3, False, False),
                                               (2041, 256, 128, 4, 2, True, True), (700, 64, 128, 64, 8, True, False),
                                               (6000, 1152, 1344, 5, 3, True, False), (9001, 640, 576, 16, 4, False, True),
                                               (60, 5120, 64, 4, 2, True, True), (200, 128, 1088, 48, 8, False, False), (2, 256, 192, 32, 2, False, False)])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_experts_forward(T, D, H, E, K, f32, skew, beta):
    x, wr, up, down = experts_case(T, D, H, E, K, T + D + E, skew)
    X = to_device(x, "bf16")
    Wr = to_device(wr, "f32" if f32 else "bf16")
    moe = M.MoE(T, D, E, K, hidden=H, router_dtype=M.F32 if f32 else M.BF16, training=False)
    y0 = torch.randn(T, D, device="cuda").bfloat16()
    Y = y0.clone()
    wup, wdown = quantized(up), quantized(down)
    moe.forward_mxfp4(X, Wr, wup, wdown, Y, beta)
    assert moe.device_status() == 0
    idx, w = moe.read("idx"), moe.read("w").astype(np.float64)
    logits = x @ wr.T
    np.testing.assert_array_equal(moe.read("logits").astype(np.float64), logits)
    np.testing.assert_array_equal(idx, np.argsort(-logits, 1, kind="stable")[:, :K])
    y, mag = experts_ref(x, up, down, idx, w)
    want = y + beta * exact64(y0)
    got = exact64(Y)
    # bf16 rounding of every gated row and of the sum (half a step each, 2^-8 of the magnitude), and a hidden element that lies
    # within fp32 error of a rounding border may fall to the other side: such elements are one in 10^5, so whole rows may
    # differ by one step of one element; held to the norm, as everywhere in this suite
    far = np.abs(got - want) > 2.0 ** -8 * (np.abs(want) + mag) * 1.01 + 1e-6
    assert far.mean() < 1e-2, far.mean()
    assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(np.abs(want) + mag)
    Y2 = y0.clone()
    moe.forward_mxfp4(X, Wr, M.Mxfp4Weights(wup), M.Mxfp4Weights(wdown), Y2, beta)
    assert torch.equal(Y, Y2)


def ln_case(rows, dim, seed, zero_row=True):
    rng = np.random.default_rng(seed)
    x = 0.3 + 1.2 * rng.standard_normal((rows, dim)) * np.exp(0.5 * rng.standard_normal((rows, dim // 32))).repeat(32, 1)
    if zero_row and rows > 2:
        x[1] = 0.0                                        # variance 0: rstd = 1 / sqrt(eps)
    return (to_device(x, "bf16"), to_device(0.1 * rng.standard_normal((rows, dim)), "bf16"),
            torch.from_numpy((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32)).cuda(),
            torch.from_numpy((0.2 * rng.standard_normal(dim)).astype(np.float32)).cuda())


LN_SHAPES = [(1, 32), (5, 64), (333, 96), (64, 128), (37, 160), (1, 256), (300, 288), (9, 512), (2047, 1280), (130, 2048), (33, 2080), (70, 4096), (17, 4128),
             (11, 8192), (5000, 32), (1, 8192)]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,dim", LN_SHAPES)
def test_ln_forward_act8_is_ln_forward_and_the_checkpoint_of_x(rows, dim, fmt):
    X, _, gamma, beta = ln_case(rows, dim, rows + dim)
    Y, Y0 = torch.full_like(X, 7), torch.zeros_like(X)
    mean, rstd, mean0, rstd0 = (torch.full((rows,), 7.0, device="cuda") for _ in range(4))
    codes, scales, c0, s0 = poisoned(rows * dim), poisoned(rows * dim // 32), poisoned(rows * dim), poisoned(rows * dim // 32)
    M.ln_forward_act8(X, gamma, beta, Y, mean, rstd, codes, scales, FMT8[fmt])
    M.ln_forward(X, gamma, beta, Y0, mean0, rstd0)
    M.act8_save(X, c0, s0, FMT8[fmt])
    assert torch.equal(Y, Y0) and torch.equal(mean, mean0) and torch.equal(rstd, rstd0)
    assert torch.equal(codes, c0) and torch.equal(scales, s0)


def ln_backward_ref(x, dy, gamma, mean, rstd):
    d = x.shape[1]
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * gamma
    dx = rstd[:, None] * (g - g.sum(1, keepdims=True) / d - xh * ((g * xh).sum(1, keepdims=True) / d))
    return dx, (dy * xh).sum(0), dy.sum(0), xh, g


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,dim", LN_SHAPES + [(4099, 256), (1200, 768)])
def test_ln_backward_act8_against_float64(rows, dim, fmt):
    X, dY, gamma, beta = ln_case(rows, dim, rows + dim)
    Y = torch.empty_like(X)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    codes, scales = poisoned(rows * dim), poisoned(rows * dim // 32)
    M.ln_forward_act8(X, gamma, beta, Y, mean, rstd, codes, scales, FMT8[fmt])
    dX = torch.full((rows + 1, dim), 7.0, device="cuda").bfloat16()
    dg, db = torch.full((dim,), float("nan"), device="cuda"), torch.full((dim,), float("nan"), device="cuda")
    need = M.ln_backward_act8_scratch_bytes(rows, dim)
    scratch = poisoned(need)
    M.ln_backward_act8(codes, scales, dY, gamma, mean, rstd, dX[:rows], dg, db, scratch, FMT8[fmt])
    assert (scratch[need:] == SENTINEL).all() and (dX[rows] == 7).all()
    x = R.values(codes.cpu().numpy()[:rows * dim].reshape(rows, dim), scales.cpu().numpy()[:rows * dim // 32].reshape(rows, -1), fmt)
    dy, g64, m64, r64 = exact64(dY), exact64(gamma), exact64(mean), exact64(rstd)
    dx, wg, wb, xh, g = ln_backward_ref(x, dy, g64, m64, r64)
    u = 2.0 ** -24
    # xh: rounded scale * rstd, mean * rstd and sum: 3 u of |x rstd| + |mean rstd|. Row sums: D terms, each partial sum off by u of
    # the magnitudes, and the errors of the terms. dx: those, 4 more roundings, and half a step of bf16.
    mx = (np.abs(x) + np.abs(m64)[:, None]) * r64[:, None]
    ea = (dim + 4) * u * np.abs(g).sum(1, keepdims=True) / dim
    eb = ((dim + 4) * u * (np.abs(g * xh)).sum(1, keepdims=True) + 4 * u * (np.abs(g) * mx).sum(1, keepdims=True)) / dim
    mag = r64[:, None] * (np.abs(g) + np.abs(g).sum(1, keepdims=True) / dim + mx * np.abs(g * xh).sum(1, keepdims=True) / dim)
    tol = 2.0 ** -8 * np.abs(dx) + r64[:, None] * (ea + eb * mx) + 8 * u * mag
    assert (np.abs(exact64(dX[:rows]) - dx) <= tol * 1.01).all()
    # column sums: `rows` terms, and the errors of the terms
    assert (np.abs(exact64(dg) - wg) <= (rows + 4) * u * np.abs(dy * xh).sum(0) + 4 * u * (np.abs(dy) * mx).sum(0)).all()
    assert (np.abs(exact64(db) - wb) <= (rows + 4) * u * np.abs(dy).sum(0)).all()
    again = [torch.empty_like(t) for t in (dX, dg, db)]
    M.ln_backward_act8(codes, scales, dY, gamma, mean, rstd, again[0][:rows], again[1], again[2], poisoned(need), FMT8[fmt])
    assert torch.equal(again[0][:rows], dX[:rows]) and torch.equal(again[1], dg) and torch.equal(again[2], db)


def test_many_calls_queued_on_one_stream():
    """Dense layers of every form queued without a wait between them, 20 deep and more: the same bits as one at a time."""
    torch.manual_seed(5)
    cases = []
    for rows, n, k in [(16384, 1024, 1024), (777, 512, 1024), (1, 2048, 1024), (8192, 1024, 512)]:
        wc, wsc = poisoned(n * k // 2), poisoned(M.mxfp4_scale_bytes(n, k))
        M.quantize_mxfp4(torch.randn(n, k, device="cuda"), wc, wsc)
        X = torch.randn(rows, k, device="cuda").bfloat16()
        Y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        cases.append((X, M.Mxfp4Weights([(wc, wsc, n, k)]), Y, poisoned(M.linear_mxfp4_work_bytes(rows, k))))
    want = []
    for X, W, Y, work in cases:
        M.linear_mxfp4(X, W, Y, work)
        torch.cuda.synchronize()
        want.append(Y.clone())
        Y.fill_(float("nan"))
    for depth in (3, 20, 100):
        for X, W, Y, work in cases:
            for _ in range(depth):
                M.linear_mxfp4(X, W, Y, work)
        for _ in range(depth):
            for X, W, Y, work in cases:
                M.linear_mxfp4(X, W, Y, work)
        torch.cuda.synchronize()
        for (_, _, Y, _), y in zip(cases, want):
            assert torch.equal(Y, y)
            Y.fill_(float("nan"))


def test_many_experts_passes_queued_on_one_stream():
    torch.manual_seed(6)
    T, D, H, E, K = 4096, 256, 512, 4, 2
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    up = M.Mxfp4Weights(quantized([w.numpy() for w in torch.randn(E, H, D) * 0.05]))
    down = M.Mxfp4Weights(quantized([w.numpy() for w in torch.randn(E, D, H) * 0.05]))
    Wr = (torch.randn(E, D, device="cuda") * 0.05).bfloat16()
    X = torch.randn(T, D, device="cuda").bfloat16()
    calls = [(X, torch.empty_like(X)), (X[:300], torch.empty_like(X[:300])), (X[:7], torch.empty_like(X[:7]))]      # many, some, few rows
    want = []
    for x, y in calls:
        moe.forward_mxfp4(x, Wr, up, down, y, 0.0, tokens=len(x))
        torch.cuda.synchronize()
        want.append(y.clone())
        y.zero_()
    for depth in (3, 20, 100):
        for x, y in calls:
            for _ in range(depth):
                moe.forward_mxfp4(x, Wr, up, down, y, 0.0, tokens=len(x))
        for _ in range(depth):
            for x, y in calls:
                moe.forward_mxfp4(x, Wr, up, down, y, 0.0, tokens=len(x))
        assert moe.device_status() == 0
        for (_, y), w in zip(calls, want):
            assert torch.equal(y, w)
            y.zero_()
