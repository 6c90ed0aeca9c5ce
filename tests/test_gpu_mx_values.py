"""What a value of the microscaled operators may depend on, and how exactly it is held: sums of a token's experts, tokens in any
batch, normalised values of rows whose mean is far above their deviation."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tmt_moe_b200 as M
from oracle import oracle as O
from test_gpu_mx import FMT8, exact64, experts_case, ln_backward_ref, quantized, to_device

pytestmark = pytest.mark.gpu


def raw(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def bf(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


def wide(shape, seed, scale=1.0):
    """Blocks of many magnitudes: the sums of their products then take values all over, not a few thousand of a coarse grid."""
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    e = torch.randint(-8, 1, (*shape[:-1], shape[-1] // 32), generator=g, device="cuda").repeat_interleave(32, -1)
    return (bf(shape, seed, 2 * scale).float() * torch.exp2(e.float())).bfloat16()


def wide_weights(E, n, k, seed):
    return M.Mxfp4Weights(quantized(wide((E, n, k), seed, 0.1).float().cpu().numpy()))


def bf64(w):
    return O.bf16_to_f32(O.f32_to_bf16(np.asarray(w, np.float32))).astype(np.float64)


def experts64(x, up, down, idx, w):
    """float64 forward for the routing the handle chose, and the magnitudes that the fp32 sums of its down products run over."""
    xq = R.q(x, "e2m1")
    y, mag = np.zeros(x.shape), np.zeros(x.shape)
    for e in range(len(up)):
        t, j = np.where(idx == e)
        if not len(t):
            continue
        p = xq[t] @ R.q(bf64(up[e]), "e2m1").T
        h, dq, g = R.q(p / (1 + np.exp(-p)), "e2m1"), R.q(bf64(down[e]), "e2m1").T, w[t, j][:, None]
        np.add.at(y, t, g * (h @ dq))
        np.add.at(mag, t, g * (np.abs(h) @ np.abs(dq)))
    return y, mag


# few rows per expert, 128 x 128 tiles, CTA pairs (more than three turns of tiles)
EXPERTS = [(40, 128, 128, 16, 4), (300, 128, 64, 12, 8), (300, 320, 192, 3, 3), (9000, 512, 512, 4, 2)]


@pytest.mark.parametrize("beta", [0.0, -0.5])
@pytest.mark.parametrize("T,D,H,E,K", EXPERTS)
def test_the_experts_of_a_token_are_added_in_fp32(T, D, H, E, K, beta):
    x, wr, up, down = experts_case(T, D, H, E, K, T + K)
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    y0 = bf((T, D), 3)
    Y = y0.clone()
    moe.forward_mxfp4(to_device(x, "bf16"), to_device(wr, "bf16"), quantized(up), quantized(down), Y, beta)
    assert moe.device_status() == 0
    y, mag = experts64(x, up, down, moe.read("idx"), moe.read("w").astype(np.float64))
    want = y + beta * exact64(y0)
    # one rounding to bf16 (half a step), and in front of it H products added in fp32, then the gate, K rows and the residual
    tol = 2.0 ** -8 * np.abs(want) + (H + K + 4) * 2.0 ** -23 * (mag + np.abs(beta * exact64(y0)))
    bad = (np.abs(exact64(Y) - want) > tol).any(1)
    # An element of the hidden row that lies within fp32 error of the border between two codes may fall to the other side, which moves the
    # whole token. That error is D 2^-23 of sum |x||w|, at most about 10^-4 of a block's scale, borders are half a scale apart, a token has
    # H K elements: below 5 % of the tokens here, by the bound (far fewer in fact). Rows rounded to bf16 before they are added miss it everywhere.
    assert bad.mean() <= 0.05, bad.mean()


def test_a_token_does_not_depend_on_the_values_of_its_neighbours():
    """Every sixteenth token has pre-activations far below zero: the others keep their bits."""
    T, D, H, E, K = 65536, 256, 4096, 16, 2                          # 5 10^8 hidden elements: a last bit moves one in 10^7 to another code
    up, down = wide_weights(E, H, D, 1), wide_weights(E, D, H, 2)
    X, Wr, Y = wide((T, D), 3, 2.0), bf((E, D), 4, 0.05), torch.zeros(T, D, device="cuda").bfloat16()
    keep = torch.arange(T, device="cuda") % 16 != 5
    for tokens in (T, 300, 40):                                      # CTA pairs, tiles, few rows
        moe = M.MoE(T, D, E, K, hidden=H, training=False)
        moe.forward_mxfp4(X, Wr, up, down, Y, 0.0, tokens=tokens)
        want = Y.clone()
        big = torch.where(keep[:, None], X, X * 2048)                # the same experts: logits scaled by a power of two
        moe.forward_mxfp4(big, Wr, up, down, Y, 0.0, tokens=tokens)
        assert moe.device_status() == 0
        n = keep[:tokens]
        assert torch.equal(Y[:tokens][n], want[:tokens][n]) and not torch.equal(Y[:tokens], want[:tokens])


def test_a_token_does_not_depend_on_the_size_of_its_batch():
    """CTA pairs for the whole batch, 128 x 128 tiles and the few-row kernel for parts of it: the same bits."""
    T, D, H, E, K = 24000, 128, 4096, 16, 2
    up, down = wide_weights(E, H, D, 1), wide_weights(E, D, H, 2)
    X, Wr, want = wide((T, D), 3, 2.0), bf((E, D), 4, 0.05), torch.zeros(T, D, device="cuda").bfloat16()
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    moe.forward_mxfp4(X, Wr, up, down, want, 0.0)
    for step, n in ((300, T), (40, T), (1, 200)):
        Y = torch.zeros_like(want)
        for t in range(0, n, step):
            moe.forward_mxfp4(X[t:t + step], Wr, up, down, Y[t:t + step], 0.0, tokens=step)
        assert moe.device_status() == 0
        assert torch.equal(Y[:n], want[:n]), step


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,dim", [(5, 32), (37, 96), (130, 256), (64, 1280), (9, 4096)])
def test_a_constant_row_has_normalised_values_of_zero(rows, dim, fmt):
    """x - mean is zero, whatever x is: no rounding of mean * rstd may be left over."""
    c = np.resize([1.75, -7.0, 448.0, 1.25 * 2.0 ** 11, 1.25 * 2.0 ** -9, -1.75 * 2.0 ** 20], rows)
    X, dY = to_device(np.repeat(c[:, None], dim, 1), "bf16"), bf((rows, dim), 5)
    gamma, beta = bf((dim,), 6).float(), bf((dim,), 7).float()
    Y, dX = torch.empty_like(X), torch.empty_like(X)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    codes, scales, scratch = raw(rows * dim), raw(rows * dim // 32), raw(M.ln_backward_act8_scratch_bytes(rows, dim))
    M.ln_forward_act8(X, gamma, beta, Y, mean, rstd, codes, scales, FMT8[fmt])
    np.testing.assert_array_equal(exact64(mean), c)                  # sums of at most 4096 equal values of a few bits: exact
    rstd.fill_(300.1)                                                # as if eps were a little larger: a number of 24 bits
    top = exact64(rstd)[0]
    dg, db = torch.full((dim,), 7.0, device="cuda"), torch.empty(dim, device="cuda")
    M.ln_backward_act8(codes, scales, dY, gamma, mean, rstd, dX, dg, db, scratch, FMT8[fmt])
    assert (dg == 0).all()
    g = exact64(dY) * exact64(gamma)
    want = top * (g - g.mean(1, keepdims=True))
    # half a step of bf16; a sum of dim terms in fp32, and three more roundings
    tol = 2.0 ** -8 * np.abs(want) + top * 2.0 ** -24 * ((dim + 4) * np.abs(g).mean(1, keepdims=True) + 4 * np.abs(g))
    assert (np.abs(exact64(dX) - want) <= tol).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,dim", [(37, 96), (300, 512), (21, 2080)])
def test_layernorm_gradient_of_rows_far_from_zero(rows, dim, fmt):
    """A mean some thousand deviations away: the normalised value keeps the bits that x - mean has."""
    rng = np.random.default_rng(rows)
    x = np.repeat(np.resize([2560.0, -1792.0, 0.4375], rows)[:, None], dim, 1)          # what the checkpoint holds of such a row
    m64 = to_device(x[:, 0] * (1 + 2.0 ** -11 * rng.standard_normal(rows)), "f32")
    codes, scales = (torch.from_numpy(a).cuda().reshape(-1) for a in R.quantize(x, fmt))
    rstd = to_device(np.abs(3.0 / (x[:, 0] - exact64(m64))) * 0.3, "f32")              # xh of about 1: the statistics are an input
    dY, gamma = bf((rows, dim), 8), bf((dim,), 9).float()
    dX, dg, db = torch.empty(rows, dim, device="cuda").bfloat16(), torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    M.ln_backward_act8(codes, scales, dY, gamma, m64, rstd, dX, dg, db, raw(M.ln_backward_act8_scratch_bytes(rows, dim)), FMT8[fmt])
    dy = exact64(dY)
    dx, wg, wb, xh, g = ln_backward_ref(x, dy, exact64(gamma), exact64(m64), exact64(rstd))
    u = 2.0 ** -24
    # x - mean and its product with rstd: two roundings of xh itself; column sums of `rows` terms
    assert (np.abs(exact64(dg) - wg) <= (rows + 4) * u * np.abs(dy * xh).sum(0)).all()
    s = np.abs(g * xh).sum(1, keepdims=True) / dim
    tol = 2.0 ** -8 * np.abs(dx) + (dim + 8) * u * exact64(rstd)[:, None] * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(xh) * s)
    assert (np.abs(exact64(dX) - dx) <= tol).all()
