"""The microscaled operators as a program uses them: one after the other, on streams of its own, side by side, recorded into
graphs, with bad values in a batch, at sizes past 32 bits, and with arguments that are refused."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tmt_moe_b200 as M
from test_gpu_mx import FMT8, exact64, experts_case, experts_ref, ln_backward_ref, quantized, to_device

pytestmark = pytest.mark.gpu


def raw(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def bf(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


class Layer:
    """One linear layer with its input, output and work buffer."""

    def __init__(self, rows, n, k, seed, stream=None, out=torch.bfloat16):
        W = bf((n, k), seed, 0.05)
        c, s = raw(n * k // 2), raw(M.mxfp4_scale_bytes(n, k))
        M.quantize_mxfp4(W, c, s)
        self.W = M.Mxfp4Weights([(c, s, n, k)])
        self.X, self.Y = bf((rows, k), seed + 1), torch.zeros(rows, n, dtype=out, device="cuda")
        self.work, self.stream = raw(M.linear_mxfp4_work_bytes(rows, k)), stream
        torch.cuda.synchronize()

    def run(self):
        M.linear_mxfp4(self.X, self.W, self.Y, self.work, stream=self.stream)
        return self.Y

    def value(self):
        """A copy of what a call gives: the copy runs on another stream than the call, so it waits."""
        self.run()
        torch.cuda.synchronize()
        return self.Y.clone()


FORMS = [(5, 520, 320), (3, 264, 2112), (300, 264, 448), (9500, 512, 64)]          # few rows, few against a long k, some, many


class Decoder:
    """LayerNorm with checkpoint -> experts with residual -> head, and the LayerNorm's gradient from the checkpoint."""

    def __init__(self, T, D, H, E, K, V, stream):
        self.stream = stream
        self.X, self.dY = bf((T, D), 1), bf((T, D), 2, 0.1)
        self.gamma, self.beta = 1 + 0.1 * bf((D,), 3).float(), 0.1 * bf((D,), 4).float()
        self.N, self.R, self.dX = torch.empty_like(self.X), torch.empty_like(self.X), torch.empty_like(self.X)
        self.mean, self.rstd = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        self.codes, self.scales = raw(T * D), raw(T * D // 32)
        self.Wr = bf((E, D), 5, 0.05)
        self.w64 = [w.numpy() for w in torch.randn(E, H, D, generator=torch.Generator().manual_seed(6)) * 0.05], \
                   [w.numpy() for w in torch.randn(E, D, H, generator=torch.Generator().manual_seed(7)) * 0.05]
        self.up, self.down = (M.Mxfp4Weights(quantized(w)) for w in self.w64)
        self.moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=stream.cuda_stream)
        hc, hs = raw(V * D // 2), raw(M.mxfp4_scale_bytes(V, D))
        self.Wh = bf((V, D), 8, 0.05)
        M.quantize_mxfp4(self.Wh, hc, hs)
        self.head = M.Mxfp4Weights([(hc, hs, V, D)])
        self.L = torch.empty(T, V, device="cuda")
        self.work = raw(M.linear_mxfp4_work_bytes(T, D))
        self.B, self.dg, self.db = torch.empty_like(self.X), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
        self.scratch = raw(M.ln_backward_act8_scratch_bytes(T, D))
        torch.cuda.synchronize()

    def run(self):
        s = self.stream.cuda_stream
        M.ln_forward_act8(self.X, self.gamma, self.beta, self.N, self.mean, self.rstd, self.codes, self.scales, stream=s)
        self.R.copy_(self.X)
        self.moe.forward_mxfp4(self.N, self.Wr, self.up, self.down, self.R, 1.0)
        M.linear_mxfp4(self.R, self.head, self.L, self.work, stream=s)
        M.act8_restore(self.codes, self.scales, self.B, stream=s)
        M.ln_backward_act8(self.codes, self.scales, self.dY, self.gamma, self.mean, self.rstd, self.dX, self.dg, self.db, self.scratch, stream=s)

    def outputs(self):
        return [self.N, self.R, self.L, self.B, self.dX, self.dg, self.db]


@pytest.mark.parametrize("T,D,H,E,K,V", [(3, 128, 192, 4, 2, 264), (90, 256, 128, 4, 2, 320), (2500, 320, 320, 6, 3, 520)])
def test_the_operators_in_a_row(T, D, H, E, K, V):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        m = Decoder(T, D, H, E, K, V, stream)
        m.run()
    stream.synchronize()
    assert m.moe.device_status() == 0
    # every stage against float64, from what the stage before it left
    x = exact64(m.X)
    mu = x.mean(1)
    rs = 1 / np.sqrt((x * x).mean(1) - mu * mu + 1e-5)
    want = (x - mu[:, None]) * rs[:, None] * exact64(m.gamma) + exact64(m.beta)
    # fp32 sums of D terms (error D 2^-24 relative to the magnitudes, which the variance subtracts), and half a step of bf16
    assert (np.abs(exact64(m.N) - want) <= 2.0 ** -8 * np.abs(want) + 4 * D * 2.0 ** -24 * (1 + np.abs(x) * rs[:, None])).all()
    n = exact64(m.N)
    y, mag = experts_ref(n, *(np.asarray(w, np.float64) for w in m.w64), m.moe.read("idx"), m.moe.read("w").astype(np.float64))
    r = exact64(m.R)
    assert np.linalg.norm(r - (x + y)) <= 2.0 ** -8 * np.linalg.norm(np.abs(x + y) + mag)
    a, w = R.q(r, "e2m1"), R.q(exact64(m.Wh), "e2m1")
    assert (np.abs(m.L.double().cpu().numpy() - a @ w.T) <= D * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)).all()
    back = R.q(x, "e4m3")
    np.testing.assert_array_equal(exact64(m.B), exact64(to_device(back, "bf16")))
    dx, dg, db, _, _ = ln_backward_ref(back, exact64(m.dY), exact64(m.gamma), exact64(m.mean), exact64(m.rstd))
    assert np.linalg.norm(exact64(m.dX) - dx) <= 2.0 ** -8 * np.linalg.norm(dx)
    assert np.linalg.norm(exact64(m.dg) - dg) <= (T + D) * 2.0 ** -23 * np.linalg.norm(np.abs(dg) + 1)
    assert np.linalg.norm(exact64(m.db) - db) <= (T + D) * 2.0 ** -23 * np.linalg.norm(np.abs(db) + 1)


@pytest.mark.parametrize("T", [3, 90, 2500])
def test_recorded_and_replayed_it_gives_the_same_bits(T):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        m = Decoder(T, 320, 192, 6, 3, 264, stream)
        m.run()
        eager = [t.clone() for t in m.outputs()]
        X1 = m.X.clone()
        m.X.copy_(bf(m.X.shape, 77))
        m.run()
        eager2 = [t.clone() for t in m.outputs()]
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            m.run()
        for X, want in ((X1, eager), (bf(m.X.shape, 77), eager2), (X1, eager)):
            m.X.copy_(X)
            for t in m.outputs():
                t.zero_()
            g.replay()
            stream.synchronize()
            for t, w in zip(m.outputs(), want):
                assert torch.equal(t, w)
    assert m.moe.device_status() == 0
    del g


def test_a_graph_keeps_the_weights_it_was_recorded_with():
    stream = torch.cuda.Stream()
    T, D, H, E, K = 200, 128, 192, 4, 2
    with torch.cuda.stream(stream):
        sets = [(M.Mxfp4Weights(quantized(torch.randn(E, H, D).numpy() * 0.05)), M.Mxfp4Weights(quantized(torch.randn(E, D, H).numpy() * 0.05)))
                for _ in range(3)]
        X, Wr, Y = bf((T, D), 1), bf((E, D), 2, 0.05), torch.empty(T, D, device="cuda").bfloat16()
        moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=stream.cuda_stream)
        stream.synchronize()

        def eager(i):
            moe.forward_mxfp4(X, Wr, *sets[i], Y, 0.0)
            return Y.clone()

        def record(i):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                Y.zero_()
                moe.forward_mxfp4(X, Wr, *sets[i], Y, 0.0)
            return g

        # the first call of a handle, and new weights, cannot be recorded; the capture goes on without them
        def refused(i):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                Y.zero_()
                with pytest.raises(M.MoeError, match="recorded"):
                    moe.forward_mxfp4(X, Wr, *sets[i], Y, 0.0)
        refused(0)
        want = [eager(0)]
        g0 = record(0)
        refused(1)
        want.append(eager(1))
        assert not torch.equal(want[0], want[1])
        g1 = record(1)
        want.append(eager(2))
        for g, w in ((g0, want[0]), (g1, want[1]), (g0, want[0])):
            Y.zero_()
            g.replay()
            assert torch.equal(Y, w)
            assert torch.equal(eager(2), want[2])
        # other contents at the same addresses are what the next call multiplies
        for (c, s, n, k) in sets[2][0]._keep:
            c.copy_(torch.randint(0, 256, (c.numel(),), device="cuda", dtype=torch.uint8))
        changed = eager(2)
        assert not torch.equal(changed, want[2])
        fresh = M.MoE(T, D, E, K, hidden=H, training=False, stream=stream.cuda_stream)
        fresh.forward_mxfp4(X, Wr, *sets[2], Y, 0.0)
        assert torch.equal(Y, changed)
    stream.synchronize()
    del g0, g1


@pytest.mark.parametrize("rows,n,k", FORMS)
def test_on_a_stream_of_its_own_an_operator_waits_for_that_stream(rows, n, k):
    stream = torch.cuda.Stream()
    layer = Layer(rows, n, k, 11, stream.cuda_stream)
    fresh = bf(layer.X.shape, 5)
    torch.cuda.synchronize()
    want0 = layer.value()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        layer.X.copy_(fresh)
        layer.run()
        got = layer.Y.clone()
        layer.Y.zero_()
    stream.synchronize()
    layer.X.copy_(fresh)
    layer.stream = None
    torch.cuda.synchronize()
    assert torch.equal(got, layer.run()) and not torch.equal(got, want0)


def test_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    layers = [[Layer(*f, 20 + i, s.cuda_stream) for i, f in enumerate(FORMS)] for s in streams]
    want = [[l.value() for l in ls] for ls in layers]
    torch.cuda.synchronize()
    for ls in layers:
        for l in ls:
            l.Y.zero_()
    torch.cuda.synchronize()
    for turn in range(30):
        for i in range(len(FORMS)):
            layers[0][i].run()
            layers[1][(i + turn) % len(FORMS)].run()
    torch.cuda.synchronize()
    for ls, ws in zip(layers, want):
        for l, w in zip(ls, ws):
            assert torch.equal(l.Y, w)


def test_two_graphs_may_share_a_work_buffer():
    stream = torch.cuda.Stream()
    a, b = Layer(300, 264, 448, 1, stream.cuda_stream), Layer(290, 136, 448, 2, stream.cuda_stream)
    b.work = a.work
    with torch.cuda.stream(stream):
        want = [a.run().clone(), b.run().clone()]
        stream.synchronize()
        graphs = []
        for l in (a, b):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                l.run()
        for order in ((0, 1), (1, 0), (0, 0, 1, 1, 0)):
            a.Y.zero_(), b.Y.zero_(), a.work.fill_(0xA5)
            for i in order:
                graphs[i].replay()
            assert torch.equal(a.Y, want[0]) and torch.equal(b.Y, want[1])
    stream.synchronize()
    del graphs


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("rows,n,k", FORMS)
def test_a_bad_value_stays_in_its_row_of_a_product(rows, n, k, bad):
    layer = Layer(rows, n, k, 3)
    want = layer.run().clone()
    hit = sorted({0, rows // 2, rows - 1})
    for r in hit[1:]:
        layer.X[r, (r * 37) % k] = bad
    got = layer.run()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[hit[1:]] = False
    assert torch.equal(got[keep], want[keep]) and got[~keep].isnan().all()
    # a bad weight: its column alone
    c, s, _, _ = layer.W._keep[0]
    W = bf((n, k), 3, 0.05)
    W[n - 2, k - 1] = bad
    M.quantize_mxfp4(W, c, s)
    got = layer.run()
    cols = torch.arange(n, device="cuda") != n - 2
    assert torch.equal(got[keep][:, cols], want[keep][:, cols]) and got[:, n - 2].isnan().all()


@pytest.mark.parametrize("T", [3, 90, 2500])
def test_a_bad_token_of_a_batch_leaves_the_others_alone(T):
    D, H, E, K = 128, 192, 4, 2
    up, down = quantized(torch.randn(E, H, D).numpy() * 0.05), quantized(torch.randn(E, D, H).numpy() * 0.05)
    X, Wr, Y = bf((T, D), 1), bf((E, D), 2, 0.05), torch.zeros(T, D, device="cuda").bfloat16()
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    want = Y.clone()
    X[T // 2, 5] = float("nan")
    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    assert moe.device_status() == 0
    idx = np.sort(moe.read("idx"), 1)
    assert (idx[:, 1:] > idx[:, :-1]).all() and idx.min() >= 0 and idx.max() < E          # different experts, the bad token's too
    keep = torch.arange(T, device="cuda") != T // 2
    # the bad token moves others within their groups, which changes no sum of theirs
    assert torch.equal(Y[keep], want[keep]) and Y[T // 2].isnan().all()


def test_a_batch_padded_behind_its_last_token_stays_untouched():
    D, H, E, K = 128, 192, 4, 2
    up, down = quantized(torch.randn(E, H, D).numpy() * 0.05), quantized(torch.randn(E, D, H).numpy() * 0.05)
    X, Wr = bf((3000, D), 1), bf((E, D), 2, 0.05)
    moe = M.MoE(3000, D, E, K, hidden=H, training=False)
    for T in (1, 17, 31, 257, 2500):
        Y = torch.full((3000, D), 7.0, device="cuda").bfloat16()
        moe.forward_mxfp4(X, Wr, up, down, Y, 0.0, tokens=T)
        alone = M.MoE(T, D, E, K, hidden=H, training=False)
        Z = torch.empty(T, D, device="cuda").bfloat16()
        alone.forward_mxfp4(X[:T], Wr, up, down, Z, 0.0)
        assert (Y[T:] == 7).all() and torch.equal(Y[:T], Z)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_layernorm_gradient_against_differences(fmt):
    rows, dim = 4, 96
    rng = np.random.default_rng(9)
    x0 = R.q(0.5 + rng.standard_normal((rows, dim)), fmt)          # values the checkpoint holds exactly
    X, dY = to_device(x0, "bf16"), to_device(0.3 * rng.standard_normal((rows, dim)), "bf16")
    assert np.array_equal(exact64(X), x0)
    gamma, beta = to_device(1 + 0.2 * rng.standard_normal(dim), "f32"), to_device(0.2 * rng.standard_normal(dim), "f32")
    Y, dX = torch.empty_like(X), torch.empty_like(X)
    mean, rstd, dg, db = (torch.empty(n, device="cuda") for n in (rows, rows, dim, dim))
    codes, scales, scratch = raw(rows * dim), raw(rows * dim // 32), raw(M.ln_backward_act8_scratch_bytes(rows, dim))
    M.ln_forward_act8(X, gamma, beta, Y, mean, rstd, codes, scales, FMT8[fmt])
    M.ln_backward_act8(codes, scales, dY, gamma, mean, rstd, dX, dg, db, scratch, FMT8[fmt])
    dy, ga, be = exact64(dY), exact64(gamma), exact64(beta)

    def loss(x, ga=ga, be=be):                                      # per row; a row's gradient depends on that row alone
        mu = x.mean(1, keepdims=True)
        return (dy * ((x - mu) / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + 1e-5) * ga + be)).sum(1)

    def difference(h):
        out = np.empty((rows, dim))
        for i in range(dim):
            e = np.zeros((1, dim))
            e[0, i] = h
            out[:, i] = (loss(x0 + e) - loss(x0 - e)) / (2 * h)
        return out
    d1, d2 = difference(2e-3), difference(1e-3)
    # a central difference is off by c h^2: |d1 - d2| = 3 c h^2 bounds the error of d2; its own rounding is 2^-50 |loss| / h.
    # The kernel: half a step of bf16, and fp32 sums of dim terms in front of it (statistics of the forward pass included).
    xh = (x0 - x0.mean(1, keepdims=True)) / x0.std(1, keepdims=True)
    g = np.abs(dy * ga)
    mag = (g + g.mean(1, keepdims=True) + np.abs(xh) * (g * np.abs(xh)).mean(1, keepdims=True)) / x0.std(1, keepdims=True)
    tol = 2.0 ** -8 * np.abs(d2) + np.abs(d1 - d2) + 1e-9 + 4 * dim * 2.0 ** -24 * mag
    assert (np.abs(exact64(dX) - d2) <= tol).all()
    for got, kw in ((dg, "ga"), (db, "be")):                        # the loss is linear in gamma and beta: differences are exact
        base = {"ga": ga, "be": be}[kw]
        want = np.array([(loss(x0, **{kw: base + np.eye(dim)[i]}) - loss(x0, **{kw: base - np.eye(dim)[i]})).sum() / 2 for i in range(dim)])
        scale = np.abs(dy * xh).sum(0) if kw == "ga" else np.abs(dy).sum(0)
        assert (np.abs(exact64(got) - want) <= 4 * (dim + rows) * 2.0 ** -24 * (scale + np.abs(dy).sum(0)) + 1e-12).all()


def test_empty_batches_do_nothing():
    X, Y = torch.empty(0, 128, device="cuda").bfloat16(), torch.empty(0, 16, device="cuda")
    e = torch.empty(0, dtype=torch.uint8, device="cuda")
    c, s = raw(16 * 64), raw(M.mxfp4_scale_bytes(16, 128))
    f0, g = torch.empty(0, device="cuda"), torch.ones(128, device="cuda")
    M.quantize_mxfp4(X, e, e)
    M.dequantize_mxfp4(e, e, X)
    M.linear_mxfp4(X, (c, s, 16, 128), Y, e)
    M.matmul_mxfp4(e, e, (c, s, 16, 128), Y)
    M.act8_save(X, e, e)
    M.act8_restore(e, e, X)
    M.ln_forward_act8(X, g, g, X, f0, f0, e, e)
    torch.cuda.synchronize()


def test_calls_that_are_refused():
    L = Layer(300, 264, 448, 1)
    c, s, n, k = L.W._keep[0]
    odd = torch.empty(300 * 448 + 8, device="cuda").bfloat16()[1:300 * 448 + 1].view(300, 448)
    host = torch.empty(300, 448).bfloat16()
    T, D = 300, 64
    ln = [bf((T, D), 1), torch.ones(D, device="cuda"), torch.ones(D, device="cuda"), bf((T, D), 2), torch.empty(T, device="cuda"), torch.empty(T, device="cuda"),
          raw(T * D), raw(T * D // 32)]
    moe = M.MoE(8, 64, 2, 1, hidden=64, training=False)
    up = quantized(torch.randn(2, 64, 64).numpy())
    x8, wr = bf((8, 64), 1), bf((2, 64), 2)
    bad = [
        ("boundary", lambda: M.linear_mxfp4(odd, L.W, L.Y, L.work)),
        ("host", lambda: M.linear_mxfp4(host, L.W, L.Y, L.work)),
        ("host", lambda: M.linear_mxfp4(host.pin_memory(), L.W, L.Y, L.work)),
        ("work", lambda: M.linear_mxfp4(L.X, L.W, L.Y, L.work[:-1])),
        ("boundary", lambda: M.linear_mxfp4(L.X, L.W, L.Y, torch.cat([L.work, L.work])[4:])),
        ("int32", lambda: M.linear_mxfp4(L.X, L.W, L.Y, L.work, status=torch.zeros(1, device="cuda"))),
        ("host", lambda: M.linear_mxfp4(L.X, L.W, L.Y, L.work, status=torch.zeros(1, dtype=torch.int32))),
        ("boundary", lambda: M.quantize_mxfp4(odd, raw(300 * 224), raw(M.mxfp4_scale_bytes(300, 448)))),
        ("host", lambda: M.act8_save(host, raw(300 * 448), raw(300 * 14))),
        ("host", lambda: M.act8_restore(raw(300 * 448), raw(300 * 14), host)),
        ("host", lambda: M.ln_forward_act8(ln[0].cpu(), *ln[1:])),
        ("format", lambda: M.ln_forward_act8(*ln, fmt=3)),
        ("host", lambda: M.ln_backward_act8(ln[6], ln[7], ln[3], ln[1], ln[4].cpu(), ln[5], ln[0], ln[1], ln[2], raw(M.ln_backward_act8_scratch_bytes(T, D)))),
        ("per expert", lambda: moe.forward_mxfp4(x8, wr, up[:1], up, x8, 0.0)),
        ("shape", lambda: moe.forward_mxfp4(x8, wr, quantized(torch.randn(2, 128, 64).numpy()), up, bf((8, 64), 3), 0.0)),
        ("host", lambda: moe.forward_mxfp4(x8.cpu(), wr, up, up, bf((8, 64), 3), 0.0)),
        ("tokens", lambda: moe.forward_mxfp4(bf((9, 64), 1), wr, up, up, bf((9, 64), 3), 0.0, tokens=9)),
        ("training", lambda: M.MoE(8, 64, 2, 1, hidden=64, training=True).forward_mxfp4(x8, wr, up, up, bf((8, 64), 3), 0.0)),
    ]
    for word, call in bad:
        with pytest.raises(M.MoeError, match=word):
            call()
    torch.cuda.synchronize()
    assert L.run().isfinite().all()


def test_matrices_past_32_bits():
    rows, cols = (1 << 21) + 37, 1088                               # 2.28e9 elements
    block = bf((4099, cols), 1)
    X = block.repeat(-(-rows // 4099), 1)[:rows].contiguous()
    probe = np.array([0, (1 << 31) // cols, (1 << 31) // cols + 1, rows - 130, rows - 1])
    part = exact64(X[probe])
    codes, scales = raw(rows * cols // 2), raw(M.mxfp4_scale_bytes(rows, cols))
    M.quantize_mxfp4(X, codes, scales)
    wc, ws = R.quantize(part, "e2m1")
    np.testing.assert_array_equal(codes.view(rows, -1)[probe].cpu().numpy(), R.pack4(wc))
    Y = torch.empty_like(X)
    M.dequantize_mxfp4(codes, scales, Y)
    np.testing.assert_array_equal(exact64(Y[probe]), R.values(wc, ws, "e2m1"))
    c8, s8 = raw(rows * cols), raw(rows * cols // 32)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    gamma, beta = torch.rand(cols, device="cuda") + 0.5, torch.rand(cols, device="cuda")
    M.ln_forward_act8(X, gamma, beta, Y, mean, rstd, c8, s8)
    wc, ws = R.quantize(part, "e4m3")
    np.testing.assert_array_equal(c8.view(rows, -1)[probe].cpu().numpy(), wc)
    np.testing.assert_array_equal(s8.view(rows, -1)[probe].cpu().numpy(), ws)
    small = [torch.empty(4099, cols, device="cuda").bfloat16(), torch.empty(4099, device="cuda"), torch.empty(4099, device="cuda")]
    M.ln_forward(block, gamma, beta, *small)
    where = torch.from_numpy(probe).cuda()
    assert torch.equal(Y[where], small[0][where % 4099]) and torch.equal(rstd[where], small[2][where % 4099])
    dX, dg, db = torch.empty_like(X), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    M.ln_backward_act8(c8, s8, Y, gamma, mean, rstd, dX, dg, db, raw(M.ln_backward_act8_scratch_bytes(rows, cols)))
    want = ln_backward_ref(R.values(wc, ws, "e4m3"), exact64(Y[where]), exact64(gamma), exact64(mean[where]), exact64(rstd[where]))[0]
    assert np.linalg.norm(exact64(dX[where]) - want) <= 2.0 ** -8 * np.linalg.norm(want)
    M.act8_restore(c8, s8, X)
    np.testing.assert_array_equal(exact64(X[where]), exact64(to_device(R.values(wc, ws, "e4m3"), "bf16")))


def test_a_product_whose_output_passes_32_bits():
    rows, n, k = (1 << 21) + 37, 1088, 64
    layer = Layer(rows, n, k, 5)
    layer.run()
    probe = torch.tensor([0, (1 << 31) // n, (1 << 31) // n + 1, rows - 200, rows - 1], device="cuda")
    few = Layer(5, n, k, 5)
    few.X.copy_(layer.X[probe])
    assert torch.equal(layer.Y[probe], few.run())


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n,k", [(1, 1024, 4096), (2, 8, 8192), (3, 264, 2112), (5, 2504, 1792), (7, 4104, 4096), (16, 128, 2048), (31, 520, 1856), (32, 1024, 4096)])
def test_few_rows_against_a_long_k(rows, n, k, out):
    layer = Layer(rows, n, k, rows, out=out)
    layer.Y = torch.full((rows + 1, n), 7.0, dtype=out, device="cuda")[:rows]
    got = layer.run().clone()
    c, s, _, _ = layer.W._keep[0]
    wv = torch.empty(n, k, device="cuda")
    M.dequantize_mxfp4(c, s, wv)
    a, w = R.q(exact64(layer.X), "e2m1"), exact64(wv)
    want, tol = a @ w.T, k * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)        # additions in fp32, then one rounding
    tol = tol + (2.0 ** -8 * np.abs(want) if out == torch.bfloat16 else 0)
    assert (np.abs(exact64(got) - want) <= tol * 1.01).all()
    for _ in range(3):
        assert torch.equal(layer.run(), got)
    assert (layer.Y._base[rows] == 7).all()
    # the product of the same codes
    codes, scales, Y = raw(rows * k // 2), raw(M.mxfp4_scale_bytes(rows, k)), torch.empty_like(got)
    M.quantize_mxfp4(layer.X, codes, scales)
    M.matmul_mxfp4(codes, scales, layer.W, Y)
    assert torch.equal(Y, got)


@pytest.mark.parametrize("T,D,H,E,K", [(60, 256, 512, 16, 2), (100, 192, 64, 13, 1), (40, 5120, 64, 16, 2), (25, 64, 4224, 16, 2), (2000, 192, 128, 8, 2)])
def test_most_tokens_pick_the_same_expert(T, D, H, E, K):
    """One expert has most of the rows, more than a pass of the few-row product takes, the others few or none."""
    x, wr, up, down = experts_case(T, D, H, E, K, T)
    x[:, 0], wr[:, 0], wr[E - 1, 0] = 4.0, 0.0, 2.0
    X, Wr, Y = to_device(x, "bf16"), to_device(wr, "bf16"), torch.zeros(T, D, device="cuda").bfloat16()
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    moe.forward_mxfp4(X, Wr, quantized(up), quantized(down), Y, 0.0)
    assert moe.device_status() == 0
    idx, w = moe.read("idx"), moe.read("w").astype(np.float64)
    # the other logits have a deviation of about 0.05 sqrt(D): at the longest rows some of them pass this expert's 8
    assert (idx[:, 0] == E - 1).mean() > 0.5
    y, mag = experts_ref(x, up, down, idx, w)
    assert np.linalg.norm(exact64(Y) - y) <= 2.0 ** -8 * np.linalg.norm(np.abs(y) + mag)


def test_every_form_recorded_side_by_side_and_replayed():
    """The layers fork onto two streams inside one recording and join again."""
    side = [torch.cuda.Stream() for _ in range(2)]
    layers = [Layer(*f, 40 + i, s.cuda_stream) for s in side for i, f in enumerate(FORMS)]
    want = [l.value() for l in layers]
    torch.cuda.synchronize()
    main, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(main):
        with torch.cuda.graph(g, stream=main):
            for s in side:
                s.wait_stream(main)
            for _ in range(3):
                for l in layers:
                    l.run()
            for s in side:
                main.wait_stream(s)
        for _ in range(5):
            for l in layers:
                l.Y.zero_()
            g.replay()
            for l, w in zip(layers, want):
                assert torch.equal(l.Y, w)
    main.synchronize()
    del g


def test_handles_of_two_streams_at_once():
    D, H, E, K = 256, 192, 4, 2
    up, down = M.Mxfp4Weights(quantized(torch.randn(E, H, D).numpy() * 0.05)), M.Mxfp4Weights(quantized(torch.randn(E, D, H).numpy() * 0.05))
    Wr = bf((E, D), 2, 0.05)
    runs = []
    for i, T in enumerate((7, 300, 2500, 9)):
        s = torch.cuda.Stream()
        moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=s.cuda_stream)
        runs.append((moe, bf((T, D), 30 + i), torch.zeros(T, D, device="cuda").bfloat16()))
    torch.cuda.synchronize()
    want = []
    for moe, X, Y in runs:
        moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
        assert moe.device_status() == 0
        want.append(Y.clone())
        torch.cuda.synchronize()
        Y.zero_()
    torch.cuda.synchronize()
    for _ in range(30):
        for moe, X, Y in runs:
            moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    torch.cuda.synchronize()
    for (moe, _, Y), w in zip(runs, want):
        assert moe.device_status() == 0 and torch.equal(Y, w)


def test_a_long_mixed_queue_on_three_streams():
    """Thousands of products of every form, CTA pairs among them, dense on two streams and grouped on a third, without a wait in between."""
    rng = np.random.default_rng(3)
    side = [torch.cuda.Stream() for _ in range(2)]
    shapes = [(1, 2048, 1024), (2, 1024, 4096), (777, 520, 448), (4096, 2048, 2048), (9500, 1024, 64)]
    layers = [[Layer(*f, 60 + i, s.cuda_stream) for i, f in enumerate(shapes)] for s in side]
    want = [[l.value() for l in ls] for ls in layers]
    s = torch.cuda.Stream()
    T, D, H, E, K = 6000, 256, 512, 16, 4
    moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=s.cuda_stream)
    up, down = M.Mxfp4Weights(quantized(torch.randn(E, H, D).numpy() * 0.05)), M.Mxfp4Weights(quantized(torch.randn(E, D, H).numpy() * 0.05))
    X, Wr, Y = bf((T, D), 1), bf((E, D), 2, 0.05), torch.zeros(T, D, device="cuda").bfloat16()
    torch.cuda.synchronize()
    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    torch.cuda.synchronize()
    y = Y.clone()
    torch.cuda.synchronize()
    for _ in range(10):
        for _ in range(400):
            i = rng.integers(0, 11)
            if i == 10:
                moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
            else:
                layers[i % 2][i // 2].run()
        torch.cuda.synchronize()
        assert moe.device_status() == 0 and torch.equal(Y, y)
        for ls, ws in zip(layers, want):
            for l, w in zip(ls, ws):
                assert torch.equal(l.Y, w)
                l.Y.zero_()
        Y.zero_()
        torch.cuda.synchronize()
        for ls in layers:
            for l in ls:
                l.run()
        moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
