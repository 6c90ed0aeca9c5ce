"""Weights that the kernel right in front writes: products wait for it, also the small ones that start while it is still running."""
import pytest
import torch

import tmt_moe_b200 as M

pytestmark = pytest.mark.gpu


def raw(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def bf(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


# few rows (the product alone, values or codes), few rows against a long k, one turn of tiles, CTA pairs
@pytest.mark.parametrize("rows,n,k", [(1, 2048, 1024), (8, 520, 320), (3, 264, 4096), (300, 264, 448), (9500, 1024, 64)])
@pytest.mark.parametrize("recorded", [False, True])
def test_a_weight_is_quantised_right_before_its_product(rows, n, k, recorded):
    ws = [bf((n, k), 10 + i, 0.05) for i in range(6)]
    c, s = raw(n * k // 2), raw(M.mxfp4_scale_bytes(n, k))
    W = M.Mxfp4Weights([(c, s, n, k)])
    X, work = bf((rows, k), 1), raw(M.linear_mxfp4_work_bytes(rows, k))
    ys = [torch.zeros(rows, n, device="cuda") for _ in ws]
    want = []
    for w in ws:
        M.quantize_mxfp4(w, c, s)
        torch.cuda.synchronize()
        M.linear_mxfp4(X, W, ys[0], work)
        torch.cuda.synchronize()
        want.append(ys[0].clone())
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def turn():                                          # one buffer for all of them: each product also has to be done before the next weight
        for w, y in zip(ws, ys):
            M.quantize_mxfp4(w, c, s, stream=stream.cuda_stream)
            M.linear_mxfp4(X, W, y, work, stream=stream.cuda_stream)
    with torch.cuda.stream(stream):
        run, g = turn, None
        if recorded:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                turn()
            run = g.replay
        for _ in range(20):
            for y in ys:
                y.zero_()
            run()
            for y, w in zip(ys, want):
                assert torch.equal(y, w)
    stream.synchronize()
    del run, g


def test_experts_weights_are_quantised_right_before_the_pass():
    D, H, E, K = 256, 512, 8, 2
    masters = [[bf((E, H, D), 20 + i, 0.05), bf((E, D, H), 30 + i, 0.05)] for i in range(3)]
    bufs = [[(raw(n * k // 2), raw(M.mxfp4_scale_bytes(n, k)), n, k) for _ in range(E)] for n, k in ((H, D), (D, H))]
    up, down = (M.Mxfp4Weights(b) for b in bufs)
    Wr = bf((E, D), 2, 0.05)
    stream = torch.cuda.Stream()
    for T in (3, 40, 700):
        X, Y = bf((T, D), T), torch.zeros(T, D, device="cuda").bfloat16()
        moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=stream.cuda_stream)
        torch.cuda.synchronize()

        def fill(m):
            for product in (1, 0):                       # the up weights last: the pass reads them first
                for e in range(E):
                    M.quantize_mxfp4(m[product][e], *bufs[product][e][:2], stream=stream.cuda_stream)
        want = []
        with torch.cuda.stream(stream):
            for m in masters:
                fill(m)
                stream.synchronize()
                moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
                want.append(Y.clone())
            for _ in range(20):
                for m, w in zip(masters, want):
                    fill(m)
                    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
                    assert torch.equal(Y, w)
        stream.synchronize()
        assert moe.device_status() == 0
