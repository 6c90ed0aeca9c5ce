"""Every kernel of the 4-bit products as a program uses them. Which kernel a shape takes is asked of the library, so that a rule that moves
fails here instead of leaving a kernel untested."""
import pytest
import torch

import test_gpu_mx as B
import test_gpu_mx_use as U
import tmt_moe_b200 as M

pytestmark = pytest.mark.gpu

PAIRS = [(9500, 1024, 64), (2300, 4104, 320), (4096, 2056, 64), (5000, 1544, 1344), (2049, 4096, 2048)]
FORMS = [(5, 520, 320), (3, 264, 2112), (300, 264, 448), (9500, 1024, 64)]
TAKES = [M.MXFP4_FEW_ROWS, M.MXFP4_FEW_ROWS, M.MXFP4_TILES, M.MXFP4_PAIRS]


@pytest.fixture(autouse=True)
def forms():
    assert [M.linear_mxfp4_form(*f) for f in FORMS] == TAKES
    assert {M.linear_mxfp4_form(*f) for f in PAIRS} == {M.MXFP4_PAIRS}


def experts_take(form, T, D, H, E, K):
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    assert [moe.forward_mxfp4_form(p) for p in (0, 1)] == [form, form]


def test_what_the_library_says_of_a_shape():
    assert M.linear_mxfp4_form(1, 2048, 1024) == M.MXFP4_FEW_ROWS and M.linear_mxfp4_form(16384, 4096, 1024) == M.MXFP4_PAIRS
    for bad in ((0, 8, 64), (4, 12, 64), (4, 8, 96)):
        with pytest.raises(M.MoeError):
            M.linear_mxfp4_form(*bad)
    moe = M.MoE(64, 1024, 16, 2, hidden=2048, training=False)
    assert moe.forward_mxfp4_form(0) == M.MXFP4_FEW_ROWS
    for product, tokens in ((2, 4), (-1, 4), (0, 0), (0, 65)):
        with pytest.raises(M.MoeError):
            moe.forward_mxfp4_form(product, tokens)
    with pytest.raises(M.MoeError, match="training"):
        M.MoE(64, 64, 2, 1, hidden=64, training=True).forward_mxfp4_form(0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n,k", PAIRS)
def test_pairs_are_exact_where_fp32_is(rows, n, k, dtype):
    B.test_matmul_is_exact_where_fp32_is(rows, n, k, dtype)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("rows,n,k", [PAIRS[0], PAIRS[3]])
def test_a_bad_value_stays_in_its_row_and_column_of_a_pairs_tile(rows, n, k, bad):
    U.test_a_bad_value_stays_in_its_row_of_a_product(rows, n, k, bad)


@pytest.mark.parametrize("col", [0, 63, 64, 191, 192, 255, 256, 700])
def test_a_bad_weight_leaves_the_columns_of_both_accumulators_alone(col):
    """The accumulators of a pair share 64 columns: 192 .. 255 of one tile are the first columns of the next."""
    rows, n, k = PAIRS[0]
    layer = U.Layer(rows, n, k, 3)
    want = layer.run().clone()
    c, s, _, _ = layer.W._keep[0]
    W = U.bf((n, k), 3, 0.05)
    W[col, 7] = float("nan")
    M.quantize_mxfp4(W, c, s)
    got = layer.run()
    keep = torch.arange(n, device="cuda") != col
    assert torch.equal(got[:, keep], want[:, keep]) and got[:, col].isnan().all()


def test_pairs_wait_for_the_stream_they_are_given():
    U.test_on_a_stream_of_its_own_an_operator_waits_for_that_stream(*PAIRS[0])


def test_every_form_on_two_streams_at_once(monkeypatch):
    monkeypatch.setattr(U, "FORMS", FORMS)
    U.test_two_streams_at_once()


def test_every_form_recorded_side_by_side(monkeypatch):
    monkeypatch.setattr(U, "FORMS", FORMS)
    U.test_every_form_recorded_side_by_side_and_replayed()


@pytest.mark.parametrize("rows,n,k", [PAIRS[0], PAIRS[1]])
def test_pairs_recorded_alone(rows, n, k):
    stream = torch.cuda.Stream()
    layer = U.Layer(rows, n, k, 9, stream.cuda_stream)
    want = layer.value()
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            layer.run()
        for _ in range(5):
            layer.Y.zero_()
            g.replay()
            assert torch.equal(layer.Y, want)
    stream.synchronize()
    del g


def test_the_operators_in_a_row_on_pairs():
    T, D, H, E, K, V = 9000, 320, 320, 6, 3, 1032
    experts_take(M.MXFP4_PAIRS, T, D, H, E, K)
    assert M.linear_mxfp4_form(T, V, D) == M.MXFP4_PAIRS
    U.test_the_operators_in_a_row(T, D, H, E, K, V)


def test_recorded_and_replayed_on_pairs():
    experts_take(M.MXFP4_PAIRS, 9800, 320, 192, 6, 3)
    U.test_recorded_and_replayed_it_gives_the_same_bits(9800)


@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_a_bad_token_of_a_batch_on_pairs(bad):
    T, D, H, E, K = 15000, 256, 256, 4, 2
    experts_take(M.MXFP4_PAIRS, T, D, H, E, K)
    up, down = (M.Mxfp4Weights(B.quantized(U.bf(shape, 1, 0.05).float().cpu().numpy())) for shape in ((E, H, D), (E, D, H)))
    X, Wr, Y = U.bf((T, D), 1), U.bf((E, D), 2, 0.05), torch.zeros(T, D, device="cuda").bfloat16()
    moe = M.MoE(T, D, E, K, hidden=H, training=False)
    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    want = Y.clone()
    hit = [0, 77, T // 2, T - 1]
    for t in hit:
        X[t, (5 * t) % D] = bad
    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    assert moe.device_status() == 0
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[hit] = False
    assert torch.equal(Y[keep], want[keep]) and Y[~keep].isnan().all()


def test_a_replay_reads_weights_that_the_caller_has_dropped():
    """Lists handed in directly: the handle keeps those that a graph was recorded with."""
    stream = torch.cuda.Stream()
    T, D, H, E, K = 200, 128, 192, 4, 2

    def weights(seed):
        return [B.quantized(U.bf(shape, seed, 0.05).float().cpu().numpy()) for shape in ((E, H, D), (E, D, H))]
    with torch.cuda.stream(stream):
        X, Wr, Y = U.bf((T, D), 1), U.bf((E, D), 2, 0.05), torch.empty(T, D, device="cuda").bfloat16()
        moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=stream.cuda_stream)
        w = weights(3)
        moe.forward_mxfp4(X, Wr, *w, Y, 0.0)
        want = Y.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            moe.forward_mxfp4(X, Wr, *w, Y, 0.0)
        del w
        other = weights(4)
        moe.forward_mxfp4(X, Wr, *other, Y, 0.0)
        assert not torch.equal(Y, want)
        junk = [torch.full((n * k // 2,), 0x77, dtype=torch.uint8, device="cuda") for n, k in ((H, D), (D, H)) for _ in range(4 * E)]      # takes freed memory
        g.replay()
        assert torch.equal(Y, want)
    stream.synchronize()
    del g, junk


def test_a_long_mixed_queue_compares_its_last_turn_too():
    """Every form on two streams and the experts on a third, queued without a wait in between; nothing goes before all of it is done."""
    side = [torch.cuda.Stream() for _ in range(2)]
    layers = [[U.Layer(*f, 60 + i, s.cuda_stream) for i, f in enumerate(FORMS + PAIRS[1:3])] for s in side]
    want = [[l.value() for l in ls] for ls in layers]
    s = torch.cuda.Stream()
    T, D, H, E, K = 15000, 256, 256, 4, 2
    moe = M.MoE(T, D, E, K, hidden=H, training=False, stream=s.cuda_stream)
    up, down = (M.Mxfp4Weights(B.quantized(U.bf(shape, 1, 0.05).float().cpu().numpy())) for shape in ((E, H, D), (E, D, H)))
    X, Wr, Y = U.bf((T, D), 1), U.bf((E, D), 2, 0.05), torch.zeros(T, D, device="cuda").bfloat16()
    torch.cuda.synchronize()
    moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
    torch.cuda.synchronize()
    y = Y.clone()
    for turn in range(3):
        for ls in layers:
            for l in ls:
                l.Y.zero_()
        Y.zero_()
        torch.cuda.synchronize()
        for i in range(100):
            for j in range(len(layers[0])):
                layers[0][j].run()
                layers[1][(i + j) % len(layers[1])].run()
            if i % 4 == turn:
                moe.forward_mxfp4(X, Wr, up, down, Y, 0.0)
        torch.cuda.synchronize()
        assert moe.device_status() == 0 and torch.equal(Y, y)
        for ls, ws in zip(layers, want):
            for l, w in zip(ls, ws):
                assert torch.equal(l.Y, w)
