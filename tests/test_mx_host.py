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


STATE_CHECK = r"""
#include <cassert>
#include <cstdlib>
#include <new>
#include "mx_state.h"
int main() {
    using tmt::MxState;
    int left = 0;                                    // allocations that still succeed
    auto alloc = [&](size_t bytes) -> void* { if (left-- <= 0) throw std::bad_alloc(); return std::calloc(1, bytes); };
    const std::vector<const void*> a = {&left}, b = {&a};
    for (int fail = 0; fail < 2; ++fail)
        for (int recorded = 0; recorded < 2; ++recorded) {
            MxState m;
            left = 2;
            m.open_tables(3, 2, alloc);
            m.key = a; m.recorded = recorded;
            CUtensorMap* const t = m.tables; const uint8_t** const s = m.scale_tab;
            assert(t && s);
            left = fail;                             // memory for none, or for the first of the two
            bool threw = false;
            try { m.open_tables(3, 2, alloc); m.key = b; } catch (const std::bad_alloc&) { threw = true; }
            assert(threw == (recorded == 1));
            assert(m.tables == t && m.scale_tab == s);                   // never one table of each list
            if (threw) {
                assert(m.key.empty() && m.recorded);                     // the first list is not taken for what they hold
                left = 2;
                m.open_tables(3, 2, alloc);
                assert(m.tables != t && m.scale_tab != s && !m.recorded && m.key.empty());
            }
        }
}
"""


def test_tables_of_weights_when_memory_runs_out(M, tmp_path):
    """After an allocation that failed the tables stand for no list of weights, and a recorded graph's are left alone."""
    import os
    import subprocess
    src = tmp_path / "check.cpp"
    src.write_text(STATE_CHECK)
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(M.__file__))), "csrc")
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.run(["g++", "-std=c++17", "-I", csrc, "-I", cuda, str(src), "-o", str(tmp_path / "check")], check=True)
    subprocess.run([str(tmp_path / "check")], check=True)


def test_the_front_end_keeps_recorded_weights_alive(M, monkeypatch):
    """A graph goes on reading the weights it was recorded with, whatever later calls are given and the caller drops."""
    import gc
    import weakref
    from test_front_end_dry_run import FakeLib

    class Lib(FakeLib):
        recorded = 0

        def __getattr__(self, name):
            if name == "tmt_moe_mxfp4_recorded":
                return lambda h: self.recorded
            return FakeLib.__getattr__(self, name)
    lib = Lib()
    monkeypatch.setattr(M, "_lib", lib)
    E, D, H = 2, 64, 128
    moe = M.MoE(8, D, E, 1, hidden=H, training=False)
    X, Y, Wr = torch.zeros(8, D, dtype=torch.bfloat16), torch.zeros(8, D, dtype=torch.bfloat16), torch.zeros(E, D, dtype=torch.bfloat16)

    def weights():
        return [[(torch.zeros(n * k // 2, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), n, k) for _ in range(E)] for n, k in ((H, D), (D, H))]

    def call(w):
        moe.forward_mxfp4(X, Wr, w[0], w[1], Y)
        return weakref.ref(w[0][0][0]), weakref.ref(w[1][E - 1][1])

    def alive(refs):
        gc.collect()
        return [r() is not None for r in refs]
    a = call(weights())
    assert alive(a) == [True, True]                      # the handle's table points at them
    lib.recorded = 1
    b = call(weights())                                  # a was recorded, b is not
    lib.recorded = 0
    assert alive(a) == [True, True]
    c = call(weights())
    assert alive(a) == [True, True] and alive(b) == [False, False] and alive(c) == [True, True]
    kept = M.Mxfp4Weights(weights()[0]), M.Mxfp4Weights(weights()[1])
    lib.recorded = 1
    for _ in range(3):
        moe.forward_mxfp4(X, Wr, *kept, Y)               # c counts as recorded once, kept needs no entry while it is the last
    assert len(moe._mx_recorded) == 2 and alive(c) == [True, True]
    moe.close()
    assert alive(a) + alive(c) == [False] * 4


def test_the_front_end_refuses_sizes_that_would_wrap(M, monkeypatch):
    """A size past 32 bits reaches a C int as its low half: a matrix of 2^32 + 64 columns would be taken for one of 64."""
    from test_front_end_dry_run import FakeLib
    monkeypatch.setattr(M, "_lib", FakeLib())            # accepts whatever it is given

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")
    n = 2 ** 32 + 64
    by = meta(2 ** 40, dtype=torch.uint8)
    f = meta(2 ** 40, dtype=torch.float32)
    W = (by, by, 8, 64)
    wide, tall, y = meta(1, n), meta(n, 64), meta(n, 8)
    calls = [lambda: M.quantize_mxfp4(wide, by, by), lambda: M.dequantize_mxfp4(by, by, wide), lambda: M.act8_save(wide, by, by),
             lambda: M.act8_restore(by, by, wide), lambda: M.linear_mxfp4(tall, W, y, by), lambda: M.matmul_mxfp4(by, by, W, y),
             lambda: M.ln_forward_act8(tall, f, f, tall, f, f, by, by), lambda: M.ln_forward_act8(wide, f, f, wide, f, f, by, by),
             lambda: M.ln_backward_act8(by, by, tall, f, f, f, tall, f, f, by), lambda: M.linear_mxfp4(meta(4, 64), (by, by, n, 64), meta(4, n), by),
             lambda: M.Mxfp4Weights([(by, by, 8, n)]), lambda: M.Mxfp4Weights([(by, by, -8, 64)]), lambda: M.matmul_mxfp4(by, by, W, meta())]
    for call in calls:
        with pytest.raises(M.MoeError):
            call()
    M.quantize_mxfp4(tall, by, by)                       # the casts count rows in 64 bits
    M.act8_restore(by, by, tall)


def test_sizes_at_the_end_of_the_column_range(M):
    k = 2 ** 31 - 64
    assert M.mxfp4_scale_bytes(1, k) == M.mxfp4_scale_bytes(128, k) == 2 ** 24 * 512
    assert M.linear_mxfp4_work_bytes(1, k) == k // 2 + 2 ** 24 * 512


def test_products_refuse_a_k_whose_sum_outlasts_the_bounded_waits(M):
    import ctypes
    lib, p = M.load(), 1 << 20
    for k in (2 ** 28 + 64, 2 ** 31 - 64):
        W = M._Mxfp4WeightDesc(p, p, 8, k)
        for rc in (lib.tmt_moe_matmul_mxfp4(p, p, 4, ctypes.byref(W), p, 0, None, None),
                   lib.tmt_moe_linear_mxfp4(p, 0, 4, ctypes.byref(W), p, 0, p, 1 << 62, None, None), lib.tmt_moe_linear_mxfp4_form(4, 8, k)):
            assert rc == -1 and b"at most" in lib.tmt_moe_last_error()
