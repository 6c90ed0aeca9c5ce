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
