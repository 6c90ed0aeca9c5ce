// What a handle keeps for tmt_moe_forward_mxfp4 (mx_moe.cu), allocated at its first call: the grouped rows and their SiLU outputs as
// 4-bit blocks, the gated outputs of the experts in fp32, and the per-expert tables of the weights last handed in.
#pragma once
#include <cuda.h>

#include <cstddef>
#include <cstdint>
#include <vector>

namespace tmt {

struct MxState {
    uint8_t *x_codes = nullptr, *x_scales = nullptr, *h_codes = nullptr, *h_scales = nullptr;
    float* y_rows = nullptr;
    bool buffers = false;                          // all of the above are there and have been filled
    CUtensorMap x_map = {}, h_map = {}, x_sf = {}, h_sf = {}, y_out = {};
    CUtensorMap* tables = nullptr;                 // per-expert weight maps (mx_moe.cu)
    const uint8_t** scale_tab = nullptr;           // [2][E]
    std::vector<const void*> key;                  // the pointers the tables were built from; empty: from none
    bool recorded = false;                         // a graph was recorded with these tables

    // Tables that may be written for another list of weights: those of before, or fresh ones where a recorded graph reads those of
    // before. alloc(bytes) throws when there is no memory. The tables stand for no list until the caller sets `key` again, so that
    // whatever throws in between, the next call writes them anew instead of taking them for what they are not.
    template <class Alloc>
    void open_tables(size_t maps, size_t scales, Alloc alloc) {
        key.clear();
        if (tables && !recorded) return;
        CUtensorMap* t = static_cast<CUtensorMap*>(alloc(maps * sizeof(CUtensorMap)));
        const uint8_t** s = static_cast<const uint8_t**>(alloc(scales * sizeof(uint8_t*)));
        tables = t;
        scale_tab = s;
        recorded = false;
    }
};

}  // namespace tmt
