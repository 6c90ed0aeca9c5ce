// Products of 4-bit microscaled matrices (mx_gemm.cu): Y[r, j] = sum_k A[r, k] W[j, k], dense or grouped by expert.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace tmt {

enum MxEpilogue : int {
    kMxBf16 = 0,     // out = bf16(acc), rows x n
    kMxF32 = 1,      // out = acc, rows x n
    kMxUp = 2,       // out = 4-bit codes of silu(acc), out_scales = their scale tiles
    kMxDown = 3,     // out = row_scale[row] * acc, fp32: a token's rows are added before anything is rounded
};

struct MxGemm {
    CUtensorMap act, w;                 // codes as bytes, 128-byte boxes (mx_make_map)
    const CUtensorMap* w_maps;          // grouped: one map per expert in device memory (then `w` is not used)
    // scale tiles of the activations (group starts are multiples of 128 rows, of 256 for kMxPair) and of the weights
    const uint8_t* act_scales;          // kMxMany
    const uint8_t* w_scales;            // dense
    const uint8_t* const* w_scales_tab; // grouped: per expert, device table
    CUtensorMap act_sf, w_sf;           // kMxPair: the same as 3-D maps {tile of 512 bytes, tiles along k, 128-row bands}
    const CUtensorMap* w_sf_maps;       // grouped
    int rows;                           // dense: rows of A
    int n, k;                           // rows and columns of one weight matrix: n % 8 == 0, k % 64 == 0
    int experts;                        // 0: dense
    const int* poff; const int* counts; // grouped: first row and number of rows of every expert's group (device)
    long row_limit;                     // rows of the activation buffer: a group that would pass it is skipped and reported
    int epi;
    void* out; uint8_t* out_scales; const float* row_scale;
    CUtensorMap out_map;                // kMxPair: the output (not used by kMxUp)
    int* status;
    int form;                           // MxForm
};

// Forms of the product: one CTA per 128 x 128 tile; CTA pairs on 256 x 256 tiles.
enum MxForm : int { kMxMany = 0, kMxPair = 1 };
// The form for `rows` activation rows in `groups` groups of about equal size, n outputs; pad: rows that group starts are multiples of.
int mx_form(long rows, int groups, int n, int k, int num_sms, int pad);

// 128-row boxes for the codes of both operands; 128-row bands per box of the scale maps (pair form).
constexpr int kMxBoxRows = 128;
constexpr int kMxActBands = 1, kMxWeightBands = 2;      // 128-row bands per box of the scale maps

// 2-D byte map {cols / 2, rows} with boxes of 128 bytes x box_rows, 128-byte swizzle, zero fill.
void mx_make_map(CUtensorMap* m, const void* codes, uint64_t rows, int cols, int box_rows);
// 3-D map of scale tiles, boxes of 2 tiles along k x `bands` bands.
void mx_make_scale_map(CUtensorMap* m, const void* scales, uint64_t rows, int cols, int bands);
// Map of a row-major output for the staged stores of the pair form: boxes of 128 bytes x 32 rows, 128-byte swizzle.
void mx_make_out_map(CUtensorMap* m, void* out, uint64_t rows, int n, bool f32);
cudaError_t launch_mx_gemm(const MxGemm& p, int num_sms, cudaStream_t stream);
cudaError_t launch_mx_gemm_2cta(const MxGemm& p, int num_sms, cudaStream_t stream);

}  // namespace tmt
