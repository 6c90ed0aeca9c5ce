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
    kMxDown = 3,     // out = bf16(row_scale[row] * acc)
};

struct MxGemm {
    CUtensorMap act, w;                 // codes as bytes, 128-byte boxes (mx_act_map / mx_weight_map)
    const CUtensorMap* w_maps;          // grouped: one map per expert in device memory (then `w` is not used)
    const uint8_t* act_scales;          // scale tiles of the activations; group starts are multiples of 128 rows
    const uint8_t* w_scales;            // dense
    const uint8_t* const* w_scales_tab; // grouped: per expert, device table
    int rows;                           // dense: rows of A
    int n, k;                           // rows and columns of one weight matrix: n % 8 == 0, k % 64 == 0
    int experts;                        // 0: dense
    const int* poff; const int* counts; // grouped: first row and number of rows of every expert's group (device)
    long row_limit;                     // rows of the activation buffer: a group that would pass it is skipped and reported
    int epi;
    void* out; uint8_t* out_scales; const float* row_scale;
    int* status;
    bool few_rows;                      // weights on the 128-row side of the MMA (mx_few_rows)
};

constexpr int kMxMapRows = 128;         // rows per box of the weight maps and of the activation maps of the many-row form
constexpr int kMxFewRows = 32;          // rows per box of the activation maps of the few-row form

// rows_per_group: average rows a weight matrix meets in this call.
bool mx_few_rows(long rows_per_group);
// 2-D byte map {cols / 2, rows} with boxes of 128 bytes x box_rows, 128-byte swizzle, zero fill.
void mx_make_map(CUtensorMap* m, const void* codes, uint64_t rows, int cols, int box_rows);
cudaError_t launch_mx_gemm(const MxGemm& p, int num_sms, cudaStream_t stream);

}  // namespace tmt
