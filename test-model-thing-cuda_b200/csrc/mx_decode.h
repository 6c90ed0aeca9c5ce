// 4-bit products with few rows per weight matrix (mx_decode.cu): dense layers of up to 32 rows, decode steps of the experts.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace tmt {

enum MxSource : int {
    kMxSrcBf16 = 0, kMxSrcF32 = 1,     // rows of values, quantised on the way in
    kMxSrcTiles = 2,                   // codes, scale tiles (include/tmt_mx.h)
    kMxSrcRows = 3,                    // codes, scale bytes row-major (cols / 32 rounded up to a multiple of 4 per row)
};

struct MxDecode {
    CUtensorMap w, w_sf;               // dense: codes in boxes of 128 rows, scale tiles in boxes of 2 x 1 band
    const CUtensorMap* w_maps;         // grouped: one per expert, device memory
    const CUtensorMap* w_sf_maps;
    const void* src; const uint8_t* src_scales; int src_kind;
    unsigned src_mul;                  // grouped: assignment a reads row a * src_mul >> 16 (mx_row_factor)
    int rows;                          // dense: rows
    const int* idx; int n_asg; int experts;      // grouped: expert of every assignment (experts = 0: dense)
    int n, k;
    int split;                         // dense: blocks (a cluster) that share k; grouped: 1
    int epi;                           // MxEpilogue; kMxUp: out_scales row-major as kMxSrcRows; grouped outputs: one row per assignment
    void* out; uint8_t* out_scales;
    const float* gate;                 // kMxDown: per assignment
    int* status;
    bool early;                        // the next kernel waits by itself: it may be scheduled at once
    bool weights_ready;                // a kernel between the weights' writer and this one has waited for it (griddepcontrol.wait), or this one's launch does
};

// a * factor >> 16 == a / divisor for a < 2048, divisor <= 8: the excess a * (factor - 65536 / divisor) / 65536 is below a / 65536 < 1 / 8.
inline unsigned mx_row_factor(int divisor) { return (65536u + (unsigned)divisor - 1) / (unsigned)divisor; }

constexpr int kMxDecodeRows = 32;      // rows per pass
constexpr int kMxDecodeMaxAsg = 2048, kMxDecodeMaxK = 8192;

// Dense: the number of blocks that share k, and whether this kernel takes the product (codes: the rows come as codes).
int mx_decode_split(int n, int k, int num_sms);
bool mx_decode_dense(long rows, int k, int split, bool codes);
// Grouped: whether this kernel takes both products of the experts; k: the longer of their two.
bool mx_decode_grouped(long rows, int groups, int k);
cudaError_t launch_mx_decode(const MxDecode& p, cudaStream_t stream);

}  // namespace tmt
