// Launcher of the 4-bit quantiser (mx_cast.cu) for the operators that quantise on the way in.
#pragma once
#include <cuda_runtime.h>

namespace tmt {
// X (rows, cols) bf16 or fp32 -> codes, scale tiles; rows >= 1. early: the next kernel may be scheduled at once (it waits itself).
cudaError_t launch_mx4_quantize(const void* X, bool f32, long long rows, int cols, void* codes, void* scales, cudaStream_t s, bool early);
}  // namespace tmt
