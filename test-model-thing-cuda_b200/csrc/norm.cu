// LayerNorm in front of the MoE block (tmt-cuda/src/norm.cu:8-110): forward with one warp per row, backward with 256
// threads walking 128 rows (row reductions through shuffles and shared memory, column sums kept in registers and added
// across blocks in a fixed order). Both passes read every input once: bound by HBM.
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../../include/tmt_norm.h"
#include "common.cuh"
#include "mx.cuh"
#include "mx_host.h"

namespace {

using namespace tmt;

constexpr int kFwdWarps = 8;            // rows per forward block
constexpr int kFwdMaxVec = 32;          // vectors a lane may own: dim <= 32 * 32 * 8 = 8192
constexpr int kBwdThreads = 256;
constexpr int kBwdRows = 128;           // rows per backward block
constexpr int kBwdMaxVec = 4;           // vectors a thread may own: dim <= 256 * 4 * 8 = 8192
constexpr float kEps = 1e-5f;

__device__ __forceinline__ void unpack8(const uint4 v, float (&f)[8]) {
    f[0] = bf_lo(v.x); f[1] = bf_hi(v.x); f[2] = bf_lo(v.y); f[3] = bf_hi(v.y);
    f[4] = bf_lo(v.z); f[5] = bf_hi(v.z); f[6] = bf_lo(v.w); f[7] = bf_hi(v.w);
}
__device__ __forceinline__ float butterfly(float v) {
    v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, 16));
    v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, 8));
    v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, 2));
    v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return v;
}

// One warp per row (rows taken grid-stride); the row stays in registers between the statistics and the output (one
// read of X) and the next row is fetched before the current one is reduced.
// FMT: mx::kE4M3 / mx::kE5M2 leaves an 8-bit checkpoint of the row as well (a block of 32 is the vectors of 4 neighbouring
// lanes): one byte more per element written, and no second read of X. 0: none.
// Bound: HBM; 131072 x 2048 takes 196 us without a checkpoint (5.5 TB/s) and 251 to 279 with one (4.8 to 5.4), 131072 x 1024 100 and 124; rows
// below 256 columns leave lanes idle: 131072 x 32 44, x 64 45, x 128 45, x 256 51 with one. Several rows a
// warp without the fetch ahead: 175 and 246 at 2048, but 10.6 and 17.0 instead of 8.8 and 11.6 at 8000 x 1024; the codes
// packed in the first pass, next to the sums: 291 at 2048 (registers).
template <int NV, int FMT>
__global__ void __launch_bounds__(kFwdWarps * 32) ln_fwd_kernel(const uint16_t* __restrict__ X, const float* __restrict__ gamma,
                                                                const float* __restrict__ beta, uint16_t* __restrict__ Y,
                                                                float* __restrict__ mean, float* __restrict__ rstd, int rows, int D,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const int nvec = D >> 3;
    const long stride = (long)gridDim.x * kFwdWarps;
    long r = (long)blockIdx.x * kFwdWarps + (threadIdx.x >> 5);
    if (r >= rows) return;
    const float fd = (float)D;
    constexpr bool kPrefetch = NV <= 8;              // wider rows would not fit two copies in registers
    uint4 raw[NV], nxt[kPrefetch ? NV : 1];
    auto fetch = [&](long row, auto& dst) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = lane + i * 32;
            if (v < nvec) dst[i] = ldg16(X + row * D + v * 8);
        }
    };
    if constexpr (kPrefetch) fetch(r, raw);
    for (; r < rows; r += stride) {
        if constexpr (kPrefetch) {
            if (r + stride < rows) fetch(r + stride, nxt);  // the next row travels while this one is reduced and written
        } else {
            fetch(r, raw);
        }
        float sum = 0.0f, sq = 0.0f;
        uint32_t amax[FMT != 0 ? NV : 1];                // largest magnitude of a lane's vector (bf16 magnitudes order like their bits)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = lane + i * 32;
            if (FMT != 0) amax[FMT != 0 ? i : 0] = 0;
            if (v < nvec) {
                float f[8];
                unpack8(raw[i], f);
#pragma unroll
                for (int q = 0; q < 8; ++q) { sum = __fadd_rn(sum, f[q]); sq = __fmaf_rn(f[q], f[q], sq); }
                if constexpr (FMT != 0) {
                    const uint32_t m = __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu));
                    amax[i] = max(m >> 16, m & 0xffffu) << 16;
                }
            }
        }
        sum = butterfly(sum);
        sq = butterfly(sq);
        const float m = __fdiv_rn(sum, fd);
        const float var = __fsub_rn(__fdiv_rn(sq, fd), __fmul_rn(m, m));
        const float rs = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(var, kEps)));
        if (lane == 0) { mean[r] = m; rstd[r] = rs; }
        uint16_t* y = Y + r * D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = lane + i * 32;
            if (v < nvec) {
                float f[8];
                unpack8(raw[i], f);
                const float4 g0 = __ldg(reinterpret_cast<const float4*>(gamma + v * 8)), g1 = __ldg(reinterpret_cast<const float4*>(gamma + v * 8) + 1);
                const float4 b0 = __ldg(reinterpret_cast<const float4*>(beta + v * 8)), b1 = __ldg(reinterpret_cast<const float4*>(beta + v * 8) + 1);
                // packed pairs: each half is the scalar operation, rounded to nearest, so the bits are those stated in the header
                const float2 gg[4] = {make_float2(g0.x, g0.y), make_float2(g0.z, g0.w), make_float2(g1.x, g1.y), make_float2(g1.z, g1.w)};
                const float2 bb[4] = {make_float2(b0.x, b0.y), make_float2(b0.z, b0.w), make_float2(b1.x, b1.y), make_float2(b1.z, b1.w)};
                const float2 nm = make_float2(-m, -m), r2 = make_float2(rs, rs);
                uint32_t o[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 t = __ffma2_rn(__fmul2_rn(__fadd2_rn(make_float2(f[2 * q], f[2 * q + 1]), nm), r2), gg[q], bb[q]);
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[q]) : "f"(t.y), "f"(t.x));
                }
                stg16(y + v * 8, make_uint4(o[0], o[1], o[2], o[3]));
            }
            if constexpr (FMT != 0) {                    // dim is a multiple of 32: the four lanes of a block agree on v < nvec
                uint32_t a = amax[i];
                a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
                a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
                if (v < nvec) {
                    const uint32_t sb = mx::scale_byte<FMT>(a);
                    const float inv = mx::inv_scale(sb);
                    float f[8];
                    unpack8(raw[i], f);
                    const float2 i2 = make_float2(inv, inv);
                    float2 p[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) p[q] = __fmul2_rn(make_float2(f[2 * q], f[2 * q + 1]), i2);
                    uint32_t lo = mx::pack_f8x4<FMT>(p[0].x, p[0].y, p[1].x, p[1].y);
                    uint32_t hi = mx::pack_f8x4<FMT>(p[2].x, p[2].y, p[3].x, p[3].y);
                    if (sb == 255u) { lo = 0; hi = 0; }
                    *reinterpret_cast<uint2*>(codes + r * D + v * 8) = make_uint2(lo, hi);
                    if ((lane & 3) == 0) scales[r * (D >> 5) + (v >> 2)] = (uint8_t)sb;
                }
            }
        }
        if constexpr (kPrefetch) {
#pragma unroll
            for (int i = 0; i < NV; ++i) raw[i] = nxt[i];
        }
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// Block = 256 threads x kBwdRows rows. Thread t owns the vectors t, t + 256, ... of every row. The rows travel through a
// ring of P rows in shared memory filled by cp.async; every thread copies exactly the 16-byte pieces it will read itself,
// so the ring needs no block barrier, and P rows per block (times the resident blocks) are in flight whatever the register
// budget. Rows are reduced RI at a time (their shuffles overlap, one block barrier serves all of them). The arithmetic
// per row and the row order of the column sums are those of a row-by-row loop.
template <int NV, int P, int RI, bool KEEP>
__global__ void __launch_bounds__(kBwdThreads) ln_bwd_kernel(const uint16_t* __restrict__ X, const uint16_t* __restrict__ dY,
                                                             const float* __restrict__ gamma, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, uint16_t* __restrict__ dX,
                                                             float* __restrict__ part, int rows, int D) {
    static_assert(P % RI == 0, "the ring is refilled RI rows at a time");
    extern __shared__ __align__(16) uint8_t ring_raw[];       // [P][dY, X][NV][256] x 16 bytes
    __shared__ __align__(16) float red[2][RI][2][kBwdThreads / 32];   // [parity of the iteration][row][s1, s2][warp]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nvec = D >> 3;
    const float fd = (float)D;
    constexpr uint32_t kSlot = 2 * NV * kBwdThreads * 16;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_raw) + threadIdx.x * 16;
    float gam[NV][8], dg[NV][8], db[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * kBwdThreads;
#pragma unroll
        for (int q = 0; q < 8; ++q) { gam[i][q] = v < nvec ? gamma[v * 8 + q] : 0.0f; dg[i][q] = 0.0f; db[i][q] = 0.0f; }
    }
    const long r0 = (long)blockIdx.x * kBwdRows;
    const long r_end = r0 + kBwdRows < rows ? r0 + kBwdRows : rows;
    auto issue = [&](long r, int slot) {         // one commit group per row, also for rows past the end (keeps the count uniform)
        if (r < r_end) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int v = threadIdx.x + i * kBwdThreads;
                if (v < nvec) {
                    cp_async16(ring + slot * kSlot + (uint32_t)(i * kBwdThreads * 16), dY + r * D + v * 8);
                    cp_async16(ring + slot * kSlot + (uint32_t)((NV + i) * kBwdThreads * 16), X + r * D + v * 8);
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < P; ++j) issue(r0 + j, j);
    float cm[RI], crs[RI];
#pragma unroll
    for (int j = 0; j < RI; ++j) { const long r = r0 + j; cm[j] = r < r_end ? mean[r] : 0.0f; crs[j] = r < r_end ? rstd[r] : 0.0f; }
    int it = 0, slot0 = 0;
    for (long rb = r0; rb < r_end; rb += RI, ++it) {
        float nm[RI], nrs[RI];
#pragma unroll
        for (int j = 0; j < RI; ++j) { const long r = rb + RI + j; nm[j] = r < r_end ? mean[r] : 0.0f; nrs[j] = r < r_end ? rstd[r] : 0.0f; }
        cp_async_wait<P - RI>();                   // the RI oldest rows have landed (each thread waits for its own copies)
        uint4 cdy[RI][NV], cx[RI][NV];
        float kg[KEEP ? RI : 1][NV][8], kxh[KEEP ? RI : 1][NV][8];     // KEEP: g and xh stay in registers for the second half
        float s1[RI], s2[RI], nmr[RI];
#pragma unroll
        for (int j = 0; j < RI; ++j) nmr[j] = -__fmul_rn(cm[j], crs[j]);      // xh = fma(x, rstd, -mean * rstd)
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            s1[j] = 0.0f; s2[j] = 0.0f;
            if (rb + j < r_end) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int v = threadIdx.x + i * kBwdThreads;
                    if (v < nvec) {
                        cdy[j][i] = lds16(ring + (slot0 + j) * kSlot + (uint32_t)(i * kBwdThreads * 16));
                        cx[j][i] = lds16(ring + (slot0 + j) * kSlot + (uint32_t)((NV + i) * kBwdThreads * 16));
                        float dy[8], x[8];
                        unpack8(cdy[j][i], dy);
                        unpack8(cx[j][i], x);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const float xh = __fmaf_rn(x[q], crs[j], nmr[j]);
                            const float g = __fmul_rn(dy[q], gam[i][q]);
                            if constexpr (KEEP) { kg[j][i][q] = g; kxh[j][i][q] = xh; }
                            s1[j] = __fadd_rn(s1[j], g);
                            s2[j] = __fmaf_rn(g, xh, s2[j]);
                            dg[i][q] = __fmaf_rn(dy[q], xh, dg[i][q]);
                            db[i][q] = __fadd_rn(db[i][q], dy[q]);
                        }
                    }
                }
            }
        }
        // the slots just read are free (this thread was their only reader): refill them with the rows P ahead
#pragma unroll
        for (int j = 0; j < RI; ++j) issue(rb + P + j, slot0 + j);
#pragma unroll
        for (int j = 0; j < RI; ++j) { s1[j] = butterfly(s1[j]); s2[j] = butterfly(s2[j]); }
        const int par = it & 1;                        // two buffers: the next iteration may write while a slow warp still reads
        if (lane == 0) {
#pragma unroll
            for (int j = 0; j < RI; ++j) { red[par][j][0][warp] = s1[j]; red[par][j][1][warp] = s2[j]; }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const long r = rb + j;
            if (r < r_end) {
                static_assert(kBwdThreads / 32 == 8, "the warp sums of a row are read as two float4");
                const float4* rp = reinterpret_cast<const float4*>(&red[par][j][0][0]);
                const float4 u0 = rp[0], u1 = rp[1], w0 = rp[2], w1 = rp[3];
                const float p1[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w}, p2[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
                float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) { t1 = __fadd_rn(t1, p1[w]); t2 = __fadd_rn(t2, p2[w]); }
                const float a = __fdiv_rn(t1, fd), b = __fdiv_rn(t2, fd);
                const float c0 = -__fmul_rn(crs[j], a), c1 = -__fmul_rn(crs[j], b);     // dx = fma(xh, -rstd*b, fma(g, rstd, -rstd*a))
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int v = threadIdx.x + i * kBwdThreads;
                    if (v < nvec) {
                        float o[8];
                        if constexpr (KEEP) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) o[q] = __fmaf_rn(kxh[j][i][q], c1, __fmaf_rn(kg[j][i][q], crs[j], c0));
                        } else {
                            float dy[8], x[8];
                            unpack8(cdy[j][i], dy);
                            unpack8(cx[j][i], x);
#pragma unroll
                            for (int q = 0; q < 8; ++q) {        // g and xh again, by the same operations
                                const float xh = __fmaf_rn(x[q], crs[j], nmr[j]);
                                const float g = __fmul_rn(dy[q], gam[i][q]);
                                o[q] = __fmaf_rn(xh, c1, __fmaf_rn(g, crs[j], c0));
                            }
                        }
                        stg16(dX + r * D + v * 8, make_uint4(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]), pack_bf2(o[4], o[5]), pack_bf2(o[6], o[7])));
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < RI; ++j) { cm[j] = nm[j]; crs[j] = nrs[j]; }
        slot0 += RI;
        if (slot0 == P) slot0 = 0;
    }
    cp_async_wait<0>();
    // block partial sums: part[block][0][D] = dGamma, part[block][1][D] = dBeta
    float* pg = part + (size_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * kBwdThreads;
        if (v < nvec) {
#pragma unroll
            for (int q = 0; q < 8; ++q) { pg[v * 8 + q] = dg[i][q]; pg[D + v * 8 + q] = db[i][q]; }
        }
    }
}

template <int NV, int P, int RI, bool KEEP>
cudaError_t launch_ln_bwd(int blocks, cudaStream_t s, const uint16_t* x, const uint16_t* dy, const float* gamma, const float* mean,
                          const float* rstd, uint16_t* dx, float* part, int rows, int dim) {
    const size_t smem = (size_t)P * 2 * NV * kBwdThreads * 16;
    cudaError_t e = cudaFuncSetAttribute(ln_bwd_kernel<NV, P, RI, KEEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    ln_bwd_kernel<NV, P, RI, KEEP><<<blocks, kBwdThreads, smem, s>>>(x, dy, gamma, mean, rstd, dx, part, rows, dim);
    return cudaGetLastError();
}

// Column d: block partial sums in block order.
__global__ void ln_bwd_reduce_kernel(const float* __restrict__ part, int blocks, int D, float* __restrict__ dGamma,
                                     float* __restrict__ dBeta) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= 2 * D) return;
    float s = 0.0f;
    int b = 0;
    for (; b + 32 <= blocks; b += 32) {       // 32 loads in flight, then added in block order
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __ldg(part + (size_t)(b + j) * 2 * D + i);
#pragma unroll
        for (int j = 0; j < 32; ++j) s = __fadd_rn(s, v[j]);
    }
    for (; b < blocks; ++b) s = __fadd_rn(s, part[(size_t)b * 2 * D + i]);
    if (i < D) dGamma[i] = s; else dBeta[i - D] = s;
}

int bwd_blocks(int rows) { return (rows - 1) / kBwdRows + 1; }

void check_shape(int rows, int dim, int max_dim) {
    if (rows < 1 || dim < 8 || dim % 8 || dim > max_dim)
        throw std::runtime_error("need rows >= 1 and dim a multiple of 8, at most " + std::to_string(max_dim));
}

template <int FMT>
void launch_ln_fwd(const void* X, const float* gamma, const float* beta, void* Y, float* mean, float* rstd, int rows, int dim,
                   uint8_t* codes, uint8_t* scales, void* stream) {
    const int nv = (dim / 8 + 31) / 32;
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int want = (rows - 1) / kFwdWarps + 1;
    const dim3 grid(std::max(1, std::min(want, std::max(sms, 1) * 6))), block(kFwdWarps * 32);      // a multiple of the SM count
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint16_t* x = static_cast<const uint16_t*>(X);
    uint16_t* y = static_cast<uint16_t*>(Y);
    if (nv <= 2) ln_fwd_kernel<2, FMT><<<grid, block, 0, s>>>(x, gamma, beta, y, mean, rstd, rows, dim, codes, scales);
    else if (nv <= 4) ln_fwd_kernel<4, FMT><<<grid, block, 0, s>>>(x, gamma, beta, y, mean, rstd, rows, dim, codes, scales);
    else if (nv <= 8) ln_fwd_kernel<8, FMT><<<grid, block, 0, s>>>(x, gamma, beta, y, mean, rstd, rows, dim, codes, scales);
    else if (nv <= 16) ln_fwd_kernel<16, FMT><<<grid, block, 0, s>>>(x, gamma, beta, y, mean, rstd, rows, dim, codes, scales);
    else ln_fwd_kernel<kFwdMaxVec, FMT><<<grid, block, 0, s>>>(x, gamma, beta, y, mean, rstd, rows, dim, codes, scales);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw std::runtime_error(std::string("LayerNorm forward launch failed: ") + cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int tmt_ln_forward(const void* X, const float* gamma, const float* beta, void* Y, float* mean, float* rstd, int rows, int dim,
                   void* stream) {
    try {
        if (!X || !gamma || !beta || !Y || !mean || !rstd) throw std::runtime_error("null argument");
        check_shape(rows, dim, 32 * kFwdMaxVec * 8);
        launch_ln_fwd<0>(X, gamma, beta, Y, mean, rstd, rows, dim, nullptr, nullptr, stream);
        return 0;
    } catch (const std::exception& e) { set_error("%s", e.what()); return -1; }
}

int tmt_ln_forward_act8(const void* X, const float* gamma, const float* beta, void* Y, float* mean, float* rstd, void* codes,
                        void* scales, int format, int rows, int dim, void* stream) {
    MX_GUARD({
        if (rows == 0) return 0;
        check_shape(rows, dim, 32 * kFwdMaxVec * 8);
        if (dim % 32) throw std::runtime_error("an 8-bit checkpoint needs dim to be a multiple of 32");
        check_tensors({X, gamma, beta, Y, codes, scales});
        check_tensors({mean, rstd}, 4);
        uint8_t* c = static_cast<uint8_t*>(codes);
        uint8_t* sc = static_cast<uint8_t*>(scales);
        if (format == mx::kE4M3) launch_ln_fwd<mx::kE4M3>(X, gamma, beta, Y, mean, rstd, rows, dim, c, sc, stream);
        else if (format == mx::kE5M2) launch_ln_fwd<mx::kE5M2>(X, gamma, beta, Y, mean, rstd, rows, dim, c, sc, stream);
        else throw std::runtime_error("format must be TMT_ACT8_E4M3 or TMT_ACT8_E5M2");
    })
}

size_t tmt_ln_backward_scratch_bytes(int rows, int dim) {
    if (rows < 1 || dim < 8) return 0;
    return (size_t)bwd_blocks(rows) * 2 * dim * sizeof(float);
}

int tmt_ln_backward(const void* X, const void* dY, const float* gamma, const float* mean, const float* rstd, void* dX,
                    float* dGamma, float* dBeta, int rows, int dim, void* scratch, void* stream) {
    try {
        if (!X || !dY || !gamma || !mean || !rstd || !dX || !dGamma || !dBeta || !scratch) throw std::runtime_error("null argument");
        check_shape(rows, dim, kBwdThreads * kBwdMaxVec * 8);
        const int nv = (dim / 8 + kBwdThreads - 1) / kBwdThreads;
        const int blocks = bwd_blocks(rows);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const uint16_t* x = static_cast<const uint16_t*>(X);
        const uint16_t* dy = static_cast<const uint16_t*>(dY);
        uint16_t* dx = static_cast<uint16_t*>(dX);
        float* part = static_cast<float*>(scratch);
        cudaError_t e;
        // dim <= 2048: four rows per iteration with g and xh kept in registers between the two halves (measured fastest of
        // {2, 4} rows x {kept, recomputed} x ring depth {8, 16}: 0.44-0.61 ms on 131072 x 2048)
        if (nv <= 1) e = launch_ln_bwd<1, 8, 4, true>(blocks, s, x, dy, gamma, mean, rstd, dx, part, rows, dim);
        else if (nv <= 2) e = launch_ln_bwd<2, 4, 2, false>(blocks, s, x, dy, gamma, mean, rstd, dx, part, rows, dim);
        else e = launch_ln_bwd<kBwdMaxVec, 2, 1, false>(blocks, s, x, dy, gamma, mean, rstd, dx, part, rows, dim);
        if (e != cudaSuccess) throw std::runtime_error(std::string("LayerNorm backward launch failed: ") + cudaGetErrorString(e));
        ln_bwd_reduce_kernel<<<(2 * dim + 63) / 64, 64, 0, s>>>(part, blocks, dim, dGamma, dBeta);
        e = cudaGetLastError();
        if (e != cudaSuccess) throw std::runtime_error(std::string("LayerNorm backward launch failed: ") + cudaGetErrorString(e));
        return 0;
    } catch (const std::exception& e) { set_error("%s", e.what()); return -1; }
}

}  // extern "C"
