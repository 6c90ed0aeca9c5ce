// LayerNorm backward from an 8-bit checkpoint of its input (include/tmt_norm.h).
//
//   xh = (x - mean) * rstd,  g = dy * gamma,  a = sum(g) / D,  b = sum(g * xh) / D
//   dx = rstd * (g - a - xh * b),   dGamma[d] = sum over rows of dy * xh,   dBeta[d] = sum over rows of dy
//
// x is never written out: an element enters as its code, and xh = fma(code, scale * rstd, -mean * rstd).
// A team walks a contiguous range of rows; a thread owns 8 neighbouring columns (16 bytes of dY, 8 bytes of codes) of every row,
// so gamma and the column sums stay in its registers. A team is a block of ceil(dim / 256) warps, or for dim < 256 the
// smallest power of two of lanes that covers a row. RI rows are reduced together: their 2 * RI row sums go through one
// transposing butterfly (each step halves the values a lane carries: 9 shuffles for 8 sums instead of 40) and one barrier,
// and the next RI rows are already on their way into registers. The products run on the packed fp32 pair instructions.
// The column sums of the teams are added by a second kernel in a fixed order: results do not depend on timing.
// Bound: HBM, 5.03 bytes per element (2 + 33/32 read, 2 written).
#include <algorithm>

#include "../../include/tmt_norm.h"
#include "launch_pdl.cuh"
#include "mx.cuh"
#include "mx_host.h"

namespace tmt {
namespace {

using namespace mx;

constexpr int kMaxDim = 8192;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float2 bc(float v) { return make_float2(v, v); }
__device__ __forceinline__ uint32_t pack2(float2 v) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
    return r;
}

struct Raw { uint4 dy; uint2 x; uint32_t sb; float mean, rstd; };

// Sums of N = 4 or 8 values over the 32 lanes of a warp. Afterwards lane l holds the sum of value l / (32 / N).
template <int N>
__device__ __forceinline__ float transpose_sum(float (&v)[N], int lane) {
    int bit = 16;
#pragma unroll
    for (int n = N / 2; n >= 1; n >>= 1, bit >>= 1) {
        const bool up = (lane & bit) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float send = up ? v[i] : v[i + n];
            const float keep = up ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(kFull, send, bit);
        }
    }
    float s = v[0];
    for (; bit >= 1; bit >>= 1) s += __shfl_xor_sync(kFull, s, bit);
    return s;
}

// L: lanes of a team (32: the whole block). RI: rows reduced together. MAXT: most threads of a block.
template <int FMT, int L, int RI, int MAXT>
__global__ void __launch_bounds__(MAXT) ln_bwd_act8_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                           const uint16_t* __restrict__ dY, const float* __restrict__ gamma,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           uint16_t* __restrict__ dX, float* __restrict__ part, int rows, int D,
                                                           int rows_per_team) {
    constexpr int NS = 2 * RI;
    __shared__ float red[2][NS][32];             // [parity][row sums][warp]
    pdl_begin();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int team = L == 32 ? (int)blockIdx.x : (int)(blockIdx.x * blockDim.x + threadIdx.x) / L;
    const int v = L == 32 ? (int)threadIdx.x : lane % L;           // this thread's vector of 8 columns
    const bool col_ok = v * 8 < D;
    const float inv_d = 1.0f / (float)D;
    float2 gam[4], dg[4], db[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        gam[i] = col_ok ? make_float2(gamma[v * 8 + 2 * i], gamma[v * 8 + 2 * i + 1]) : bc(0.0f);
        dg[i] = bc(0.0f); db[i] = bc(0.0f);
    }
    const long r0 = (long)team * rows_per_team;
    const long r1 = min(r0 + rows_per_team, (long)rows);
    auto fetch = [&](long r, Raw& w) {
        w.dy = make_uint4(0, 0, 0, 0); w.x = make_uint2(0, 0); w.sb = 127; w.mean = 0.0f; w.rstd = 0.0f;
        if (r < r1) {
            w.mean = __ldg(mean + r); w.rstd = __ldg(rstd + r);
            if (col_ok) {
                w.dy = ldg16_stream(dY + r * D + v * 8);
                w.x = __ldg(reinterpret_cast<const uint2*>(codes + r * D + v * 8));
                w.sb = __ldg(scales + r * (D >> 5) + (v >> 2));
            }
        }
    };
    Raw nxt[RI];
#pragma unroll
    for (int j = 0; j < RI; ++j) fetch(r0 + j, nxt[j]);
    int par = 0;
    // every lane of a warp makes the same number of turns (sub-warp teams differ in their last rows alone)
    for (int turn = 0; turn * RI < rows_per_team; ++turn, par ^= 1) {
        const long rb = r0 + turn * RI;
        if (L == 32 && rb >= r1) break;
        float2 g[RI][4], xh[RI][4];
        float rs[RI], s[NS];
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const Raw w = nxt[j];
            rs[j] = w.rstd;
            const float2 sc = bc(scale_value(w.sb) * w.rstd), c = bc(-w.mean * w.rstd);
            const uint32_t dw[4] = {w.dy.x, w.dy.y, w.dy.z, w.dy.w}, xw[2] = {w.x.x, w.x.y};
            float2 s1 = bc(0.0f), s2 = bc(0.0f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 dy = make_float2(bf_lo(dw[i]), bf_hi(dw[i]));
                xh[j][i] = __ffma2_rn(unpack_f8x2<FMT>((uint16_t)(xw[i >> 1] >> (16 * (i & 1)))), sc, c);
                g[j][i] = __fmul2_rn(dy, gam[i]);
                s1 = __fadd2_rn(s1, g[j][i]);
                s2 = __ffma2_rn(g[j][i], xh[j][i], s2);
                dg[i] = __ffma2_rn(dy, xh[j][i], dg[i]);
                db[i] = __fadd2_rn(db[i], dy);
            }
            s[2 * j] = s1.x + s1.y; s[2 * j + 1] = s2.x + s2.y;
        }
#pragma unroll
        for (int j = 0; j < RI; ++j) fetch(rb + RI + j, nxt[j]);
        float tot[NS];
        if constexpr (L == 32) {
            float mine = transpose_sum<NS>(s, lane);                   // value lane / (32 / NS)
            if (warps > 1) {
                if (lane % (32 / NS) == 0) red[par][lane / (32 / NS)][warp] = mine;
                __syncthreads();                                       // the other parity is free: one barrier a turn is enough
                mine = 0.0f;
                for (int w = lane % (32 / NS); w < warps; w += 32 / NS) mine += red[par][lane / (32 / NS)][w];
#pragma unroll
                for (int o = 1; o < 32 / NS; o <<= 1) mine += __shfl_xor_sync(kFull, mine, o);
            }
#pragma unroll
            for (int k = 0; k < NS; ++k) tot[k] = __shfl_sync(kFull, mine, k * (32 / NS));
        } else {
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                tot[k] = s[k];
#pragma unroll
                for (int o = L / 2; o >= 1; o >>= 1) tot[k] += __shfl_xor_sync(kFull, tot[k], o);
            }
        }
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const float2 r2 = bc(rs[j]), ca = bc(-rs[j] * (tot[2 * j] * inv_d)), cb = bc(-rs[j] * (tot[2 * j + 1] * inv_d));
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = pack2(__ffma2_rn(xh[j][i], cb, __ffma2_rn(g[j][i], r2, ca)));
            if (rb + j < r1 && col_ok) stg16(dX + (rb + j) * D + v * 8, make_uint4(o[0], o[1], o[2], o[3]));
        }
    }
    if (col_ok) {
        float* p = part + (size_t)team * 2 * D + v * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *reinterpret_cast<float2*>(p + 2 * i) = dg[i];
            *reinterpret_cast<float2*>(p + D + 2 * i) = db[i];
        }
    }
}

// Column i of [dGamma | dBeta]: 32 partial sums over the teams (teams y, y + 32, ...), then those in a tree.
__global__ void __launch_bounds__(1024) ln_bwd_act8_reduce_kernel(const float* __restrict__ part, int teams, int D,
                                                                  float* __restrict__ dGamma, float* __restrict__ dBeta) {
    __shared__ float sh[32][33];
    pdl_begin();
    pdl_wait();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + x;                             // 2 * D is a multiple of 32
    float s = 0.0f;
    for (int t = y; t < teams; t += 32) s += part[(size_t)t * 2 * D + i];
    sh[y][x] = s;
    __syncthreads();
    s = sh[x][y];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    const int c = blockIdx.x * 32 + y;
    if (x == 0) { if (c < D) dGamma[c] = s; else dBeta[c - D] = s; }
}

struct Plan { int lanes, threads, blocks, teams, rows_per_team; };

// From the shape alone (148 SMs): the scratch size and the order of the sums do not depend on where the call runs.
Plan plan(int rows, int dim) {
    constexpr int kSms = 148, kMinRows = 8;
    Plan p;
    const int vec = dim / 8;
    p.lanes = 32;
    while (p.lanes / 2 >= vec) p.lanes /= 2;
    const int warps = (vec + 31) / 32;
    p.threads = p.lanes < 32 ? 128 : warps * 32;
    const int per_block = p.lanes < 32 ? p.threads / p.lanes : 1;
    const int resident = std::max(1, std::min(24, 16 / warps)) * kSms * (p.lanes < 32 ? 4 : 1);
    const int want = (rows + kMinRows * per_block - 1) / (kMinRows * per_block);
    p.blocks = std::max(1, std::min(want, resident));
    p.teams = p.blocks * per_block;
    p.rows_per_team = (rows + p.teams - 1) / p.teams;
    return p;
}

template <int FMT, int L, int RI, int MAXT>
cudaError_t launch_t(const Plan& p, cudaStream_t s, const uint8_t* codes, const uint8_t* scales, const uint16_t* dY, const float* gamma,
                     const float* mean, const float* rstd, uint16_t* dX, float* part, int rows, int dim) {
    return launch_pdl(ln_bwd_act8_kernel<FMT, L, RI, MAXT>, dim3(p.blocks), dim3(p.threads), 0, s, codes, scales, dY, gamma, mean, rstd, dX, part,
                      rows, dim, p.rows_per_team);
}

template <int FMT, class... A>
cudaError_t launch_f(const Plan& p, A... a) {
    switch (p.lanes) {
        case 4: return launch_t<FMT, 4, 4, 128>(p, a...);
        case 8: return launch_t<FMT, 8, 4, 128>(p, a...);
        case 16: return launch_t<FMT, 16, 4, 128>(p, a...);
        default: break;
    }
    if (p.threads <= 256) return launch_t<FMT, 32, 4, 256>(p, a...);
    if (p.threads <= 512) return launch_t<FMT, 32, 4, 512>(p, a...);
    return launch_t<FMT, 32, 2, 1024>(p, a...);
}

}  // namespace
}  // namespace tmt

using namespace tmt;

extern "C" {

size_t tmt_ln_backward_act8_scratch_bytes(int rows, int dim) {
    if (rows < 1 || dim < 32 || dim % 32 || dim > kMaxDim) return 0;
    return (size_t)plan(rows, dim).teams * 2 * dim * sizeof(float);
}

int tmt_ln_backward_act8(const void* codes, const void* scales, int format, const void* dY, const float* gamma, const float* mean,
                         const float* rstd, void* dX, float* dGamma, float* dBeta, int rows, int dim, void* scratch, void* stream) {
    MX_GUARD({
        if (rows < 1 || dim < 32 || dim % 32 || dim > kMaxDim)
            throw std::runtime_error("need rows >= 1 and dim a multiple of 32, at most " + std::to_string(kMaxDim));
        if (format != kE4M3 && format != kE5M2) throw std::runtime_error("format must be TMT_ACT8_E4M3 or TMT_ACT8_E5M2");
        check_tensors({codes, scales, dY, dX, scratch});
        check_tensors({gamma, mean, rstd, dGamma, dBeta}, 4);
        const Plan p = plan(rows, dim);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const uint8_t* c = static_cast<const uint8_t*>(codes);
        const uint8_t* sc = static_cast<const uint8_t*>(scales);
        const uint16_t* dy = static_cast<const uint16_t*>(dY);
        uint16_t* dx = static_cast<uint16_t*>(dX);
        float* part = static_cast<float*>(scratch);
        cuda_ok(format == kE4M3 ? launch_f<kE4M3>(p, s, c, sc, dy, gamma, mean, rstd, dx, part, rows, dim)
                                : launch_f<kE5M2>(p, s, c, sc, dy, gamma, mean, rstd, dx, part, rows, dim), "ln_backward_act8 launch");
        cuda_ok(launch_pdl(ln_bwd_act8_reduce_kernel, dim3(2 * dim / 32), dim3(1024), 0, s, part, p.teams, dim, dGamma, dBeta), "ln_backward_act8 launch");
    })
}

}  // extern "C"
