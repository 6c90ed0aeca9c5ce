// LayerNorm backward from an 8-bit checkpoint of its input (include/tmt_norm.h).
//
//   xh = (x - mean) * rstd,  g = dy * gamma,  a = sum(g) / D,  b = sum(g * xh) / D
//   dx = rstd * (g - a - xh * b),   dGamma[d] = sum over rows of dy * xh,   dBeta[d] = sum over rows of dy
//
// x is never written out: an element enters as its code, and xh = fma(code, scale, -mean) * rstd: code * scale is exact, so x - mean is
// rounded once, and a row whose mean is far above its deviation keeps its bits (fma(code, scale * rstd, -mean * rstd) would leave the
// rounding of mean * rstd in a constant row).
// A team walks a contiguous range of rows; a thread owns one vector of 8 columns (16 bytes of dY, 8 bytes of codes) of every row
// (V = 2 vectors, half a row apart, where dim > 2048), so gamma and the column sums stay in its registers. A team is a block of
// ceil(dim / 256) warps; for dim < 256 it is the smallest power of two of lanes that covers a row. RI rows are reduced together:
// their 2 * RI row sums go through one transposing butterfly (each step halves the values a lane carries: 9 shuffles for 8
// sums instead of 40) and one barrier. Rows travel through a ring of P rows in shared memory filled by cp.async; every thread
// copies exactly the pieces it will read itself, so the ring needs no barrier, and its depth costs no registers. The products run
// on the packed fp32 pair instructions.
// Measured at 131072 x 2048 (e4m3): 272 to 285 us = 4.9 TB/s, 0.75 of the copy rate; bound by latency at 16 warps an SM (128 registers a
// thread): issue slots are 57 % busy, DRAM 55 to 75 %. Other widths, 131072 rows, us beside the floor: 32 columns 68 | 3, 64: 48 | 7, 128: 46 | 13,
// 256: 53 | 26 (these by the column-sum kernel, which has 2 * dim / 32 blocks for the sums of up to 16384 teams), 1024: 142 | 105, 2080: 353 | 212;
// 65536 x 4096 290 | 209, 32768 x 8192 290 | 209 (one block of up to 512 threads an SM, 36 bytes spilled). Two rows a turn and
// three blocks an SM: 284-315; rows dealt round instead of in ranges: 380; two vectors a thread and four blocks: 375; the
// row fetched ahead into registers instead of the ring: 343-365.
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

template <int V> struct Raw { uint32_t sb[V]; float mean, rstd; };      // what of a row does not go through the ring

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}

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

// V: vectors of a thread. L: lanes of a team (32: the whole block). RI: rows reduced together. P: rows of the ring (one commit group each), a multiple of RI.
// MAXT: most threads of a block, MINB: blocks an SM holds at that size.
template <int FMT, int V, int L, int RI, int P, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) ln_bwd_act8_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                           const uint16_t* __restrict__ dY, const float* __restrict__ gamma,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           uint16_t* __restrict__ dX, float* __restrict__ part, int rows, int D,
                                                           int teams) {
    static_assert(P % RI == 0, "the ring is refilled RI rows at a time");
    constexpr int NS = 2 * RI;                               // row sums of a turn
    extern __shared__ __align__(16) uint8_t ring_raw[];      // [P] x [V] x { 16 bytes of dY, 8 of codes } per thread
    __shared__ float red[2][NS][32];             // [parity][row sums][warp]
    pdl_wait();
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int team = L == 32 ? (int)blockIdx.x : (int)(blockIdx.x * blockDim.x + threadIdx.x) / L;
    const int c0 = (L == 32 ? (int)threadIdx.x : lane % L) * 8;    // first column of this thread's first vector
    const int cstep = blockDim.x * 8;                              // from there to the second
    bool ok[V];
    float2 gam[V][4], dg[V][4], db[V][4];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        ok[k] = c0 + k * cstep < D;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* p = gamma + c0 + k * cstep + 2 * i;
            gam[k][i] = ok[k] ? make_float2(p[0], p[1]) : bc(0.0f);
            dg[k][i] = bc(0.0f); db[k][i] = bc(0.0f);
        }
    }
    const float inv_d = 1.0f / (float)D;
    const int rpt = (rows - 1) / teams + 1;          // rows of a team
    const long first = (long)team * rpt;
    const int n = (int)max(0L, min((long)rpt, rows - first));
    const uint32_t vec_bytes = blockDim.x * 24, slot_bytes = V * vec_bytes;
    const uint32_t ring_dy = (uint32_t)__cvta_generic_to_shared(ring_raw) + threadIdx.x * 16;
    const uint32_t ring_x = (uint32_t)__cvta_generic_to_shared(ring_raw) + blockDim.x * 16 + threadIdx.x * 8;
    // running addresses: of the next row to copy, to fetch, to write
    const uint16_t* p_dy = dY + first * D + c0;
    const uint8_t* p_x = codes + first * D + c0;
    const uint8_t* p_sb = scales + first * (D >> 5) + (c0 >> 5);
    const float* p_mean = mean + first;
    const float* p_rstd = rstd + first;
    uint16_t* p_dx = dX + first * D + c0;
    const int step_sb = D >> 5;
    int copied = 0, fetched = 0;
    auto issue = [&](int slot) {                     // one commit group per row, also past the end: the count stays uniform
        if (copied < n) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (ok[k]) {
                    copy16(ring_dy + slot * slot_bytes + k * vec_bytes, p_dy + k * cstep);
                    copy8(ring_x + slot * slot_bytes + k * vec_bytes, p_x + k * cstep);
                }
        }
        copy_commit();
        ++copied; p_dy += D; p_x += D;
    };
    auto fetch = [&](Raw<V>& w) {
        w.mean = 0.0f; w.rstd = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) w.sb[k] = 127;
        if (fetched < n) {
            w.mean = __ldg(p_mean); w.rstd = __ldg(p_rstd);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (ok[k]) w.sb[k] = __ldg(p_sb + k * (cstep >> 5));
        }
        ++fetched; ++p_mean; ++p_rstd; p_sb += step_sb;
    };
#pragma unroll
    for (int j = 0; j < P; ++j) issue(j);
    Raw<V> nxt[RI];                                  // one turn ahead
#pragma unroll
    for (int j = 0; j < RI; ++j) fetch(nxt[j]);
    int par = 0, slot0 = 0;
    // every lane of a warp makes the same number of turns (sub-warp teams differ in their last rows alone)
    const int n_max = L == 32 ? n : rpt;
    for (int i0 = 0; i0 < n_max; i0 += RI, par ^= 1) {
        float2 g[RI][V][4], xh[RI][V][4];
        float rs[RI], s[NS];
        copy_wait<P - RI>();                         // the RI oldest rows have landed (each thread waits for its own copies)
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const Raw<V> w = nxt[j];
            rs[j] = w.rstd;
            const float2 minus_mean = bc(-w.mean), r2 = bc(w.rstd);
            float2 s1 = bc(0.0f), s2 = bc(0.0f);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                uint4 dy4 = make_uint4(0, 0, 0, 0);
                uint2 x8 = make_uint2(0, 0);
                if (i0 + j < n && ok[k]) {
                    const uint32_t at = (slot0 + j) * slot_bytes + k * vec_bytes;
                    dy4 = lds16(ring_dy + at); x8 = lds8(ring_x + at);
                }
                const float2 sc = bc(scale_value(w.sb[k]));
                const uint32_t dw[4] = {dy4.x, dy4.y, dy4.z, dy4.w}, xw[2] = {x8.x, x8.y};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 dy = make_float2(bf_lo(dw[i]), bf_hi(dw[i]));
                    xh[j][k][i] = __fmul2_rn(__ffma2_rn(unpack_f8x2<FMT>((uint16_t)(xw[i >> 1] >> (16 * (i & 1)))), sc, minus_mean), r2);
                    g[j][k][i] = __fmul2_rn(dy, gam[k][i]);
                    s1 = __fadd2_rn(s1, g[j][k][i]);
                    s2 = __ffma2_rn(g[j][k][i], xh[j][k][i], s2);
                    dg[k][i] = __ffma2_rn(dy, xh[j][k][i], dg[k][i]);
                    db[k][i] = __fadd2_rn(db[k][i], dy);
                }
            }
            s[2 * j] = s1.x + s1.y; s[2 * j + 1] = s2.x + s2.y;
        }
        // the slots just read are free (this thread was their only reader)
#pragma unroll
        for (int j = 0; j < RI; ++j) { issue(slot0 + j); fetch(nxt[j]); }
        slot0 = slot0 + RI == P ? 0 : slot0 + RI;
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
#pragma unroll
            for (int k = 0; k < V; ++k) {
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = pack2(__ffma2_rn(xh[j][k][i], cb, __ffma2_rn(g[j][k][i], r2, ca)));
                if (i0 + j < n && ok[k]) stg16(p_dx + k * cstep, make_uint4(o[0], o[1], o[2], o[3]));
            }
            p_dx += D;
        }
    }
    copy_wait<0>();
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (ok[k]) {
            float* p = part + (size_t)team * 2 * D + c0 + k * cstep;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<float2*>(p + 2 * i) = dg[k][i];
                *reinterpret_cast<float2*>(p + D + 2 * i) = db[k][i];
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

struct Plan { int lanes, threads, blocks, teams; };

// From the shape alone (148 SMs): the scratch size and the order of the sums do not depend on where the call runs.
Plan plan(int rows, int dim) {
    constexpr int kSms = 148, kMinRows = 8;
    Plan p;
    const int threads = (dim / (dim <= 2048 ? 8 : 16) + 31) / 32 * 32;
    p.lanes = 32;
    while (dim <= 256 && p.lanes / 2 >= dim / 8) p.lanes /= 2;
    p.threads = p.lanes < 32 ? 128 : threads;
    const int per_block = p.lanes < 32 ? p.threads / p.lanes : 1;
    const int resident = std::max(1, std::min(24, 512 / p.threads)) * kSms;      // 16 warps an SM hold 128 registers each
    const int want = (rows - 1) / (kMinRows * per_block) + 1;
    p.blocks = std::max(1, std::min(want, resident));
    p.teams = p.blocks * per_block;
    return p;
}

template <int FMT, int V, int L, int RI, int P, int MAXT, int MINB>
cudaError_t launch_t(const Plan& p, cudaStream_t s, const uint8_t* codes, const uint8_t* scales, const uint16_t* dY, const float* gamma,
                     const float* mean, const float* rstd, uint16_t* dX, float* part, int rows, int dim) {
    auto kernel = ln_bwd_act8_kernel<FMT, V, L, RI, P, MAXT, MINB>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P * MAXT * 24 * V);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3(p.blocks), dim3(p.threads), (size_t)P * p.threads * 24 * V, s, codes, scales, dY, gamma, mean, rstd, dX, part,
                      rows, dim, p.teams);
}

template <int FMT, class... A>
cudaError_t launch_f(const Plan& p, int dim, A... a) {
    switch (p.lanes) {
        case 4: return launch_t<FMT, 1, 4, 4, 8, 128, 4>(p, a...);
        case 8: return launch_t<FMT, 1, 8, 4, 8, 128, 4>(p, a...);
        case 16: return launch_t<FMT, 1, 16, 4, 8, 128, 4>(p, a...);
        default: break;
    }
    if (dim <= 256) return launch_t<FMT, 1, 32, 4, 8, 32, 16>(p, a...);
    if (dim <= 2048) return launch_t<FMT, 1, 32, 4, 8, 256, 2>(p, a...);
    return launch_t<FMT, 2, 32, 2, 4, 512, 1>(p, a...);
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
        cuda_ok(format == kE4M3 ? launch_f<kE4M3>(p, dim, s, c, sc, dy, gamma, mean, rstd, dx, part, rows, dim)
                                : launch_f<kE5M2>(p, dim, s, c, sc, dy, gamma, mean, rstd, dx, part, rows, dim), "ln_backward_act8 launch");
        cuda_ok(launch_pdl(ln_bwd_act8_reduce_kernel, dim3(2 * dim / 32), dim3(1024), 0, s, part, p.teams, dim, dGamma, dBeta), "ln_backward_act8 launch");
    })
}

}  // extern "C"
