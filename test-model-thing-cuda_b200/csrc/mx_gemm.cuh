// Device pieces shared by the two 4-bit product kernels (mx_gemm.cu, mx_gemm_2cta.cu): descriptors, groups and tiles.
#pragma once
#include "mx.cuh"
#include "mx_gemm.h"
#include "tc_util.cuh"

namespace tmt {
namespace mxg {

using namespace tc;
using namespace mx;

constexpr int kKB = 256;                 // elements of k per pipeline stage: one 128-byte swizzle row, two scale tiles
constexpr int kMaxExperts = 256;

// Instruction descriptor: e2m1 operands, e8m0 scales, both K-major, m rows x n columns. The scale ids (0 or 2) pick the
// blocks 0-1 or 2-3 of a scale tile, i.e. the first or second 64 elements of its 128.
__device__ __forceinline__ uint32_t mxf4_idesc(uint32_t m, uint32_t n) { return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24); }
__device__ __forceinline__ uint32_t mxf4_ids(uint32_t id) { return (id << 4) | (id << 29); }
// 512-byte scale tile in shared memory: 32 rows of 16 bytes, 8-row groups 128 bytes apart, no swizzle
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)(16u >> 4) << 16) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46);
}
// a scale tile into 4 columns of tensor memory: 32 lanes x 16 bytes, repeated for the four lane quarters
__device__ __forceinline__ void scale_copy(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {      // this address in another CTA of the cluster
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
struct Groups {                          // in shared memory: the experts' groups and their tiles on the activation side
    int first[kMaxExperts + 1];          // first activation tile of each group
    int poff[kMaxExperts], count[kMaxExperts];
};
struct Tile {
    int expert, row0, rows, w0;          // activation rows [row0, row0 + rows), weight rows from w0
};

template <int TA>                        // activation rows of a tile
__device__ __forceinline__ void load_groups(const MxGemm& p, Groups& g) {
    if (p.experts == 0) {
        if (threadIdx.x == 0) { g.first[0] = 0; g.first[1] = ceil_div(p.rows, TA); g.poff[0] = 0; g.count[0] = p.rows; }
        return;
    }
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
        const int r0 = p.poff[e];
        int c = p.counts[e];
        if (r0 < 0 || (r0 & 127) || c < 0 || (long)r0 + c > p.row_limit) { report(p.status, kErrSlotRange); c = 0; }
        g.poff[e] = r0; g.count[e] = c;
    }
    __syncthreads();
    if (threadIdx.x < 32) {              // prefix sum over the experts, 32 at a time
        int base = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + threadIdx.x;
            const int t = e < p.experts ? (g.count[e] + TA - 1) / TA : 0;
            int incl = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if ((int)threadIdx.x >= o) incl += v;
            }
            if (e < p.experts) g.first[e] = base + incl - t;
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (threadIdx.x == 0) g.first[p.experts] = base;
    }
}
template <int TA, int TW>
__device__ __forceinline__ bool get_tile(const MxGemm& p, const Groups& g, int t, int w_tiles, Tile& ti) {
    const int ng = p.experts == 0 ? 1 : p.experts;
    const int at = t / w_tiles;
    if (at >= g.first[ng]) return false;
    int lo = 0, hi = ng;                 // last expert whose first tile is <= at and that has tiles
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (g.first[mid] <= at) lo = mid; else hi = mid; }
    const int off = (at - g.first[lo]) * TA;
    ti.expert = lo;
    ti.row0 = g.poff[lo] + off;
    ti.rows = min(TA, g.count[lo] - off);
    ti.w0 = (t - at * w_tiles) * TW;
    return true;
}

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Starts the load of 64 columns of the warp's 32 lanes; the registers hold them after tmem_wait64.
__device__ __forceinline__ void tmem_start64(uint32_t addr, uint32_t (&r)[64]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[32 * h + 0]), "=r"(r[32 * h + 1]), "=r"(r[32 * h + 2]), "=r"(r[32 * h + 3]), "=r"(r[32 * h + 4]), "=r"(r[32 * h + 5]),
              "=r"(r[32 * h + 6]), "=r"(r[32 * h + 7]), "=r"(r[32 * h + 8]), "=r"(r[32 * h + 9]), "=r"(r[32 * h + 10]), "=r"(r[32 * h + 11]),
              "=r"(r[32 * h + 12]), "=r"(r[32 * h + 13]), "=r"(r[32 * h + 14]), "=r"(r[32 * h + 15]), "=r"(r[32 * h + 16]), "=r"(r[32 * h + 17]),
              "=r"(r[32 * h + 18]), "=r"(r[32 * h + 19]), "=r"(r[32 * h + 20]), "=r"(r[32 * h + 21]), "=r"(r[32 * h + 22]), "=r"(r[32 * h + 23]),
              "=r"(r[32 * h + 24]), "=r"(r[32 * h + 25]), "=r"(r[32 * h + 26]), "=r"(r[32 * h + 27]), "=r"(r[32 * h + 28]), "=r"(r[32 * h + 29]),
              "=r"(r[32 * h + 30]), "=r"(r[32 * h + 31])
            : "r"(addr + 32 * h) : "memory");
}
// After the wait no use of the registers may move above it.
__device__ __forceinline__ void tmem_wait64(uint32_t (&r)[64]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

__device__ __forceinline__ float exp2_fast(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp_fast(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// silu of a block of 32 accumulators, in place. The special-function unit sets the pace of this epilogue (16 results a clock and SM): two
// neighbours share one reciprocal, 1 / a = b / (a b), so that an element costs 1.5 of its results instead of 2. a b stays finite,
// and its reciprocal a normal number, while both exponents are below 43; a block that holds an element below -43 takes the plain form.
// The choice is the block's own (a thread holds it whole), never the warp's, whose other lanes are other tokens; silu_lane is the same
// function with a block in the lanes of a warp, bit for bit. So a token's hidden row is the same in any batch.
constexpr float kMinusLog2e = -1.4426950408889634f, kSiluPairMin = -43.0f;
__device__ __forceinline__ void silu32(float (&f)[32]) {
    float lo = fminf(f[0], f[1]);
#pragma unroll
    for (int i = 2; i < 32; i += 2) lo = fminf(fminf(lo, f[i]), f[i + 1]);
    if (lo > kSiluPairMin) {                             // false for a NaN in every element alone; others propagate through either form
        const float2 c = make_float2(kMinusLog2e, kMinusLog2e), one = make_float2(1.0f, 1.0f);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 x = make_float2(f[i], f[i + 1]);
            float2 e = __fmul2_rn(x, c);
            e = __fadd2_rn(make_float2(exp2_fast(e.x), exp2_fast(e.y)), one);
            const float r = rcp_fast(e.x * e.y);
            f[i] = x.x * (r * e.y);
            f[i + 1] = x.y * (r * e.x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = f[i] * sigmoid_fast(f[i]);
    }
}
__device__ __forceinline__ float silu_lane(float x) {
    const float e = __fadd_rn(exp2_fast(__fmul_rn(x, kMinusLog2e)), 1.0f), other = __shfl_xor_sync(0xffffffffu, e, 1);
    const float r = rcp_fast(__fmul_rn(e, other));
    return __any_sync(0xffffffffu, x <= kSiluPairMin) ? x * sigmoid_fast(x) : __fmul_rn(x, __fmul_rn(r, other));
}
// One block of 32 -> its 4-bit codes, element 0 in the lowest nibble of q[0]; returns the scale byte.
__device__ __forceinline__ uint32_t quantize32(const float (&f)[32], uint32_t (&q)[4]) {
    float m = 0.0f;                                      // NaN-propagating maximum of the magnitudes
#pragma unroll
    for (int i = 0; i < 32; i += 2)
        asm("{\n\t.reg .f32 a, b;\n\tabs.f32 a, %1;\n\tabs.f32 b, %2;\n\tmax.NaN.f32 a, a, b;\n\tmax.NaN.f32 %0, %0, a;\n\t}" : "+f"(m) : "f"(f[i]), "f"(f[i + 1]));
    const uint32_t sb = scale_byte<kE2M1>(__float_as_uint(m));
    const float inv = inv_scale(sb);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = f[8 * j + i] * inv;
        q[j] = sb == 255u ? 0u : pack_e2m1x8(g);
    }
    return sb;
}

}  // namespace mxg
}  // namespace tmt
