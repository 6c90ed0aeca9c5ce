// Matrices into microscaled blocks and back (include/tmt_mx.h): 4-bit weights and activations, 8-bit checkpoints.
//
// A warp takes 256 neighbouring elements of a row, 8 per lane, so that a block of 32 is 4 lanes: one 16-byte load per lane
// (two for fp32), the block's largest magnitude by two shuffles, one store of 4 (e2m1) or 8 bytes (e4m3, e5m2) per lane. Every
// byte moves once; bound by HBM. In 4 bits a warp takes the same 256 columns of the rows r, r + 32, r + 64 and r + 96 of a band of 128,
// whose scale words are neighbours in the scale tile (single words, one row a warp, took 150 us instead of 114 at 131072 x 2048). Several
// such chunks are in flight per warp where there are enough of them (U). Rows below 256 columns leave lanes idle: 131072 x 64 takes 18 us
// in either direction and format, beside a floor of 3 to 4, as 131072 x 256 does (20 | 13 to 16).
// `early`: lets the next kernel of the stream be scheduled at once (launch_pdl.cuh). Only where that kernel is known to wait
// before it reads anything: the product of a dense layer, whose barriers and tensor memory are then ready when this kernel ends.
#include <cuda_runtime.h>

#include "../../include/tmt_mx.h"
#include "launch_pdl.cuh"
#include "mx.cuh"
#include "mx_cast.h"
#include "mx_host.h"

namespace tmt {
namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 256;             // elements a warp takes at a time

template <bool F32> struct Vec8 { uint4 a, b; };
template <> struct Vec8<false> { uint4 a; };

template <bool F32>
__device__ __forceinline__ Vec8<F32> load8(const void* X, size_t at) {
    Vec8<F32> v;
    if constexpr (F32) {
        const float* p = static_cast<const float*>(X) + at;
        v.a = ldg16_stream(p); v.b = ldg16_stream(p + 4);
    } else {
        v.a = ldg16_stream(static_cast<const uint16_t*>(X) + at);
    }
    return v;
}
template <bool F32>
__device__ __forceinline__ uint32_t spread(const Vec8<F32>& v, float (&f)[8]) {
    if constexpr (F32) return spread8(v.a, v.b, f);
    else return spread8(v.a, f);
}

template <int FMT, bool F32, int U>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const void* __restrict__ X, unsigned rows, int cols, unsigned chunks,
                                                               unsigned per_row, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, bool early) {
    pdl_wait();
    if (early) pdl_begin();
    const int lane = threadIdx.x & 31;
    const unsigned c0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * U;
    size_t at[U]; unsigned row[U]; int col[U]; bool ok[U];
    Vec8<F32> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned c = FMT == kE2M1 ? c0 / U : c0 + u;
        row[u] = c / per_row;
        col[u] = (int)(c - row[u] * per_row) * kChunk + lane * 8;
        if (FMT == kE2M1) row[u] = (row[u] >> 5) * 128 + (row[u] & 31) + u * 32;      // rows r, r + 32, r + 64, r + 96 of a band
        ok[u] = c < chunks && row[u] < rows && col[u] < cols;                             // cols is a multiple of 32: whole blocks
        at[u] = (size_t)row[u] * cols + col[u];
        v[u] = Vec8<F32>{};
        if (ok[u]) v[u] = load8<F32>(X, at[u]);
    }
    uint32_t word[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (FMT != kE2M1 && c0 + u >= chunks) break;          // whole warps leave together
        float f[8];
        const uint32_t m = spread<F32>(v[u], f);
        if constexpr (FMT == kE2M1) {
            const uint32_t q = quantize8_e2m1(f, m, ok[u], lane, word[u]);
            if (ok[u]) *reinterpret_cast<uint32_t*>(codes + at[u] / 2) = q;
        } else {
            const uint32_t sb = scale_block<FMT>(f, m);
            uint32_t lo = pack_f8x4<FMT>(f[0], f[1], f[2], f[3]), hi = pack_f8x4<FMT>(f[4], f[5], f[6], f[7]);
            if (sb == 255u) { lo = 0; hi = 0; }
            if (ok[u]) {
                *reinterpret_cast<uint2*>(codes + at[u]) = make_uint2(lo, hi);
                if ((lane & 3) == 0) scales[at[u] >> 5] = (uint8_t)sb;
            }
        }
    }
    if constexpr (FMT == kE2M1) {
        // the four words of rows r .. r + 96 are neighbours in the scale tile: one 16-byte store (rows past the last: 0, inside the tile)
        static_assert(FMT != kE2M1 || U == 4, "one row of each quarter of a band");
        if ((lane & 15) == 0 && ok[0])
            stg16(scales + scale_word(row[0], col[0] >> 7, scale_tiles_k(cols)), make_uint4(word[0], word[1], word[2], word[3]));
    }
}

template <int FMT, bool F32, int U>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                 unsigned rows, int cols, unsigned chunks, unsigned per_row,
                                                                 void* __restrict__ Y) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const unsigned c0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * U;
    size_t at[U]; bool ok[U]; uint2 q[U]; uint32_t sb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned c = c0 + u, row = c / per_row;
        const int col = (int)(c - row * per_row) * kChunk + lane * 8;
        ok[u] = c < chunks && col < cols;
        at[u] = (size_t)row * cols + col;
        q[u] = make_uint2(0, 0); sb[u] = 0;
        if (ok[u]) {
            if constexpr (FMT == kE2M1) {
                q[u].x = __ldg(reinterpret_cast<const uint32_t*>(codes + at[u] / 2));
                sb[u] = __ldg(scales + scale_word(row, col >> 7, scale_tiles_k(cols)) + ((col >> 5) & 3));
            } else {
                q[u] = __ldg(reinterpret_cast<const uint2*>(codes + at[u]));
                sb[u] = __ldg(scales + (at[u] >> 5));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!ok[u]) continue;
        float f[8];
        if constexpr (FMT == kE2M1) unpack_e2m1x8(q[u].x, f);
        else {
            const uint32_t w[2] = {q[u].x, q[u].y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 p = unpack_f8x2<FMT>((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
                f[2 * i] = p.x; f[2 * i + 1] = p.y;
            }
        }
        const float s = scale_value(sb[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= s;
        if constexpr (F32) {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(Y) + at[u]);
            dst[0] = make_float4(f[0], f[1], f[2], f[3]);
            dst[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            stg16(static_cast<uint16_t*>(Y) + at[u], make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7])));
        }
    }
}

struct Grid { unsigned chunks, per_row; int u; dim3 grid; };

// bands: chunks are counted over 32 rows of every band of 128 (4-bit quantiser: a warp takes four rows of a band at once)
Grid plan(long long rows, int cols, bool bands = false) {
    Grid g;
    g.per_row = (unsigned)ceil_div(cols, kChunk);
    if (rows > 0x7fffffffLL / g.per_row) throw std::runtime_error("rows * cols exceeds the supported range");
    if (bands) {
        const long long r = rows / 128 * 32 + (rows % 128 < 32 ? rows % 128 : 32);
        g.chunks = (unsigned)(r * g.per_row);
        g.u = 4;
        g.grid = dim3((g.chunks + kWarps - 1) / kWarps);
        return g;
    }
    g.chunks = (unsigned)(rows * g.per_row);
    // few chunks: one per warp, spread over the SMs; many: four loads in flight per lane
    g.u = g.chunks < 16384u ? 1 : 4;
    g.grid = dim3((g.chunks + kWarps * g.u - 1) / (kWarps * g.u));
    return g;
}

template <int FMT>
cudaError_t quantize_t(const void* X, bool f32, long long rows, int cols, uint8_t* codes, uint8_t* scales, cudaStream_t s, bool early = false) {
    const Grid g = plan(rows, cols, FMT == kE2M1);
    auto go = [&](auto kernel) { return launch_pdl(kernel, g.grid, dim3(kThreads), 0, s, X, (unsigned)rows, cols, g.chunks, g.per_row, codes, scales, early); };
    if constexpr (FMT == kE2M1) return f32 ? go(mx_quantize_kernel<FMT, true, 4>) : go(mx_quantize_kernel<FMT, false, 4>);
    else {
        if (f32) return g.u == 1 ? go(mx_quantize_kernel<FMT, true, 1>) : go(mx_quantize_kernel<FMT, true, 4>);
        return g.u == 1 ? go(mx_quantize_kernel<FMT, false, 1>) : go(mx_quantize_kernel<FMT, false, 4>);
    }
}

template <int FMT>
cudaError_t dequantize_t(const uint8_t* codes, const uint8_t* scales, long long rows, int cols, void* Y, bool f32, cudaStream_t s) {
    const Grid g = plan(rows, cols);
    auto go = [&](auto kernel) { return launch_pdl(kernel, g.grid, dim3(kThreads), 0, s, codes, scales, (unsigned)rows, cols, g.chunks, g.per_row, Y); };
    if (f32) return g.u == 1 ? go(mx_dequantize_kernel<FMT, true, 1>) : go(mx_dequantize_kernel<FMT, true, 4>);
    return g.u == 1 ? go(mx_dequantize_kernel<FMT, false, 1>) : go(mx_dequantize_kernel<FMT, false, 4>);
}

void check_shape(long long rows, int cols, int multiple, int dtype) {
    if (rows < 0 || cols < multiple || cols % multiple)
        throw std::runtime_error("need rows >= 0 and cols a positive multiple of " + std::to_string(multiple));
    if (dtype != TMT_MOE_BF16 && dtype != TMT_MOE_F32) throw std::runtime_error("dtype must be TMT_MOE_BF16 or TMT_MOE_F32");
}
void check_format(int format) {
    if (format != TMT_ACT8_E4M3 && format != TMT_ACT8_E5M2) throw std::runtime_error("format must be TMT_ACT8_E4M3 or TMT_ACT8_E5M2");
}

}  // namespace

cudaError_t launch_mx4_quantize(const void* X, bool f32, long long rows, int cols, void* codes, void* scales, cudaStream_t s, bool early) {
    return quantize_t<kE2M1>(X, f32, rows, cols, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), s, early);
}

}  // namespace tmt

using namespace tmt;

extern "C" {

size_t tmt_moe_mxfp4_scale_bytes(long long rows, int cols) {
    return rows < 0 || cols < 64 || cols % 64 ? 0 : mx::scale_bytes((long)rows, cols);
}

int tmt_moe_quantize_mxfp4(const void* X, int dtype, long long rows, int cols, void* codes, void* scales, void* stream) {
    MX_GUARD({
        check_shape(rows, cols, 64, dtype);
        if (rows == 0) return 0;
        check_tensors({X, codes, scales});
        cuda_ok(launch_mx4_quantize(X, dtype == TMT_MOE_F32, rows, cols, codes, scales, static_cast<cudaStream_t>(stream), false), "quantize_mxfp4 launch");
    })
}

int tmt_moe_dequantize_mxfp4(const void* codes, const void* scales, long long rows, int cols, void* Y, int dtype, void* stream) {
    MX_GUARD({
        check_shape(rows, cols, 64, dtype);
        if (rows == 0) return 0;
        check_tensors({codes, scales, Y});
        cuda_ok(dequantize_t<mx::kE2M1>(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, cols, Y,
                                        dtype == TMT_MOE_F32, static_cast<cudaStream_t>(stream)), "dequantize_mxfp4 launch");
    })
}

int tmt_moe_act8_save(const void* X, int dtype, long long rows, int cols, int format, void* codes, void* scales, void* stream) {
    MX_GUARD({
        check_shape(rows, cols, 32, dtype);
        check_format(format);
        if (rows == 0) return 0;
        check_tensors({X, codes, scales});
        uint8_t* c = static_cast<uint8_t*>(codes);
        uint8_t* sc = static_cast<uint8_t*>(scales);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool f32 = dtype == TMT_MOE_F32;
        cuda_ok(format == TMT_ACT8_E4M3 ? quantize_t<mx::kE4M3>(X, f32, rows, cols, c, sc, s) : quantize_t<mx::kE5M2>(X, f32, rows, cols, c, sc, s),
                "act8_save launch");
    })
}

int tmt_moe_act8_restore(const void* codes, const void* scales, long long rows, int cols, int format, void* Y, int dtype, void* stream) {
    MX_GUARD({
        check_shape(rows, cols, 32, dtype);
        check_format(format);
        if (rows == 0) return 0;
        check_tensors({codes, scales, Y});
        const uint8_t* c = static_cast<const uint8_t*>(codes);
        const uint8_t* sc = static_cast<const uint8_t*>(scales);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool f32 = dtype == TMT_MOE_F32;
        cuda_ok(format == TMT_ACT8_E4M3 ? dequantize_t<mx::kE4M3>(c, sc, rows, cols, Y, f32, s) : dequantize_t<mx::kE5M2>(c, sc, rows, cols, Y, f32, s),
                "act8_restore launch");
    })
}

}  // extern "C"
