// Microscaled blocks: 32 neighbouring elements of a row and one power-of-two scale. Device arithmetic shared by the
// casts, the LayerNorm checkpoints and the GEMM epilogues.
//
//   value_i = q_i * 2^(byte - 127),  byte in [0, 254];  byte 255: the block held an infinity or NaN and stands for NaN
//
// Scale rule: the smallest power of two at which no element passes the type's largest value V (6, 448 or 57344). With
// amax = (1 + m) * 2^(E - 127) and V = v * 2^emax, 1 <= v < 2, that exponent is E - emax, one more where 1 + m > v: two
// integer operations on the bits of amax, exact, no division and no logarithm. (The published microscaling formats
// leave the scale to the producer; rounding its exponent down instead would clip up to a quarter of the block's largest
// element in e2m1.) Elements are then rounded to nearest, ties to even; nothing saturates. Multiplying by a power of two
// is exact in fp32 but for results below 2^-126, which lie far under half of the smallest step of every element type.
#pragma once
#include "common.cuh"

namespace tmt {
namespace mx {

enum Fmt : int { kE2M1 = 0, kE4M3 = 1, kE5M2 = 2 };      // kE4M3 / kE5M2 as TMT_ACT8_E4M3 / TMT_ACT8_E5M2
constexpr int kBlock = 32;

template <int FMT> struct FmtTraits;
template <> struct FmtTraits<kE2M1> { static constexpr int emax = 2; static constexpr uint32_t frac = 0x400000u; };    // 6 = 1.5 * 2^2
template <> struct FmtTraits<kE4M3> { static constexpr int emax = 8; static constexpr uint32_t frac = 0x600000u; };    // 448 = 1.75 * 2^8
template <> struct FmtTraits<kE5M2> { static constexpr int emax = 15; static constexpr uint32_t frac = 0x600000u; };   // 57344 = 1.75 * 2^15

// Scale byte of a block from the fp32 bits of its largest magnitude (taken as an integer maximum of |x|'s bits, so that
// infinities and NaN, whose bits are the largest, are seen).
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int b = (int)(amax_bits >> 23) - FmtTraits<FMT>::emax + ((amax_bits & 0x7fffffu) > FmtTraits<FMT>::frac ? 1 : 0);
    return (uint32_t)max(b, 0);
}
// 2^(127 - byte): always a normal number for byte <= 254. 0 for byte 255, with which a finite element becomes code 0
// (and the others are masked by the caller): the bytes of a non-finite block are the same whatever it held.
__device__ __forceinline__ float inv_scale(uint32_t byte) { return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); byte 0 is 2^-127, a subnormal, byte 255 is NaN
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
}

// 8 floats -> 8 e2m1 codes, element 0 in the lowest nibble
__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&f)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}
// 4 floats -> 4 bytes of e4m3 / e5m2
template <int FMT>
__device__ __forceinline__ uint32_t pack_f8x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    if constexpr (FMT == kE4M3) {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    } else {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    }
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// two packed bytes -> two floats (exact: both types are subsets of fp16)
template <int FMT>
__device__ __forceinline__ float2 unpack_f8x2(uint16_t v) {
    uint32_t h;
    if constexpr (FMT == kE4M3) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
    else asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(v));
    float2 f;
    asm("{\n\t.reg .f16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
// 8 e2m1 codes -> 8 floats
__device__ __forceinline__ void unpack_e2m1x8(uint32_t w, float (&f)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("{\n\t.reg .f16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}" : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "r"(h[i]));
}

// 8 values of a row (16 bytes of bf16, 32 of fp32) as floats; returns the fp32 bits of the largest magnitude among them
__device__ __forceinline__ uint32_t spread8(const uint4& a, float (&f)[8]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    uint32_t m = 0;                                           // two 16-bit maxima: magnitudes of bf16 order like their bits
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf_lo(w[i]); f[2 * i + 1] = bf_hi(w[i]); m = __vmaxu2(m, w[i] & 0x7fff7fffu); }
    return max(m >> 16, m & 0xffffu) << 16;
}
__device__ __forceinline__ uint32_t spread8(const uint4& a, const uint4& b, float (&f)[8]) {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { f[i] = __uint_as_float(w[i]); m = max(m, w[i] & 0x7fffffffu); }
    return m;
}
// Scale byte of a block held by 4 neighbouring lanes, 8 elements each, which are brought to units of the scale; m: the lane's largest.
template <int FMT>
__device__ __forceinline__ uint32_t scale_block(float (&f)[8], uint32_t m) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t sb = scale_byte<FMT>(m);
    const float inv = inv_scale(sb);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= inv;
    return sb;
}
// The lane's 8 codes, and the word of scale bytes of the 4 blocks its 16 lanes hold (blocks of lanes that are not ok: 0).
__device__ __forceinline__ uint32_t quantize8_e2m1(float (&f)[8], uint32_t m, bool ok, int lane, uint32_t& word) {
    const uint32_t sb = scale_block<kE2M1>(f, m);
    word = ok ? sb << (8 * ((lane >> 2) & 3)) : 0u;
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    return sb == 255u ? 0u : pack_e2m1x8(f);
}

// ---- 4-bit matrices: where the scale bytes lie ----
// The tensor cores read the scales of 128 rows x 4 blocks (128 columns) as one 512-byte tile: byte
// (row % 32) * 16 + (row % 128 / 32) * 4 + block % 4, copied to tensor memory as it is. A matrix keeps them in that
// order: tiles of a 128-row band one after the other, band after band; rows and blocks are padded to whole tiles.
constexpr int kScaleTile = 512;
// Sizes go up to the end of the int range, so rounding up starts from one less. a >= 1.
__host__ __device__ __forceinline__ constexpr int ceil_div(int a, int b) { return (a - 1) / b + 1; }
__host__ __device__ __forceinline__ int scale_tiles_k(int cols) { return ceil_div(cols, 128); }
__host__ __device__ __forceinline__ size_t scale_bytes(long rows, int cols) {
    return (size_t)((rows + 127) / 128) * scale_tiles_k(cols) * kScaleTile;
}
// address of the 4-byte word that holds the blocks 4t .. 4t+3 of a row
__host__ __device__ __forceinline__ size_t scale_word(long row, int t, int tiles_k) {
    return ((size_t)(row >> 7) * tiles_k + t) * kScaleTile + (size_t)(row & 31) * 16 + (size_t)((row & 127) >> 5) * 4;
}

}  // namespace mx
}  // namespace tmt
