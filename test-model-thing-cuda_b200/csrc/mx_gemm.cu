// Products of 4-bit microscaled matrices on the block-scaled tensor-core instruction of sm_100a
// (tcgen05.mma kind::mxf4, e2m1 operands, one e8m0 scale per 32 elements of each operand).
//
//   acc[i, j] = sum over blocks b of  sP[i, b] sQ[j, b]  sum over the block of qP qQ
//
// Operand P, on the 128-row side of the MMA, are activations, Q, on its column side, weights.
//
// Codes travel by TMA in boxes of 128 bytes (256 elements of k) with the 128-byte swizzle, exactly as a bf16 operand of 64
// elements would; an MMA takes 64 elements (32 bytes). Scales travel as whole 512-byte tiles (128 rows x 4 blocks) by untiled
// bulk copies into shared memory and from there by tcgen05.cp (32 lanes x 16 bytes, repeated for the four lane quarters) into
// tensor memory, 4 columns per tile; the MMA reads two of the four blocks, picked by the scale ids of its descriptor. An MMA and
// the copies issued before it by the same thread run in order, so the scale columns need no second buffer.
//
// Warps: 0 = TMA producer of P, 1 = MMA issuer and TMEM owner, 2..9 = epilogue (two groups of four, 64 outputs each), 10 = TMA
// producer of Q. Persistent over tiles of 128 x 128, two accumulators in tensor memory. Every wait is bounded, as in the bf16 kernels.
//
// This form serves products of up to a few turns of tiles (mx_form below; mx_gemm_2cta.cu takes the larger ones). They are bound by
// latency: a launch, the first loads, a tile's products and its epilogue, one after the other. 128 x 1024 -> 1024 takes 4.3 us, 777 x
// 1344 -> 2504 5.4 us (bf16 out) and 6.0 us (fp32 out), each k block of 256 about 0.3 us of it.
#include <stdexcept>
#include <string>

#include "launch_pdl.cuh"
#include "mx_gemm.cuh"

namespace tmt {
namespace {

using namespace mxg;

constexpr int kBP = 128;                 // rows of a tile on the P side
constexpr int kThreads = 352;
constexpr int kOutBox = 32 * 128;        // staged outputs of a warp: its 32 rows x 128 bytes

constexpr int kBQ = 128;                 // and on the Q side
constexpr int kCodesP = kBP * 128, kCodesQ = kBQ * 128;
constexpr int kSf = 2 * kScaleTile;      // scale tiles of either side
constexpr int kStageBytes = kCodesP + kCodesQ + 2 * kSf;
constexpr int kStages = (220 * 1024 - 8 * kOutBox) / kStageBytes;
constexpr int kSmem = kStages * kStageBytes + 8 * kOutBox + 1024;
constexpr uint32_t kSfCol = 2 * kBQ;     // scale columns follow the two accumulators
constexpr uint32_t kTmemCols = 512;
static_assert(kSfCol + 16 <= kTmemCols, "tensor memory");

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_mxf4(uint32_t tmem_d, uint64_t dp, uint64_t dq, uint32_t idesc, uint32_t sfp, uint32_t sfq, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(dp), "l"(dq), "r"(idesc), "r"(sfp), "r"(sfq), "r"(accumulate) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// The epilogue of one warp: 32 rows (its TMEM lanes) and 64 of the tile's 128 outputs. The accumulator is handed back once its
// 64 columns are in registers. Outputs go through 4 KB of shared memory per warp, so that 8 lanes store the 128 bytes of a row
// together: a lane per row, 16 bytes each into 32 rows, took 1.4 us more for the fp32 outputs of a single turn of tiles.
template <int EPI>
__device__ __forceinline__ void drain_tile(const MxGemm& p, const Tile& ti, uint32_t tm, int quarter, int group, uint32_t buf, uint32_t tempty, int lane) {
    const int row0 = ti.row0 + quarter * 32, rows = ti.rows - quarter * 32, col0 = ti.w0 + group * 64;
    const long row = (long)row0 + lane;
    float gate = 0.0f;
    if constexpr (EPI == kMxDown) gate = lane < rows ? p.row_scale[row] : 0.0f;
    uint32_t v[64];
    tmem_start64(tm + group * 64, v);
    tmem_wait64(v);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(tempty);
    if (rows <= 0 || col0 >= p.n) return;
    if constexpr (EPI == kMxUp) {            // silu, then two blocks of 32: 32 bytes of codes and two scale bytes per row
        uint32_t scales = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float f[32];
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[32 * b + i]);
            silu32(f);
            const uint32_t sb = quantize32(f, q);
            if (lane < rows) stg16(static_cast<uint8_t*>(p.out) + row * (p.n / 2) + col0 / 2 + 16 * b, make_uint4(q[0], q[1], q[2], q[3]));
            scales |= sb << (8 * b);
        }
        if (lane < rows)
            *reinterpret_cast<uint16_t*>(p.out_scales + scale_word(row, col0 >> 7, scale_tiles_k(p.n)) + ((col0 >> 5) & 3)) = (uint16_t)scales;
    } else {
        constexpr int kBytes = EPI == kMxBf16 ? 2 : 4, kBoxCols = 128 / kBytes;
        uint8_t* out = static_cast<uint8_t*>(p.out);
#pragma unroll
        for (int x0 = 0; x0 < 64; x0 += kBoxCols) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (EPI == kMxF32) w[i] = v[x0 + 4 * q + i];
                    else if constexpr (EPI == kMxDown) w[i] = __float_as_uint(gate * __uint_as_float(v[x0 + 4 * q + i]));
                    else w[i] = pack_pair(__uint_as_float(v[8 * q + 2 * i]), __uint_as_float(v[8 * q + 2 * i + 1]));
                }
                st_shared16(buf + lane * 128 + ((q ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            const int c = lane & 7;
            const bool col_ok = col0 + x0 + c * (16 / kBytes) < p.n;       // n is a multiple of 8: whole 16-byte pieces
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + (lane >> 3);
                if (r < rows && col_ok) stg16(out + ((long)(row0 + r) * p.n + col0 + x0) * kBytes + c * 16, lds16(buf + r * 128 + ((c ^ (r & 7)) << 4)));
            }
            __syncwarp();
        }
    }
}

template <int EPI>
__global__ void __launch_bounds__(kThreads, 1) mx_gemm_kernel(const __grid_constant__ MxGemm p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], tfull_bar[2], tempty_bar[2];
    __shared__ Groups groups;
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t codes_p = base, codes_q = base + kStages * kCodesP, sf_p = codes_q + kStages * kCodesQ, sf_q = sf_p + kStages * kSf;
    volatile int* abort_flag = &abort_s;

    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < kStages; ++s) { mbar_init(smem_u32(&full_bar[s]), 2); mbar_init(smem_u32(&empty_bar[s]), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(smem_u32(&tfull_bar[a]), 1); mbar_init(smem_u32(&tempty_bar[a]), 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_begin();                         // not before: the next kernel could take the tensor memory this one is about to ask for
    }
    pdl_wait();
    load_groups<kBP>(p, groups);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;
    const int w_tiles = ceil_div(p.n, kBQ);
    const int nkb = ceil_div(p.k, kKB);
    const int tiles_k = scale_tiles_k(p.k);

    if (warp == 0 || warp == 10) {
        // ---------------- producers: codes box and scale tiles of one operand per stage ----------------
        if (lane == 0) {
            const bool is_p = warp == 0;
            int s = 0; uint32_t ph = 0;
            uint32_t issued = 0, last_parity = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok; t += gridDim.x) {
                Tile ti;
                if (!get_tile<kBP, kBQ>(p, groups, t, w_tiles, ti)) break;
                const CUtensorMap* map;
                const uint8_t* sc;
                int row;
                if (is_p) {
                    map = &p.act; sc = p.act_scales; row = ti.row0;
                } else {
                    map = p.w_maps ? p.w_maps + ti.expert : &p.w;
                    sc = p.w_scales_tab ? p.w_scales_tab[ti.expert] : p.w_scales;
                    row = ti.w0;
                    if (p.w_maps) tensormap_acquire(map);
                }
                const size_t band = (size_t)(row >> 7) * tiles_k;      // first scale tile of the tile's 128 rows
                for (int kb = 0; kb < nkb; ++kb) {
                    ok = mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, p.status);
                    if (!ok) break;
                    const uint32_t fb = smem_u32(&full_bar[s]);
                    const uint32_t sf_bytes = (uint32_t)min(2, tiles_k - 2 * kb) * kScaleTile;
                    static_assert(kCodesP == kCodesQ, "one box size for both operands");
                    mbar_expect_tx(fb, kCodesP + sf_bytes);
                    tma_load_2d((is_p ? codes_p : codes_q) + s * kCodesP, map, fb, kb * 128, row);
                    bulk_load((is_p ? sf_p : sf_q) + s * kSf, sc + (band + 2 * kb) * kScaleTile, sf_bytes, fb);
                    issued |= 1u << s;
                    last_parity = (last_parity & ~(1u << s)) | (ph << s);
                    if (++s == kStages) { s = 0; ph ^= 1; }
                }
            }
            if (!ok)       // aborting: wait (bounded) until the copies already issued have landed
                for (int q = 0; q < kStages; ++q) {
                    if (!(issued >> q & 1)) continue;
                    const long long t0 = clock64();
                    while (!mbar_try_wait(smem_u32(&full_bar[q]), (last_parity >> q) & 1) && clock64() - t0 < kWaitCycles) {}
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA issuer: the whole warp runs the loop, one elected lane issues ----------------
        const uint32_t sfp_t = tmem_base + kSfCol, sfq_t = sfp_t + 8;
        const uint32_t idesc0 = mxf4_idesc(kBP, kBQ);
        int s = 0; uint32_t ph = 0;
        int acc = 0; uint32_t acc_ph = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok; t += gridDim.x) {
            Tile ti;
            if (!get_tile<kBP, kBQ>(p, groups, t, w_tiles, ti)) break;
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&tempty_bar[acc]), acc_ph ^ 1, abort_flag, p.status));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * kBQ;
            for (int kb = 0; kb < nkb; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full_bar[s]), ph, abort_flag, p.status));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t dp = make_desc(codes_p + s * kCodesP, false, 0), dq = make_desc(codes_q + s * kCodesQ, false, 0);
                    const int steps = min(4, (p.k - kb * kKB) / 64);
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        if (2 * a < steps) {
                            scale_copy(sfp_t + a * 4, scale_desc(sf_p + s * kSf + a * kScaleTile));
                            scale_copy(sfq_t + a * 4, scale_desc(sf_q + s * kSf + a * kScaleTile));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j < steps) {
                            mma_mxf4(d_tmem, dp + (uint64_t)(j * 2), dq + (uint64_t)(j * 2), idesc0 | mxf4_ids((j & 1) * 2), sfp_t + (j >> 1) * 4,
                                     sfq_t + (j >> 1) * 4, (kb | j) != 0);
                        }
                    tc_commit(smem_u32(&empty_bar[s]));
                }
                __syncwarp();
                if (++s == kStages) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            if (elect_one()) tc_commit(smem_u32(&tfull_bar[acc]));
            __syncwarp();
            if (++acc == 2) { acc = 0; acc_ph ^= 1; }
        }
        __syncwarp();
    } else {
        // ---------------- epilogue ----------------
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        const uint32_t buf = sf_q + kStages * kSf + (uint32_t)(warp - 2) * kOutBox;
        int acc = 0; uint32_t acc_ph = 0;
        for (int t = blockIdx.x;; t += gridDim.x) {
            Tile ti;
            if (!get_tile<kBP, kBQ>(p, groups, t, w_tiles, ti)) break;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&tfull_bar[acc]), acc_ph, abort_flag, p.status))) break;
            tc_fence_after();
            const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * kBQ);
            drain_tile<EPI>(p, ti, tm, quarter, group, buf, smem_u32(&tempty_bar[acc]), lane);
            if (++acc == 2) { acc = 0; acc_ph ^= 1; }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

template <int EPI>
cudaError_t launch_t(const MxGemm& p, int grid, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(mx_gemm_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    return launch_pdl(mx_gemm_kernel<EPI>, dim3(grid), dim3(kThreads), kSmem, stream, p);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    if (!fn) throw std::runtime_error("cuTensorMapEncodeTiled is not available from this driver");
    return fn;
}

}  // namespace

// Pairs where the single CTAs' tiles would take more than one turn of the SMs and k is long, or more than three turns.
// Dense layers, us, single CTAs / pairs by the number of 128 x 128 tiles (148 SMs):
//     1024 -> 1024    256: 10.3 / 10.6    384: 12.1 / 13.2    512: 14.3 / 13.7    1024: 24.3 / 21.9
//     1024 -> 4096    256:  8.2 /  9.2    384: 10.5 / 11.2    512: 12.3 / 11.4    1024: 19.6 / 16.5
//     2048 -> 2048    128:  8.2 / 10.7    192: 13.1 / 11.2    256: 13.2 / 11.8     512: 20.0 / 16.5
//     4096 -> 1024    128: 13.3 / 15.3    160: 19.8 / 16.3    256: 22.6 / 19.0     512: 44.1 / 32.3
//     4096 -> 4096    128: 11.3 / 13.1    256: 19.0 / 14.3    384: 25.1 / 20.6    1024: 53.7 / 37.2
int mx_form(long rows, int groups, int n, int k, int num_sms, int pad) {
    const long each = (rows + groups - 1) / groups;
    const long tiles = groups * ((each + 127) / 128) * (long)ceil_div(n, 128);
    return pad % 256 == 0 && tiles > (k >= 2048 ? 1 : 3) * num_sms ? kMxPair : kMxMany;
}

namespace {
void encode(CUtensorMap* m, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion l2) {
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = encode_fn()(m, type, rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, l2,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed for a 4-bit product (" + std::to_string((int)r) + ")");
}
}  // namespace

void mx_make_map(CUtensorMap* m, const void* codes, uint64_t rows, int cols, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols / 2, rows}, strides[1] = {(cuuint64_t)cols / 2};
    const cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
    encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

void mx_make_scale_map(CUtensorMap* m, const void* scales, uint64_t rows, int cols, int bands) {
    const cuuint64_t tiles_k = (cuuint64_t)scale_tiles_k(cols);
    const cuuint64_t dims[3] = {kScaleTile / 4, tiles_k, (rows + 127) / 128}, strides[2] = {kScaleTile, tiles_k * kScaleTile};
    const cuuint32_t box[3] = {kScaleTile / 4, 2u, (cuuint32_t)bands};
    encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

void mx_make_out_map(CUtensorMap* m, void* out, uint64_t rows, int n, bool f32) {
    const cuuint64_t dims[2] = {(cuuint64_t)n, rows}, strides[1] = {(cuuint64_t)n * (f32 ? 4 : 2)};
    const cuuint32_t box[2] = {f32 ? 32u : 64u, 32u};
    encode(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

cudaError_t launch_mx_gemm(const MxGemm& p, int num_sms, cudaStream_t stream) {
    if (p.form == kMxPair) return launch_mx_gemm_2cta(p, num_sms, stream);
    switch (p.epi) {
        case kMxBf16: return launch_t<kMxBf16>(p, num_sms, stream);
        case kMxF32: return launch_t<kMxF32>(p, num_sms, stream);
        case kMxUp: return launch_t<kMxUp>(p, num_sms, stream);
        case kMxDown: return launch_t<kMxDown>(p, num_sms, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace tmt
