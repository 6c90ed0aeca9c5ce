// Products of 4-bit microscaled matrices with many rows: CTA-pair MMAs (tcgen05.mma cta_group::2, kind::mxf4), two CTAs of
// a cluster on one tile of 256 activation rows x 256 outputs. See mx_gemm.cu for the operand and scale layouts.
//
// Why a pair. A 4-bit MMA consumes operand bytes at the rate of a bf16 one: a 128 x 128 tile of one CTA needs 128 bytes per
// clock and SM from L2, a 256 x 256 tile of a pair 64 (each CTA stages its 128 activation rows and half of the weight rows),
// where L2 gives about 72 (as measured for the bf16 pair kernel). Scales add 6 bytes per clock: a CTA stages the tiles of its own
// 128 activation rows and of all 256 weight rows, because each CTA's tensor memory holds the scales of what it multiplies.
//
// Shared memory is the next bound: an MMA of 256 columns reads 4 KB of A and 4 KB of its B half per 128 clocks in each CTA, and
// TMA writes 35 KB per 512 clocks: 134 of the 128 bytes a clock it can do. (Columns in two MMAs of 128 read A twice: measured
// 764 instead of about 540 clocks per k block.)
//
// Tensor memory. Two fp32 accumulators of 256 columns would fill all 512 columns and leave none for the scales (24 a stage, two
// stages in turn, so that copies run under the MMAs of the stage before: measured 908 -> 764 clocks in the form above). So the
// accumulators overlap by 64 columns: [0, 256) and [192, 448). The epilogue takes those 64 into registers first and hands them
// over; the next tile's MMAs start then, about 400 clocks after the last MMA of the tile before, and run under the rest.
//
// Warps of a CTA: 0 = TMA of activation codes, 1 = MMA issuer (leader CTA only) and TMEM owner, 2..9 = epilogue (two groups of
// four, two runs of 64 columns each), 10 = TMA of weight codes, 11 = TMA of scales (a TMA instruction keeps its warp busy for some
// 200 clocks). An epilogue thread owns a row: it loads 64 columns, hands them back, and works from registers; outputs are staged
// in shared memory and written by TMA stores.
// Measured (1 TF/s = 10^12 FLOP/s; operands of random codes): 16384 x 8192 -> 8192 5350 TF/s, held by the power limit at 1.3 to 1.4 GHz (7530 TF/s
// on zeros, at 1.965 GHz: 640 clocks per k block of 512 ideal); 65536 x 2048 -> 2048 118 to 135 us = 4070 to 4660 TF/s; 16384 x 1024 -> 4096 36 to 42 us = 3300 to 3800 TF/s
// (the longer times with other products right before and after),
// 4000 clocks per tile of 2048 ideal: some 500 between the last product of a tile and the first of the next, the rest waits
// for operands while the outputs (64 KB a tile and CTA) leave through the same L2 (without the stores: 33 us).
// Waits are bounded as in the bf16 kernels; both CTAs always reach the closing cluster barrier before tensor memory is freed.
#include "mx_gemm.cuh"

namespace tmt {
namespace {

using namespace mxg;

constexpr int kRows = 128;               // activation rows, and weight rows, per CTA
constexpr int kCols = 256;               // outputs of a tile
constexpr int kStages = 5;
constexpr int kCodesA = kRows * 128, kCodesW = kRows * 128;
constexpr int kSfA = 2 * kScaleTile, kSfW = 4 * kScaleTile;
constexpr int kStageBytes = kCodesA + kCodesW + kSfA + kSfW;
constexpr int kOutBox = 32 * 128;        // one staged box of outputs: a warp's 32 rows x 128 bytes
constexpr int kSmem = kStages * kStageBytes + 8 * kOutBox + 1024;
static_assert(kSmem + 4096 <= 232448, "227 KB of shared memory, about 3 KB of it static");
constexpr int kOverlap = 64;             // columns the two accumulators share: the last of the first, the first of the second
constexpr uint32_t kAcc1 = kCols - kOverlap, kSfCol = kAcc1 + kCols, kSfCols = 24, kTmemCols = 512;
static_assert(kSfCol + 2 * kSfCols <= kTmemCols, "tensor memory");
constexpr int kThreads = 384;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// No memory is handed over with these arrivals, only tensor memory (ordered by the tcgen05 fences), so they carry no release at
// cluster scope: with one, a warp waited some 1100 clocks for its earlier writes before the next tile's MMAs could start.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Loads into this CTA's shared memory, counted on the leader's barrier.
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void scale_copy_pair(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this offset in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) mx_gemm_2cta_kernel(const __grid_constant__ MxGemm p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], tfull_bar[2], tempty_bar[2], shared_bar[2];
    __shared__ Groups groups;
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const bool leader = rank == 0;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t codes_a = base, codes_w = codes_a + kStages * kCodesA, sf_a = codes_w + kStages * kCodesW, sf_w = sf_a + kStages * kSfA;
    const uint32_t out_s = sf_w + kStages * kSfW;
    volatile int* abort_flag = &abort_s;

    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < kStages; ++s) { mbar_init(smem_u32(&full_bar[s]), 3); mbar_init(smem_u32(&empty_bar[s]), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(smem_u32(&tfull_bar[a]), 1); mbar_init(smem_u32(&tempty_bar[a]), 16); mbar_init(smem_u32(&shared_bar[a]), 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    cluster_sync();            // the pair's allocation is one act of both CTAs: both are there, with their barriers, before it
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    load_groups<2 * kRows>(p, groups);
    tc_fence_before();
    __syncthreads();
    cluster_sync();            // both hold their tensor memory
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;
    const int w_tiles = ceil_div(p.n, kCols);
    const int nkb = ceil_div(p.k, kKB);
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    // Loop control of the producers and of the MMA warp goes through warp votes: the compiler then knows it to be uniform and
    // keeps descriptors, coordinates and addresses in uniform registers, where these instructions take them from.
    const int tiles = groups.first[p.experts == 0 ? 1 : p.experts] * w_tiles;

    if (warp == 0 || warp >= 10) {
        // ---------------- TMA producers (both CTAs) ----------------
        int s = 0; uint32_t ph = 0;
        uint32_t issued = 0, last_parity = 0;
        bool ok = true;
        for (int t = pair; __any_sync(kFull, ok && t < tiles); t += npairs) {
            Tile ti;
            get_tile<2 * kRows, kCols>(p, groups, t, w_tiles, ti);
            const int w0 = (t % w_tiles) * kCols;
            const CUtensorMap* map = warp == 0 ? &p.act : p.w_maps ? p.w_maps + ti.expert : &p.w;
            const CUtensorMap* sf_map = p.w_sf_maps ? p.w_sf_maps + ti.expert : &p.w_sf;
            if (p.w_maps && lane == 0) { if (warp == 10) tensormap_acquire(map); else if (warp == 11) tensormap_acquire(sf_map); }
            __syncwarp();
            const int row = (warp == 0 ? ti.row0 : w0) + rank * kRows;
            const uint32_t dst0 = warp == 0 ? codes_a : codes_w;
            const int band_a = (ti.row0 >> 7) + rank, band_w = w0 >> 7;
            const uint32_t bytes = warp == 11 ? kSfA + kSfW : kCodesA;
            static_assert(kCodesA == kCodesW, "one box size for both operands");
            for (int kb = 0; kb < nkb; ++kb) {
                ok = __all_sync(kFull, mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, p.status));
                if (!ok) break;
                const uint32_t fb_local = smem_u32(&full_bar[s]), fb = map_to_cta(fb_local, 0);
                if (elect_one()) {
                    if (leader) mbar_expect_tx(fb_local, 2 * bytes);           // both CTAs' bytes
                    if (warp != 11) load_2d(dst0 + s * kCodesA, map, fb, kb * 128, row);
                    else {
                        load_3d(sf_a + s * kSfA, &p.act_sf, fb, 0, 2 * kb, band_a);
                        load_3d(sf_w + s * kSfW, sf_map, fb, 0, 2 * kb, band_w);
                    }
                }
                __syncwarp();
                issued |= 1u << s;
                last_parity = (last_parity & ~(1u << s)) | (ph << s);
                if (++s == kStages) { s = 0; ph ^= 1; }
            }
        }
        if (!ok && leader && lane == 0)       // aborting: the leader's barriers count both CTAs' copies; wait (bounded) for what was announced
            for (int q = 0; q < kStages; ++q) {
                if (!(issued >> q & 1)) continue;
                const long long t0 = clock64();
                while (!mbar_try_wait(smem_u32(&full_bar[q]), (last_parity >> q) & 1) && clock64() - t0 < kWaitCycles) {}
            }
        __syncwarp();
    } else if (warp == 1) {
        if (leader) {
            // ---------------- MMA issuer: the whole warp runs the loop, one elected lane issues ----------------
            const uint32_t idesc = mxf4_idesc(2 * kRows, kCols);
            int s = 0; uint32_t ph = 0;
            uint32_t sf = 0;                           // which of the two sets of scale columns
            int acc = 0; uint32_t acc_ph = 0;
            bool ok = true;
            for (int t = pair; __any_sync(kFull, ok && t < tiles); t += npairs) {
                // this accumulator's last tile has been drained, and the columns it shares with the tile before this one have
                ok = __all_sync(kFull, mbar_wait(smem_u32(&tempty_bar[acc]), acc_ph ^ 1, abort_flag, p.status));
                if (ok && t != pair)
                    ok = __all_sync(kFull, mbar_wait(smem_u32(&shared_bar[acc ^ 1]), acc == 0 ? acc_ph ^ 1 : acc_ph, abort_flag, p.status));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem_base + (acc ? kAcc1 : 0u);
                for (int kb = 0; kb < nkb; ++kb) {
                    ok = __all_sync(kFull, mbar_wait(smem_u32(&full_bar[s]), ph, abort_flag, p.status));
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t sc = tmem_base + kSfCol + sf * kSfCols;       // 8 columns of activation scales, 16 of weight scales
#pragma unroll
                        for (int a = 0; a < 2; ++a) {
                            scale_copy_pair(sc + a * 4, scale_desc(sf_a + s * kSfA + a * kScaleTile));
                            scale_copy_pair(sc + 8 + a * 8, scale_desc(sf_w + s * kSfW + a * kScaleTile));
                            scale_copy_pair(sc + 8 + a * 8 + 4, scale_desc(sf_w + s * kSfW + (2 + a) * kScaleTile));
                        }
                        const uint64_t da = make_desc(codes_a + s * kCodesA, false, 0), db = make_desc(codes_w + s * kCodesW, false, 0);
                        auto mma = [&](int j) {
                            mma_pair(d, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), idesc | mxf4_ids((j & 1) * 2), sc + (j >> 1) * 4, sc + 8 + (j >> 1) * 8,
                                     (kb | j) != 0);
                        };
                        const int steps = (p.k - kb * kKB) / 64;
                        mma(0);
                        if (steps >= 4) { mma(1); mma(2); mma(3); }
                        else {
                            if (steps > 1) mma(1);
                            if (steps > 2) mma(2);
                        }
                        commit_pair(smem_u32(&empty_bar[s]));
                    }
                    __syncwarp();
                    sf ^= 1;
                    if (++s == kStages) { s = 0; ph ^= 1; }
                }
                if (!ok) break;
                if (elect_one()) commit_pair(smem_u32(&tfull_bar[acc]));
                __syncwarp();
                acc ^= 1;
                if (acc == 0) acc_ph ^= 1;
            }
        }
        __syncwarp();
    } else {
        // ---------------- epilogue (both CTAs) ----------------
        // A warp owns 32 rows (its lane quarter) and, by its group, two runs of 64 outputs; group 0 takes the shared columns, first.
        // Every warp stages and stores on its own: no barrier between warps. (One staged chunk of 32 columns for four warps,
        // with a group barrier and one TMA store per chunk, took about 5900 clocks a tile; this form about 1100.)
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        const uint32_t buf = out_s + (uint32_t)(warp - 2) * kOutBox;
        int acc = 0; uint32_t acc_ph = 0;
        for (int t = pair;; t += npairs) {
            Tile ti;
            if (!get_tile<2 * kRows, kCols>(p, groups, t, w_tiles, ti)) break;
            if (!__all_sync(kFull, mbar_wait(smem_u32(&tfull_bar[acc]), acc_ph, abort_flag, p.status))) break;
            tc_fence_after();
            const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16) + (acc ? kAcc1 : 0u);
            const int row0 = ti.row0 + rank * kRows + quarter * 32;
            const int rows = ti.rows - rank * kRows - quarter * 32;       // of this warp's 32, may be <= 0
            const long row = (long)row0 + lane;
            float gate = 1.0f;
            if constexpr (EPI == kMxDown) gate = lane < rows ? p.row_scale[row] : 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                // the runs start at these outputs: accumulator 0 shares its columns 192.. (group 0's first run), accumulator 1 its columns 0..
                const int run = c == 0 ? (group ? (acc ? 128 : 64) : (acc ? 0 : 192)) : (group ? (acc ? 192 : 128) : (acc ? 64 : 0));
                uint32_t v[64];
                tmem_start64(tm + run, v);
                tmem_wait64(v);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (c == 1) arrive_cluster(map_to_cta(smem_u32(&tempty_bar[acc]), 0));
                    else if (group == 0) arrive_cluster(map_to_cta(smem_u32(&shared_bar[acc]), 0));       // the next tile's MMAs may start
                }
                const int col0 = ti.w0 + run;
                if (rows <= 0 || col0 >= p.n) continue;
                if constexpr (EPI == kMxUp) {
                    // silu, then two blocks of 32: 32 bytes of codes (one sector) and two scale bytes per row, written directly
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
                    if (lane < rows)       // runs start on an even block
                        *reinterpret_cast<uint16_t*>(p.out_scales + scale_word(row, col0 >> 7, scale_tiles_k(p.n)) + ((col0 >> 5) & 3)) = (uint16_t)scales;
                } else {
                    constexpr int kBoxCols = EPI == kMxBf16 ? 64 : 32;      // 128 bytes a row
#pragma unroll
                    for (int x0 = 0; x0 < 64; x0 += kBoxCols) {
                        if (col0 + x0 >= p.n) continue;
                        if (lane == 0) bulk_wait_read<0>();                // the store before has read the box
                        __syncwarp();
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
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) { tma_store_2d(&p.out_map, buf, col0 + x0, row0); bulk_commit(); }
                    }
                }
            }
            acc ^= 1;
            if (acc == 0) acc_ph ^= 1;
        }
        if (lane == 0) bulk_wait_all();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();            // the peer may still be reading this CTA's shared memory or signalling its barriers
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
    __syncthreads();
    // Neither leaves before both have freed theirs: without this barrier and the one before the allocation, about one launch in 40000 of a
    // busy queue stood still, one CTA inside its allocation, the other waiting for it.
    cluster_sync();
}

template <int EPI>
cudaError_t launch_t(const MxGemm& p, int grid, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(mx_gemm_2cta_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    // An ordinary launch: a kernel of this length has little to gain from the early start of the short kernels' chains.
    mx_gemm_2cta_kernel<EPI><<<grid, kThreads, kSmem, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mx_gemm_2cta(const MxGemm& p, int num_sms, cudaStream_t stream) {
    const int grid = num_sms & ~1;      // whole pairs
    switch (p.epi) {
        case kMxBf16: return launch_t<kMxBf16>(p, grid, stream);
        case kMxF32: return launch_t<kMxF32>(p, grid, stream);
        case kMxUp: return launch_t<kMxUp>(p, grid, stream);
        case kMxDown: return launch_t<kMxDown>(p, grid, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace tmt
