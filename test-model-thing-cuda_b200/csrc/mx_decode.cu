// 4-bit products with few rows per weight matrix: bound by how fast the weights arrive, and below that by the latency of a chain of
// short kernels.
//
// A block (with a long k and few matrices: a cluster, each block a share of k) owns 128 weight rows of one matrix, the 128-row side of the MMA; the matrix's activation rows are its columns, 32 at a
// time. It asks for all of its weights (up to the shared memory there is: 64 bytes per row and 128 of k) before it knows whether and by whom
// the matrix is used, so that every weight of the product is on its way at once: in the experts' chain at its start, while the kernel before it
// is still running (the chain's first kernel has waited for whoever wrote them); a dense layer's only after it has waited, since the kernel
// before it may be the one that writes them, and writes are promised to be visible after griddepcontrol.wait alone (1 row, 1024 -> 2048, in a
// queue of such layers: 4.6 us; 4.3 when it did not wait, which read weights that might still be on their way). Meanwhile sixteen
// warps find the matrix's rows in the router's index table (grouped) and bring them in: as values, which they quantise here, or
// as codes. There is no separate quantising or dispatching kernel, and no row moves through memory twice.
// Activations stay in shared memory for the whole of k in the order the MMA reads them (128-byte swizzle, scale tiles).
// An epilogue thread owns an output: a block of 32 outputs of one row is a warp, its largest magnitude one warp reduction.
//
// Warps: 0..15 = rows in, then epilogue (four lane quarters x every fourth group of rows); 16 = TMA of the weights; 17 = MMA issuer, TMEM owner.
// Every wait is bounded, as in the other kernels.
#include "launch_pdl.cuh"
#include "mx_decode.h"
#include "mx_gemm.cuh"

namespace tmt {
namespace {

using namespace mxg;

constexpr int kRowWarps = 16, kTmaWarp = kRowWarps, kMmaWarp = kRowWarps + 1, kThreads = 32 * (kRowWarps + 2);
constexpr int kRows = kMxDecodeRows;
constexpr int kCodesW = 128 * 128, kSfW = 2 * kScaleTile, kStageW = kCodesW + kSfW;      // one k block of 256
constexpr int kCodesA = kRows * 128, kSfA = 2 * kScaleTile, kStageA = kCodesA + kSfA;
constexpr int kMaxStages = 16;
constexpr int kSmemMax = 222 * 1024;
// two accumulators, two sets of activation scale columns, weight scale columns of up to kMaxStages k blocks; two blocks fit an SM
constexpr uint32_t kSfACol = 2 * kRows, kSfWCol = kSfACol + 16, kTmemCols = 256;
static_assert(kSfWCol + 8 * kMaxStages <= kTmemCols, "tensor memory");
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void st_shared4(uint32_t addr, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void tmem_ld4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ float ld_cluster(uint32_t addr, int rank) {       // the word at this offset of another block of the cluster
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(addr, (uint32_t)rank)) : "memory");
    return v;
}

// A piece of one row: one k block of 256 elements, 8 per lane, on its way into registers.
template <int SRC>
struct Piece {
    static constexpr int kAhead = SRC == kMxSrcF32 ? 2 : SRC == kMxSrcBf16 ? 3 : 6;      // pieces in flight: 16, 12 or 12 registers
    uint4 a, b;
    uint32_t sw;
    __device__ __forceinline__ void fetch(const MxDecode& p, long row, int kb, int tiles_k, int lane) {      // kb: of the whole row
        const int col = kb * kKB + lane * 8;
        a = make_uint4(0, 0, 0, 0); sw = 0;
        if constexpr (SRC == kMxSrcF32) b = a;
        if (col < p.k) {
            if constexpr (SRC == kMxSrcBf16) a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.src) + row * p.k + col);
            else if constexpr (SRC == kMxSrcF32) {
                const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p.src) + row * p.k + col);
                a = s[0]; b = s[1];
            } else {
                a.x = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.src) + (row * p.k + col) / 2);
                const size_t at = SRC == kMxSrcTiles ? scale_word(row, col >> 7, tiles_k) : ((size_t)row * tiles_k + (col >> 7)) * 4;
                sw = *reinterpret_cast<const uint32_t*>(p.src_scales + at);
            }
        }
    }
    // codes into their swizzled place, scale words into the tiles
    __device__ __forceinline__ void put(uint32_t act, int r, int kb, int lane) const {
        uint32_t q = a.x, word = sw;
        if constexpr (SRC == kMxSrcBf16 || SRC == kMxSrcF32) {
            float f[8];
            uint32_t m;
            if constexpr (SRC == kMxSrcF32) m = spread8(a, b, f);
            else m = spread8(a, f);
            q = quantize8_e2m1(f, m, true, lane, word);
        }
        const uint32_t stage = act + kb * kStageA;
        st_shared4(stage + r * 128 + ((((uint32_t)lane >> 2) ^ (uint32_t)(r & 7)) << 4) + (lane & 3) * 4, q);
        if ((lane & 15) == 0) st_shared4(stage + kCodesA + (lane >> 4) * kScaleTile + r * 16, word);
    }
};

// Brings the rows [r0, r0 + nr) of the pass in: a warp takes every sixteenth piece, its next ones already on their way. The code of a
// kernel this short arrives from L2 as it runs, so the loop is kept small rather than unrolled. (Handing the k blocks to the
// MMAs one by one, k block by k block, gained nothing: the pieces then came in as much later as the products ended sooner.)
template <int SRC>
__device__ __forceinline__ void rows_in(const MxDecode& p, const uint16_t* list, int r0, int nr, int kb0, int nkb, uint32_t act, int warp, int lane) {
    const int tiles_k = scale_tiles_k(p.k), pieces = nr * nkb;
    // (row, k block) of the piece being stored and of the one being fetched: sixteen pieces further each time
    const int dr = kRowWarps / nkb, dk = kRowWarps - dr * nkb;
    int r = warp / nkb, kb = warp - r * nkb, fr = r, fk = kb, fu = warp;
    constexpr int A = Piece<SRC>::kAhead;
    Piece<SRC> x[A];
    auto fetch = [&](Piece<SRC>& d) {
        if (fu < pieces) d.fetch(p, p.experts ? (int)(list[r0 + fr] * p.src_mul >> 16) : r0 + fr, kb0 + fk, tiles_k, lane);
        fu += kRowWarps;
        fr += dr; fk += dk;
        if (fk >= nkb) { fk -= nkb; ++fr; }
    };
#pragma unroll
    for (int i = 0; i < A; ++i) fetch(x[i]);
#pragma unroll 1
    for (int u = warp; u < pieces; u += kRowWarps) {
        x[0].put(act, r, kb, lane);
#pragma unroll
        for (int i = 0; i + 1 < A; ++i) x[i] = x[i + 1];
        fetch(x[A - 1]);
        r += dr; kb += dk;
        if (kb >= nkb) { kb -= nkb; ++r; }
    }
}

// One output (lane) of the rows r0 .. r0 + nr - 1 (columns of the accumulator), four at a time, every fourth group per set of warps: the chains
// of a group overlap, and what a group computes past the last row is not stored.
template <int EPI>
__device__ __forceinline__ void drain(const MxDecode& p, const uint16_t* list, int r0, int nr, uint32_t tm, int set, int col, int lane) {
    const bool col_ok = col < p.n;
#pragma unroll 1
    for (int g = set * 4; g < nr; g += kRowWarps) {
        uint32_t v[4], q[4], sb[4];
        tmem_ld4(tm + g, v);
        long row[4];
        float gate[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + min(g + i, nr - 1);
            row[i] = p.experts ? list[r] : r;
            gate[i] = EPI == kMxDown ? p.gate[row[i]] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = __uint_as_float(v[i]);
            if constexpr (EPI == kMxUp) {        // the warp's 32 outputs are one block
                const float s = silu_lane(x);
                sb[i] = scale_byte<kE2M1>(__reduce_max_sync(kFull, __float_as_uint(s) & 0x7fffffffu));
                const float f[8] = {s * inv_scale(sb[i]), 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                q[i] = sb[i] == 255u ? 0u : (pack_e2m1x8(f) & 15u) << (4 * (lane & 7));
                q[i] |= __shfl_xor_sync(kFull, q[i], 1);
                q[i] |= __shfl_xor_sync(kFull, q[i], 2);
                q[i] |= __shfl_xor_sync(kFull, q[i], 4);
            } else if constexpr (EPI == kMxBf16) q[i] = f2bf(x);
            else q[i] = __float_as_uint(EPI == kMxDown ? x * gate[i] : x);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (g + i >= nr || !col_ok) continue;
            if constexpr (EPI == kMxUp) {
                if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + (row[i] * p.n + col) / 2) = q[i];
                if (lane == 0) p.out_scales[(size_t)row[i] * scale_tiles_k(p.n) * 4 + (col >> 5)] = (uint8_t)sb[i];
            } else if constexpr (EPI == kMxBf16) static_cast<uint16_t*>(p.out)[row[i] * p.n + col] = (uint16_t)q[i];
            else static_cast<float*>(p.out)[row[i] * p.n + col] = __uint_as_float(q[i]);
        }
        __syncwarp();
    }
}

// The rows of expert e among the assignments, in order. Every warp makes the list for itself (all write the same entries), which
// takes no barrier between them.
__device__ __forceinline__ int make_list(const MxDecode& p, int e, uint16_t* list, int lane) {
    int n = 0;
    for (int a0 = 0; a0 < p.n_asg; a0 += 128) {
        int x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a0 + i * 32 + lane < p.n_asg ? p.idx[a0 + i * 32 + lane] : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned m = __ballot_sync(kFull, x[i] == e);
            if (x[i] == e) list[n + __popc(m & ((1u << lane) - 1))] = (uint16_t)(a0 + i * 32 + lane);
            n += __popc(m);
        }
    }
    __syncwarp();
    return n;
}

// SPLIT: the blocks of a cluster share k.
template <int SRC, int EPI, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2) mx_decode_kernel(const __grid_constant__ MxDecode p, int stages) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], rows_bar, acc_bar[2], free_bar[2], mma_bar;
    __shared__ uint16_t list[kMxDecodeMaxAsg];
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w_tiles = ceil_div(p.n, 128);
    const int split = SPLIT ? p.split : 1, part = SPLIT ? (int)blockIdx.x % split : 0, tile = SPLIT ? (int)blockIdx.x / split : (int)blockIdx.x;
    const int e = SPLIT ? 0 : tile / w_tiles, w0 = (SPLIT ? tile : tile % w_tiles) << 7;
    const int nkb_all = ceil_div(p.k, kKB);
    const int kb0 = SPLIT ? nkb_all * part / split : 0, nkb = SPLIT ? nkb_all * (part + 1) / split - kb0 : nkb_all;      // this block's share of k
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t codes_w = base, act = codes_w + stages * kCodesW, sf_w = act + nkb * kStageA;      // 1024-byte multiples throughout
    volatile int* abort_flag = &abort_s;

    const CUtensorMap* map = p.w_maps ? p.w_maps + e : &p.w;
    const CUtensorMap* sf_map = p.w_sf_maps ? p.w_sf_maps + e : &p.w_sf;
    auto load_stage = [&](int s, int kb) {
        const uint32_t fb = smem_u32(&full_bar[s]);
        mbar_expect_tx(fb, kStageW);
        tma_load_2d(codes_w + s * kCodesW, map, fb, (kb0 + kb) * 128, w0);
        tma_load_3d(sf_w + s * kSfW, sf_map, fb, 0, 2 * (kb0 + kb), w0 >> 7);
    };
    // With fewer assignments than experts most blocks would ask in vain: they look first.
    const bool ahead = p.experts == 0 || p.n_asg >= p.experts;
    auto load_first = [&](int& issued) {
        for (; issued < min(stages, nkb); ++issued) load_stage(issued, issued);
    };
    int issued = 0;                          // loads so far (lane 0 of the TMA warp)
    if (warp == kTmaWarp && lane == 0) {
        abort_s = 0;
        for (int s = 0; s < stages; ++s) { mbar_init(smem_u32(&full_bar[s]), 1); mbar_init(smem_u32(&empty_bar[s]), 1); }
        mbar_init(smem_u32(&rows_bar), kRowWarps); mbar_init(smem_u32(&mma_bar), 1);
        for (int a = 0; a < 2; ++a) { mbar_init(smem_u32(&acc_bar[a]), 1); mbar_init(smem_u32(&free_bar[a]), kRowWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (p.w_maps) { tensormap_acquire(map); tensormap_acquire(sf_map); }
        if (ahead && p.weights_ready) load_first(issued);
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        if (p.early) pdl_begin();            // not before: the next kernel could take the tensor memory this one is about to ask for
    }
    __syncwarp();
    pdl_wait();
    if (warp == kTmaWarp && lane == 0 && ahead) load_first(issued);
    __syncwarp();
    const int count = p.experts ? make_list(p, e, list, lane) : p.rows;
    const int passes = (count + kRows - 1) / kRows;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;

    if (warp == kTmaWarp) {
        // ---------------- weights: k blocks beyond the first `stages`, and again in further passes when they do not all stay ----------------
        if (lane == 0) {
            const int total = passes == 0 ? 0 : stages < nkb ? passes * nkb : nkb;
            bool ok = true;
            for (; issued < total; ++issued) {
                const int s = issued % stages;
                if (issued >= stages) ok = mbar_wait(smem_u32(&empty_bar[s]), (uint32_t)(issued / stages - 1) & 1u, abort_flag, p.status);
                if (!ok) break;
                load_stage(s, issued % nkb);
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issuer ----------------
        const uint32_t idesc = mxf4_idesc(128, kRows);
        const bool resident = stages >= nkb;     // all of k stays: a stage is filled once, further passes find it there
        int it = 0;
        bool ok = true;
        if (resident) {                          // the weights' scales go to tensor memory before the rows are in
            for (int kb = 0; kb < nkb && passes > 0 && ok; ++kb) ok = __all_sync(kFull, mbar_wait(smem_u32(&full_bar[kb]), 0, abort_flag, p.status));
            tc_fence_after();
            if (passes > 0 && ok && elect_one())
                for (int kb = 0; kb < nkb; ++kb)
#pragma unroll
                    for (int a = 0; a < 2; ++a) scale_copy(tmem_base + kSfWCol + kb * 8 + a * 4, scale_desc(sf_w + kb * kSfW + a * kScaleTile));
            __syncwarp();
        }
        for (int ps = 0; __any_sync(kFull, ok && ps < passes); ++ps) {
            ok = __all_sync(kFull, mbar_wait(smem_u32(&rows_bar), ps & 1, abort_flag, p.status) &&
                                       mbar_wait(smem_u32(&free_bar[ps & 1]), ((ps >> 1) & 1) ^ 1, abort_flag, p.status));
            if (!ok) break;
            tc_fence_after();
            for (int kb = 0; kb < nkb; ++kb, ++it) {
                const int s = resident ? kb : it % stages;
                if (!resident) {
                    ok = __all_sync(kFull, mbar_wait(smem_u32(&full_bar[s]), (it / stages) & 1, abort_flag, p.status));
                    if (!ok) break;
                    tc_fence_after();
                }
                if (elect_one()) {
                    const uint32_t sf_at = tmem_base + kSfACol + (it & 1) * 8, sfw_at = tmem_base + kSfWCol + (resident ? kb : it & 1) * 8;
                    const uint32_t stage_a = act + kb * kStageA;
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        if (!resident) scale_copy(sfw_at + a * 4, scale_desc(sf_w + s * kSfW + a * kScaleTile));
                        scale_copy(sf_at + a * 4, scale_desc(stage_a + kCodesA + a * kScaleTile));
                    }
                    const uint64_t dw = make_desc(codes_w + s * kCodesW, false, 0), da = make_desc(stage_a, false, 0);
                    const int steps = (p.k - (kb0 + kb) * kKB) / 64;
                    auto step = [&](int j) {
                        mma(tmem_base + (ps & 1) * kRows, dw + (uint64_t)(j * 2), da + (uint64_t)(j * 2), idesc | mxf4_ids((j & 1) * 2),
                            sfw_at + (j >> 1) * 4, sf_at + (j >> 1) * 4, (kb | j) != 0);
                    };
                    step(0);
                    if (steps >= 4) { step(1); step(2); step(3); }
                    else {
                        if (steps > 1) step(1);
                        if (steps > 2) step(2);
                    }
                    if (!resident) tc_commit(smem_u32(&empty_bar[s]));
                    if (kb == nkb - 1) { tc_commit(smem_u32(&acc_bar[ps & 1])); tc_commit(smem_u32(&mma_bar)); }
                }
                __syncwarp();
            }
        }
        __syncwarp();
    } else {
        // ---------------- rows in, then epilogue ----------------
        bool ok = true;
        for (int ps = 0; ps < passes && ok; ++ps) {
            const int r0 = ps * kRows, nr = min(kRows, count - r0);
            if (ps > 0) ok = __all_sync(kFull, mbar_wait(smem_u32(&mma_bar), (ps - 1) & 1, abort_flag, p.status));      // the last pass's rows have been read
            if (!ok) break;
            rows_in<SRC>(p, list, r0, nr, kb0, nkb, act, warp, lane);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&rows_bar));
            ok = __all_sync(kFull, mbar_wait(smem_u32(&acc_bar[ps & 1]), (ps >> 1) & 1, abort_flag, p.status));
            if (!ok) break;
            tc_fence_after();
            const int quarter = warp & 3, set = warp >> 2;
            if constexpr (SPLIT) {                   // this share of the sums, for the cluster (the weights of stage 0 have been read)
                for (int g = set * 4; g < nr; g += kRowWarps) {
                    uint32_t v[4];
                    tmem_ld4(tmem_base + ((uint32_t)(quarter * 32) << 16) + (ps & 1) * kRows + g, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) st_shared4(codes_w + (g + i) * 512 + (quarter * 32 + lane) * 4, v[i]);
                }
            } else drain<EPI>(p, list, r0, nr, tmem_base + ((uint32_t)(quarter * 32) << 16) + (ps & 1) * kRows, set, w0 + quarter * 32 + lane, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&free_bar[ps & 1]));
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (SPLIT) {
        // Row r is added up by the block r % split, its shares in the order of k. Every thread of every block comes by here, also
        // after a wait that ran out.
        cluster_sync();
        if (warp < kRowWarps && w0 + (int)(threadIdx.x & 127) < p.n)
            for (int r = part + split * (int)(threadIdx.x >> 7); r < p.rows; r += split * (kRowWarps / 4)) {
                const uint32_t at = codes_w + r * 512 + (threadIdx.x & 127) * 4;
                float x = 0.0f;
                for (int q = 0; q < split; ++q) x += ld_cluster(at, q);
                const size_t to = (size_t)r * p.n + w0 + (threadIdx.x & 127);
                if constexpr (EPI == kMxF32) static_cast<float*>(p.out)[to] = x;
                else static_cast<uint16_t*>(p.out)[to] = f2bf(x);
            }
        __syncwarp();
        cluster_sync();            // the others have read this block's share
    }
    if (warp == kTmaWarp && lane == 0) {
        // No copy may still be on its way into this block's shared memory. The MMA warp has waited for all of them, but in a block
        // without rows, or when a wait ran out: wait (bounded) for the last load of every stage.
        if (passes == 0 || *abort_flag)
            for (int f = max(0, issued - stages); f < issued; ++f) {
                const long long t0 = clock64();
                while (!mbar_try_wait(smem_u32(&full_bar[f % stages]), (uint32_t)(f / stages) & 1u) && clock64() - t0 < kWaitCycles) {}
            }
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

template <int SRC, int EPI, bool SPLIT>
cudaError_t launch_t(const MxDecode& p, cudaStream_t stream) {
    const int nkb = ceil_div(ceil_div(p.k, kKB), p.split);      // the largest share
    const int room = (kSmemMax - 1024 - nkb * kStageA) / kStageW;
    const int stages = room < nkb ? (room < kMaxStages ? room : kMaxStages) : (nkb < kMaxStages ? nkb : kMaxStages);
    const size_t smem = 1024 + (size_t)nkb * kStageA + (size_t)stages * kStageW;
    const auto kernel = mx_decode_kernel<SRC, EPI, SPLIT>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e != cudaSuccess) return e;
    const int blocks = ceil_div(p.n, 128) * (p.experts ? p.experts : p.split);
    if constexpr (!SPLIT) return launch_pdl(kernel, dim3(blocks), dim3(kThreads), smem, stream, p, stages);
    // a cluster per tile
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p, stages);
}
template <int SRC>
cudaError_t launch_dense(const MxDecode& p, cudaStream_t stream) {
    if (SRC == kMxSrcTiles || p.split > 1) return p.epi == kMxF32 ? launch_t<SRC, kMxF32, true>(p, stream) : launch_t<SRC, kMxBf16, true>(p, stream);
    if constexpr (SRC != kMxSrcTiles) return p.epi == kMxF32 ? launch_t<SRC, kMxF32, false>(p, stream) : launch_t<SRC, kMxBf16, false>(p, stream);
}

}  // namespace

// A block alone takes k in turn, about 1.6 us per 1024 of it: from 2048 on a cluster shares it, as far as there are SMs. 1 row, us:
//     n x k        alone  shared               n x k        alone  shared
//     2048 x 2048    6.3     5.6               4096 x 4096   10.0     7.3
//     1024 x 4096   10.0     5.6               1024 x 8192   16.9     6.5
// Below 2048 a block alone is done sooner than any cluster was (1024 x 1024: 4.4): it starts early, which clusters go without.
int mx_decode_split(int n, int k, int num_sms) {
    const int tiles = ceil_div(n, 128), nkb = ceil_div(k, kKB);
    int split = 1;
    while (split < 8 && nkb >= 8 && 4 * split <= nkb && tiles <= num_sms / (2 * split)) split *= 2;
    return split;
}

// Every block brings all rows in for itself, 0.03 us per row and 256 of its share of k, where quantising once and 128 x 128 tiles
// cost the same for 1 row as for 128. Dense layers, us, few rows (1, 8, 16, 24, 32) | tiles:
//      320 -> 4096   3.7   3.9   4.4   5.0   5.5 |  4.9         4096 -> 1024   5.6   5.8   6.4   7.0   7.5 |  9.9
//     1024 -> 1024   4.4   5.0   5.9   6.9   7.9 |  5.4         4096 -> 4096   7.3   7.4   8.5   9.7  10.6 | 10.4
//     2048 -> 2048   5.6   5.8   6.4   7.1   7.7 |  7.3         8192 -> 1024   6.5   6.8   7.9   8.9   9.9 | 15.2
// and of codes, where only a k long enough to be shared pays:
//     1024 -> 1024   6.2   6.7   7.5   8.3   9.2 |  3.8         4096 -> 4096   7.4   7.5   7.9   8.6   9.3 |  8.7
//     2048 -> 2048   5.6   5.9   6.4   6.9   7.3 |  5.8         8192 -> 1024   6.6   6.8   7.5   8.2   8.9 | 13.5
bool mx_decode_dense(long rows, int k, int split, bool codes) {
    if (k > kMxDecodeMaxK || rows > kMxDecodeRows) return false;
    const long nkb = ceil_div(k, kKB), work = rows * ((nkb + split - 1) / split);
    if (codes) return split > 1 && work <= 8 * nkb - 64;
    return work <= (split > 1 ? 8 * nkb - 24 : 40);
}

// Experts, us for the whole pass, this kernel | scan, dispatch and tiles, by rows per expert:
//     16 experts 1024 -> 2048:   2 rows 24.3 | 31.5     8 rows 26.5 | 32.0    16 rows 36.5 | 36.1    32 rows 53 | 37
//      4 experts  512 -> 1024:   2 rows 18.1 | 23.4     8 rows 20.0 | 23.2    16 rows 21.9 | 23.6    32 rows 30 | 23
bool mx_decode_grouped(long rows, int groups, int k) {
    const long nkb = ceil_div(k, kKB);
    return rows <= kMxDecodeMaxAsg && k <= kMxDecodeMaxK && rows <= 20L * groups && rows * nkb <= 80L * groups;
}

cudaError_t launch_mx_decode(const MxDecode& p, cudaStream_t stream) {
    if (p.epi == kMxUp) return launch_t<kMxSrcBf16, kMxUp, false>(p, stream);
    if (p.epi == kMxDown) return launch_t<kMxSrcRows, kMxDown, false>(p, stream);
    switch (p.src_kind) {
        case kMxSrcBf16: return launch_dense<kMxSrcBf16>(p, stream);
        case kMxSrcF32: return launch_dense<kMxSrcF32>(p, stream);
        case kMxSrcTiles: return launch_dense<kMxSrcTiles>(p, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace tmt
