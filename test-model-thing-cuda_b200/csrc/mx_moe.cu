// Entry points of the 4-bit products (include/tmt_mx.h): the dense layer, and the block's forward pass with both expert
// products on 4-bit blocks. Router and offset tables are those of tmt_moe_forward; then come the quantising dispatch below, two
// grouped products (mx_gemm.cu, mx_gemm_2cta.cu: up writes q4(silu(.)) straight from its accumulators, down applies the gate
// weight) and the combine below. With few rows per expert (mx_decode.cu) there is no dispatch.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../../include/tmt_mx.h"
#include "gemm.cuh"
#include "launch_pdl.cuh"
#include "moe_internal.h"
#include "mx.cuh"
#include "mx_cast.h"
#include "mx_decode.h"
#include "mx_gemm.h"
#include "mx_host.h"

namespace tmt {
namespace {

using namespace mx;

// The status of products that are given no word of their own; the second word is where the self-test's kernel says it ended.
__device__ int g_status[2];

// Their address on the current device.
int* shared_status() {
    static std::atomic<int*> known[64];
    return per_device(known, [](int) {
        void* p = nullptr;
        cuda_ok(cudaGetSymbolAddress(&p, g_status), "cudaGetSymbolAddress");
        return static_cast<int*>(p);
    });
}

constexpr int kDispatchWarps = 8;
constexpr int kMaxTopk = 8;

// One warp per token: the row is read and quantised once, its codes and scale words are written to the token's K rows of
// the experts' groups (topk * 0.53 bytes per element instead of the bf16 dispatch's topk * 2). 131072 rows of 2048, 4 experts
// each: 241 us = 4.6 TB/s; bound by its stores of 128 bytes (with four loads of a lane in flight instead of one: 263). Rows between
// a group's end and its padding keep what they held: the products neither use nor write them.
__global__ void __launch_bounds__(kDispatchWarps * 32) mx_dispatch_kernel(const RouteDims d, const RouteBufs b, const uint16_t* __restrict__ X,
                                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    extern __shared__ int table[];       // [E] first row of this router block's assignments to each expert
    pdl_begin();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned full = 0xffffffffu;
    // kTokBlock is a multiple of the 8 tokens of this block, so one router block covers them all
    const long t0 = (long)blockIdx.x * kDispatchWarps;
    const int rb = (int)(t0 / kTokBlock);
    for (int e = threadIdx.x; e < d.E; e += blockDim.x) table[e] = b.poff[e] + b.block_base[(long)rb * d.E + e];
    __syncthreads();
    const long t = t0 + warp;
    if (t >= d.T) return;
    int slot = -1;
    if (lane < d.K) {
        const int e = b.idx[t * d.K + lane];
        if (e < 0 || e >= d.E) report(b.status, kErrSlotRange);
        else {
            slot = table[e] + b.rank[t * d.K + lane];
            if (slot < 0 || slot >= d.cap) { report(b.status, kErrSlotRange); slot = -1; }
            else {
                b.slotw[slot] = b.w[t * d.K + lane];
                b.tok_of_slot[slot] = (int)t;
            }
        }
        b.slot_of[t * d.K + lane] = slot;        // -1: the combine leaves the row out
    }
    int slots[kMaxTopk];
#pragma unroll
    for (int j = 0; j < kMaxTopk; ++j) slots[j] = __shfl_sync(full, slot, j);
    const uint16_t* src = X + t * d.D;
    const int tiles_k = scale_tiles_k(d.D);
    for (int c0 = 0; c0 < d.D; c0 += 256) {
        const int col = c0 + lane * 8;
        const bool ok = col < d.D;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (ok) x = ldg16(src + col);
        float f[8];
        uint32_t word;
        const uint32_t m = spread8(x, f), q = quantize8_e2m1(f, m, ok, lane, word);
        if (ok) {
#pragma unroll
            for (int j = 0; j < kMaxTopk; ++j)
                if (j < d.K && slots[j] >= 0) {
                    *reinterpret_cast<uint32_t*>(codes + ((long)slots[j] * d.D + col) / 2) = q;
                    if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + scale_word(slots[j], col >> 7, tiles_k)) = word;
                }
        }
    }
}

// Y[t] = beta * Y[t] + the token's K gated rows, fp32 rows added in fp32 in the order of its experts and rounded once. (Rows of bf16,
// as the bf16 block keeps them, are half the bytes: at 131072 tokens x 4 of 2048 columns the product and this kernel took 925 + 400 us
// with them, and take 1150 + 728 now (6.6 TB/s); the output was off by 2.4e-3 of its norm, now by the 1.7e-3 of its own rounding.) A lane takes 4
// columns and has two vectors of every row in flight before it adds, with the row count known to the compiler; a row of blocks
// (blockIdx.y) takes every gridDim.y-th run of 256 columns, so that a few tokens spread over the SMs. DIRECT: the rows lie in the order of
// the assignments (few-row products), else where the dispatch put them.
template <int K, bool DIRECT>
__global__ void __launch_bounds__(kDispatchWarps * 32) mx_combine_kernel(const RouteDims d, const RouteBufs b, const float* __restrict__ Yg,
                                                                         uint16_t* __restrict__ Y, float beta) {
    pdl_wait();
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const long t = (long)blockIdx.x * kDispatchWarps + (threadIdx.x >> 5);
    if (t >= d.T) return;
    const float* rows[K];
    unsigned skip = 0;
    if constexpr (DIRECT) {
#pragma unroll
        for (int j = 0; j < K; ++j) rows[j] = Yg + (t * K + j) * d.D;
    } else {
        int slot = lane < K ? b.slot_of[t * K + lane] : 0;
        const bool bad = slot < 0 || slot >= d.cap;           // a slot the dispatch refused: the row is left out
        if (bad) { report(b.status, kErrSlotRange); slot = 0; }
        skip = __ballot_sync(0xffffffffu, bad);
#pragma unroll
        for (int j = 0; j < K; ++j) rows[j] = Yg + (long)__shfl_sync(0xffffffffu, slot, j) * d.D;
    }
    uint16_t* dst = Y + t * d.D;
    auto add = [&](int v, const uint4 (&x)[K], const uint2& y) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (beta != 0.0f) { acc[0] = beta * bf_lo(y.x); acc[1] = beta * bf_hi(y.x); acc[2] = beta * bf_lo(y.y); acc[3] = beta * bf_hi(y.y); }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (!DIRECT && (skip >> j & 1)) continue;
            acc[0] += __uint_as_float(x[j].x); acc[1] += __uint_as_float(x[j].y);
            acc[2] += __uint_as_float(x[j].z); acc[3] += __uint_as_float(x[j].w);
        }
        *reinterpret_cast<uint2*>(dst + v) = make_uint2(pack_bf2(acc[0], acc[1]), pack_bf2(acc[2], acc[3]));
    };
    for (int v = (int)blockIdx.y * 256 + lane * 4; v < d.D; v += 256 * (int)gridDim.y) {
        const bool two = v + 128 < d.D;
        uint4 x0[K], x1[K];
        uint2 y0 = make_uint2(0, 0), y1 = y0;
#pragma unroll
        for (int j = 0; j < K; ++j) x0[j] = ldg16_stream(rows[j] + v);
        if (beta != 0.0f) y0 = *reinterpret_cast<const uint2*>(dst + v);
        if (two) {
#pragma unroll
            for (int j = 0; j < K; ++j) x1[j] = ldg16_stream(rows[j] + v + 128);
            if (beta != 0.0f) y1 = *reinterpret_cast<const uint2*>(dst + v + 128);
        }
        add(v, x0, y0);
        if (two) add(v + 128, x1, y1);
    }
}
template <bool DIRECT>
cudaError_t launch_mx_combine(const RouteDims& d, const RouteBufs& b, const float* Yg, uint16_t* Y, float beta, cudaStream_t s) {
    const dim3 grid((d.T + kDispatchWarps - 1) / kDispatchWarps, DIRECT ? (d.D + 255) / 256 : 1), block(kDispatchWarps * 32);
    switch (d.K) {
        case 1: return launch_pdl(mx_combine_kernel<1, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 2: return launch_pdl(mx_combine_kernel<2, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 3: return launch_pdl(mx_combine_kernel<3, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 4: return launch_pdl(mx_combine_kernel<4, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 5: return launch_pdl(mx_combine_kernel<5, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 6: return launch_pdl(mx_combine_kernel<6, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 7: return launch_pdl(mx_combine_kernel<7, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        case 8: return launch_pdl(mx_combine_kernel<8, DIRECT>, grid, block, 0, s, d, b, Yg, Y, beta);
        default: return cudaErrorInvalidValue;
    }
}

// Per-expert maps: of each product the codes, and the scale tiles in boxes of one band (decode form) and of two (pair form).
enum Table : int { kTabCodes = 0, kTabScales1, kTabScales2, kTabsPerProduct, kTables = 2 * kTabsPerProduct };

void* alloc(tmt_moe* h, size_t bytes) {
    void* p = nullptr;
    cuda_ok(cudaMalloc(&p, bytes), "cudaMalloc");
    h->allocs.push_back(p);
    h->bytes += bytes;
    return p;
}

void make_buffers(tmt_moe* h) {
    MxState& m = h->mx;
    const int D = h->d.dim, H = h->d.hidden;
    const long cap = h->dims.cap;
    // what an earlier call got before memory ran out is kept
    auto need = [&](auto*& p, size_t n) { if (!p) p = static_cast<std::remove_reference_t<decltype(p)>>(alloc(h, n * sizeof *p)); };
    need(m.x_codes, (size_t)cap * D / 2);
    need(m.x_scales, scale_bytes(cap, D));
    need(m.h_codes, (size_t)cap * H / 2);
    need(m.h_scales, scale_bytes(cap, H));
    need(m.y_rows, (size_t)cap * D);
    mx_make_map(&m.x_map, m.x_codes, cap, D, kMxBoxRows);
    mx_make_map(&m.h_map, m.h_codes, cap, H, kMxBoxRows);
    mx_make_scale_map(&m.x_sf, m.x_scales, cap, D, kMxActBands);
    mx_make_scale_map(&m.h_sf, m.h_scales, cap, H, kMxActBands);
    mx_make_out_map(&m.y_out, m.y_rows, cap, D, true);
    // the padding rows' scale bytes are read with the others (their products are never used): give them a value
    cuda_ok(cudaMemsetAsync(m.x_scales, 0, scale_bytes(cap, D), h->stream), "cudaMemsetAsync");
    cuda_ok(cudaMemsetAsync(m.h_scales, 0, scale_bytes(cap, H), h->stream), "cudaMemsetAsync");
    m.buffers = true;
}

bool capturing(cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    cuda_ok(cudaStreamIsCapturing(s, &st), "cudaStreamIsCapturing");
    return st != cudaStreamCaptureStatusNone;
}

// Per-expert maps and scale pointers of the weights handed in, uploaded when they are not those of the call before. (They are
// addresses and shapes only; what the weights hold is read at every call.) A recorded graph goes on reading the tables it was
// recorded with: those are never written again, the next list of weights gets tables of its own.
void refresh_tables(tmt_moe* h, const tmt_mxfp4_weight* Wup, const tmt_mxfp4_weight* Wdown) {
    const int E = h->d.experts;
    MxState& m = h->mx;
    std::vector<const void*> key(4 * (size_t)E);
    for (int e = 0; e < E; ++e) { key[e] = Wup[e].scales; key[E + e] = Wdown[e].scales; key[2 * E + e] = Wup[e].codes; key[3 * E + e] = Wdown[e].codes; }
    const bool recording = capturing(h->stream);
    if (key == m.key) {
        m.recorded |= recording;
        return;
    }
    if (recording)
        throw std::runtime_error("forward_mxfp4: the first call on a handle, and the first one with other weights, cannot be recorded into a graph; make one outside the capture");
    if (!m.buffers) make_buffers(h);
    m.open_tables(kTables * (size_t)E, 2 * (size_t)E, [&](size_t bytes) { return alloc(h, bytes); });
    for (const void* p : key) check_tensors({p});
    std::vector<CUtensorMap> maps(kTables * (size_t)E);
    for (int product = 0; product < 2; ++product)
        for (int e = 0; e < E; ++e) {
            const tmt_mxfp4_weight& w = product == 0 ? Wup[e] : Wdown[e];
            CUtensorMap* t = maps.data() + (size_t)product * kTabsPerProduct * E + e;
            mx_make_map(t + (size_t)kTabCodes * E, w.codes, w.rows, w.cols, kMxBoxRows);
            mx_make_scale_map(t + (size_t)kTabScales1 * E, w.scales, w.rows, w.cols, 1);
            mx_make_scale_map(t + (size_t)kTabScales2 * E, w.scales, w.rows, w.cols, kMxWeightBands);
        }
    cuda_ok(cudaMemcpyAsync(m.tables, maps.data(), maps.size() * sizeof(CUtensorMap), cudaMemcpyHostToDevice, h->stream), "cudaMemcpyAsync");
    cuda_ok(cudaMemcpyAsync(m.scale_tab, key.data(), 2 * (size_t)E * sizeof(void*), cudaMemcpyHostToDevice, h->stream), "cudaMemcpyAsync");
    cuda_ok(cudaStreamSynchronize(h->stream), "cudaStreamSynchronize");      // the host vectors are about to go
    m.key = key;
}

// The kernel of an expert product with n outputs and k inputs. With few rows per expert both products take the few-row kernel.
int experts_form(const tmt_moe* h, int tokens, int n, int k) {
    const long rows = (long)tokens * h->d.topk;
    if (mx_decode_grouped(rows, h->d.experts, std::max(h->d.dim, h->d.hidden))) return TMT_MXFP4_FEW_ROWS;
    return mx_form(rows, h->d.experts, n, k, h->num_sms, h->pad) == kMxPair ? TMT_MXFP4_PAIRS : TMT_MXFP4_TILES;
}

void forward_mx(tmt_moe* h, const void* X, const void* Wr, const tmt_mxfp4_weight* Wup, const tmt_mxfp4_weight* Wdown, void* Y,
                float beta, int tokens) {
    const int D = h->d.dim, H = h->d.hidden, E = h->d.experts, K = h->d.topk;
    if (H == 0 || h->d.training || h->d.ep_world > 1) throw std::runtime_error("MXFP4 forward needs hidden > 0, training = 0 and a single rank");
    if (!X || !Wr || !Wup || !Wdown || !Y) throw std::runtime_error("null argument");
    if (tokens < 1 || tokens > h->d.tokens) throw std::runtime_error("tokens outside [1, desc.tokens]");
    for (int e = 0; e < E; ++e)
        if (Wup[e].rows != H || Wup[e].cols != D || Wdown[e].rows != D || Wdown[e].cols != H)
            throw std::runtime_error("MXFP4 weight shape does not match the handle");
    cuda_ok(cudaSetDevice(h->d.device), "cudaSetDevice");
    check_tensors({X, Wr, Y});
    refresh_tables(h, Wup, Wdown);
    MxState& m = h->mx;
    h->dims.T = tokens;
    h->last_tokens = tokens;
    route_only(h, static_cast<const uint16_t*>(X), Wr);
    if (experts_form(h, tokens, H, D) == TMT_MXFP4_FEW_ROWS) {
        // Few rows per expert: no dispatch; up finds and quantises its rows itself and writes one row per assignment, down reads those.
        MxDecode q;
        memset(&q, 0, sizeof q);
        q.idx = h->rb.idx; q.n_asg = tokens * K; q.experts = E; q.status = h->rb.status; q.early = true; q.split = 1;
        q.weights_ready = true;              // the router's first kernel waits before it lets the next one start
        q.src = X; q.src_kind = kMxSrcBf16; q.src_mul = mx_row_factor(K);
        q.w_maps = m.tables + (size_t)kTabCodes * E; q.w_sf_maps = m.tables + (size_t)kTabScales1 * E;
        q.n = H; q.k = D; q.epi = kMxUp; q.out = m.h_codes; q.out_scales = m.h_scales;
        prof_mark(h, kPhGemmUp);
        cuda_ok(launch_mx_decode(q, h->stream), "mx up launch");
        q.src = m.h_codes; q.src_scales = m.h_scales; q.src_kind = kMxSrcRows; q.src_mul = mx_row_factor(1);
        q.w_maps += (size_t)kTabsPerProduct * E; q.w_sf_maps += (size_t)kTabsPerProduct * E;
        q.n = D; q.k = H; q.epi = kMxDown; q.out = m.y_rows; q.out_scales = nullptr; q.gate = h->rb.w;
        prof_mark(h, kPhGemmDown);
        cuda_ok(launch_mx_decode(q, h->stream), "mx down launch");
        prof_mark(h, kPhCombine);
        cuda_ok(launch_mx_combine<true>(h->dims, h->rb, m.y_rows, static_cast<uint16_t*>(Y), beta, h->stream), "combine launch");
        prof_mark(h, -1);
        h->launches += 3;
        h->have_forward = true;
        return;
    }
    prof_mark(h, kPhDispatch);
    cuda_ok(launch_pdl(mx_dispatch_kernel, dim3((tokens + kDispatchWarps - 1) / kDispatchWarps), dim3(kDispatchWarps * 32), E * sizeof(int),
                       h->stream, h->dims, h->rb, static_cast<const uint16_t*>(X), m.x_codes, m.x_scales), "mx dispatch launch");
    MxGemm p;
    memset(&p, 0, sizeof p);
    p.experts = E; p.poff = h->rb.poff; p.counts = h->rb.counts; p.row_limit = h->dims.cap;
    p.status = h->rb.status;
    // a product's view of the per-expert tables
    auto weights = [&](int product) {
        const CUtensorMap* t = m.tables + (size_t)product * kTabsPerProduct * E;
        p.w_maps = t + (size_t)kTabCodes * E;
        p.w_sf_maps = t + (size_t)kTabScales2 * E;
        p.w_scales_tab = m.scale_tab + (size_t)product * E;
    };
    p.n = H; p.k = D; p.epi = kMxUp; p.out = m.h_codes; p.out_scales = m.h_scales;
    p.form = experts_form(h, tokens, p.n, p.k) == TMT_MXFP4_PAIRS ? kMxPair : kMxMany;
    p.act = m.x_map; p.act_scales = m.x_scales; p.act_sf = m.x_sf;
    weights(0);
    prof_mark(h, kPhGemmUp);
    cuda_ok(launch_mx_gemm(p, h->num_sms, h->stream), "mx up launch");
    p.n = D; p.k = H; p.epi = kMxDown; p.out = m.y_rows; p.out_scales = nullptr; p.out_map = m.y_out; p.row_scale = h->rb.slotw;
    p.form = experts_form(h, tokens, p.n, p.k) == TMT_MXFP4_PAIRS ? kMxPair : kMxMany;
    p.act = m.h_map; p.act_scales = m.h_scales; p.act_sf = m.h_sf;
    weights(1);
    prof_mark(h, kPhGemmDown);
    cuda_ok(launch_mx_gemm(p, h->num_sms, h->stream), "mx down launch");
    prof_mark(h, kPhCombine);
    cuda_ok(launch_mx_combine<false>(h->dims, h->rb, m.y_rows, static_cast<uint16_t*>(Y), beta, h->stream), "combine launch");
    prof_mark(h, -1);
    h->launches += 4;
    h->have_forward = true;
}

// A tile's sum over k is one chain of about 0.3 us per 256, and the epilogue's wait for it is bounded (two seconds): 2^28 take 0.3 s.
constexpr int kMaxK = 1 << 28;
void check_weight(int rows, int cols) {
    if (rows < 8 || rows % 8 || cols < 64 || cols % 64) throw std::runtime_error("MXFP4 weight: rows must be a positive multiple of 8, cols of 64");
    if (cols > kMaxK) throw std::runtime_error("MXFP4 weight: cols must be at most " + std::to_string(kMaxK));
}
void check_weight(const tmt_mxfp4_weight* W) {
    if (!W) throw std::runtime_error("null argument");
    check_weight(W->rows, W->cols);
}

// The kernel of a dense product; codes: the rows come as codes.
int dense_form(int rows, int n, int k, bool codes) {
    const int sms = sm_count();
    if (mx_decode_dense(rows, k, mx_decode_split(n, k, sms), codes)) return TMT_MXFP4_FEW_ROWS;
    return mx_form(rows, 1, n, k, sms, 256) == kMxPair ? TMT_MXFP4_PAIRS : TMT_MXFP4_TILES;
}

// Up to 32 rows, from values or from codes.
void few_rows(const void* src, const void* scales, int kind, int rows, const tmt_mxfp4_weight& W, void* Y, int dtype, int* status, cudaStream_t s) {
    MxDecode p;
    memset(&p, 0, sizeof p);
    mx_make_map(&p.w, W.codes, W.rows, W.cols, kMxBoxRows);
    mx_make_scale_map(&p.w_sf, W.scales, W.rows, W.cols, 1);
    p.src = src; p.src_scales = static_cast<const uint8_t*>(scales); p.src_kind = kind;
    p.rows = rows; p.n = W.rows; p.k = W.cols;
    p.split = mx_decode_split(W.rows, W.cols, sm_count());
    p.weights_ready = p.split > 1;           // clusters are launched the ordinary way, after all that came before
    p.epi = dtype == TMT_MOE_F32 ? kMxF32 : kMxBf16; p.out = Y; p.status = status;
    cuda_ok(launch_mx_decode(p, s), "matmul_mxfp4 launch");
}

void matmul(const void* codes, const void* scales, int rows, const tmt_mxfp4_weight& W, void* Y, int dtype, int* status, cudaStream_t s) {
    const int form = dense_form(rows, W.rows, W.cols, true);
    if (form == TMT_MXFP4_FEW_ROWS) return few_rows(codes, scales, kMxSrcTiles, rows, W, Y, dtype, status, s);
    MxGemm p;
    memset(&p, 0, sizeof p);
    const int sms = sm_count();
    p.rows = rows; p.n = W.rows; p.k = W.cols;
    p.epi = dtype == TMT_MOE_F32 ? kMxF32 : kMxBf16; p.out = Y; p.status = status;
    p.form = form == TMT_MXFP4_PAIRS ? kMxPair : kMxMany;
    p.act_scales = static_cast<const uint8_t*>(scales); p.w_scales = static_cast<const uint8_t*>(W.scales);
    mx_make_map(&p.act, codes, rows, p.k, kMxBoxRows);
    mx_make_map(&p.w, W.codes, p.n, p.k, kMxBoxRows);
    if (p.form == kMxPair) {
        mx_make_scale_map(&p.act_sf, scales, rows, p.k, kMxActBands);
        mx_make_scale_map(&p.w_sf, W.scales, p.n, p.k, kMxWeightBands);
        mx_make_out_map(&p.out_map, Y, rows, p.n, p.epi == kMxF32);
    }
    cuda_ok(launch_mx_gemm(p, sms, s), "matmul_mxfp4 launch");
}

void check_dtype(int dtype) {
    if (dtype != TMT_MOE_BF16 && dtype != TMT_MOE_F32) throw std::runtime_error("dtype must be TMT_MOE_BF16 or TMT_MOE_F32");
}

// codes first, then the scale tiles on a 16-byte boundary (cols / 2 is a multiple of 32)
size_t codes_bytes(long long rows, int cols) { return (size_t)rows * cols / 2; }

}  // namespace
}  // namespace tmt

using namespace tmt;

extern "C" {

int tmt_moe_matmul_mxfp4(const void* A_codes, const void* A_scales, int rows, const tmt_mxfp4_weight* W, void* Y, int dtype,
                         int* status, void* stream) {
    MX_GUARD({
        check_weight(W);
        check_dtype(dtype);
        if (rows < 0) throw std::runtime_error("rows must not be negative");
        if (rows == 0) return 0;
        check_tensors({A_codes, A_scales, W->codes, W->scales, Y});
        if (status) check_tensors({status}, 4);
        else status = shared_status();
        matmul(A_codes, A_scales, rows, *W, Y, dtype, status, static_cast<cudaStream_t>(stream));
    })
}

size_t tmt_moe_linear_mxfp4_work_bytes(long long rows, int cols) {
    return rows < 0 || cols < 64 || cols % 64 ? 0 : codes_bytes(rows, cols) + mx::scale_bytes((long)rows, cols);
}

int tmt_moe_linear_mxfp4(const void* X, int x_dtype, int rows, const tmt_mxfp4_weight* W, void* Y, int y_dtype, void* work,
                         size_t work_bytes, int* status, void* stream) {
    MX_GUARD({
        check_weight(W);
        check_dtype(x_dtype);
        check_dtype(y_dtype);
        if (rows < 0) throw std::runtime_error("rows must not be negative");
        if (rows == 0) return 0;
        if (work_bytes < tmt_moe_linear_mxfp4_work_bytes(rows, W->cols)) throw std::runtime_error("work buffer too small (tmt_moe_linear_mxfp4_work_bytes)");
        check_tensors({X, W->codes, W->scales, Y, work});
        if (status) check_tensors({status}, 4);
        else status = shared_status();
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (dense_form(rows, W->rows, W->cols, false) == TMT_MXFP4_FEW_ROWS) {
            few_rows(X, nullptr, x_dtype == TMT_MOE_F32 ? kMxSrcF32 : kMxSrcBf16, rows, *W, Y, y_dtype, status, s);
            return 0;
        }
        uint8_t* codes = static_cast<uint8_t*>(work);
        uint8_t* scales = codes + codes_bytes(rows, W->cols);
        cuda_ok(launch_mx4_quantize(X, x_dtype == TMT_MOE_F32, rows, W->cols, codes, scales, s, true), "quantize_mxfp4 launch");
        matmul(codes, scales, rows, *W, Y, y_dtype, status, s);
    })
}

int tmt_moe_mxfp4_status(void) {
    try {
        int* word = shared_status();
        int v = 0;
        cuda_ok(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
        cuda_ok(cudaMemcpy(&v, word, sizeof v, cudaMemcpyDeviceToHost), "cudaMemcpy");
        if (v) cuda_ok(cudaMemset(word, 0, sizeof v), "cudaMemset");
        return v;
    } catch (const std::exception& e) { set_error("%s", e.what()); return -1; }
}

int tmt_moe_mxfp4_selftest_bounded_wait(long long limit_cycles, void* stream) {
    MX_GUARD({
        if (limit_cycles < 1 || limit_cycles > 2000000000LL) throw std::runtime_error("limit_cycles outside [1, 2e9]");
        int* words = shared_status();
        cuda_ok(launch_bounded_wait_selftest(words, limit_cycles, words + 1, static_cast<cudaStream_t>(stream)), "self-test launch");
    })
}

int tmt_moe_linear_mxfp4_form(int rows, int n, int k) {
    try {
        check_weight(n, k);
        if (rows < 1) throw std::runtime_error("rows must be positive");
        const int form = dense_form(rows, n, k, false);
        return form == TMT_MXFP4_FEW_ROWS ? form : dense_form(rows, n, k, true);        // quantised first, then a product of codes
    } catch (const std::exception& e) { set_error("%s", e.what()); return -1; }
}

int tmt_moe_forward_mxfp4_form(const tmt_moe* h, int tokens, int product) {
    if (!h) { set_error("null handle"); return -1; }
    if (tokens < 1 || tokens > h->d.tokens || product < 0 || product > 1) { set_error("tokens outside [1, desc.tokens], or product not 0 or 1"); return -1; }
    if (h->d.hidden == 0 || h->d.training || h->d.ep_world > 1) { set_error("MXFP4 forward needs hidden > 0, training = 0 and a single rank"); return -1; }
    return product == 0 ? experts_form(h, tokens, h->d.hidden, h->d.dim) : experts_form(h, tokens, h->d.dim, h->d.hidden);
}

int tmt_moe_forward_mxfp4(tmt_moe* h, const void* X, const void* Wrouter, const tmt_mxfp4_weight* Wup, const tmt_mxfp4_weight* Wdown,
                          void* Y, float beta, int tokens) {
    if (!h) { set_error("null handle"); return -1; }
    MX_GUARD(forward_mx(h, X, Wrouter, Wup, Wdown, Y, beta, tokens))
}

int tmt_moe_mxfp4_recorded(const tmt_moe* h) {
    if (!h) { set_error("null handle"); return -1; }
    return h->mx.recorded ? 1 : 0;
}

}  // extern "C"
