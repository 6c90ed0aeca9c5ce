/* C ABI of the microscaled operators around the MoE block on B200 (sm_100a): 4-bit matrices and their products, and
 * 8-bit checkpoints of activations.
 *
 * A block is 32 neighbouring elements of a row. It keeps 32 element codes and one scale byte b:
 *     value_i = code_i * 2^(b - 127),    b = 255: the block held an infinity or a NaN; all its values are NaN.
 * The scale is the smallest power of two (not below 2^-127) at which no element of the block passes the element type's
 * largest value; the elements are x / scale rounded to nearest, ties to even. Nothing saturates, and no input is refused
 * for its values.
 *     e2m1 (largest 6)      MXFP4, 4.25 bits per element: weights and activations of a product
 *     e4m3 (448), e5m2 (57344)   8.25 bits per element: what a backward pass keeps of an activation ("act8")
 *
 * 4-bit matrix (rows, cols), cols a multiple of 64: `codes` rows * cols / 2 bytes, row-major, element 2i of a row in the low
 * half of its byte i; `scales` tmt_moe_mxfp4_scale_bytes(rows, cols) bytes in the order the tensor cores read them:
 * tiles of 128 rows x 4 blocks, 512 bytes each, the tiles of a 128-row band one after the other; within a tile the byte
 * of (row, block) is (row % 32) * 16 + (row % 128 / 32) * 4 + block % 4. Bytes of rows past the last are never used.
 * 8-bit matrix (rows, cols), cols a multiple of 32: `codes` rows * cols bytes, `scales` rows * cols / 32 bytes, both row-major.
 *
 * Conventions as in tmt_moe.h and tmt_norm.h: 0 / -1, message from tmt_moe_last_error(), device pointers, 16-byte aligned
 * (what cudaMalloc returns is), nothing allocates, nothing synchronises, nothing calls exit(). Work is queued on `stream`
 * of the current device; a tensor that lies on another device or in host memory is refused. Outputs and workspaces overlap
 * neither each other nor an input.
 * Calls without a handle may run side by side on several streams (they share no state but the word of tmt_moe_mxfp4_status),
 * and may be captured into a graph.
 * rows = 0 is allowed where no handle is involved and does nothing.
 *
 * Kernels of these operators may be scheduled while the one before them on the stream is still running (programmatic launch;
 * TMT_MOE_PDL=0 in the environment switches it off). They wait for it before they touch what it may write, weights among it: any tensor
 * may be written by the call, copy or kernel right before the one that reads it. */
#ifndef TMT_MX_H
#define TMT_MX_H

#include <stddef.h>
#include <stdint.h>

#include "tmt_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Formats of the 8-bit checkpoints. */
enum { TMT_ACT8_E4M3 = 1, TMT_ACT8_E5M2 = 2 };

/* Kernels of a 4-bit product: few rows per weight matrix, 128 x 128 tiles, CTA pairs on 256 x 256 tiles. */
enum { TMT_MXFP4_FEW_ROWS = 0, TMT_MXFP4_TILES = 1, TMT_MXFP4_PAIRS = 2 };

/* A 4-bit weight matrix W (rows = outputs, cols = inputs), [out,in] as everywhere in tmt_moe.h. */
typedef struct tmt_mxfp4_weight {
    const void* codes;
    const void* scales;
    int rows, cols;
} tmt_mxfp4_weight;

/* Bytes of the scale buffer of a 4-bit (rows, cols) matrix; 0 for a shape that is not supported. */
size_t tmt_moe_mxfp4_scale_bytes(long long rows, int cols);

/* X (rows, cols), dtype TMT_MOE_BF16 or TMT_MOE_F32 -> 4-bit blocks. cols: a multiple of 64. One matrix per call: a list of
 * experts' matrices is quantised one by one, each into a buffer of its own. */
int tmt_moe_quantize_mxfp4(const void* X, int dtype, long long rows, int cols, void* codes, void* scales, void* stream);
/* 4-bit blocks -> Y (rows, cols), exact in both dtypes (bf16: but for values below its smallest normal number). */
int tmt_moe_dequantize_mxfp4(const void* codes, const void* scales, long long rows, int cols, void* Y, int dtype, void* stream);

/* Y = A W^T with both operands in 4-bit blocks, on the block-scaled tensor-core instruction: products exact, sums in fp32,
 * rounded once to `dtype`. A (rows, W->cols), Y (rows, W->rows) row-major and dense; W->rows: a multiple of 8, W->cols: a
 * multiple of 64, at most 2^28. How k is shared among blocks depends on `rows`, and with it the last bits of a sum. status
 * (device int): receives a code of tmt_moe_device_status when a bounded wait ran out (Y is then not complete); never cleared
 * here. NULL: the library's own word of the device receives it, see tmt_moe_mxfp4_status. */
int tmt_moe_matmul_mxfp4(const void* A_codes, const void* A_scales, int rows, const tmt_mxfp4_weight* W, void* Y, int dtype,
                         int* status, void* stream);

/* A dense layer: X (rows, W->cols) bf16 or fp32 is quantised into `work` (tmt_moe_linear_mxfp4_work_bytes bytes, contents
 * before and after the call do not matter) and multiplied. Two calls that may run at the same time need a work buffer each. */
size_t tmt_moe_linear_mxfp4_work_bytes(long long rows, int cols);
int tmt_moe_linear_mxfp4(const void* X, int x_dtype, int rows, const tmt_mxfp4_weight* W, void* Y, int y_dtype, void* work,
                         size_t work_bytes, int* status, void* stream);
/* The first code that a product without a status word of its own has recorded on the current device since the last call of this
 * function, 0 when there is none; -1 on an error. Waits for the device (so not while a stream is being captured), and clears
 * the word. */
int tmt_moe_mxfp4_status(void);
/* Failure-detection self-test of that word: queues one block that waits on a barrier nothing arrives on, limit_cycles clock cycles
 * long, through the same bounded wait as the products. tmt_moe_mxfp4_status then gives 2. */
int tmt_moe_mxfp4_selftest_bounded_wait(long long limit_cycles, void* stream);
/* Which kernel the layer's product takes on the current device (for profiles and tests); -1 for a shape that is not supported. */
int tmt_moe_linear_mxfp4_form(int rows, int n, int k);

/* tmt_moe_forward with both expert products on 4-bit blocks (hidden > 0, training = 0, a single rank). The router, the gate
 * weights, the statistics and the residual (beta) are those of tmt_moe_forward, bit for bit; a token's row is quantised on its
 * way into its experts' groups; P = q4(X) Wup^T, then q4(silu(P)) straight from the fp32 accumulators, then gate *
 * (q4(silu(P)) Wdown^T): fp32, a token's rows and the residual added in fp32 and rounded once to bf16. (The bf16 block rounds
 * every gated row before it adds; here a handle keeps them as fp32, 4 bytes for each of its grouped rows' elements.) A token's
 * output depends on its own row alone, bit for bit: not on its neighbours, nor on how many tokens a call has. Wup / Wdown:
 * HOST arrays of E descriptors whose device memory must stay valid while the handle uses them. The first call on a handle
 * allocates its buffers, and a call with other pointers than the last one uploads a table and waits for it: both are refused
 * while the handle's stream is being captured. Other calls may be recorded; a graph keeps the weights' addresses it was
 * recorded with, whatever later calls are given. */
int tmt_moe_forward_mxfp4(tmt_moe* h, const void* X, const void* Wrouter, const tmt_mxfp4_weight* Wup,
                          const tmt_mxfp4_weight* Wdown, void* Y, float beta, int tokens);
/* Which kernel the up (product 0) and the down product (1) of a call with `tokens` tokens take; -1 for arguments out of
 * range and for a handle without this pass. */
int tmt_moe_forward_mxfp4_form(const tmt_moe* h, int tokens, int product);
/* 1 when the weights last handed to tmt_moe_forward_mxfp4 were recorded into a graph (which goes on reading them), else 0; -1 for a
 * null handle. */
int tmt_moe_mxfp4_recorded(const tmt_moe* h);

/* 8-bit checkpoint of an activation X (rows, cols), and back. format: TMT_ACT8_E4M3 or TMT_ACT8_E5M2; cols: a multiple of 32. */
int tmt_moe_act8_save(const void* X, int dtype, long long rows, int cols, int format, void* codes, void* scales, void* stream);
int tmt_moe_act8_restore(const void* codes, const void* scales, long long rows, int cols, int format, void* Y, int dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif
