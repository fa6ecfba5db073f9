/* C ABI of libmono_linear.so: the block-FP8 products of a decoder layer outside of the one-launch MoE kernel of prefill_mono.h:
 * rows to 8 bits, dense projections, and experts of any geometry. Plain pointers and sizes only; every launch is asynchronous on
 * the caller's stream, allocates nothing and keeps nothing between calls. All tensors are on the current device, contiguous
 * unless a stride is given.
 *
 * Return codes: 0 launched; MONO_LIN_* below, before any CUDA call was made; > 0 cudaError_t.
 *
 * Numbers: a row of K values has ceil(K / 128) groups of 128. With m the largest magnitude of a group (1 where that is below
 * 2^-100) its scale is m / 448 and its codes are e4m3 of x * (448 / m), to nearest; a group that holds an infinity or a NaN has the
 * scale NaN. Weights [N, K] in e4m3 have one fp32 scale for each block of 128 x 128, [ceil(N / 128), ceil(K / 128)].
 * K is a multiple of 16; codes and weights begin on 16-byte boundaries.
 *
 * status: two 32-bit words of device memory, zeroed by their owner: what a kernel finds wrong with numbers that only the device
 * knows (codes in csrc/linear/linear.cuh) and where; the first one stays. The access itself is left out or kept in bounds.
 */
#ifndef MONO_LINEAR_H_
#define MONO_LINEAR_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* mono_lin_stream_t; /* cudaStream_t */

#define MONO_LIN_NULL (-301)      /* a required pointer is null */
#define MONO_LIN_BAD_SIZE (-302)  /* a size is out of its range */
#define MONO_LIN_ALIGNMENT (-303) /* a pointer or a stride does not begin where it has to */
#define MONO_LIN_DRIVER (-304)    /* the driver has no tensor maps, or refuses one */

#define MONO_LIN_MAX_EXPERTS 1024
#define MONO_LIN_MAX_TOP 64
#define MONO_LIN_FEW_ROWS 16

/* x: bf16 [rows, cols] (with silu [rows, 2 cols]: silu of the first half times the second), row_stride elements apart, a multiple of 8. codes: e4m3
 * [rows, cols]; scales: fp32 [rows, ceil(cols / 128)]. */
int mono_lin_quantize(const void* x, int64_t row_stride, int64_t rows, int cols, int silu, uint8_t* codes, float* scales,
                      mono_lin_stream_t stream);

/* Product of rows [rows, k] with a weight [n, k]. Exactly one of out and codes_out is given.
 * out: [rows, n], bf16 or (out_fp32) fp32, plus residual (bf16 [rows, n]) unless null.
 * codes_out, scales_out: silu of columns [0, n / 2) times columns [n / 2, n), as rows [rows, n / 2]; n / 2 is a multiple of 128.
 * after_quantize: the launch before this one on the stream is the mono_lin_quantize that makes codes and scales, and nothing else
 * that this one reads or writes is in use there: this one may then begin before that one has ended, and waits for it by itself. */
int mono_lin_product(const uint8_t* codes, const float* scales, int64_t rows, const uint8_t* weight, const float* weight_scale, int n, int k,
                     void* out, int out_fp32, const void* residual, uint8_t* codes_out, float* scales_out, int after_quantize,
                     uint32_t* status, mono_lin_stream_t stream);

/* The same of few rows in 16 bits (x and row_stride as in mono_lin_quantize), quantised inside the launch: the codes are those of mono_lin_quantize. For
 * the sizes of which mono_lin_takes_rows says 1: up to MONO_LIN_FEW_ROWS rows, where n and k leave each CTA no more than it has room for. */
int mono_lin_takes_rows(int rows, int n, int k, int silu);
int mono_lin_product_rows(const void* x, int64_t row_stride, int rows, const uint8_t* weight, const float* weight_scale, int n, int k, void* out,
                          int out_fp32, const void* residual, uint8_t* codes_out, float* scales_out, uint32_t* status, mono_lin_stream_t stream);

/* Division of a batch among experts. ids: [tokens, top], int32 or (ids_64) int64; negative: computed elsewhere. Slots (token, place) are
 * sorted by expert, those of one expert in ascending order, into rows: offsets int32 [experts + 1], the first row of each
 * expert's run; tokens_out int32 [tokens * top], the token of each row, -1 behind the last run; positions int32 [tokens, top],
 * the row of each slot or -1. */
int mono_lin_plan(const void* ids, int ids_64, int64_t tokens, int top, int experts, int32_t* offsets, int32_t* tokens_out, int32_t* positions,
                  uint32_t* status, mono_lin_stream_t stream);

/* Products of runs of rows with a weight for each: row i, offsets[e] <= i < offsets[e + 1], with weight[e] of [experts, n, k]
 * (scales [experts, ceil(n / 128), ceil(k / 128)]). Row i has the codes and scales of row tokens[i] of [x_rows, k], or of row i where
 * tokens is null. out bf16 [rows, n], or codes_out and scales_out as above; rows outside of all runs are not written. */
int mono_lin_experts(const uint8_t* codes, const float* scales, int64_t x_rows, const int32_t* tokens, const int32_t* offsets, int64_t rows,
                     int experts, const uint8_t* weight, const float* weight_scale, int n, int k, void* out, uint8_t* codes_out,
                     float* scales_out, uint32_t* status, mono_lin_stream_t stream);

/* out bf16 [tokens, cols] = sum over j of weights[t, j] * partial[positions[t, j]] (bf16 [rows, cols]; slots at -1 add nothing) plus
 * residual (bf16) unless null; in fp32, j ascending, rounded once. cols is a multiple of 8. */
int mono_lin_combine(const void* partial, int64_t rows, const int32_t* positions, const float* weights, int64_t tokens, int top, int cols,
                     const void* residual, void* out, uint32_t* status, mono_lin_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MONO_LINEAR_H_ */
