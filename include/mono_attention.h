/* C ABI of libmono_attention.so: the attention half of a decoder layer next to the MoE layer of prefill_mono.h, over a paged
 * key/value cache held in 4 bits. Plain pointers and sizes only; every launch is asynchronous on the caller's stream, allocates
 * nothing and keeps nothing between calls. All tensors are on the current device; bf16 rows begin on 16-byte boundaries
 * (strides are in elements, multiples of 8).
 *
 * Return codes: 0 launched; MONO_ATTN_* below, before any CUDA call was made; > 0 cudaError_t.
 *
 * status: two 32-bit words of device memory, zeroed by their owner. What a kernel finds wrong with indexes and lengths that
 * only the device knows (codes in csrc/attention/kv4_format.cuh) is reported there, the first one stays; the access itself is
 * left out or kept in bounds.
 *
 * Cache: uint8 [num_pages, kv_heads, page_size / 16, 17 * head_dim]; the order inside a block of 16 tokens is in
 * csrc/attention/kv4_format.cuh. page_size is a power of two from 16 to 1024, head_dim 64, 128 or 256. A slot is
 * page * page_size + place in the page.
 */
#ifndef MONO_ATTENTION_H_
#define MONO_ATTENTION_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* mono_attn_stream_t; /* cudaStream_t */

#define MONO_ATTN_NULL (-201)         /* a required pointer is null */
#define MONO_ATTN_BAD_SIZE (-202)     /* a size is out of its range */
#define MONO_ATTN_BAD_HEAD_DIM (-203) /* head_dim is not 64, 128 or 256 */
#define MONO_ATTN_WORKSPACE (-204)    /* workspace smaller than mono_attn_workspace_bytes() */

#define MONO_ATTN_SMS 148             /* persistent grids are this many times the CTAs that fit an SM */
#define MONO_ATTN_COUNTERS (4 * MONO_ATTN_SMS)
#define MONO_ATTN_MAX_REQUESTS 16384

/* Positions, slots, requests and block-table entries of a step's tokens. cached, fresh: int32 [batch], tokens in the cache
 * and tokens of this step. table: int32 [batch, width]; the entries of the pages that a request has are read, those of the
 * pages that it gets are written. free_pages: int32 [free_count]; the next one handed out is free_pages[*taken],
 * entries for which there is none left become -1 (*taken_out is then above free_count).
 * Out: query_start int32 [batch + 1], seq_lens int32 [batch], positions int32, slots int64 and requests int32 [tokens]
 * (rows behind the last token: 0, -1, -1), taken_out int32 [1]. A token without a page gets slot -1. */
int mono_attn_plan(const int32_t* cached, const int32_t* fresh, int batch, int32_t* table, int width, const int32_t* free_pages,
                   int free_count, const int32_t* taken, int page_size, int tokens, int32_t* query_start, int32_t* seq_lens,
                   int32_t* positions, int64_t* slots, int32_t* requests, int32_t* taken_out, uint32_t* status,
                   mono_attn_stream_t stream);

/* Norm and rotation of q [tokens, q_heads, head_dim] and k [tokens, kv_heads, head_dim], bf16, into contiguous q_out, k_out.
 * Weights bf16 or fp32 [head_dim] (plus one with unit_offset). table: fp32 [table_rows, rotary_dim], cosines then sines;
 * rotary_dim a multiple of 16, up to head_dim. With cache (else null): the keys and v are stored in it at slots (int64
 * [tokens], -1 = not stored), and k_out may be null. */
int mono_attn_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                           int64_t k_head_stride, const void* q_weight, const void* k_weight, int weights_fp32, int unit_offset,
                           float eps, const float* table, int table_rows, int rotary_dim, int interleaved,
                           const int32_t* positions, int tokens, int q_heads, int kv_heads, int head_dim, void* q_out,
                           void* k_out, const void* v, int64_t v_token_stride, int64_t v_head_stride, uint8_t* cache,
                           int64_t num_pages, int page_size, const int64_t* slots, uint32_t* status, mono_attn_stream_t stream);

/* k and v [tokens, kv_heads, head_dim], bf16, into the cache at slots (-1 = not stored; no slot twice). */
int mono_attn_kv4_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                         int64_t v_head_stride, int tokens, int kv_heads, int head_dim, uint8_t* cache, int64_t num_pages,
                         int page_size, const int64_t* slots, uint32_t* status, mono_attn_stream_t stream);

/* What the cache holds at slots, as contiguous bf16 [tokens, kv_heads, head_dim] (fastest on 32-byte
 * boundaries); zeros for slot -1. */
int mono_attn_kv4_read(const uint8_t* cache, int64_t num_pages, int page_size, const int64_t* slots, int tokens, int kv_heads,
                       int head_dim, void* k_out, void* v_out, uint32_t* status, mono_attn_stream_t stream);

/* Attention of q [tokens, q_heads, head_dim] over the cache, into contiguous bf16 out and, unless null, fp32 lse [tokens,
 * q_heads] (natural log). Rows query_start[b] .. query_start[b + 1] are the last ones of sequence b, seq_lens[b] long with them;
 * each sees the keys up to its own place, with window > 0 the last `window` of them. Keys and values of a page that is missing from block_table (an
 * entry outside the cache, which is reported) are zeros. Rows of no request are not written.
 * scale is finite. max_query_len: an upper bound of the queries of a request; it chooses kernels, results do not depend on it.
 * workspace: mono_attn_workspace_bytes(), its first 4 * MONO_ATTN_COUNTERS bytes zero before the first launch (each launch
 * leaves them zero); launches that share it must not overlap. */
size_t mono_attn_workspace_bytes(void);
int mono_attn_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const uint8_t* cache,
                            int64_t num_pages, int page_size, const int32_t* block_table, int table_width,
                            const int32_t* seq_lens, const int32_t* query_start, int batch, int tokens, int max_query_len,
                            int q_heads, int kv_heads, int head_dim, float scale, int window, void* out, float* lse,
                            void* workspace, size_t workspace_bytes, uint32_t* status, mono_attn_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* MONO_ATTENTION_H_ */
