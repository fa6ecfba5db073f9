// What the two attention kernels over the 4-bit cache share: their arguments, the clamped lengths of a request, which kernel
// takes it, and the even division of all work among the CTAs.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  j <= place of i (and > place of i - window);
// query i of n sits at place len - n + i of its sequence. A row that sees nothing is zero, its log-sum-exp -infinity.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include "kv4_format.cuh"
#include "../../../include/mono_attention.h"

namespace mono {
namespace kv4 {

struct AttnArgs {
  const __nv_bfloat16* q;
  const uint8_t* cache;
  const int32_t *table, *seq_lens, *query_start;
  __nv_bfloat16* out;
  float* lse;                                // or null
  float* partial;                            // of items that several CTAs share
  uint32_t* counters;                        // arrivals at such items: zero before and after a launch
  uint32_t* status;
  int64_t q_ts, q_hs, num_pages;
  int tokens, batch, width, hq, hk, group, shift, window, split_rows;
  float scale_log2;                          // scale * log2(e)
  uint32_t group_inv;                        // (2^32 - 1) / group
};

struct Request {
  int first, n, len;                         // first query row, queries, length of the sequence
};

__device__ __forceinline__ int by_group(const AttnArgs& a, int x) { return divide(x, a.group, a.group_inv); }

// The lengths of request b, whatever the arrays hold within the buffers that there are.
__device__ __forceinline__ Request request_of(const AttnArgs& a, int b, bool tell) {
  int s = a.query_start[b], e = a.query_start[b + 1], len = a.seq_lens[b];
  const int cap = static_cast<int>(min(static_cast<int64_t>(a.width) << a.shift, static_cast<int64_t>(0x7FFF0000)));
  if (tell) {
    if (s < 0 || e < s || e > a.tokens || len < 0) report(a.status, kBadLength, b);
    if (len > cap) report(a.status, kTooLong, b);
  }
  s = min(max(s, 0), a.tokens);
  e = min(max(e, s), a.tokens);
  return {s, e - s, min(max(len, 0), cap)};
}

// Page of column `col` of request b. An entry outside the cache is reported: -1, whose keys and values are zeros. Any page that there is might be
// another request's.
__device__ __forceinline__ int page_of(const AttnArgs& a, int b, int col) {
  const int p = __ldg(a.table + static_cast<int64_t>(b) * a.width + min(col, a.width - 1));
  if (p >= 0 && p < a.num_pages) return p;
  report(a.status, kBadPage, b);
  return -1;
}

// The two kernels: requests of up to a.split_rows query rows for a KV head, and those of more.
int decode(const AttnArgs& a, int head_dim, int rows, cudaStream_t stream);
int prompt(const AttnArgs& a, int head_dim, cudaStream_t stream);
size_t decode_partial_floats();
size_t prompt_partial_floats();

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

}  // namespace kv4
}  // namespace mono
