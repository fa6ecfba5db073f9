// Positions, cache slots, requests and block-table entries of a step's tokens, from the lengths of its requests.
//
//   held_b = ceil(cached_b / P), need_b = ceil((cached_b + new_b) / P); request b takes need_b - held_b pages from the free
//   list, in the order of the requests; its i-th new token is at position cached_b + i, slot table[b, pos / P] * P + pos % P.
//
// One launch without any exchange between CTAs: each scans the lengths itself (a few thousand integers from L2), then does
// one token per thread. A token in a page that this step hands out takes the page from the free list, not from the table, so
// nothing is read that another CTA writes. Bound by latency: one read of the lengths, two scans, one gather. A call takes 7.1 us for one
// request as for 37 chunks of 16384 tokens: the host's share of it, checks, one allocation and the launch, is what is left.
#include <cuda_runtime.h>
#include "kv4_format.cuh"
#include "../../../include/mono_attention.h"

namespace mono {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRequests = MONO_ATTN_MAX_REQUESTS;
// Longest sequence; longer ones are reported and cut. Then no place, page or column leaves 32 bits, whatever the lengths are, and sums over requests
// stay at the largest integer instead of turning negative (starts that fall would give a token a place outside its request).
constexpr int kLongest = 0x7FFF0000;
__device__ __forceinline__ int add(int x, int y) { return static_cast<int>(min(static_cast<uint32_t>(x) + static_cast<uint32_t>(y), 0x7FFFFFFFu)); }

struct PlanArgs {
  const int32_t *cached, *fresh;
  int32_t* table;
  const int32_t *free_pages, *taken;
  int32_t *query_start, *seq_lens, *positions, *requests, *taken_out;
  int64_t* slots;
  uint32_t* status;
  int batch, width, free_count, shift, tokens;
};

__global__ __launch_bounds__(kThreads) void plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* start = sm;                       // [batch + 1] first token of each request
  int32_t* first = sm + a.batch + 1;         // [batch + 1] pages handed out before it
  __shared__ int32_t wsum[2][kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << a.shift;
  int base_t = 0, base_p = 0;
  bool bad = false, too_long = false;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0, f = 0;
    if (b < a.batch) {
      int c = a.cached[b];
      n = a.fresh[b];
      bad |= c < 0 || n < 0;
      c = max(c, 0);
      n = max(n, 0);
      too_long |= c > kLongest || n > kLongest - c;
      c = min(c, kLongest);
      n = min(n, kLongest - c);
      f = ((c + n + page - 1) >> a.shift) - ((c + page - 1) >> a.shift);
    }
    int sn = n, sf = f;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, sn, d), y = __shfl_up_sync(0xFFFFFFFFu, sf, d);
      if (lane >= d) { sn = add(sn, x); sf = add(sf, y); }
    }
    if (lane == 31) { wsum[0][warp] = sn; wsum[1][warp] = sf; }
    __syncthreads();
    int on = base_t, of = base_p, tn = 0, tf = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int x = wsum[0][w], y = wsum[1][w];
      if (w < warp) { on = add(on, x); of = add(of, y); }
      tn = add(tn, x);
      tf = add(tf, y);
    }
    const int n_before = __shfl_up_sync(0xFFFFFFFFu, sn, 1), f_before = __shfl_up_sync(0xFFFFFFFFu, sf, 1);
    if (b < a.batch) { start[b] = lane ? add(on, n_before) : on; first[b] = lane ? add(of, f_before) : of; }
    base_t = add(base_t, tn);
    base_p = add(base_p, tf);
    __syncthreads();
  }
  if (tid == 0) { start[a.batch] = base_t; first[a.batch] = base_p; }
  __syncthreads();
  const int total = base_t, taken = a.taken[0];
  if (blockIdx.x == 0 && tid == 0) {
    const int64_t behind = static_cast<int64_t>(taken) + base_p;
    a.taken_out[0] = static_cast<int>(min(behind, static_cast<int64_t>(INT32_MAX)));
    a.query_start[a.batch] = total;
    if (total > a.tokens) kv4::report(a.status, kv4::kTooManyTokens, total);
    if (taken < 0 || behind > a.free_count) kv4::report(a.status, kv4::kNoPages, static_cast<uint32_t>(behind));
  }
  if (bad && blockIdx.x == 0) kv4::report(a.status, kv4::kBadLength, tid);
  if (too_long && blockIdx.x == 0) kv4::report(a.status, kv4::kTooLong, tid);

  // one warp for a request: its length, its start, the entries of its new pages
  for (int b = blockIdx.x * kWarps + warp; b < a.batch; b += gridDim.x * kWarps) {
    const int c = min(max(a.cached[b], 0), kLongest), n = start[b + 1] - start[b];
    if (lane == 0) {
      a.seq_lens[b] = c + n;
      a.query_start[b] = start[b];
    }
    const int held = (c + page - 1) >> a.shift, f = first[b + 1] - first[b];
    if (held + f > a.width && lane == 0 && n > 0) kv4::report(a.status, kv4::kTooLong, b);
    for (int j = lane; j < min(f, a.width - held); j += 32) {
      const int64_t at = static_cast<int64_t>(taken) + first[b] + j;
      // none left: not what the row held for an earlier request
      a.table[static_cast<int64_t>(b) * a.width + held + j] = at >= 0 && at < a.free_count ? a.free_pages[at] : -1;
    }
  }

  // one thread for a token: the request by bisection of the starts
  for (int t = blockIdx.x * kThreads + tid; t < a.tokens; t += gridDim.x * kThreads) {
    int pos = 0, req = -1;
    int64_t slot = -1;
    if (t < total) {
      int lo = 0, hi = a.batch;              // start[lo] <= t < start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
      }
      req = lo;
      const int c = min(max(a.cached[req], 0), kLongest), held = (c + page - 1) >> a.shift;
      pos = c + t - start[req];
      const int col = pos >> a.shift;
      int pg = -1;
      if (col < held) {
        if (col < a.width) pg = a.table[static_cast<int64_t>(req) * a.width + col];
        if (pg < 0) kv4::report(a.status, col < a.width ? kv4::kBadPage : kv4::kTooLong, req);
      } else {
        const int64_t at = static_cast<int64_t>(taken) + first[req] + col - held;
        if (col < a.width && at >= 0 && at < a.free_count) pg = a.free_pages[at];
      }
      if (pg >= 0) slot = (static_cast<int64_t>(pg) << a.shift) + (pos & (page - 1));
    }
    a.positions[t] = pos;
    a.requests[t] = req;
    a.slots[t] = slot;
  }
}

}  // namespace
}  // namespace mono

extern "C" int mono_attn_plan(const int32_t* cached, const int32_t* fresh, int batch, int32_t* table, int width,
                              const int32_t* free_pages, int free_count, const int32_t* taken, int page_size, int tokens,
                              int32_t* query_start, int32_t* seq_lens, int32_t* positions, int64_t* slots, int32_t* requests,
                              int32_t* taken_out, uint32_t* status, mono_attn_stream_t stream) {
  using namespace mono;
  if (batch < 1 || batch > kMaxRequests || width < 1 || free_count < 0 || tokens < 0) return MONO_ATTN_BAD_SIZE;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return MONO_ATTN_BAD_SIZE;
  if (!cached || !fresh || !table || (free_count && !free_pages) || !taken || !query_start || !seq_lens || !taken_out || !status ||
      (tokens && (!positions || !slots || !requests)))
    return MONO_ATTN_NULL;
  PlanArgs a{cached, fresh, table, free_pages, taken, query_start, seq_lens, positions, requests, taken_out, slots, status,
             batch, width, free_count, __builtin_ctz(page_size), tokens};
  const size_t smem = 2 * (batch + 1) * sizeof(int32_t);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const int work = tokens > batch * 32 ? tokens : batch * 32;
  const int grid = (work + kThreads - 1) / kThreads;
  plan_kernel<<<grid < 148 ? grid : 148, kThreads, smem, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
