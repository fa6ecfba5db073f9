// Entry of the attention over the 4-bit cache: checks, and which kernels are launched.
#include <cfloat>
#include <cmath>
#include "kv4_attention.cuh"

namespace mono {
namespace kv4 {
// Query rows for a KV head up to which a request goes to the kernel of few rows, whose time grows with the rows, while the other
// one's hardly does up to its 128 or 256. Few (request, KV head) items leave each to many CTAs, whose states the kernel of many rows takes
// longer to join. Measured, in us (kernel of few rows / of many, heads of 128, groups of 8): 32 requests to 8192 with 4 KV heads, 32
// rows 79 / 95, 48 rows 106 / 98; 16 such requests, 48 rows 60 / 61; 4 requests to 16384, 64 rows 46 / 52, 128 rows 68 / 68;
// one to 65536, 128 rows 95 / 115. Heads of 256: 32 rows 85 / 76, 16 requests 48 rows 68 / 62; 4 to 16384, 128 rows 79 / 128.
constexpr int kSplitRows = 40, kSplitRowsFew = 128, kFewItems = 32;
}  // namespace kv4
}  // namespace mono

extern "C" size_t mono_attn_workspace_bytes(void) {
  const size_t a = mono::kv4::decode_partial_floats(), b = mono::kv4::prompt_partial_floats();
  return MONO_ATTN_COUNTERS * sizeof(uint32_t) + (a > b ? a : b) * sizeof(float);
}

extern "C" int mono_attn_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const uint8_t* cache,
                                       int64_t num_pages, int page_size, const int32_t* block_table, int table_width,
                                       const int32_t* seq_lens, const int32_t* query_start, int batch, int tokens,
                                       int max_query_len, int q_heads, int kv_heads, int head_dim, float scale, int window,
                                       void* out, float* lse, void* workspace, size_t workspace_bytes, uint32_t* status,
                                       mono_attn_stream_t stream) {
  using namespace mono::kv4;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MONO_ATTN_BAD_HEAD_DIM;
  if (batch < 0 || tokens < 0 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || table_width < 1 || num_pages < 1 ||
      window < 0 || max_query_len < 0 || !(fabsf(scale) <= FLT_MAX) || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return MONO_ATTN_BAD_SIZE;
  if (static_cast<int64_t>(kv_heads) * page_size / 16 * block_bytes(head_dim) > INT32_MAX) return MONO_ATTN_BAD_SIZE;   // bytes of a page
  if (batch == 0 || tokens == 0) return 0;
  if (!q || !cache || !block_table || !seq_lens || !query_start || !out || !workspace || !status) return MONO_ATTN_NULL;
  if (workspace_bytes < mono_attn_workspace_bytes()) return MONO_ATTN_WORKSPACE;
  AttnArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.cache = cache;
  a.table = block_table; a.seq_lens = seq_lens; a.query_start = query_start;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.counters = static_cast<uint32_t*>(workspace);
  a.partial = reinterpret_cast<float*>(a.counters + MONO_ATTN_COUNTERS);
  a.status = status;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.num_pages = num_pages;
  a.tokens = tokens; a.batch = batch; a.width = table_width; a.hq = q_heads; a.hk = kv_heads;
  a.group = q_heads / kv_heads;
  a.group_inv = 0xFFFFFFFFu / static_cast<uint32_t>(a.group);
  a.shift = __builtin_ctz(page_size);
  const int64_t longest = static_cast<int64_t>(table_width) * page_size;
  a.window = window >= longest ? 0 : window;  // as wide as any sequence: none
  a.scale_log2 = scale * 1.4426950408889634f;
  // max_query_len is only a bound: without the kernel of many rows the other one takes every request
  const int64_t most = static_cast<int64_t>(max_query_len < tokens ? max_query_len : tokens) * a.group;
  const int split = batch * static_cast<int64_t>(kv_heads) < kFewItems ? kSplitRowsFew : kSplitRows;
  const bool many = most > split && a.group <= 128;
  // every request has the largest number of queries (as one alone does): all of them are the other kernel's
  const bool all = many && static_cast<int64_t>(max_query_len) * batch <= tokens;
  a.split_rows = all ? 0 : many ? split : INT32_MAX;
  if (all) return prompt(a, head_dim, stream);
  if (const int rc = decode(a, head_dim, most > split ? split : static_cast<int>(most), stream)) return rc;
  return many ? prompt(a, head_dim, stream) : 0;
}
