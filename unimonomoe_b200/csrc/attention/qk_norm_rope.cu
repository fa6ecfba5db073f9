// Root-mean-square norm of every query and key head with the position rotation in the same pass, and, where a cache is given,
// the rotated keys and the values stored in it.
//
//   y = x / sqrt(mean(x^2) + eps) * w   (w or 1 + w);   (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin) on the first R dims,
//   pairs (i, i + R/2), or (2i, 2i+1) in the interleaved form.
//
// Sums and products in fp32, one rounding to bf16 at the end. The cache quantises the key after that rounding, so that it
// holds the same codes as a key stored from the tensor.
//
// Bound by memory: 4 bytes a value, read and written once. 8192 tokens of 36 heads of 128 take 33.2 us, 4.7 TB/s, where a copy
// of as many bytes takes 26.8; behind memory it is instructions, some 130 for a lane's eight dims with what it shares among four heads. With the
// keys and values stored in the cache, a fifth of the rows, 47 us: more than the two apart (33.2 and 8.3), for eight dims to a lane take more
// instructions to quantise than kv4_append's sixteen, and value rows run through the norm as well. What it saves is a launch, where tokens are few.
#include <cuda_runtime.h>
#include "kv4_format.cuh"
#include "../../../include/mono_attention.h"

namespace mono {
namespace {

constexpr int kWarps = 8;

struct RopeArgs {
  const __nv_bfloat16 *q, *k, *v;
  const void *wq, *wk;
  const float* table;
  const int32_t* positions;
  __nv_bfloat16 *q_out, *k_out;
  uint8_t* cache;
  const int64_t* slots;
  uint32_t* status;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, slot_count;
  int tokens, hq, hk, heads, rotary, table_rows, shift, q_units, per;   // units of a token: of its queries, all
  uint32_t per_inv;
  float eps;
  bool interleaved, unit, w_fp32;
};

// The lane's eight weights: four from `at`, four from `then`.
__device__ __forceinline__ void load_weight(const RopeArgs& a, const void* w, int at, int then, float (&x)[8]) {
  if (a.w_fp32) {
    const float4 p = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at), q = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + then);
    x[0] = p.x; x[1] = p.y; x[2] = p.z; x[3] = p.w; x[4] = q.x; x[5] = q.y; x[6] = q.z; x[7] = q.w;
  } else {
    const uint2 p = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + at), q = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + then);
    kv4::unpack_bf16x8(make_uint4(p.x, p.y, q.x, q.y), x);
  }
  if (a.unit)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += 1.0f;
}

// An infinity reaches the dim that it turns against; dims that do not turn only share a lane's products (0 times it) with it, and are done again here, each
// on its own. (A NaN reaches them all.) The cache's groups of 64 need it not: one value that is not a number makes all of a group so.
// A call that begins anew, so that the kernel keeps nothing for it but a predicate.
template <int D, int U>
__device__ __noinline__ void beside_infinity(const RopeArgs& a) {
  constexpr int L = D / 8, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, unit = static_cast<int>(blockIdx.x) * kWarps + static_cast<int>(threadIdx.x >> 5);
  const int token = unit / a.per, part = unit % a.per;
  const bool queries = part < a.q_units;
  __nv_bfloat16* const out = queries ? a.q_out + static_cast<int64_t>(token) * a.hq * D : a.k_out ? a.k_out + static_cast<int64_t>(token) * a.hk * D : nullptr;
  const __nv_bfloat16* const in = queries ? a.q + token * a.q_ts : a.k + token * a.k_ts;
  float w[8];
  load_weight(a, queries ? a.wq : a.wk, 8 * l, 8 * l + 4, w);
  for (int i = 0; i < U; ++i) {
    const int h = (queries ? part : part - a.q_units) * R * U + lane / L + i * R;
    if (h >= (queries ? a.hq : a.hk) || !out) continue;
    const uint4* row = reinterpret_cast<const uint4*>(in + h * (queries ? a.q_hs : a.k_hs));
    float x[8], sum = 0.0f;                 // of magnitudes: infinite only with an infinity and no NaN
    for (int n = 0; n < L; ++n) {
      kv4::unpack_bf16x8(row[n], x);
      for (int d = 0; d < 8; ++d) sum += fabsf(x[d]) * 0x1p-10f;
    }
    if (sum != INFINITY) continue;
    kv4::unpack_bf16x8(row[l], x);
    for (int d = 0; d < 8; ++d) x[d] = x[d] * 0.0f * w[d];
    *reinterpret_cast<uint4*>(out + h * D + 8 * l) = kv4::pack_bf16x8(x);
  }
}

// A row (one head of one token) is held by D/8 lanes, eight dims each; a warp does 32/(D/8) heads of one token at a time, U times, either of
// the queries or of the keys (and values). Where halves turn against each other a lane below the rotary dims has four dims of each
// half, so that both of a pair and their one cosine and sine are in one lane; else its eight dims are adjacent. What is stored in
// the cache is brought into that order. Pairs (x0, x1) become r (x0 w0 c - x1 w1 s), r (x1 w1 c + x0 w0 s) with the products of the
// weights made once for all heads; two pairs to an instruction.
// Five CTAs to an SM (48 registers, one of them spilled for heads of 128 and 256): 8192 tokens of 36 heads of 128 33.2 us; four 35.5; six 37.3. Storing,
// four (64 registers, none spilled): 47.4 us, of 40 heads of 64 with 8 stored 31.0; five (100 to 116 bytes spilled) 47.2 and 33.0.
template <int D, int U, bool STORE>
__global__ __launch_bounds__(kWarps * 32, STORE ? 4 : 5) void rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = D / 8, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
  const int unit = static_cast<int>(blockIdx.x) * kWarps + static_cast<int>(threadIdx.x >> 5);
  const int token = kv4::divide(unit, a.per, a.per_inv);
  if (token >= a.tokens) return;            // the whole warp
  const int part = unit - token * a.per;
  const bool queries = part < a.q_units;
  const int h0 = (queries ? part : part - a.q_units) * R * U + sub, heads = queries ? a.hq : a.heads - a.hq;   // of the queries, or of keys and values
  const int half = a.rotary >> 1;
  const bool turns = 8 * l < a.rotary, split = turns && !a.interleaved;
  const int at = split ? 4 * l : 8 * l, then = split ? at + half : at + 4;

  uint4 raw[U];
  if (queries) {
    const __nv_bfloat16* p = a.q + token * a.q_ts;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const __nv_bfloat16* x = p + min(h0 + i * R, heads - 1) * a.q_hs;
      const uint2 y = __ldg(reinterpret_cast<const uint2*>(x + at)), z = __ldg(reinterpret_cast<const uint2*>(x + then));
      raw[i] = make_uint4(y.x, y.y, z.x, z.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = min(h0 + i * R, heads - 1);
      const bool is_v = STORE && h >= a.hk;
      const __nv_bfloat16* x = is_v ? a.v + token * a.v_ts + (h - a.hk) * a.v_hs : a.k + token * a.k_ts + h * a.k_hs;
      const uint2 y = __ldg(reinterpret_cast<const uint2*>(x + (is_v ? 8 * l : at))), z = __ldg(reinterpret_cast<const uint2*>(x + (is_v ? 8 * l + 4 : then)));
      raw[i] = make_uint4(y.x, y.y, z.x, z.y);
    }
  }
  int pos = __ldg(a.positions + token);
  if (pos < 0 || pos >= a.table_rows) {
    if (lane == 0) kv4::report(a.status, kv4::kBadPosition, static_cast<uint32_t>(token));
    pos = 0;
  }
  float4 co = make_float4(1.0f, 1.0f, 1.0f, 1.0f), si = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // of the lane's four pairs
  if (turns) {
    const float* row = a.table + static_cast<int64_t>(pos) * a.rotary + 4 * l;
    co = __ldg(reinterpret_cast<const float4*>(row));
    si = __ldg(reinterpret_cast<const float4*>(row + half));
  }
  // first and second of the pairs: (x[j], x[j + 4]), or neighbours; their weights times the cosines, times the sines
  float2 c0[2], c1[2], s0[2], s1[2];
  {
    float w[8];
    load_weight(a, queries ? a.wq : a.wk, at, then, w);
    const float c[4] = {co.x, co.y, co.z, co.w}, s[4] = {si.x, si.y, si.z, si.w};
    const bool near = a.interleaved;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 w0 = near ? make_float2(w[4 * j], w[4 * j + 2]) : make_float2(w[2 * j], w[2 * j + 1]);
      const float2 w1 = near ? make_float2(w[4 * j + 1], w[4 * j + 3]) : make_float2(w[2 * j + 4], w[2 * j + 5]);
      const float2 cj = make_float2(c[2 * j], c[2 * j + 1]), sj = make_float2(s[2 * j], s[2 * j + 1]);
      c0[j] = kv4::mul2(w0, cj);
      c1[j] = kv4::mul2(w1, cj);
      s0[j] = kv4::mul2(w0, sj);
      s1[j] = kv4::mul2(w1, make_float2(-sj.x, -sj.y));
    }
  }

  int64_t slot = -1;
  if constexpr (STORE) {
    slot = a.slots[token];
    if (slot >= a.slot_count || slot < -1) {
      if (lane == 0) kv4::report(a.status, kv4::kBadSlot, static_cast<uint32_t>(token));
      slot = -1;
    }
  }
  __nv_bfloat16* out = queries ? a.q_out + static_cast<int64_t>(token) * a.hq * D : a.k_out + static_cast<int64_t>(token) * a.hk * D;
  const int outs = queries ? a.hq : STORE && a.k_out == nullptr ? 0 : a.hk;   // heads that are written
  bool infinite = false;                    // a head with an infinity in it (or squares beyond fp32): a root of infinity, everything times 0

#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = h0 + i * R;
    const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float2 x0[2], x1[2];                    // first and second of pairs 2 j, 2 j + 1
    if (a.interleaved) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 p = kv4::bf16x2(v[2 * j]), q = kv4::bf16x2(v[2 * j + 1]);
        x0[j] = make_float2(p.x, q.x);
        x1[j] = make_float2(p.y, q.y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x0[j] = kv4::bf16x2(v[j]);
        x1[j] = kv4::bf16x2(v[j + 2]);
      }
    }
    float2 sq = kv4::mul2(x0[0], x0[0]);
    sq = kv4::fma2(x0[1], x0[1], sq);
    sq = kv4::fma2(x1[0], x1[0], sq);
    sq = kv4::fma2(x1[1], x1[1], sq);
    float ss = sq.x + sq.y;
#pragma unroll
    for (int d = 1; d < L; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
    const float2 r = kv4::both(rsqrtf(ss * (1.0f / D) + a.eps));
    infinite |= r.x == 0.0f;
    float2 y0[2], y1[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      y0[j] = kv4::mul2(kv4::fma2(x0[j], c0[j], kv4::mul2(x1[j], s1[j])), r);
      y1[j] = kv4::mul2(kv4::fma2(x1[j], c1[j], kv4::mul2(x0[j], s0[j])), r);
    }
    uint4 rounded;
    if (a.interleaved)
      rounded = make_uint4(kv4::pack_bf16x2(y0[0].x, y1[0].x), kv4::pack_bf16x2(y0[0].y, y1[0].y), kv4::pack_bf16x2(y0[1].x, y1[1].x), kv4::pack_bf16x2(y0[1].y, y1[1].y));
    else
      rounded = make_uint4(kv4::pack_bf16x2(y0[0].x, y0[0].y), kv4::pack_bf16x2(y0[1].x, y0[1].y), kv4::pack_bf16x2(y1[0].x, y1[0].y), kv4::pack_bf16x2(y1[1].x, y1[1].y));
    if (h < outs) {
      __nv_bfloat16* o = out + h * D;
      *reinterpret_cast<uint2*>(o + at) = make_uint2(rounded.x, rounded.y);
      *reinterpret_cast<uint2*>(o + then) = make_uint2(rounded.z, rounded.w);
    }
    if constexpr (STORE) {
      if (queries) continue;                // the whole warp
      const bool is_v = h >= a.hk;
      // dims 8 l .. 8 l + 7 of a key: the lower pieces of lanes 2 l and 2 l + 1, or the upper ones of those that lie half further back
      uint4 row = is_v ? raw[i] : rounded;
      if (!a.interleaved) {
        const bool upper = 8 * l >= half;
        const int from = sub * L + (upper ? (8 * l - half) / 4 : 2 * l), src = turns ? from : lane, src2 = turns ? from + 1 : lane;
        uint32_t p[8];
        p[0] = __shfl_sync(0xFFFFFFFFu, rounded.x, src); p[1] = __shfl_sync(0xFFFFFFFFu, rounded.y, src);
        p[2] = __shfl_sync(0xFFFFFFFFu, rounded.x, src2); p[3] = __shfl_sync(0xFFFFFFFFu, rounded.y, src2);
        p[4] = __shfl_sync(0xFFFFFFFFu, rounded.z, src); p[5] = __shfl_sync(0xFFFFFFFFu, rounded.w, src);
        p[6] = __shfl_sync(0xFFFFFFFFu, rounded.z, src2); p[7] = __shfl_sync(0xFFFFFFFFu, rounded.w, src2);
        if (turns && !is_v) row = upper ? make_uint4(p[4], p[5], p[6], p[7]) : make_uint4(p[0], p[1], p[2], p[3]);
      }
      float sc;
      const uint32_t word = kv4::quantise8(row, sc);
      if (slot >= 0 && h < heads) {
        const int head = is_v ? h - a.hk : h;
        kv4::store8<D>(a.cache + kv4::block_at<D>(slot, head, a.hk, a.shift), static_cast<int>(slot & 15), is_v, l, word, sc);
      }
    }
  }
  if (infinite && !turns) beside_infinity<D, U>(a);
}

template <int D, int U, bool STORE>
int launch(RopeArgs a, cudaStream_t stream) {
  const int rows = 32 / (D / 8) * U;
  a.q_units = (a.hq + rows - 1) / rows;
  a.per = a.q_units + (a.heads - a.hq + rows - 1) / rows;
  a.per_inv = 0xFFFFFFFFu / static_cast<uint32_t>(a.per);
  const int64_t units = static_cast<int64_t>(a.tokens) * a.per;
  if (units > INT32_MAX - 64) return MONO_ATTN_BAD_SIZE;
  rope_kernel<D, U, STORE><<<static_cast<unsigned>((units + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <int D>
int launch_d(const RopeArgs& a, bool store, cudaStream_t stream) {
  constexpr int U = 4;                      // 8192 tokens of 36 heads of 128, four CTAs to an SM: 1: 55 us, 2: 39, 4: 35.5, 8: 37
  return store ? launch<D, U, true>(a, stream) : launch<D, U, false>(a, stream);
}

}  // namespace
}  // namespace mono

extern "C" int mono_attn_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                      int64_t k_token_stride, int64_t k_head_stride, const void* q_weight, const void* k_weight,
                                      int weights_fp32, int unit_offset, float eps, const float* table, int table_rows,
                                      int rotary_dim, int interleaved, const int32_t* positions, int tokens, int q_heads,
                                      int kv_heads, int head_dim, void* q_out, void* k_out, const void* v,
                                      int64_t v_token_stride, int64_t v_head_stride, uint8_t* cache, int64_t num_pages,
                                      int page_size, const int64_t* slots, uint32_t* status, mono_attn_stream_t stream) {
  using namespace mono;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MONO_ATTN_BAD_HEAD_DIM;
  if (tokens < 0 || q_heads < 1 || kv_heads < 1 || rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16) return MONO_ATTN_BAD_SIZE;
  if (!q || !k || !q_weight || !k_weight || !positions || !q_out || (!k_out && !cache) || !status || (rotary_dim && (!table || table_rows < 1)))
    return MONO_ATTN_NULL;
  if (cache && (!v || !slots)) return MONO_ATTN_NULL;
  if (cache && (num_pages < 1 || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))) return MONO_ATTN_BAD_SIZE;
  if (tokens == 0) return 0;
  RopeArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.wq = q_weight;
  a.wk = k_weight;
  a.table = table;
  a.positions = positions;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.k_out = static_cast<__nv_bfloat16*>(k_out);
  a.cache = cache;
  a.slots = slots;
  a.status = status;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.k_ts = k_token_stride; a.k_hs = k_head_stride;
  a.v_ts = v_token_stride; a.v_hs = v_head_stride;
  a.slot_count = num_pages * page_size;
  a.tokens = tokens; a.hq = q_heads; a.hk = kv_heads;
  a.heads = q_heads + kv_heads * (cache ? 2 : 1);
  a.rotary = rotary_dim;
  a.table_rows = rotary_dim ? table_rows : INT32_MAX;
  a.shift = cache ? __builtin_ctz(page_size) : 4;
  a.eps = eps;
  a.interleaved = interleaved != 0; a.unit = unit_offset != 0; a.w_fp32 = weights_fp32 != 0;
  const bool store = cache != nullptr;
  return head_dim == 64    ? launch_d<64>(a, store, stream)
         : head_dim == 128 ? launch_d<128>(a, store, stream)
                           : launch_d<256>(a, store, stream);
}
