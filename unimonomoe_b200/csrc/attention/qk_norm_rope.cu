// Root-mean-square norm of every query and key head with the position rotation in the same pass, and, where a cache is given,
// the rotated keys and the values stored in it.
//
//   y = x / sqrt(mean(x^2) + eps) * w   (w or 1 + w);   (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin) on the first R dims,
//   pairs (i, i + R/2), or (2i, 2i+1) in the interleaved form.
//
// Sums and products in fp32, one rounding to bf16 at the end. The cache quantises the key after that rounding, so that it
// holds the same codes as a key stored from the tensor.
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
  int tokens, hq, hk, heads, rotary, table_rows, shift;
  float eps;
  bool interleaved, unit, w_fp32;
};

__device__ __forceinline__ void load_weight(const void* w, bool fp32, bool unit, int at, float (&x)[8]) {
  if (fp32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    kv4::unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + at), x);
  }
  if (unit)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += 1.0f;
}

// A row (one head of one token) is held by D/8 lanes, eight dims each; a warp does 32/(D/8) heads of one token at a time, U times.
template <int D, int U, bool STORE>
__global__ __launch_bounds__(kWarps * 32) void rope_kernel(const RopeArgs a) {
  constexpr int L = D / 8, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
  const int per = (a.heads + R * U - 1) / (R * U);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t token = unit / per;
  if (token >= a.tokens) return;            // the whole warp
  const int h0 = static_cast<int>(unit - token * per) * R * U + sub;

  uint4 raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = min(h0 + i * R, a.heads - 1);
    const __nv_bfloat16* p = h < a.hq          ? a.q + token * a.q_ts + h * a.q_hs
                             : h < a.hq + a.hk ? a.k + token * a.k_ts + (h - a.hq) * a.k_hs
                                               : a.v + token * a.v_ts + (h - a.hq - a.hk) * a.v_hs;
    raw[i] = *reinterpret_cast<const uint4*>(p + 8 * l);
  }

  // cosines and sines of this lane's eight dims (four pairs in the interleaved form); outside the rotary dims 1 and 0
  const int half = a.rotary >> 1, d0 = 8 * l;
  const bool turns = d0 < a.rotary;
  float co[8], si[8];
  int pos = a.positions[token];
  if (pos < 0 || pos >= a.table_rows) {
    if (lane == 0) kv4::report(a.status, kv4::kBadPosition, static_cast<uint32_t>(token));
    pos = 0;
  }
  if (turns) {
    const float* row = a.table + static_cast<int64_t>(pos) * a.rotary;
    if (a.interleaved) {
      const float4 c = *reinterpret_cast<const float4*>(row + d0 / 2), s = *reinterpret_cast<const float4*>(row + half + d0 / 2);
      co[0] = co[1] = c.x; co[2] = co[3] = c.y; co[4] = co[5] = c.z; co[6] = co[7] = c.w;
      si[0] = -s.x; si[1] = s.x; si[2] = -s.y; si[3] = s.y; si[4] = -s.z; si[5] = s.z; si[6] = -s.w; si[7] = s.w;
    } else {
      const float* c = row + (d0 < half ? d0 : d0 - half);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 x = reinterpret_cast<const float4*>(c)[j], y = reinterpret_cast<const float4*>(c + half)[j];
        const float sign = d0 < half ? -1.0f : 1.0f;
        co[4 * j] = x.x; co[4 * j + 1] = x.y; co[4 * j + 2] = x.z; co[4 * j + 3] = x.w;
        si[4 * j] = sign * y.x; si[4 * j + 1] = sign * y.y; si[4 * j + 2] = sign * y.z; si[4 * j + 3] = sign * y.w;
      }
    }
  }
  const int partner = a.interleaved ? l : d0 < half ? l + half / 8 : l - half / 8;
  const int src = sub * L + (turns ? partner : l);

  int64_t slot = -1;
  if constexpr (STORE) {
    slot = a.slots[token];
    if (slot >= a.slot_count || slot < -1) {
      if (lane == 0) kv4::report(a.status, kv4::kBadSlot, static_cast<uint32_t>(token));
      slot = -1;
    }
  }

#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = h0 + i * R;
    const bool is_v = STORE && h >= a.hq + a.hk, is_q = h < a.hq;
    float x[8];
    kv4::unpack_bf16x8(raw[i], x);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
    for (int d = 1; d < L; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
    const float r = rsqrtf(ss * (1.0f / D) + a.eps);
    float w[8];
    load_weight(is_q ? a.wq : a.wk, a.w_fp32, a.unit, d0, w);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x[j] * r * w[j];
    if (a.interleaved) {
      if (turns) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float y0 = y[j], y1 = y[j + 1];
          y[j] = fmaf(y0, co[j], y1 * si[j]);
          y[j + 1] = fmaf(y1, co[j + 1], y0 * si[j + 1]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float other = __shfl_sync(0xFFFFFFFFu, y[j], src);
        if (turns) y[j] = fmaf(y[j], co[j], other * si[j]);
      }
    }
    const uint4 rounded = is_v ? raw[i] : kv4::pack_bf16x8(y);
    if (is_q || (h < a.hq + a.hk && a.k_out)) {
      __nv_bfloat16* o = is_q ? a.q_out + (token * a.hq + h) * D : a.k_out + (token * a.hk + h - a.hq) * D;
      *reinterpret_cast<uint4*>(o + d0) = rounded;
    }
    if constexpr (STORE) {
      float z[8], s;
      kv4::unpack_bf16x8(rounded, z);
      const uint32_t word = kv4::quantise8(z, 0xFFFFFFFFu, s);
      if (slot >= 0 && !is_q && h < a.heads) {
        const int head = is_v ? h - a.hq - a.hk : h - a.hq;
        kv4::store8<D>(a.cache + kv4::block_at<D>(slot, head, a.hk, a.shift), static_cast<int>(slot & 15), is_v, l, word, s);
      }
    }
  }
}

template <int D, int U, bool STORE>
int launch(const RopeArgs& a, cudaStream_t stream) {
  const int rows = 32 / (D / 8) * U, per = (a.heads + rows - 1) / rows;
  const int64_t blocks = (static_cast<int64_t>(a.tokens) * per + kWarps - 1) / kWarps;
  rope_kernel<D, U, STORE><<<static_cast<unsigned>(blocks), kWarps * 32, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <int D>
int launch_d(const RopeArgs& a, bool store, cudaStream_t stream) {
  constexpr int U = 4;
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
