// Keys and values into the 4-bit cache, and what they stand for back out of it, by slot.
// 2 bytes a value on one side, 17/32 on the other. 16384 tokens with 4 heads of 128, 42.6 MB, take 12.5 us to store and 8.7 us to read; a copy
// of as many bytes takes 7.4. Stored, bound by instructions (the largest magnitude and scale of a group, a quotient for each value), which
// is why a lane has 16 dims: with eight, 160 instructions for each eight instead of some 100, it took 15.9, and 10.5 to read.
// That a token's values lie 64 bytes apart costs nothing: stored like keys they take as long.
#include <cuda_runtime.h>
#include "kv4_format.cuh"
#include "../../../include/mono_attention.h"

namespace mono {
namespace {

constexpr int kWarps = 8;

struct StoreArgs {
  const __nv_bfloat16 *k, *v;               // stored, or
  __nv_bfloat16 *k_out, *v_out;             // read
  uint8_t* cache;
  const int64_t* slots;
  uint32_t* status;
  int64_t k_ts, k_hs, v_ts, v_hs, slot_count;
  int tokens, step, heads, shift;           // step: half of the tokens
  uint32_t per_inv;                         // of the rows of a token
  bool wide;                                // outputs begin on 32-byte boundaries
};

// 32 bytes on a 32-byte boundary in one go, else in two of 16, each at every other 16, which touch all sectors twice: 16384 tokens
// with 4 heads of 128 are read in 8.7 us instead of 12.7. (Loads of 32 bytes gain nothing: the second of two finds its sector in L1.)
__device__ __forceinline__ void store32(__nv_bfloat16* p, const uint4& v, const uint4& w, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = v;
    reinterpret_cast<uint4*>(p)[1] = w;
  }
}

// Rows are (token, head, key or value), D/16 lanes each, two words of the cache to a lane: side by side for a key, 64 bytes apart for a
// value. A thread has U rows, of the same head of tokens `step` apart, so that what belongs to the head is worked out once.
template <int D, int U, bool READ>
__global__ __launch_bounds__(kWarps * 32) void store_kernel(const StoreArgs a) {
  constexpr int L = D / 16, Scales = 4 * D / kv4::kGroup;    // lanes of a row; bytes of a token's scales
  const int l = threadIdx.x % L, row = static_cast<int>(blockIdx.x * (kWarps * 32 / L) + threadIdx.x / L), per = 2 * a.heads;
  if (row - static_cast<int>(threadIdx.x % 32) / L >= a.step * per) return;   // the whole warp
  const int first = kv4::divide(min(row, a.step * per - 1), per, a.per_inv), h = min(row, a.step * per - 1) - first * per;
  const bool value = h >= a.heads, real = row < a.step * per;
  const int head = value ? h - a.heads : h, scale_to = kv4::scale_at<D>(0, value, l >> 2), second = value ? 64 : 4;
  const kv4::WordPlace<D> place(value, 2 * l);
  int64_t slot[U];
  bool fine[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    fine[i] = real && first + i * a.step < a.tokens;
    slot[i] = fine[i] ? __ldg(a.slots + first + i * a.step) : -1;
  }
  uint4 raw[U][2];
  if constexpr (!READ) {
    const int64_t ts = value ? a.v_ts : a.k_ts;
    const __nv_bfloat16* from = (value ? a.v + head * a.v_hs : a.k + head * a.k_hs) + first * ts + 16 * l;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n) raw[i][n] = fine[i] ? __ldg(reinterpret_cast<const uint4*>(from + i * (a.step * ts)) + n) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (static_cast<uint64_t>(slot[i]) >= static_cast<uint64_t>(a.slot_count)) {
      if (slot[i] != -1 && l == 0) kv4::report(a.status, kv4::kBadSlot, static_cast<uint32_t>(first + i * a.step));
      slot[i] = -1;
    }
  if constexpr (READ) {
    uint32_t word[U][2], scale[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      word[i][0] = word[i][1] = 0x88888888u;
      scale[i] = 0;
      if (slot[i] >= 0) {
        const uint8_t* blk = a.cache + kv4::block_at<D>(slot[i], head, a.heads, a.shift);
        const int r = static_cast<int>(slot[i]) & 15;
        const uint8_t* at = blk + place.at(r);
        word[i][0] = __ldg(reinterpret_cast<const uint32_t*>(at));
        word[i][1] = __ldg(reinterpret_cast<const uint32_t*>(at + second));
        scale[i] = __ldg(reinterpret_cast<const uint16_t*>(blk + scale_to + r * Scales));
      }
    }
    __nv_bfloat16* to = (value ? a.v_out : a.k_out) + (static_cast<int64_t>(first) * a.heads + head) * D + 16 * l;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (fine[i]) store32(to + i * (static_cast<int64_t>(a.step) * a.heads * D), kv4::dequantise8(word[i][0], scale[i]), kv4::dequantise8(word[i][1], scale[i]), a.wide);
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float s;
      uint32_t word[2];
      kv4::quantise(raw[i], word, s);
      if (slot[i] >= 0) {
        uint8_t* blk = a.cache + kv4::block_at<D>(slot[i], head, a.heads, a.shift);
        const int r = static_cast<int>(slot[i]) & 15;
        uint8_t* at = blk + place.at(r);
        *reinterpret_cast<uint32_t*>(at) = word[0];
        *reinterpret_cast<uint32_t*>(at + second) = word[1];
        if ((l & 3) == 0) *reinterpret_cast<uint16_t*>(blk + scale_to + r * Scales) = static_cast<uint16_t>(__float_as_uint(s) >> 16);
      }
    }
  }
}

template <int D, bool READ>
int launch(StoreArgs& a, cudaStream_t stream) {
  // 16384 tokens stored, read: U = 1 14.5, 9.8 us; 2 12.5, 8.7; 4 13.1, 9.8
  constexpr int U = 2, Rows = kWarps * 32 / (D / 16);
  a.step = (a.tokens + U - 1) / U;
  store_kernel<D, U, READ><<<static_cast<unsigned>((static_cast<int64_t>(a.step) * 2 * a.heads + Rows - 1) / Rows), kWarps * 32, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

int check(int tokens, int heads, int head_dim, int64_t num_pages, int page_size) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MONO_ATTN_BAD_HEAD_DIM;
  if (tokens < 0 || heads < 1 || num_pages < 1 || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return MONO_ATTN_BAD_SIZE;
  return static_cast<int64_t>(tokens) * heads * 2 > INT32_MAX - 4096 ? MONO_ATTN_BAD_SIZE : 0;
}

}  // namespace
}  // namespace mono

extern "C" int mono_attn_kv4_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                    int64_t v_token_stride, int64_t v_head_stride, int tokens, int kv_heads, int head_dim,
                                    uint8_t* cache, int64_t num_pages, int page_size, const int64_t* slots, uint32_t* status,
                                    mono_attn_stream_t stream) {
  using namespace mono;
  if (const int rc = check(tokens, kv_heads, head_dim, num_pages, page_size)) return rc;
  if (!k || !v || !cache || !slots || !status) return MONO_ATTN_NULL;
  if (tokens == 0) return 0;
  StoreArgs a{};
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.cache = cache; a.slots = slots; a.status = status;
  a.k_ts = k_token_stride; a.k_hs = k_head_stride; a.v_ts = v_token_stride; a.v_hs = v_head_stride;
  a.slot_count = num_pages * page_size;
  a.tokens = tokens;
  a.per_inv = 0xFFFFFFFFu / static_cast<uint32_t>(2 * kv_heads);
  a.heads = kv_heads;
  a.shift = __builtin_ctz(page_size);
  return head_dim == 64 ? launch<64, false>(a, stream) : head_dim == 128 ? launch<128, false>(a, stream) : launch<256, false>(a, stream);
}

extern "C" int mono_attn_kv4_read(const uint8_t* cache, int64_t num_pages, int page_size, const int64_t* slots, int tokens,
                                  int kv_heads, int head_dim, void* k_out, void* v_out, uint32_t* status,
                                  mono_attn_stream_t stream) {
  using namespace mono;
  if (const int rc = check(tokens, kv_heads, head_dim, num_pages, page_size)) return rc;
  if (!k_out || !v_out || !cache || !slots || !status) return MONO_ATTN_NULL;
  if (tokens == 0) return 0;
  StoreArgs a{};
  a.k_out = static_cast<__nv_bfloat16*>(k_out);
  a.v_out = static_cast<__nv_bfloat16*>(v_out);
  a.wide = !((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 31);
  a.cache = const_cast<uint8_t*>(cache); a.slots = slots; a.status = status;
  a.slot_count = num_pages * page_size;
  a.tokens = tokens;
  a.per_inv = 0xFFFFFFFFu / static_cast<uint32_t>(2 * kv_heads);
  a.heads = kv_heads;
  a.shift = __builtin_ctz(page_size);
  return head_dim == 64 ? launch<64, true>(a, stream) : head_dim == 128 ? launch<128, true>(a, stream) : launch<256, true>(a, stream);
}
