// The 4-bit key/value cache: where a code and a scale lie, how a row is quantised and read back.
//
// A page of one KV head is a run of blocks of 16 tokens, 17*D bytes each (D = head size, NG = D/64 groups of 64 dims):
//   [0, 8D)      key codes      [8D, 16D)   value codes      [16D, 17D)  scales, per token NG of the key then NG of the value
// A group x of 64 values is stored as a scale s and codes c in [-7, 7], kept as c + 8 in half a byte:
//   s = round to five significant bits of max|x| / 7, within [2^-60, 2^60];   c = clamp(rint(x / s), -7, 7);   value s * c
// Five bits of s and three of c make s * c exact in bfloat16: nothing is rounded when a key or value is read back, and
// the matrix unit works on the values themselves. Rounding s moves it by at most 1/32, the largest value of a
// group by at most 7/32 of a step.
// A group that holds an infinity or a NaN gets the scale NaN: what reads it sees that it was not finite.
//
// Codes lie in the order in which the lanes of a warp use them as the A operand of mma.m16n8k16 (lane = 4 g + t holds rows g
// and g + 8, columns 2t, 2t+1, 2t+8, 2t+9), 16 bytes to a lane at a time, so that a block is loaded with full-width
// shared-memory reads free of bank conflicts and no code is moved between lanes:
//   keys:   token r = g or g + 8, dims 64 gi + 16 t + (0..15): two words for each of the two tokens and each group
//   values: dims 64 gi + 8 g + (0..7) of tokens 2t, 2t+1, 2t+8, 2t+9: one word for each token and group
// The order of the products inside a sum is free, so dims may stand in any column as long as the query's do too.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>

namespace mono {
namespace kv4 {

constexpr int kGroup = 64;
constexpr int kTokens = 16;               // tokens of a block
constexpr float kScaleMin = 0x1p-60f, kScaleMax = 0x1p60f;

__host__ __device__ constexpr int block_bytes(int d) { return 17 * d; }

// Byte of the word that holds dims 8 l .. 8 l + 7 of token r, from the start of its block.
template <int D>
__device__ __forceinline__ int key_word(int r, int l) {
  constexpr int NG = D / kGroup;
  const int o = (r >> 3) * 8 * NG + (2 * (l >> 3) + (l & 1)) * 4;
  return (o >> 4) * 512 + ((r & 7) * 4 + ((l & 7) >> 1)) * 16 + (o & 15);
}
template <int D>
__device__ __forceinline__ int value_word(int r, int l) {
  constexpr int NG = D / kGroup;
  const int o = ((r >> 3) * 2 + (r & 1)) * 4 * NG + (l >> 3) * 4;
  return 8 * D + (o >> 4) * 512 + ((l & 7) * 4 + ((r >> 1) & 3)) * 16 + (o & 15);
}
template <int D>
__device__ __forceinline__ int scale_at(int r, bool value, int gi) {
  constexpr int NG = D / kGroup;
  return 16 * D + r * 4 * NG + (value ? 2 * NG : 0) + gi * 2;
}

// First byte of the block of `slot` (page * page_size + offset) for one head; page_shift = log2(page_size).
template <int D>
__device__ __forceinline__ int64_t block_at(int64_t slot, int head, int heads, int page_shift) {
  // numbers of blocks fit 32 bits: 2^32 of the smallest ones are 4 TB
  const int shift = page_shift - 4;
  const uint32_t sub = static_cast<uint32_t>(slot >> 4), page = sub >> shift;
  return static_cast<int64_t>(sub + page * (static_cast<uint32_t>(heads - 1) << shift) + (static_cast<uint32_t>(head) << shift)) * block_bytes(D);
}

// key_word or value_word of a lane whose row is a key (or a value) throughout, for many tokens: linear in three parts of r.
template <int D>
struct WordPlace {
  int first, pair, odd;                     // the place for r = 0; what a step of r >> 1 & 3, of r & 1 adds
  __device__ __forceinline__ WordPlace(bool value, int l)
      : first(value ? value_word<D>(0, l) : key_word<D>(0, l)), pair(value ? value_word<D>(2, 0) - value_word<D>(0, 0) : key_word<D>(2, 0)),
        odd(value ? value_word<D>(1, 0) - value_word<D>(0, 0) : key_word<D>(1, 0)) {}
  __device__ __forceinline__ int at(int r) const { return first + (r >> 3) * key_word<D>(8, 0) + (r >> 1 & 3) * pair + (r & 1) * odd; }
};

// To five significant bits, ties to even. Finite, normal s.
__device__ __forceinline__ float round5(float s) {
  uint32_t b = __float_as_uint(s);
  b += 0x3FFFFu + ((b >> 19) & 1u);
  return __uint_as_float(b & ~0x7FFFFu);
}

// Pairs of fp32 in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)),
      "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 bf16x2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }

// 8 N bf16 of a row, in the 8 / N adjacent lanes that share a group: their codes as N words, and the group's scale.
// All lanes of the warp take part.
template <int N>
__device__ __forceinline__ void quantise(const uint4 (&raw)[N], uint32_t (&words)[N], float& scale) {
  // largest magnitude, as integers: a NaN is above infinity, infinity above the rest
  uint32_t m = 0;
#pragma unroll
  for (int n = 0; n < N; ++n)
    m = __vmaxu2(m, __vmaxu2(__vmaxu2(raw[n].x & 0x7FFF7FFFu, raw[n].y & 0x7FFF7FFFu), __vmaxu2(raw[n].z & 0x7FFF7FFFu, raw[n].w & 0x7FFF7FFFu)));
#pragma unroll
  for (int d = 1; d < 8 / N; d <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
  const uint32_t top = max(m << 16, m & 0xFFFF0000u);
  if (top >= 0x7F800000u) {
    scale = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int n = 0; n < N; ++n) words[n] = 0x88888888u;
    return;
  }
  // top / 7 and x / s by one step of Newton's method on the quotient with an exact residual (Markstein, 1990). With the rounded reciprocal
  // of 7 it is the rounded quotient.
  const float seven = 0.14285714924335479736f, about = __uint_as_float(top) * seven, seventh = fmaf(fmaf(about, -7.0f, __uint_as_float(top)), seven, about);
  const float s = fminf(fmaxf(round5(seventh), kScaleMin), kScaleMax);
  scale = s;
  // A quotient x / s halfway between two codes has few bits and comes out exactly with any reciprocal that is right to some 2^-20,
  // so that ties go to even as they are defined to; the others are further from there than the error. No quotient rounds to more
  // than 7, unless the scale was cut. The integers are taken from the low bits of sums with 1.5 * 2^23 + 8, whose other bits are
  // subtracted from the word at the end.
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const bool cut = seventh > kScaleMax;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const uint32_t w[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
    uint32_t word = 0u - 0x4B400000u * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = bf16x2(w[i]);
      float2 y = mul2(x, both(inv));
      y = fma2(fma2(y, both(-s), x), both(inv), y);
      if (cut) y = make_float2(fminf(fmaxf(y.x, -7.0f), 7.0f), fminf(fmaxf(y.y, -7.0f), 7.0f));
      y = add2(y, both(12582920.0f));
      word += __float_as_uint(y.x) * (1u << (8 * i)) + __float_as_uint(y.y) * (1u << (8 * i + 4));
    }
    words[n] = word;
  }
}
__device__ __forceinline__ uint32_t quantise8(const uint4& raw, float& scale) {
  const uint4 r[1] = {raw};
  uint32_t w[1];
  quantise(r, w, scale);
  return w[0];
}

// What a word of eight codes and their scale stand for, in order, exactly.
__device__ __forceinline__ uint4 dequantise8(uint32_t word, uint32_t scale) {
  // a code c + 8 as the top four bits of the mantissa under the exponent of 16 is 24 + c; (24 + c) s - 24 s in one step
  const uint32_t even = (word << 3) & 0x78787878u, odd = (word >> 1) & 0x78787878u, s2 = scale | scale << 16;
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2), n = __hmul2(s, __float2bfloat162_rn(-24.0f));
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t y = __byte_perm(even, odd, i * 0x1111 + 0x4400);            // byte i of both, twice
    y = (y & 0x00780078u) | 0x41804180u;
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&y), s, n);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// x / d for 0 <= x < 2^31 with inv = (2^32 - 1) / d: the product with the reciprocal is at most one too low.
__device__ __forceinline__ int divide(int x, int d, uint32_t inv) {
  const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(x), inv));
  return x - q * d >= d ? q + 1 : q;
}

// Stores dims 8 l .. 8 l + 7 of one row: `blk` is its block, r its token there.
template <int D>
__device__ __forceinline__ void store8(uint8_t* blk, int r, bool value, int l, uint32_t word, float scale) {
  *reinterpret_cast<uint32_t*>(blk + (value ? value_word<D>(r, l) : key_word<D>(r, l))) = word;
  if ((l & 7) == 0)
    *reinterpret_cast<uint16_t*>(blk + scale_at<D>(r, value, l >> 3)) = static_cast<uint16_t>(__float_as_uint(scale) >> 16);
}

// Device-side errors of the operators: the first one stays in the status word.
enum Status : uint32_t {
  kStatusOk = 0,
  kBadPosition = 1,      // a position outside the rotation table
  kBadSlot = 2,          // a slot outside the cache
  kBadPage = 3,          // a block-table entry outside the cache
  kTooLong = 4,          // a sequence longer than its row of the block table
  kNoPages = 5,          // more pages needed than are free
  kTooManyTokens = 6,    // more tokens than the outputs have rows
  kBadLength = 7,        // a negative length, or query offsets that fall or pass the query's rows
  kWaitTimeout = 8,      // a wait inside a kernel ran out
};
__device__ __forceinline__ void report(uint32_t* status, uint32_t code, uint32_t where) {
  if (atomicCAS(status, 0u, code) == 0u) status[1] = where;
}

__device__ __forceinline__ void unpack_bf16x8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 pack_bf16x8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

}  // namespace kv4
}  // namespace mono
