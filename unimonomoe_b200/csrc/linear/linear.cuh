// What the block-FP8 operators share: packing, the arguments of a product and the division of its
// work into units.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "../../../include/mono_linear.h"
#include "../ptx_sm100.cuh"
#include "waits.cuh"

namespace mono {
namespace lin {

constexpr int kGroup = 128;                  // columns that share a scale, rows too in a weight
constexpr int kSms = 148;

// ---- values
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 bf16x2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)),
      "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return *reinterpret_cast<const float2*>(&r);
}
// Four values as e4m3, to nearest, the first in the lowest byte; NaN stays NaN, what is past 448 becomes 448.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 minus(float2 a) { return make_float2(-a.x, -a.y); }
// exp(-a) of a from -88.72 to 90 is 2^t, t = -a log2(e): of the rounded product, and what rounding it lost put back by 1 + rest ln(2). (That alone is up
// to |t| 2^-24 of the result.) Arguments outside are cut to that.
__device__ __forceinline__ float2 exp_minus(float2 a) {
  constexpr float kLog2E = 0x1.715476p+0f, kLog2ERest = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;
  const float2 m = make_float2(fminf(fmaxf(-a.x, -90.0f), 88.72f), fminf(fmaxf(-a.y, -90.0f), 88.72f)), t = mul2(m, both(kLog2E));
  const float2 rest = fma2(m, both(kLog2ERest), fma2(m, both(kLog2E), minus(t)));
  const float2 e = make_float2(ex2_approx_ftz(t.x), ex2_approx_ftz(t.y));
  return fma2(e, mul2(rest, both(kLn2)), e);
}
// silu(a) * b into a, to fp32's precision: with the fast exponential and quotient one code in 10^5 is another. The quotient is made of a reciprocal
// with one step of Newton's method and a correction by its exact residual (Markstein, 1990), which is the rounded quotient; a sixteenth of both
// sides, so that the reciprocal of the largest exponential is a normal number. Below -88.72, where the exponential is infinite, the quotient is zero, for
// an infinite a NaN. (65.7 us for 131072 x 512; with expf, and the same to a step in its last place, 69.9.)
__device__ __forceinline__ void gate16(float2 (&a)[8], const float2 (&b)[8]) {
  constexpr float kLeast = -88.72f, kSixteenth = 0.0625f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 d = fma2(exp_minus(a[i]), both(kSixteenth), both(kSixteenth));
    const float2 n = mul2(a[i], make_float2(a[i].x < kLeast ? 0.0f : kSixteenth, a[i].y < kLeast ? 0.0f : kSixteenth));
    float2 r = make_float2(rcp_approx_ftz(d.x), rcp_approx_ftz(d.y));
    r = fma2(fma2(minus(d), r, both(1.0f)), r, r);
    const float2 q = mul2(n, r);
    a[i] = mul2(fma2(fma2(minus(q), d, n), r, q), b[i]);
  }
}
// The same of a product's sums, which are themselves off by more than the fast exponential and division are. Where exp(-a) is infinite
// or close to it (a under -87) the quotient is -0.
__device__ __forceinline__ float gated_sums(float a, float b) { return __fdividef(a, 1.0f + __expf(-a)) * b; }
// The scale of a group whose largest magnitude has the bits `m` (a NaN's are above infinity's), and what its values are multiplied by.
struct GroupScale {
  float scale, inverse;
  __device__ __forceinline__ explicit GroupScale(uint32_t m) {
    const float top = m < 0x0D800000u ? 1.0f : __uint_as_float(m);      // 2^-100
    if (m >= 0x7F800000u) {
      scale = inverse = __uint_as_float(0x7FC00000u);
    } else {
      scale = __fdiv_rn(top, 448.0f);
      inverse = __fdiv_rn(448.0f, top);
    }
  }
};
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// 16 bf16 in fp32.
__device__ __forceinline__ void unpack16(const uint4& a, const uint4& b, float2 (&v)[8]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = bf16x2(w[i]);
}
// Largest magnitude (as bits, a NaN's above all) of a group that eight neighbouring lanes share, 16 values each. All lanes of the warp take part.
__device__ __forceinline__ uint32_t top_of_group(const float2 (&v)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(v[i].x), "f"(v[i].y));
  uint32_t m = __float_as_uint(top);
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
  return m;
}
__device__ __forceinline__ uint4 codes16(const float2 (&v)[8], float inverse) {
  const float2 scale = both(inverse);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 lo = mul2(v[2 * i], scale), hi = mul2(v[2 * i + 1], scale);
    w[i] = pack_e4m3x4(lo.x, lo.y, hi.x, hi.y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- launches one after another without a gap
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Of what that launch writes: stays behind the wait, where a load that counts on memory that nobody writes might be moved in front of it.
__device__ __forceinline__ float ld_after(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void let_next_launch_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- products
struct Product {
  const uint8_t* x;                          // codes [x_rows, k]
  const float* xs;                           // their scales [x_rows, groups]
  const __nv_bfloat16* raw;                  // or the rows in 16 bits, which the kernel of few rows quantises (else null)
  int64_t raw_stride;
  const float* ws;                           // [experts][blocks][groups]
  const int32_t* offsets;                    // of the experts' runs, or null: one run of all rows
  const int32_t* tokens;                     // row of x for each row, or null: the same
  const __nv_bfloat16* residual;
  void* out;
  uint8_t* codes;
  float* scales;
  uint32_t* status;
  int64_t rows, x_rows;
  int n, k, experts, groups, blocks;
  int cols;                                  // units along n
  int fp32, vec, after;                      // out is fp32; its rows begin on 16-byte boundaries; launched beside the launch before
};

struct Run {
  int row, rows, expert, col;                // first row of the unit, its rows
};

// Units of `Tile` rows: units of a run of n rows are ceil(n / Tile), times p.cols along n. `first` (shared memory, experts + 1 words)
// holds the number of row tiles in the runs before each; filled by all threads of the CTA.
template <int Tile>
struct Division {
  const Product& p;
  const int* first;
  __device__ __forceinline__ Division(const Product& p, const int* first) : p(p), first(first) {}

  // By all threads, `threads` of them a multiple of 32, at most 1024; `sums` has 32 words. Where offsets are out of order or
  // outside the rows, there are no units. The run of row tile `tile`, where there is one, is left in `found` (shared memory; its column not) by the thread
  // that comes upon it: a search takes 1200 cycles.
  static __device__ __forceinline__ void fill(const Product& p, int* first, int* sums, int threads, int tile = -1, Run* found = nullptr) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int base = 0;
    bool bad = false;
    for (int e0 = 0; e0 < p.experts; e0 += threads) {
      int n = 0;
      int64_t a = 0, b = 0;
      if (e0 + t < p.experts) {
        a = __ldg(p.offsets + e0 + t);
        b = __ldg(p.offsets + e0 + t + 1);
        if (a < 0 || b < a || b > p.rows) {
          report(p.status, kBadOffsets, e0 + t);
          bad = true;
        } else {
          n = static_cast<int>((b - a + Tile - 1) / Tile);
        }
      }
      int s = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if (lane >= d) s += o;
      }
      if (lane == 31) sums[warp] = s;
      __syncthreads();
      const int of_warp = lane < threads / 32 ? sums[lane] : 0;
      int before = of_warp;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, before, d);
        if (lane >= d) before += o;
      }
      const int lower = __shfl_sync(0xFFFFFFFFu, before - of_warp, warp);
      const int mine = base + lower + s - n;
      if (e0 + t < p.experts) first[e0 + t] = mine;
      if (tile >= mine && tile < mine + n) {
        const int row = static_cast<int>(a) + (tile - mine) * Tile;
        *found = Run{row, min(Tile, static_cast<int>(b) - row), e0 + t, 0};
      }
      base += __shfl_sync(0xFFFFFFFFu, before, 31);
      if (e0 + threads < p.experts) __syncthreads();
    }
    if (__syncthreads_or(bad)) base = 0;
    if (t == 0) first[p.experts] = base;
    __syncthreads();
  }

  __device__ __forceinline__ int row_tiles() const { return p.offsets ? first[p.experts] : static_cast<int>((p.rows + Tile - 1) / Tile); }
  __device__ __forceinline__ int units() const { return row_tiles() * p.cols; }
  // Unit u of a dense product: bands of eight row tiles, whose rows and the weight's both stay in L2.
  __device__ __forceinline__ Run unit(int u) const {
    Run r;
    if (p.rows <= Tile) {                    // without the divisions
      r.expert = r.row = 0;
      r.rows = static_cast<int>(p.rows);
      r.col = u;
      return r;
    }
    constexpr int kBand = 8;
    const int band = u / (kBand * p.cols), high = min(kBand, row_tiles() - band * kBand), in = u - band * kBand * p.cols;
    r.expert = 0;
    r.col = in / high;
    r.row = (band * kBand + in - r.col * high) * Tile;
    r.rows = min(Tile, static_cast<int>(p.rows) - r.row);
    return r;
  }
  // Unit u by a whole warp that takes its units in order; `lo` is the expert of the one before, 0 at first. Experts' units follow one another along n, so that a
  // weight is read once for the row tiles of its run.
  __device__ __forceinline__ Run unit_after(int u, int& lo) const {
    if (p.offsets) {
      const int tile = u / p.cols, lane = threadIdx.x & 31;
      int n;
      do {
        const int e = lo + 1 + lane;
        n = __popc(__ballot_sync(0xFFFFFFFFu, e < p.experts && first[e] <= tile));
        lo += n;
      } while (n == 32);
      return of_expert(lo, tile, u - tile * p.cols);
    }
    return unit(u);
  }

 private:
  __device__ __forceinline__ Run of_expert(int e, int tile, int col) const {
    const int a = __ldg(p.offsets + e), b = __ldg(p.offsets + e + 1);
    Run r;
    r.expert = e;
    r.col = col;
    r.row = a + (tile - first[e]) * Tile;
    r.rows = max(0, min(Tile, b - r.row));
    return r;
  }
};

// ---- results
// Four columns of a row of the result, from column n on. Out of line, like all that is not the usual case: what a unit runs through
// once it finds in no cache, and every 128 bytes of code then cost it as much as some hundred cycles.
static __device__ __noinline__ void store_any(const __nv_bfloat16* residual, void* out, int cols, int fp32, int64_t at, int n, float4 v) {
  float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < cols) {
      if (residual) x[i] += __bfloat162float(residual[at + i]);
      if (fp32) static_cast<float*>(out)[at + i] = x[i];
      else static_cast<__nv_bfloat16*>(out)[at + i] = __float2bfloat16_rn(x[i]);
    }
}
__device__ __forceinline__ void store4(const Product& p, int64_t row, int n, const float4& v) {
  const int64_t at = row * p.n + n;
  if (p.vec && !p.fp32) {                    // n is a multiple of 8
    if (n < p.n) {
      float4 x = v;
      if (p.residual) {
        const uint2 r = __ldg(reinterpret_cast<const uint2*>(p.residual + at));
        const float2 a = bf16x2(r.x), b = bf16x2(r.y);
        x = make_float4(x.x + a.x, x.y + a.y, x.z + b.x, x.w + b.y);
      }
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
    }
  } else {
    store_any(p.residual, p.out, p.n, p.fp32, at, n, v);
  }
}

// Row of x that row i has; where there is none that is reported, and the first one is taken.
__device__ __forceinline__ int source_row(const Product& p, int64_t i) {
  if (!p.tokens) return static_cast<int>(i);
  const int t = __ldg(p.tokens + i);
  if (t >= 0 && t < p.x_rows) return t;
  report(p.status, kBadToken, static_cast<uint32_t>(i));
  return 0;
}

// ---- copies into shared memory
// 16 bytes, or zeros where `bytes` is 0.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// The two kernels (linear_few.cu, linear_many.cu). Groups of K in a stage of the first, and how many clusters of `split` of its CTAs run at once.
constexpr int few_groups(bool gate) { return gate ? 1 : 2; }
int few_clusters(int split);
int few_stages(int tile, bool gate);         // of the ring of a CTA
int launch_few(const Product& p, const CUtensorMap& weight, int tile, int split, int64_t clusters, cudaStream_t stream);
int launch_many(const Product& p, const CUtensorMap& weight, const CUtensorMap& x, const CUtensorMap& out, const CUtensorMap& residual, int split,
                int clusters, cudaStream_t stream);

}  // namespace lin
}  // namespace mono
