// Rows to 8 bits: a scale for each group of 128 columns, codes e4m3 (include/mono_linear.h has the definition), with silu(a) * b in
// front of it where the rows hold a and b side by side.
//
// Eight lanes share a group, 16 values (32 bytes) a lane: the largest magnitude takes three exchanges, a lane writes 16 codes at once.
// Bound by memory: 2 (4) bytes in and 1 out for a value.
#include "linear.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kThreads = 256, kPerBlock = kThreads / 8;

struct QuantizeArgs {
  const __nv_bfloat16* x;
  uint8_t* codes;
  float* scales;
  int64_t stride, items;                     // groups in all
  int cols, groups;
};

// 16 bf16 in fp32.
__device__ __forceinline__ void load16(const __nv_bfloat16* p, float2 (&v)[8]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = bf16x2(w[i]);
}

template <bool Silu>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantizeArgs a) {
  let_next_launch_begin();                   // a product that waits for these results by itself
  const int sub = threadIdx.x & 7;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kPerBlock + (threadIdx.x >> 3); ; item += static_cast<int64_t>(gridDim.x) * kPerBlock) {
    const bool have = item < a.items;
    if (!__any_sync(0xFFFFFFFFu, have)) break;
    const int64_t row = have ? item / a.groups : 0;
    const int group = have ? static_cast<int>(item - row * a.groups) : 0, col = group * kGroup + sub * 16;
    const bool mine = have && col < a.cols;
    float2 v[8] = {};
    if (mine) {
      const __nv_bfloat16* src = a.x + row * a.stride + col;
      load16(src, v);
      if constexpr (Silu) {
        float2 u[8];
        load16(src + a.cols, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = gated(v[i], u[i]);
      }
    }
    // the largest magnitude, which passes over what is not a number; that is found by products with zero
    float top = 0.0f;
    float2 zero = both(0.0f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = fmaxf(top, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
      zero = fma2(v[i], both(0.0f), zero);
    }
    uint32_t m = zero.x + zero.y == 0.0f ? __float_as_uint(top) : 0x7FC00000u;
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    const GroupScale g(m);
    if (mine) {
      const float2 scale = both(g.inverse);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 lo = mul2(v[2 * i], scale), hi = mul2(v[2 * i + 1], scale);
        w[i] = pack_e4m3x4(lo.x, lo.y, hi.x, hi.y);
      }
      *reinterpret_cast<uint4*>(a.codes + row * a.cols + col) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (have && sub == 0) a.scales[item] = g.scale;
  }
}

}  // namespace
}  // namespace mono

extern "C" int mono_lin_quantize(const void* x, int64_t row_stride, int64_t rows, int cols, int silu, uint8_t* codes, float* scales,
                                 mono_lin_stream_t stream) {
  using namespace mono;
  if (rows < 0 || cols < 16 || cols % 16 || cols > (1 << 24) || row_stride < 0) return MONO_LIN_BAD_SIZE;
  if (rows == 0) return 0;
  if (!x || !codes || !scales) return MONO_LIN_NULL;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes)) & 15 || row_stride % 8) return MONO_LIN_ALIGNMENT;
  const int groups = (cols + lin::kGroup - 1) / lin::kGroup;
  QuantizeArgs a{static_cast<const __nv_bfloat16*>(x), codes, scales, row_stride, rows * groups, cols, groups};
  const int64_t blocks = (a.items + kPerBlock - 1) / kPerBlock, most = lin::kSms * 8 * 4;
  const int grid = static_cast<int>(blocks < most ? blocks : most);
  if (silu) quantize_kernel<true><<<grid, kThreads, 0, stream>>>(a);
  else quantize_kernel<false><<<grid, kThreads, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
