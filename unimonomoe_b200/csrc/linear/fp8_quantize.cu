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
    const GroupScale g(top_of_group(v));
    if (mine) *reinterpret_cast<uint4*>(a.codes + row * a.cols + col) = codes16(v, g.inverse);
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
