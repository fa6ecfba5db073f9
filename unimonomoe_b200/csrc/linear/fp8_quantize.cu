// Rows to 8 bits: a scale for each group of 128 columns, codes e4m3 (include/mono_linear.h has the definition), with silu(a) * b in
// front of it where the rows hold a and b side by side.
//
// Eight lanes share a group, 16 values (32 bytes) a lane: the largest magnitude takes three exchanges, a lane writes 16 codes at once. Each thread goes
// from group to group, the next one's values on their way while one is quantised, its place by additions: with a division of 64 bits for
// each and no values ahead 16384 x 7168 took 67.6 us. The grid has eight CTAs for an SM, of which four run at once by their registers (53, with silu 64). Bound by
// memory, 2 bytes in and 1 out for a value: 59.6 us there, 5.9 TB/s. With silu 4 bytes in and an exponential and a quotient to fp32's precision (gate16() has the reason):
// 131072 rows of 512 in 65.7 us, 5.1 TB/s. Neither memory (57%) nor the issue slots (2.8 of 4 a cycle) are full then; 42% of the warps are too few to fill
// either. One row of 2048 takes what a launch takes.
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
  const int at_first = blockIdx.x * kPerBlock + (threadIdx.x >> 3), step = gridDim.x * kPerBlock;
  int64_t item = at_first, row = at_first / a.groups;
  int group = at_first % a.groups;
  const int rows = step / a.groups, groups = step - rows * a.groups;
  constexpr int kLoads = Silu ? 4 : 2;
  uint4 next[kLoads];
  auto fetch = [&]() {
    const int col = group * kGroup + sub * 16;
    const bool have = item < a.items && col < a.cols;
    const uint4* src = reinterpret_cast<const uint4*>(a.x + row * a.stride + col);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) next[i] = have ? __ldg(src + (i & 1) + (i >> 1) * (a.cols / 8)) : make_uint4(0, 0, 0, 0);
  };
  fetch();
  while (__any_sync(0xFFFFFFFFu, item < a.items)) {
    const bool have = item < a.items, mine = have && group * kGroup + sub * 16 < a.cols;
    const int64_t at = item, to = row * a.cols + group * kGroup + sub * 16;
    float2 v[8], u[8];
    unpack16(next[0], next[1], v);
    if constexpr (Silu) unpack16(next[2], next[3], u);
    item += step;
    row += rows;
    group += groups;
    if (group >= a.groups) {
      group -= a.groups;
      ++row;
    }
    fetch();
    if constexpr (Silu) gate16(v, u);
    const GroupScale g(top_of_group(v));
    if (mine) *reinterpret_cast<uint4*>(a.codes + to) = codes16(v, g.inverse);
    if (have && sub == 0) a.scales[at] = g.scale;
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
  const int64_t blocks = (a.items + kPerBlock - 1) / kPerBlock, most = lin::kSms * 8;
  const int grid = static_cast<int>(blocks < most ? blocks : most);
  if (silu) quantize_kernel<true><<<grid, kThreads, 0, stream>>>(a);
  else quantize_kernel<false><<<grid, kThreads, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
