// Weighted sum of each token's results: out[t] = sum_j w[t, j] * partial[position[t, j]] (+ residual), in fp32 in the order of j.
//
// Eight columns a thread; a token's rows are requested together, up to eight at a time. Bound by memory, every row is read once: 16384 tokens of 8
// rows of 2048 in 100 us, 6.0 TB/s. The grid is what runs at once, each thread goes from piece to piece: with 64 CTAs for an SM it took 109 us. (Four
// columns a thread and more of them: 129. The next piece's positions ahead, for which there are no registers: 109.)
#include "linear.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kThreads = 256, kAtOnce = 8, kResident = 3;   // CTAs of an SM, by their registers

struct CombineArgs {
  const uint4 *partial, *residual;
  uint4* out;
  const int32_t* positions;
  const float* weights;
  uint32_t* status;
  int64_t rows, items;
  int top, vecs;                             // pieces of eight columns in a row
};

__global__ void __launch_bounds__(kThreads) combine_kernel(const CombineArgs a) {
  const int at_first = blockIdx.x * kThreads + threadIdx.x, step = gridDim.x * kThreads;
  int64_t i = at_first, t = at_first / a.vecs;
  int v = at_first % a.vecs;
  const int tokens = step / a.vecs, vecs = step - tokens * a.vecs;
  for (; i < a.items; i += step, t += tokens, v += vecs) {
    if (v >= a.vecs) {
      v -= a.vecs;
      ++t;
    }
    float2 sum[4] = {};
    for (int j0 = 0; j0 < a.top; j0 += kAtOnce) {
      uint4 row[kAtOnce];
      float w[kAtOnce];
      bool have[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        have[j] = false;
        if (j0 + j < a.top) {
          const int64_t p = __ldg(a.positions + t * a.top + j0 + j);
          have[j] = p >= 0 && p < a.rows;
          if (p >= a.rows) report(a.status, kBadPosition, static_cast<uint32_t>(t));
          if (have[j]) {
            w[j] = __ldg(a.weights + t * a.top + j0 + j);
            row[j] = __ldcs(a.partial + p * a.vecs + v);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (have[j]) {
          const float2 ww = make_float2(w[j], w[j]);
          sum[0] = fma2(ww, bf16x2(row[j].x), sum[0]);
          sum[1] = fma2(ww, bf16x2(row[j].y), sum[1]);
          sum[2] = fma2(ww, bf16x2(row[j].z), sum[2]);
          sum[3] = fma2(ww, bf16x2(row[j].w), sum[3]);
        }
    }
    if (a.residual) {
      const uint4 r = __ldg(a.residual + i);
      const float2 one = make_float2(1.0f, 1.0f);
      sum[0] = fma2(one, bf16x2(r.x), sum[0]);
      sum[1] = fma2(one, bf16x2(r.y), sum[1]);
      sum[2] = fma2(one, bf16x2(r.z), sum[2]);
      sum[3] = fma2(one, bf16x2(r.w), sum[3]);
    }
    a.out[i] = make_uint4(pack_bf16x2(sum[0].x, sum[0].y), pack_bf16x2(sum[1].x, sum[1].y), pack_bf16x2(sum[2].x, sum[2].y), pack_bf16x2(sum[3].x, sum[3].y));
  }
}

}  // namespace
}  // namespace mono

extern "C" int mono_lin_combine(const void* partial, int64_t rows, const int32_t* positions, const float* weights, int64_t tokens, int top, int cols,
                                const void* residual, void* out, uint32_t* status, mono_lin_stream_t stream) {
  using namespace mono;
  if (rows < 0 || tokens < 0 || top < 1 || top > MONO_LIN_MAX_TOP || cols < 8 || cols % 8 || cols > (1 << 24)) return MONO_LIN_BAD_SIZE;
  if (tokens == 0) return 0;
  if ((!partial && rows > 0) || !positions || !weights || !out || !status) return MONO_LIN_NULL;
  if ((reinterpret_cast<uintptr_t>(partial) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(out)) & 15) return MONO_LIN_ALIGNMENT;
  CombineArgs a{static_cast<const uint4*>(partial), static_cast<const uint4*>(residual), static_cast<uint4*>(out), positions, weights, status, rows,
                tokens * (cols / 8), top, cols / 8};
  const int64_t blocks = (a.items + kThreads - 1) / kThreads, most = lin::kSms * kResident;
  combine_kernel<<<static_cast<int>(blocks < most ? blocks : most), kThreads, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
