// Division of a batch among experts: a stable counting sort of the (token, place) slots by expert.
//
// One cluster of up to eight CTAs, so that one launch does it without a grid-wide barrier or memory kept between calls. Each warp has
// a run of slots: it counts them into a row of its own of the CTA's table (lanes with the same expert find one another, the first
// of them adds), the table is summed over warps, CTAs (distributed shared memory) and experts, and the warp walks its run again
// with the cursors that it finds in its row. The order depends on nothing but the ids.
#include "linear.cuh"
#include "../pair_sm100.cuh"

namespace mono {
namespace {

using namespace lin;

struct PlanArgs {
  const void* ids;
  int32_t *offsets, *tokens, *positions;
  uint32_t* status;
  int64_t slots;
  int top, experts;
};

__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename Id>
__global__ void __launch_bounds__(1024, 1) plan_kernel(const PlanArgs a) {
  extern __shared__ uint32_t table[];        // [warps][experts], then [experts] of the CTA
  __shared__ uint32_t sums[32];
  const int E = a.experts, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = gridDim.x;
  const uint32_t rank = blockIdx.x;          // the grid is one cluster
  uint32_t *mine = table + warp * E, *total = table + warps * E;
  const int64_t parts = static_cast<int64_t>(ctas) * warps, part = static_cast<int64_t>(rank) * warps + warp;
  const int64_t each = ((a.slots + parts - 1) / parts + 31) / 32 * 32;
  const int64_t lo = min(part * each, a.slots), hi = min(lo + each, a.slots);
  const Id* ids = static_cast<const Id*>(a.ids);
  for (int i = threadIdx.x; i < warps * E; i += blockDim.x) table[i] = 0;
  __syncthreads();

  // Expert of slot i, -1 where there is none here.
  auto expert = [&](int64_t i, bool tell) {
    if (i >= hi) return -1;
    const Id id = __ldg(ids + i);
    if (id >= E && tell) report(a.status, kBadExpert, static_cast<uint32_t>(i));
    return id < 0 || id >= E ? -1 : static_cast<int>(id);
  };
  for (int64_t i0 = lo; i0 < hi; i0 += 32) {
    const int e = expert(i0 + lane, true);
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {       // of the CTA, and what lies in its lower warps
    uint32_t s = 0;
    for (int w = 0; w < warps; ++w) {
      const uint32_t n = table[w * E + e];
      table[w * E + e] = s;
      s += n;
    }
    total[e] = s;
  }
  __syncthreads();
  cluster_sync_all();
  uint32_t base = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    uint32_t all = 0, lower = 0;
    if (e < E)
      for (int c = 0; c < ctas; ++c) {
        const uint32_t n = ld_cluster(map_to_cta(smem_u32(total + e), c));
        if (c < static_cast<int>(rank)) lower += n;
        all += n;
      }
    uint32_t s = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d) s += o;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    uint32_t first = base + s - all;
    for (int w = 0; w < warp; ++w) first += sums[w];
    for (int w = 0; w < warps; ++w) base += sums[w];
    if (e < E) {
      if (rank == 0) a.offsets[e] = static_cast<int32_t>(first);
      for (int w = 0; w < warps; ++w) table[w * E + e] += first + lower;
    }
    __syncthreads();
  }
  if (rank == 0 && threadIdx.x == 0) a.offsets[E] = static_cast<int32_t>(base);
  for (int64_t i0 = lo; i0 < hi; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = expert(i, false);
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    const uint32_t row = e < 0 ? 0 : mine[e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
    if (i < hi) {
      a.positions[i] = e < 0 ? -1 : static_cast<int32_t>(row);
      if (e >= 0) a.tokens[row] = static_cast<int32_t>(i / a.top);
    }
  }
  for (int64_t i = base + static_cast<int64_t>(rank) * blockDim.x + threadIdx.x; i < a.slots; i += static_cast<int64_t>(ctas) * blockDim.x) a.tokens[i] = -1;
  __syncthreads();
  cluster_sync_all();                        // the others have read this CTA's sums
}

// Slots from which eight CTAs are faster than one.
constexpr int64_t kOneCta = 4096;

template <typename Id>
int launch(const PlanArgs& a, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  constexpr int kMost = (33 * MONO_LIN_MAX_EXPERTS) * 4;
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(plan_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  const int ctas = a.slots <= kOneCta ? 1 : 8;
  const int64_t per = (a.slots + ctas - 1) / ctas;
  const int warps = per >= 1024 ? 32 : per <= 32 * 4 ? 4 : static_cast<int>((per + 31) / 32);
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(ctas);
  c.blockDim = dim3(warps * 32);
  c.dynamicSmemBytes = static_cast<size_t>(warps + 1) * a.experts * 4;
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&c, plan_kernel<Id>, a));
}

}  // namespace
}  // namespace mono

extern "C" int mono_lin_plan(const void* ids, int ids_64, int64_t tokens, int top, int experts, int32_t* offsets, int32_t* tokens_out, int32_t* positions,
                             uint32_t* status, mono_lin_stream_t stream) {
  using namespace mono;
  if (tokens < 0 || top < 1 || top > MONO_LIN_MAX_TOP || experts < 1 || experts > MONO_LIN_MAX_EXPERTS || tokens > INT32_MAX / top) return MONO_LIN_BAD_SIZE;
  if (!offsets || !status || (tokens > 0 && (!ids || !tokens_out || !positions))) return MONO_LIN_NULL;
  const PlanArgs a{ids, offsets, tokens_out, positions, status, tokens * top, top, experts};
  return ids_64 ? launch<int64_t>(a, stream) : launch<int32_t>(a, stream);
}
