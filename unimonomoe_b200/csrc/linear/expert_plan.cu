// Division of a batch among experts: a stable counting sort of the (token, place) slots by expert.
//
// One cluster of up to sixteen CTAs, so that one launch does it without a grid-wide barrier or memory kept between calls. Each warp has
// a run of slots: it counts them into a row of its own of the CTA's table, the table is summed over warps, CTAs (distributed shared memory)
// and experts, and the warp walks its run again with the cursors that it finds in its row. Lanes with the same expert find one another
// by the bits of its number, a vote for each (the instruction made for that, match.any, takes an SM 75 cycles: 41 us for 131072 slots).
// The order depends on nothing but the ids.
//
// Bound by latency: ids, counts, sums over warps and CTAs, ids again and results follow one another. 8 slots of 256 experts take 3.0-3.2 us in a graph,
// 131072 of 128 experts 12.0, where ids and results alone would take 0.3.
#include "linear.cuh"
#include "../pair_sm100.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kSteps = 8, kCtas = 16;

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
  extern __shared__ uint32_t table[];        // [warps][experts], then [experts] of the CTA and [experts] of its first rows
  __shared__ uint32_t sums[32];
  const int E = a.experts, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = gridDim.x;
  const uint32_t rank = blockIdx.x;          // the grid is one cluster
  uint32_t *mine = table + warp * E, *total = table + warps * E, *start = total + E;
  const int bits = 32 - __clz(E - 1);         // of an expert's number
  const int64_t parts = static_cast<int64_t>(ctas) * warps, part = static_cast<int64_t>(rank) * warps + warp;
  const int64_t each = ((a.slots + parts - 1) / parts + 31) / 32 * 32;
  const int64_t lo = min(part * each, a.slots), hi = min(lo + each, a.slots);
  const Id* ids = static_cast<const Id*>(a.ids);
  for (int i = threadIdx.x; i < warps * E; i += blockDim.x) table[i] = 0;
  __syncthreads();

  // Eight steps of 32 slots from i0 on: each lane's experts, -1 where there is none here. The ids are requested together.
  auto take = [&](int64_t i0, int (&e)[kSteps], bool tell) {
    Id id[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) id[k] = i0 + 32 * k + lane < hi ? __ldg(ids + i0 + 32 * k + lane) : -1;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      if (id[k] >= E && tell) report(a.status, kBadExpert, static_cast<uint32_t>(i0 + 32 * k + lane));
      e[k] = id[k] < 0 || id[k] >= E ? -1 : static_cast<int>(id[k]);
    }
  };
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kSteps) {
    int e[kSteps];
    take(i0, e, true);
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
      if (e[k] >= 0) atomicAdd(mine + e[k], 1u);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {       // of the CTA, and what lies in its lower warps
    uint32_t s = 0;
    for (int w0 = 0; w0 < warps; w0 += 4) {  // warps are a multiple of four
      uint32_t n[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) n[w] = table[(w0 + w) * E + e];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        table[(w0 + w) * E + e] = s;
        s += n[w];
      }
    }
    total[e] = s;
  }
  __syncthreads();
  if (ctas > 1) cluster_sync_all();
  uint32_t base = 0;                         // rows of the experts before
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    uint32_t all = 0, lower = 0;
    if (e < E) {
      if (ctas == 1) {
        all = total[e];
      } else {
        uint32_t n[kCtas];
#pragma unroll
        for (int c = 0; c < kCtas; ++c) n[c] = c < ctas ? ld_cluster(map_to_cta(smem_u32(total + e), c)) : 0;
#pragma unroll
        for (int c = 0; c < kCtas; ++c) {
          if (c < static_cast<int>(rank)) lower += n[c];
          all += n[c];
        }
      }
    }
    uint32_t s = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d) s += o;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    const uint32_t of_warp = lane < warps ? sums[lane] : 0;
    uint32_t before = of_warp;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, before, d);
      if (lane >= d) before += o;
    }
    const uint32_t first = base + __shfl_sync(0xFFFFFFFFu, before - of_warp, warp) + s - all;
    base += __shfl_sync(0xFFFFFFFFu, before, 31);
    if (e < E) {
      if (rank == 0) a.offsets[e] = static_cast<int32_t>(first);
      start[e] = first + lower;
    }
    __syncthreads();
  }
  if (rank == 0 && threadIdx.x == 0) a.offsets[E] = static_cast<int32_t>(base);
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kSteps) {
    int e[kSteps];
    take(i0, e, false);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      if (i0 + 32 * k >= hi) break;
      const int64_t i = i0 + 32 * k + lane;
      uint32_t same = __ballot_sync(0xFFFFFFFFu, e[k] >= 0);         // lanes with the same expert
      for (int b = 0; b < bits; ++b) {
        const uint32_t set = __ballot_sync(0xFFFFFFFFu, e[k] >> b & 1);
        same &= e[k] >> b & 1 ? set : ~set;
      }
      const uint32_t row = e[k] < 0 ? 0 : start[e[k]] + mine[e[k]] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (e[k] >= 0 && lane == __ffs(same) - 1) mine[e[k]] += __popc(same);
      __syncwarp();
      if (i < hi) {
        a.positions[i] = e[k] < 0 ? -1 : static_cast<int32_t>(row);
        if (e[k] >= 0) a.tokens[row] = static_cast<int32_t>(static_cast<uint32_t>(i) / static_cast<uint32_t>(a.top));
      }
    }
  }
  for (int64_t i = base + static_cast<int64_t>(rank) * blockDim.x + threadIdx.x; i < a.slots; i += static_cast<int64_t>(ctas) * blockDim.x) a.tokens[i] = -1;
  __syncthreads();
  if (ctas > 1) cluster_sync_all();          // the others have read this CTA's sums
}

// Slots up to which one CTA is as fast as sixteen, which wait for one another twice: 512 slots 3.6 us and 4.8, 1024 4.4 and 5.1, 2048 5.5
// and 5.2, 8192 10.7 and 5.3.
constexpr int64_t kOneCta = 1024;

template <typename Id>
int launch(const PlanArgs& a, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  constexpr int kMost = (34 * MONO_LIN_MAX_EXPERTS) * 4;
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(plan_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(plan_kernel<Id>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  // Sixteen where the tables of two fit an SM: up to 16 warps two CTAs run on one, so that a processing cluster takes them with eight SMs free. 32 warps fill an
  // SM with their registers, and sixteen of those need sixteen SMs of one processing cluster; of eight clusters that share 148 SMs the largest has more.
  const int ctas = a.slots <= kOneCta ? 1 : 34 * a.experts * 4 <= 100 * 1024 ? kCtas : kCtas / 2;
  const int64_t per = (a.slots + ctas - 1) / ctas;
  // More warps are more rows of the table to sum: with 32 of them from 1024 slots of a CTA on 16384 slots took 7.6 us instead of 6.2, 65536 9.7
  // instead of 9.3; with 16 throughout 131072 take 13.5 instead of 12.0.
  const int warps = per >= 8192 ? 32 : per >= 1024 ? 16 : static_cast<int>((per + 255) / 256) * 4 + (per == 0 ? 4 : 0);
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(ctas);
  c.blockDim = dim3(warps * 32);
  c.dynamicSmemBytes = static_cast<size_t>(warps + 2) * a.experts * 4;
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
