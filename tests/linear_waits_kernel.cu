// Waits of csrc/linear/waits.cuh on a barrier that nobody arrives at, with a short limit: three warps by the three forms, then 200 waits more each.
#include <cuda_runtime.h>
#include "waits.cuh"

using namespace mono;
using namespace mono::lin;

__global__ void waits_kernel(uint32_t* status, uint64_t* ns, uint64_t limit) {
  __shared__ uint64_t bars[2];
  __shared__ uint32_t stop;
  if (threadIdx.x == 0) {
    mbar_init(&bars[0], 1);
    mbar_init(&bars[1], 1);
    mbar_init_fence();
    stop = 0;
  }
  __syncthreads();
  const Waits waits{&stop, status, limit};
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint64_t t0 = globaltimer_ns();
  uint64_t t1 = t0;
  for (int i = 0; i <= 200; ++i) {
    if (warp == 0) {
      waits.wait(&bars[0], 0, &bars[1], 0);
    } else if (warp == 1) {
      waits.wait_warp(&bars[0], 0);
    } else {
      if (lane == 0) waits.wait_lane(&bars[1], 0);
      __syncwarp();
    }
    if (i == 0) t1 = globaltimer_ns();
  }
  const uint64_t t2 = globaltimer_ns();
  if (lane == 0) {
    ns[(blockIdx.x * 3 + warp) * 2] = t1 - t0;
    ns[(blockIdx.x * 3 + warp) * 2 + 1] = t2 - t1;
  }
}

extern "C" int waits_launch(uint32_t* status, uint64_t* ns, int ctas, uint64_t limit) {
  waits_kernel<<<ctas, 96>>>(status, ns, limit);
  const cudaError_t e = cudaGetLastError();
  return static_cast<int>(e != cudaSuccess ? e : cudaDeviceSynchronize());
}
