// Block-FP8 products for many rows: tiles of 256 rows of x and 256 rows of the weight on clusters of two CTAs.
//
//   y[i, n] = sum_g sx[i, g] sw[n / 128, g] sum_{k in g} qx[i, k] qw[n, k]
//
// The two CTAs' tensor cores work as one (cta_group::2): each CTA holds 128 rows of x and half of the tile's weight rows, and its
// tensor memory the sums of its rows with all 256. A sum over a group of 128 goes to one of two buffers, from where eight warps
// add it, times its scales, to sums in registers: a thread has one row of x (one scale) and 128 rows of the weight (one scale, or
// the gate's and the other half's). Twelve warps a CTA:
//   0     requests weights, and rows of x where they lie in order
//   1     in the first CTA: issues the products of both
//   2, 3  bring rows of x that lie anywhere (tokens), by cp.async with the 128-byte swizzle written by hand
//   4-11  read the sums; write the results, through shared memory in whole lines
// With the gated activation a tile is 128 rows of the gate's half (the first CTA's) and the matching 128 of the other one.
//
// Why pairs: a product of 128 x 256 x 128 on one SM takes 512 cycles of its tensor core and moves 48 KB into shared memory and 48 KB
// out of it, 768 cycles at its 128 bytes a cycle; in pairs each SM has half of the weight's bytes, and both rates meet.
#include "linear.cuh"
#include "../pair_sm100.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kThreads = 384, kLoaders = 64, kReaders = 8, kRows = 128, kTile = 256;
constexpr int kHalf = kRows * kGroup, kStage = 2 * kHalf, kStages = 5, kSums = 2;
constexpr int kStaging = 4096;               // of a reader: 32 rows x 64 columns of bf16
// Registers of a thread: at launch, of the first four warps, of the readers. The readers' share comes from what the others give back.
constexpr int kRegs = 168, kRegsOther = 56, kRegsReader = 224;
static_assert(4 * kRegsOther + 8 * kRegsReader <= 12 * kRegs, "a wait for registers that are not there has no end");

struct Control {
  uint64_t full[kStages], gathered[kStages], empty[kStages], d_full[kSums], d_empty[kSums];
  uint32_t tmem, stop;
  int sums[32];
  uint32_t top[2][kRows];
  int source[kRows];
  int first[MONO_LIN_MAX_EXPERTS + 1];
};
constexpr int kSmem = kStages * kStage + kReaders * kStaging + static_cast<int>(sizeof(Control)) + 1024;
static_assert(kSmem <= 232448, "shared memory of an SM");

__device__ __forceinline__ void tma_weight_pair(const CUtensorMap* m, int k, int row, int expert, uint32_t dst, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(k), "r"(row), "r"(expert), "r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// What the peer's tensor core is to read is released to the cluster.
__device__ __forceinline__ void arrive_release_cluster(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// 64 columns of a row as bf16 into the reader's 4 KB, 16 bytes at a time at places that spread over the banks.
__device__ __forceinline__ void stage_row(uint32_t at, int lane, const float2* v) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t w[4] = {pack_bf16x2(v[4 * c].x, v[4 * c].y), pack_bf16x2(v[4 * c + 1].x, v[4 * c + 1].y), pack_bf16x2(v[4 * c + 2].x, v[4 * c + 2].y),
                           pack_bf16x2(v[4 * c + 3].x, v[4 * c + 3].y)};
    st_shared_128(at + lane * 128 + ((c ^ (lane & 7)) << 4), w);
  }
}

// 64 columns from `col` of row `row`, one row a lane; `have`: the lane has a row. The warp works together.
__device__ __forceinline__ void write_out(const Product& p, uint32_t at, int lane, int64_t row0, int rows, int col, float2* v) {
  const int64_t row = row0 + lane;
  const bool have = lane < rows;
  if (p.residual && have) {
    const __nv_bfloat16* res = p.residual + row * p.n + col;
    if (p.vec && col + 64 <= p.n) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(res) + c);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = bf16x2(w[i]);
          v[4 * c + i].x += f.x;
          v[4 * c + i].y += f.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (col + 2 * i < p.n) v[i].x += __bfloat162float(res[2 * i]);
        if (col + 2 * i + 1 < p.n) v[i].y += __bfloat162float(res[2 * i + 1]);
      }
    }
  }
  if (p.fp32) {
    if (!have) return;
    float* out = static_cast<float*>(p.out) + row * p.n + col;
    if (p.vec && col + 64 <= p.n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) reinterpret_cast<float4*>(out)[i] = make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (col + 2 * i < p.n) out[2 * i] = v[i].x;
        if (col + 2 * i + 1 < p.n) out[2 * i + 1] = v[i].y;
      }
    }
    return;
  }
  if (p.vec) {
    stage_row(at, lane, v);
    __syncwarp();
    const int c = lane & 7;
    if (col + c * 8 < p.n) {                 // n is a multiple of 8 here
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + col + c * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        if (r < rows) {
          uint4 w;
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at + r * 128 + ((c ^ (r & 7)) << 4)) : "memory");
          *reinterpret_cast<uint4*>(out + (row0 + r) * p.n) = w;
        }
      }
    }
    __syncwarp();
  } else if (have) {
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + row * p.n + col;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (col + 2 * i < p.n) out[2 * i] = __float2bfloat16_rn(v[i].x);
      if (col + 2 * i + 1 < p.n) out[2 * i + 1] = __float2bfloat16_rn(v[i].y);
    }
  }
}

template <bool Gate>
__global__ void __launch_bounds__(kThreads, 1) many_kernel(const __grid_constant__ CUtensorMap weight, const __grid_constant__ CUtensorMap rows,
                                                           const __grid_constant__ Product p) {
  extern __shared__ uint8_t raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Control& C = *reinterpret_cast<Control*>(stages + kStages * kStage + kReaders * kStaging);
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const Waits waits{&C.stop, p.status};
  const bool gather = p.tokens != nullptr;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&C.full[i], gather ? 2 : 1);  // the first CTA's bytes, and that the second has gathered its rows
      mbar_init(&C.gathered[i], kLoaders);
      mbar_init(&C.empty[i], 1);
    }
    for (int i = 0; i < kSums; ++i) {
      mbar_init(&C.d_full[i], 1);
      mbar_init(&C.d_empty[i], 2 * kReaders);
    }
    mbar_init_fence();
    C.stop = 0;
  }
  if (warp == 1) {
    tmem_alloc_pair(&C.tmem, 512);
    tmem_relinquish_pair();
  }
  if (p.offsets) Division<kTile>::fill(p, C.first, C.sums, kThreads);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                        // the peer's barriers are there before anything signals them
  tc_fence_after();

  const Division<kTile> division(p, C.first);
  const int64_t units = division.units(), step = gridDim.x / 2, u0 = blockIdx.x / 2;
  const uint32_t base = smem_u32(stages);
  auto leaders = [&](uint64_t* bar) { return map_to_cta(smem_u32(bar), 0); };

  if (warp < 4) {
    reg_dec<kRegsOther>();
    if (warp == 0) {
      if (lane == 0) {
        uint32_t n = 0;
        for (int64_t u = u0; u < units; u += step) {
          const Run r = division.unit(u);
          const int wrow = Gate ? (rank ? p.n / 2 : 0) + r.col * kRows : r.col * kTile + static_cast<int>(rank) * kRows;
          const int64_t xrow = r.row + rank * kRows;
          for (int g = 0; g < p.groups; ++g, ++n) {
            const uint32_t s = n % kStages, at = base + s * kStage, bar = leaders(&C.full[s]);
            waits.wait_lane(&C.empty[s], (n / kStages & 1) ^ 1);
            if (rank == 0) mbar_arrive_expect_tx(&C.full[s], gather ? 2 * kHalf : 4 * kHalf);
            tma_weight_pair(&weight, g * kGroup, wrow, r.expert, at + kHalf, bar);
            if (!gather) tma_load_2d_pair(&rows, g * kGroup, static_cast<uint32_t>(xrow), stages + s * kStage, bar);
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      if (rank == 0) {
        constexpr uint32_t idesc = umma_idesc_e4m3_f32(2 * kRows, kTile);
        uint32_t n = 0;
        for (int64_t u = u0; u < units; u += step)
          for (int g = 0; g < p.groups; ++g, ++n) {
            const uint32_t s = n % kStages, b = n % kSums;
            waits.wait_warp(&C.d_empty[b], (n / kSums & 1) ^ 1);
            waits.wait_warp(&C.full[s], n / kStages & 1);
            if (gather) {
              waits.wait_warp(&C.gathered[s], n / kStages & 1);
              fence_proxy_async_smem();
            }
            tc_fence_after();
            if (elect_one_sync()) {
              const uint64_t x = umma_desc_sw128(base + s * kStage), w = umma_desc_sw128(base + s * kStage + kHalf);
#pragma unroll
              for (int i = 0; i < 4; ++i) umma_f8_pair(C.tmem + b * kTile, x + i * 2, w + i * 2, idesc, i > 0);
              umma_commit_pair(&C.empty[s]);
              umma_commit_pair(&C.d_full[b]);
            }
            __syncwarp();
          }
      } else if (gather) {
        uint32_t n = 0;
        for (int64_t u = u0; u < units; u += step)
          for (int g = 0; g < p.groups; ++g, ++n) {
            waits.wait_warp(&C.gathered[n % kStages], n / kStages & 1);
            fence_proxy_async_smem();
            if (lane == 0) arrive_release_cluster(leaders(&C.full[n % kStages]));
            __syncwarp();
          }
      }
    } else if (gather) {
      const int t = threadIdx.x - 64, chunk = t & 7, r0 = t >> 3;
      constexpr int kEach = kRows / 8;
      uint32_t n = 0;
      for (int64_t u = u0; u < units; u += step) {
        const Run r = division.unit(u);
        int* src = C.source + r0;            // rows of x, -1: none; eight lanes of the warp share 16 of them
        __syncwarp();
#pragma unroll
        for (int i = chunk; i < kEach; i += 8) {
          const int at = static_cast<int>(rank) * kRows + r0 + 8 * i;
          src[8 * i] = at < r.rows ? static_cast<int>(source_row(p, r.row + at)) : -1;
        }
        __syncwarp();
        for (int g = 0; g < p.groups; ++g, ++n) {
          const uint32_t s = n % kStages;
          waits.wait(&C.empty[s], (n / kStages & 1) ^ 1);
          const int k = g * kGroup + chunk * 16;
          const uint32_t dst = base + s * kStage + r0 * 128 + ((chunk ^ (r0 & 7)) << 4);
#pragma unroll 4
          for (int i = 0; i < kEach; ++i) {
            const int row = src[8 * i];
            const bool have = row >= 0 && k < p.k;
            cp_async16_or_zero(dst + i * 1024, have ? p.x + static_cast<int64_t>(row) * p.k + k : p.x, have ? 16 : 0);
          }
          cp_async_arrive_noinc(&C.gathered[s]);
        }
      }
      cp_async_commit();
      cp_async_wait<0>();                    // of a launch that gave up, too
    }
  } else {
    reg_inc<kRegsReader>();
    wait_for_launch_before();
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t staging = base + kStages * kStage + (warp - 4) * kStaging;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t column = Gate ? half * 64 : half * 128, other = Gate ? 128 : 64;   // first 64 columns of this warp, and how far behind the others lie
    uint32_t n = 0;
    for (int64_t u = u0; u < units; u += step) {
      const Run r = division.unit(u);
      const int in = static_cast<int>(rank) * kRows + quarter * 32, mine = max(0, min(32, r.rows - in));   // rows of this warp
      const int64_t row0 = r.row + in;
      const int64_t src = lane < mine ? source_row(p, row0 + lane) : -1;
      const float* xs = p.xs + (src < 0 ? 0 : src) * p.groups;
      const int block = Gate ? r.col : min(r.col * 2 + half, p.blocks - 1);
      const float* ws = p.ws + (static_cast<int64_t>(r.expert) * p.blocks + block) * p.groups;
      const int64_t gate_step = static_cast<int64_t>(p.blocks / 2) * p.groups;
      float2 acc[2][32] = {};
      // scales two groups ahead
      float x0 = 0.0f, x1 = 0.0f, w0 = 0.0f, w1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
      if (mine > 0) {
        const int g1 = min(1, p.groups - 1);
        x0 = __ldg(xs);
        x1 = __ldg(xs + g1);
        w0 = __ldg(ws);
        w1 = __ldg(ws + g1);
        if constexpr (Gate) {
          v0 = __ldg(ws + gate_step);
          v1 = __ldg(ws + gate_step + g1);
        }
      }
      for (int g = 0; g < p.groups; ++g, ++n) {
        const uint32_t b = n % kSums;
        if (mine > 0) {
          const float sa = x0 * w0, sb = Gate ? x0 * v0 : sa;
          const int g2 = min(g + 2, p.groups - 1);
          x0 = x1;
          w0 = w1;
          x1 = __ldg(xs + g2);
          w1 = __ldg(ws + g2);
          if constexpr (Gate) {
            v0 = v1;
            v1 = __ldg(ws + gate_step + g2);
          }
          waits.wait(&C.d_full[b], n / kSums & 1);
          tc_fence_after();
          const uint32_t d = C.tmem + b * kTile + lanes + column;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[64];
            tmem_ld64(d + h * other, v);
            tmem_ld_wait();
            if (h == 1) {                    // read out: the next product may have the buffer
              tc_fence_before();
              __syncwarp();
              if (lane == 0) { if (rank) mbar_arrive_cluster(leaders(&C.d_empty[b])); else mbar_arrive(&C.d_empty[b]); }
            }
            const float2 sc = h ? make_float2(sb, sb) : make_float2(sa, sa);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[h][i] = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sc, acc[h][i]);
          }
        } else {
          waits.wait(&C.d_full[b], n / kSums & 1);
          if (lane == 0) { if (rank) mbar_arrive_cluster(leaders(&C.d_empty[b])); else mbar_arrive(&C.d_empty[b]); }
        }
      }
      if constexpr (Gate) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          acc[0][i].x = gated(acc[0][i].x, acc[1][i].x);
          acc[0][i].y = gated(acc[0][i].y, acc[1][i].y);
          m = max(m, max(magnitude(acc[0][i].x), magnitude(acc[0][i].y)));
        }
        C.top[half][quarter * 32 + lane] = m;
        named_bar_sync(2 + quarter, 64);     // the two warps that share these rows
        const GroupScale gs(max(m, C.top[half ^ 1][quarter * 32 + lane]));
        if (lane < mine) {
          uint4* out = reinterpret_cast<uint4*>(p.codes + (row0 + lane) * (p.n / 2) + r.col * kRows + half * 64);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 a = acc[0][8 * c + 2 * i], e = acc[0][8 * c + 2 * i + 1];
              w[i] = pack_e4m3x4(a.x * gs.inverse, a.y * gs.inverse, e.x * gs.inverse, e.y * gs.inverse);
            }
            out[c] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (half == 0) p.scales[(row0 + lane) * (p.n / 2 / kGroup) + r.col] = gs.scale;
        }
        named_bar_sync(2 + quarter, 64);     // both have read the magnitudes
      } else if (mine > 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = r.col * kTile + half * 128 + h * 64;
          if (col < p.n) write_out(p, staging, lane, row0, mine, col, acc[h]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                        // nothing of the peer is on its way to this CTA, or reads its memory
  tc_fence_after();
  if (C.stop) settle();
  if (warp == 1) tmem_dealloc_pair(C.tmem, 512);
}

template <bool Gate>
int launch(const Product& p, const CUtensorMap& weight, const CUtensorMap& x, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(many_kernel<Gate>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(kSms);
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = kSmem;
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&c, many_kernel<Gate>, weight, x, p));
}

}  // namespace

namespace lin {
int launch_many(const Product& p, const CUtensorMap& weight, const CUtensorMap& x, cudaStream_t stream) {
  return p.codes ? launch<true>(p, weight, x, stream) : launch<false>(p, weight, x, stream);
}
}  // namespace lin
}  // namespace mono
