// Block-FP8 products for few rows: D^T = W X^T, with 128 rows of the weight as the rows of the tensor-core product and up to Tile
// rows of x as its columns, so that the weight is read once and nothing of the product is padding beyond 16 rows of x.
//
//   y[i, n] = sum_g sx[i, g] sw[n / 128, g] sum_{k in g} qx[i, k] qw[n, k]
//
// The sum over a group of 128 is made by the tensor core (e4m3, fp32 sums in tensor memory), the scales are applied to it in
// registers: a thread has one row of the weight and some rows of x. Twelve warps, one CTA to an SM:
//   0     requests the weight, [128 rows x 128] at a time (with the gated activation the gate's and the other half's 128 rows)
//   1     issues the products, four to a group
//   2, 3  bring the rows of x, by cp.async with the 128-byte swizzle written by hand: they may lie anywhere (tokens)
//   4-11  read the sums, four warps for the 128 rows, twice for the halves of the rows of x
// The groups of K may be divided among the CTAs of a cluster, whose sums are then added in the order of the CTAs through
// distributed shared memory; the result does not depend on timing. Without that a CTA goes from unit to unit, and the weight's
// requests run ahead across them.
#include "linear.cuh"
#include "../pair_sm100.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kThreads = 384, kLoaders = 64, kReaders = 256, kRows = 128;
constexpr int kStageLimit = 200 * 1024;

template <int Tile, bool Gate>
struct Shape {
  static constexpr int Halves = Gate ? 2 : 1;
  static constexpr int Weight = Halves * kRows * kGroup, Stage = Weight + Tile * kGroup;
  static constexpr int Stages = kStageLimit / Stage < 12 ? kStageLimit / Stage : 12;
  static constexpr int Cols = Halves * Tile;                  // of a sum in tensor memory
  static constexpr int Sums = Cols * 4 <= 512 ? 4 : 2;
  static constexpr int Tmem = Cols * Sums < 32 ? 32 : Cols * Sums;
  static constexpr int Mine = Tile / 2;                       // rows of x of a thread
  static constexpr int Add = Halves * Tile * kRows * 4;       // bytes of the sums that a CTA of a cluster gives to the others
  static_assert(Add <= Stages * Stage, "they lie where the stages were");
  static_assert((Tmem & (Tmem - 1)) == 0 && Tmem <= 512, "columns of tensor memory");
};

template <int Tile>
struct Control {
  uint64_t w_full[12], x_full[12], empty[12], d_full[4], d_empty[4];
  uint32_t tmem, stop;
  int sums[32];
  uint32_t top[2][4][Tile / 2];                               // largest magnitudes, by half and warp
  alignas(16) float scale[8][2][2][Tile / 2];                             // by warp: scales of this group and the next, of both halves of a gated product
  int first[MONO_LIN_MAX_EXPERTS + 1];
};

template <int Tile, bool Gate>
constexpr int smem_bytes() { return Shape<Tile, Gate>::Stages * Shape<Tile, Gate>::Stage + static_cast<int>(sizeof(Control<Tile>)) + 1024; }

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[N]) {
  static_assert(N == 8 || N == 16, "columns at a time");
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(t) : "memory");
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(t) : "memory");
}
// 16 bytes, of which `bytes` (0 or 16) come from `src`, zeros for the rest.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_weight(const CUtensorMap* m, int k, int row, int expert, uint32_t dst, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(k), "r"(row), "r"(expert), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void store_code(uint8_t* p, float x) { *p = static_cast<uint8_t>(pack_e4m3x4(x, 0.0f, 0.0f, 0.0f)); }

// One value of the result, to its type.
__device__ __forceinline__ void store(const Product& p, int64_t row, int n, float v) {
  const int64_t at = row * p.n + n;
  if (p.residual) v += __bfloat162float(p.residual[at]);
  if (p.fp32) static_cast<float*>(p.out)[at] = v;
  else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
}

template <int Tile, bool Gate>
__global__ void __launch_bounds__(kThreads, 1) few_kernel(const __grid_constant__ CUtensorMap weight, const __grid_constant__ Product p, const int split) {
  using S = Shape<Tile, Gate>;
  extern __shared__ uint8_t raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Control<Tile>& C = *reinterpret_cast<Control<Tile>*>(stages + S::Stages * S::Stage);
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = split > 1 ? cluster_ctarank() : 0;
  const Waits waits{&C.stop, p.status};

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::Stages; ++i) {
      mbar_init(&C.w_full[i], 1);
      mbar_init(&C.x_full[i], kLoaders);
      mbar_init(&C.empty[i], 1);
    }
    for (int i = 0; i < S::Sums; ++i) {
      mbar_init(&C.d_full[i], 1);
      mbar_init(&C.d_empty[i], kReaders / 32);
    }
    mbar_init_fence();
    C.stop = 0;
  }
  if (warp == 1) {
    tmem_alloc(&C.tmem, S::Tmem);
    tmem_relinquish();
  }
  if (p.offsets) Division<Tile>::fill(p, C.first, C.sums, kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const Division<Tile> division(p, C.first);
  const int64_t units = division.units(), step = gridDim.x / split, u0 = blockIdx.x / split;
  const int g0 = p.groups * static_cast<int>(rank) / split, g1 = p.groups * static_cast<int>(rank + 1) / split;
  const uint32_t base = smem_u32(stages);

  if (warp == 0) {
    if (lane == 0) {
      uint32_t n = 0;
      for (int64_t u = u0; u < units; u += step) {
        const Run r = division.unit(u);
        for (int g = g0; g < g1; ++g, ++n) {
          const uint32_t s = n % S::Stages;
          waits.wait_lane(&C.empty[s], (n / S::Stages & 1) ^ 1);
          mbar_arrive_expect_tx(&C.w_full[s], S::Weight);
          tma_weight(&weight, g * kGroup, r.col * kRows, r.expert, base + s * S::Stage, &C.w_full[s]);
          if constexpr (Gate) tma_weight(&weight, g * kGroup, p.n / 2 + r.col * kRows, r.expert, base + s * S::Stage + kRows * kGroup, &C.w_full[s]);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    uint32_t n = 0;
    for (int64_t u = u0; u < units; u += step) {
      const Run r = division.unit(u);
      const uint32_t idesc = umma_idesc_e4m3_f32(kRows, (r.rows + 15) / 16 * 16);
      for (int g = g0; g < g1; ++g, ++n) {
        const uint32_t s = n % S::Stages, b = n % S::Sums;
        waits.wait_warp(&C.d_empty[b], (n / S::Sums & 1) ^ 1);
        waits.wait_warp(&C.w_full[s], n / S::Stages & 1);
        waits.wait_warp(&C.x_full[s], n / S::Stages & 1);
        fence_proxy_async_smem();            // rows of x were written by cp.async
        tc_fence_after();
        if (elect_one_sync()) {
          const uint32_t at = base + s * S::Stage, d = C.tmem + b * S::Cols;
          const uint64_t x = umma_desc_sw128(at + S::Weight);
#pragma unroll
          for (int h = 0; h < S::Halves; ++h) {
            const uint64_t w = umma_desc_sw128(at + h * kRows * kGroup);
#pragma unroll
            for (int i = 0; i < 4; ++i) umma_f8(d + h * Tile, w + i * 2, x + i * 2, idesc, i > 0);
          }
          umma_commit(&C.empty[s]);
          umma_commit(&C.d_full[b]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 4) {
    wait_for_launch_before();
    const int t = threadIdx.x - 64, chunk = t & 7, r0 = t >> 3;
    constexpr int kEach = Tile / 8;          // rows of a thread, eight apart
    uint32_t n = 0;
    for (int64_t u = u0; u < units; u += step) {
      const Run r = division.unit(u);
      const uint8_t* src[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int64_t row = r0 + 8 * i < r.rows ? source_row(p, r.row + r0 + 8 * i) : -1;
        src[i] = row < 0 ? nullptr : p.x + row * p.k + chunk * 16;
      }
      for (int g = g0; g < g1; ++g, ++n) {
        const uint32_t s = n % S::Stages;
        waits.wait(&C.empty[s], (n / S::Stages & 1) ^ 1);
        const bool in = g * kGroup + chunk * 16 < p.k;
        const uint32_t dst = base + s * S::Stage + S::Weight + r0 * 128 + ((chunk ^ (r0 & 7)) << 4);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (8 * i < r.rows) {              // all of the eight rows or none: what lies behind them is not read
            const bool have = in && src[i] != nullptr;
            cp_async16_or_zero(dst + i * 1024, have ? src[i] + g * kGroup : p.x, have ? 16 : 0);
          } else if (8 * i < (r.rows + 15) / 16 * 16) {
            cp_async16_or_zero(dst + i * 1024, p.x, 0);
          }
        cp_async_arrive_noinc(&C.x_full[s]);
      }
    }
    cp_async_commit();
    cp_async_wait<0>();                      // of a launch that gave up, too
  } else {
    wait_for_launch_before();
    const int quarter = warp & 3, half = (warp - 4) >> 2, w = warp - 4;
    constexpr int kPiece = S::Mine < 16 ? S::Mine : 16, kOwn = (S::Mine + 31) / 32;
    uint32_t n = 0;
    for (int64_t u = u0; u < units; u += step) {
      const Run r = division.unit(u);
      const int col = r.col * kRows + quarter * 32 + lane;             // row of the weight
      const int i0 = half * S::Mine;                                   // first row of x of this thread
      const float* ws = p.ws + (static_cast<int64_t>(r.expert) * p.blocks + r.col) * p.groups;
      const float* ws2 = ws + static_cast<int64_t>(p.blocks / 2) * p.groups;
      const float* xs[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int at = i0 + i * 32 + lane;
        const int64_t row = i * 32 + lane < S::Mine && at < r.rows ? source_row(p, r.row + at) : -1;
        xs[i] = row < 0 ? nullptr : p.xs + row * p.groups;
      }
      // scales of a group: lanes fetch those of their rows, two groups ahead, and hand them to the warp through shared memory
      float next[kOwn][2], next_w[2], next_w2[2];
      auto fetch = [&](int g, int slot) {
        const bool in = g < g1;
        next_w[slot] = in ? __ldg(ws + g) : 0.0f;
        next_w2[slot] = Gate && in ? __ldg(ws2 + g) : 0.0f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) next[i][slot] = in && xs[i] ? __ldg(xs[i] + g) : 0.0f;
      };
      fetch(g0, 0);
      fetch(g0 + 1, 1);
      float2 acc[S::Halves][S::Mine / 2] = {};
      const bool some = i0 < r.rows;
      for (int g = g0; g < g1; ++g, ++n) {
        const uint32_t b = n % S::Sums;
        const int slot = (g - g0) & 1;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (S::Mine >= 32 || lane < S::Mine) {
            const float x = slot ? next[i][1] : next[i][0];
            C.scale[w][slot][0][i * 32 + lane] = x * (slot ? next_w[1] : next_w[0]);
            if constexpr (Gate) C.scale[w][slot][1][i * 32 + lane] = x * (slot ? next_w2[1] : next_w2[0]);
          }
        if (slot) fetch(g + 2, 1); else fetch(g + 2, 0);
        waits.wait(&C.d_full[b], n / S::Sums & 1);
        tc_fence_after();
        if (some) {
          const uint32_t d = C.tmem + b * S::Cols + i0 + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
          for (int h = 0; h < S::Halves; ++h)
#pragma unroll
            for (int c = 0; c < S::Mine; c += kPiece)
              if (i0 + c < r.rows) {
                uint32_t v[kPiece];
                tmem_ld<kPiece>(d + h * Tile + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < kPiece; j += 4) {
                  const float4 sc = *reinterpret_cast<const float4*>(&C.scale[w][slot][h][c + j]);
                  float2& a0 = acc[h][(c + j) / 2];
                  float2& a1 = acc[h][(c + j) / 2 + 1];
                  a0 = fma2(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), make_float2(sc.x, sc.y), a0);
                  a1 = fma2(make_float2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), make_float2(sc.z, sc.w), a1);
                }
              }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&C.d_empty[b]);
      }

      // ---- the unit's sums are complete, for this CTA's groups
      int from = i0, count = S::Mine;                                  // rows of x whose results this thread has
      if (split > 1) {
        // every product of this CTA is through, so nobody reads the stages any more
        float* mine = reinterpret_cast<float*>(stages);
#pragma unroll
        for (int h = 0; h < S::Halves; ++h)
#pragma unroll
          for (int i = 0; i < S::Mine; ++i)
            if (i0 + i < r.rows) mine[(h * Tile + i0 + i) * kRows + quarter * 32 + lane] = i & 1 ? acc[h][i / 2].y : acc[h][i / 2].x;
        break;                               // one unit to a cluster
      }
      if constexpr (Gate) {
        uint32_t top[kOwn] = {};
#pragma unroll
        for (int i = 0; i < S::Mine; ++i) {
          float& a = i & 1 ? acc[0][i / 2].y : acc[0][i / 2].x;
          a = gated(a, i & 1 ? acc[1][i / 2].y : acc[1][i / 2].x);
          const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, magnitude(a));
          if (lane == (i & 31)) top[i / 32] = m;
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (S::Mine >= 32 || lane < S::Mine) C.top[half][quarter][i * 32 + lane] = top[i];
        named_bar_sync(2 + half, 128);
#pragma unroll
        for (int i = 0; i < S::Mine; ++i)
          if (from + i < r.rows) {
            const GroupScale gs(max(max(C.top[half][0][i], C.top[half][1][i]), max(C.top[half][2][i], C.top[half][3][i])));
            const int64_t row = r.row + from + i;
            store_code(p.codes + row * (p.n / 2) + col, (i & 1 ? acc[0][i / 2].y : acc[0][i / 2].x) * gs.inverse);
            if (quarter == 0 && lane == 0) p.scales[row * (p.n / 2 / kGroup) + r.col] = gs.scale;
          }
        named_bar_sync(2 + half, 128);       // everyone has read the magnitudes
      } else {
#pragma unroll
        for (int i = 0; i < S::Mine; ++i)
          if (i < count && from + i < r.rows && col < p.n) store(p, r.row + from + i, col, i & 1 ? acc[0][i / 2].y : acc[0][i / 2].x);
      }
    }
  }

  if (split > 1) {
    // Sums of the CTAs in their order; each CTA finishes a share of the rows of x, its 256 readers two rows at a time.
    __syncthreads();
    cluster_sync_all();
    if (warp >= 4 && u0 < units) {
      const Run r = division.unit(u0);
      const int quarter = warp & 3, half = (warp - 4) >> 2, col = r.col * kRows + quarter * 32 + lane;
      const int each = (r.rows + split - 1) / split, lo = each * static_cast<int>(rank), hi = min(lo + each, r.rows);
      const uint32_t here = base + (quarter * 32 + lane) * 4;
      for (int i = lo; i < hi; i += 2) {
        const int row = i + half;
        float v[S::Halves] = {};
        if (row < hi)
          for (int c = 0; c < split; ++c)
#pragma unroll
            for (int h = 0; h < S::Halves; ++h) v[h] += ld_cluster(map_to_cta(here + (h * Tile + row) * kRows * 4, c));
        if constexpr (Gate) {
          const float a = gated(v[0], v[1]);
          const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, magnitude(a));
          if (lane == 0) C.top[half][quarter][0] = m;
          named_bar_sync(2 + half, 128);
          const GroupScale gs(max(max(C.top[half][0][0], C.top[half][1][0]), max(C.top[half][2][0], C.top[half][3][0])));
          if (row < hi) {
            store_code(p.codes + (r.row + row) * (p.n / 2) + col, a * gs.inverse);
            if (quarter == 0 && lane == 0) p.scales[(r.row + row) * (p.n / 2 / kGroup) + r.col] = gs.scale;
          }
          named_bar_sync(2 + half, 128);
        } else if (row < hi && col < p.n) {
          store(p, r.row + row, col, v[0]);
        }
      }
    }
    __syncthreads();
    cluster_sync_all();                      // the others have read this CTA's sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (C.stop) settle();
  if (warp == 1) tmem_dealloc(C.tmem, S::Tmem);
}

template <int Tile, bool Gate>
int launch(const Product& p, const CUtensorMap& weight, int split, int64_t clusters, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  constexpr int kBytes = smem_bytes<Tile, Gate>();
  static_assert(kBytes <= 232448, "shared memory of an SM");
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(few_kernel<Tile, Gate>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(static_cast<unsigned>(clusters * split));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = kBytes;
  c.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (split > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = split;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.after) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  c.attrs = at;
  c.numAttrs = n;
  return static_cast<int>(cudaLaunchKernelEx(&c, few_kernel<Tile, Gate>, weight, p, split));
}

}  // namespace

namespace lin {
int launch_few(const Product& p, const CUtensorMap& weight, int tile, int split, int64_t clusters, cudaStream_t stream) {
  if (p.codes)
    return tile == 16 ? launch<16, true>(p, weight, split, clusters, stream) : tile == 32 ? launch<32, true>(p, weight, split, clusters, stream)
                                                                                          : launch<64, true>(p, weight, split, clusters, stream);
  return tile == 16   ? launch<16, false>(p, weight, split, clusters, stream)
         : tile == 32 ? launch<32, false>(p, weight, split, clusters, stream)
         : tile == 64 ? launch<64, false>(p, weight, split, clusters, stream)
                      : launch<128, false>(p, weight, split, clusters, stream);
}
}  // namespace lin
}  // namespace mono
