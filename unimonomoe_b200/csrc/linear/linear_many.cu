// Block-FP8 products for many rows: tiles of 128 rows of x and 256 rows of the weight.
//
//   y[i, n] = sum_g sx[i, g] sw[n / 128, g] sum_{k in g} qx[i, k] qw[n, k]
//
// A sum over a group of 128 is made by the tensor core (e4m3, fp32 in tensor memory), in two halves of 128 columns with two buffers each, from
// where eight warps add it, times its scales, to sums in registers: a thread has one row of x (one scale) and 128 rows of the weight (one
// scale, or the gate's and the other half's). Sixteen warps, one CTA to an SM:
//   0     requests weights, and rows of x where they lie in order
//   1, 2  issue the products, a half of the columns each
//   3     finds the units of experts, some ahead: the others read them from shared memory (found by each role for itself a unit cost 1600 cycles, as
//         much as two groups of K; those of one dense product are a few divisions, and taking them from there made 506 us of 483)
//   4-7   bring the scales, some groups ahead, and rows of x that lie anywhere (tokens), by cp.async with the 128-byte swizzle
//         written by hand
//   8-15  read the sums, a half of the columns each four; write the results, through shared memory by tensor stores
// With the gated activation a tile is 128 rows of the gate's half of the weight and the matching 128 of the other. Where a dense product has few tiles
// the groups of K are divided among two or four CTAs of a cluster, each of which finishes a part of the tile's rows: the others' sums of them come by bulk
// copies from shared memory to shared memory and are added to its own in the order of the CTAs, so that results do not depend on timing.
//
// Bound by the readers: of a group's 128 x 256 sums each has to be read from tensor memory, multiplied by its scale and added, some 920 cycles
// with the waits between, while the products take 512; the tensor pipe is busy half of the time. Around the groups of a unit lie 2900 cycles (first
// sums, results), 5400 with the gated activation, whose exponentials and quotients take the most of it. Measured: 16384 x 7168 x 4096 in 478-490 us (2.0
// PFLOP/s; under the power cap 535-547), 4096 x 2048 x 4096 in 50 (1.4), 8192 x 7168 x 4096 gated in 240-250; 256 experts' gated up projection (K 2048, N 1024) of 16384
// tokens in 414-440 (1.25-1.33), their down projection (K 512, N 2048) in 257 (1.07), of 3000 tokens unevenly routed in 85, where weights and results alone take 58.
// 8192 x 2048 x 4096 takes 72 us, with a residual, which is brought while the groups are summed, 84 (read a row a lane behind them 99), in fp32 87 (a row
// a lane 125), where rows of the result begin anywhere 148, with a residual 210.
// With K divided 256 rows of 7168 to 7168 columns take 25 us (undivided 37), 1024 of 4096 to 2048 19 (24); dividing costs 3.7 us in two, 5.7 in four (by stores of 16 bytes into the
// other CTA instead of bulk copies 7 to 8). Tiles of 256 x 256 by pairs of CTAs took 502 us for the first, for the gated up projection 457; twenty warps, sixteen of them readers with
// half the registers each, 580; one warp that issues for both halves, four stages with less room for results, and bands of sixteen
// row tiles made no difference or a worse one.
#include "linear.cuh"
#include "../pair_sm100.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kThreads = 512, kLoaders = 128, kReaders = 8, kRows = 128, kTile = 256;
constexpr int kMma = 1, kFinder = 3, kFirstLoader = 4, kFirstReader = 8;   // warps
constexpr int kSums = 4;                      // buffers of 128 columns, two for each half of the tile's
constexpr int kScales = 8;                   // groups whose scales are on their way or in use
constexpr int kRuns = 4;                     // units that are found and not yet done with
constexpr int kBox = 4096, kStaging = 2 * kBox;               // of a reader: 32 rows x 64 columns of bf16, twice
// Registers of a thread: at launch, of the first eight warps, of the readers. The readers' share comes from what the others give back.
constexpr int kRegs = 65536 / kThreads, kRegsOther = 48, kRegsReader = 208;
static_assert(8 * kRegsOther + 8 * kRegsReader <= 16 * kRegs, "a wait for registers that are not there has no end");

constexpr int kX = kRows * kGroup, kPart = 128 * kGroup, kStage = kX + 2 * kPart, kStages = 3;   // bytes of x, of a half of the weight's rows

struct Control {
  uint64_t full[kStages], gathered[kStages], empty[kStages], d_full[kSums], d_empty[kSums], s_full[kScales], s_empty[kScales], found[kRuns], taken[kRuns], joined, r_full[kReaders];
  Run runs[kRuns];
  uint32_t tmem, stop;
  int sums[32];
  uint32_t top[2][kRows];
  float x_scale[kScales][kRows], w_scale[kScales][2];
  int first[MONO_LIN_MAX_EXPERTS + 1];
};
// With K in four parts: the sums that come and go, 96 KB each, and room for results of the two warps that write.
static_assert(2 * 3 * (kRows / 4) * kTile * 4 + 2 * kStaging <= kStages * kStage + kReaders * kStaging, "divided sums");
static_assert(2 * 1 * (kRows / 2) * kTile * 4 + 4 * kStaging <= kStages * kStage + kReaders * kStaging, "divided sums");
constexpr int kSmem = kStages * kStage + kReaders * kStaging + static_cast<int>(sizeof(Control)) + 1024;
static_assert(kSmem <= 232448, "shared memory of an SM");

__device__ __forceinline__ void tma_weight(const CUtensorMap* m, int k, int row, int expert, uint32_t dst, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(k), "r"(row), "r"(expert), "r"(smem_u32(bar)) : "memory");
}
// A box of 64 columns x 32 rows from shared memory.
__device__ __forceinline__ void tma_store(const CUtensorMap* m, int col, int row, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(reinterpret_cast<uint64_t>(m)), "r"(col), "r"(row), "r"(src) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint4 ld_shared_128(uint32_t at) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
  return w;
}

// Shared memory into that of a CTA of the cluster, whose barrier counts it.
__device__ __forceinline__ void bulk_to_cta(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "r"(src), "r"(bytes), "r"(bar) : "memory");
}

// 128 columns from `col` on of 32 rows, of which the first `rows` are the unit's; one row a lane. Pieces of 16 bytes lie in shared memory at places
// that spread over the banks, as a tensor map with the 128-byte swizzle has them. So does the residual, if it was `brought` there. Plain: bf16 in rows
// that begin on 16 bytes, without residual; what else there is in one kernel with that costs it 3%.
template <bool Plain>
__device__ __forceinline__ void write_out(const Product& p, const CUtensorMap* out, uint32_t at, int lane, int64_t row0, int rows, int col, bool brought, float2 (&acc)[2][32]) {
  auto add = [&](int c, const uint4& r) {    // to eight columns
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = bf16x2(w[i]);
      float2& t = acc[c / 8][c % 8 * 4 + i];
      t.x += f.x;
      t.y += f.y;
    }
  };
  if (!Plain && brought) {
#pragma unroll
    for (int c = 0; c < 16; ++c) add(c, ld_shared_128(at + c / 8 * kBox + lane * 128 + (((c % 8) ^ (lane & 7)) << 4)));
    __syncwarp();
  } else if (!Plain && p.vec && p.residual && lane < rows) {
    const uint4* res = reinterpret_cast<const uint4*>(p.residual + (row0 + lane) * p.n + col);
#pragma unroll
    for (int c = 0; c < 16; ++c)
      if (col + c * 8 < p.n) add(c, __ldg(res + c));
  }
  if (Plain || (p.vec && !p.fp32)) {
    if (lane == 0) bulk_wait_read<0>();      // of the unit before
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float2* v = acc[h] + 4 * c;
        const uint32_t w[4] = {pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y)};
        st_shared_128(at + h * kBox + lane * 128 + ((c ^ (lane & 7)) << 4), w);
      }
    }
    if (rows == 32) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store(out, col, static_cast<int>(row0), at);      // what lies behind the last column is left out
        if (col + 64 < p.n) tma_store(out, col + 64, static_cast<int>(row0), at + kBox);
        bulk_commit();
      }
    } else {                                 // the next rows are another run's
      __syncwarp();
      const int c = lane & 7, half = (lane >> 3) & 1;
      if (col + half * 64 + c * 8 < p.n)
#pragma unroll 4
        for (int r = lane >> 4; r < rows; r += 2)
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + (row0 + r) * p.n + col + half * 64 + c * 8) =
              ld_shared_128(at + half * kBox + r * 128 + ((c ^ (r & 7)) << 4));
      __syncwarp();
    }
  } else if (!Plain && p.vec) {              // 64 columns of fp32 at a time
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float2 *v = acc[h] + 2 * c;
        const uint32_t w[4] = {__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y)};
        st_shared_128(at + c / 8 * kBox + lane * 128 + (((c % 8) ^ (lane & 7)) << 4), w);
      }
      const int from = col + h * 64;
      if (rows == 32) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && from < p.n) {
          tma_store(out, from, static_cast<int>(row0), at);
          if (from + 32 < p.n) tma_store(out, from + 32, static_cast<int>(row0), at + kBox);
          bulk_commit();
        }
      } else {
        __syncwarp();
        const int c = lane & 7, box = (lane >> 3) & 1, n = from + box * 32 + c * 4;
        if (n < p.n)
#pragma unroll 4
          for (int r = lane >> 4; r < rows; r += 2)
            *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + (row0 + r) * p.n + n) = ld_shared_128(at + box * kBox + r * 128 + ((c ^ (r & 7)) << 4));
        __syncwarp();
      }
    }
  } else if (!Plain) {                       // rows that begin anywhere: 32 columns at a time, a column a lane
#pragma unroll
    for (int h = 0; h < 4; ++h) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float2* v = acc[h >> 1] + (h & 1) * 16 + 2 * c;
        const uint32_t w[4] = {__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y)};
        st_shared_128(at + lane * 128 + ((c ^ (lane & 7)) << 4), w);
      }
      __syncwarp();
      const int n = col + h * 32 + lane;
      if (n < p.n)
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 8) {
          __nv_bfloat16 res[8];
          if (p.residual) {
#pragma unroll
            for (int i = 0; i < 8; ++i) res[i] = p.residual[(row0 + min(r0 + i, rows - 1)) * p.n + n];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = r0 + i;
            if (r >= rows) break;
            float x;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
            const int64_t to = (row0 + r) * p.n + n;
            if (p.residual) x += __bfloat162float(res[i]);
            if (p.fp32) static_cast<float*>(p.out)[to] = x;
            else static_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(x);
          }
        }
      __syncwarp();
    }
  }
}

template <bool Gate, bool Runs, bool Split, bool Plain>
__global__ void __launch_bounds__(kThreads, 1) many_kernel(const __grid_constant__ CUtensorMap weight, const __grid_constant__ CUtensorMap rows,
                                                           const __grid_constant__ CUtensorMap out, const __grid_constant__ CUtensorMap residual,
                                                           const __grid_constant__ Product p, const int split) {
  extern __shared__ uint8_t raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Control& C = *reinterpret_cast<Control*>(stages + kStages * kStage + kReaders * kStaging);
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const Waits waits{&C.stop, p.status};
  const bool gather = Runs && p.tokens != nullptr;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&C.full[i], 1);
      mbar_init(&C.gathered[i], kLoaders);
      mbar_init(&C.empty[i], 2);             // of both halves
    }
    for (int i = 0; i < kSums; ++i) {
      mbar_init(&C.d_full[i], 1);
      mbar_init(&C.d_empty[i], kReaders / 2);               // the four readers of a half
    }
    for (int i = 0; i < kScales; ++i) {
      mbar_init(&C.s_full[i], kLoaders);
      mbar_init(&C.s_empty[i], kReaders);
    }
    for (int i = 0; i < kRuns; ++i) {
      mbar_init(&C.found[i], 1);
      mbar_init(&C.taken[i], 1 + kLoaders / 32 + kReaders);
    }
    mbar_init(&C.joined, 1);
    for (int i = 0; i < kReaders; ++i) mbar_init(&C.r_full[i], 1);
    mbar_init_fence();
    C.stop = 0;
  }
  if (warp == kMma) {
    tmem_alloc(&C.tmem, 512);
    tmem_relinquish();
  }
  if constexpr (Runs) Division<kRows>::fill(p, C.first, C.sums, kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const Division<kRows> division(p, C.first);
  const int rank = Split ? static_cast<int>(cluster_ctarank()) : 0, of = Split ? split : 1;
  const int units = division.units(), step = gridDim.x / of, u0 = blockIdx.x / of;
  const int g0 = p.groups * rank / of, g1 = p.groups * (rank + 1) / of;     // groups of K of this CTA
  const uint32_t base = smem_u32(stages);
  // Unit u, the next one of this CTA. Where it is one of a run it is one without rows in a launch that gave up: what is in memory may be half of another.
  uint32_t nth = 0;
  auto take = [&](int u) {
    if constexpr (!Runs) {
      return division.unit(u);
    } else {
      const uint32_t slot = nth % kRuns;
      waits.wait(&C.found[slot], nth++ / kRuns & 1);
      const Run r = C.runs[slot];
      if (waits.stopped()) return Run{};
      if (lane == 0) mbar_arrive(&C.taken[slot]);
      return r;
    }
  };

  if (warp < kFirstReader) {
    reg_dec<kRegsOther>();
    if (warp == 0) {
      uint32_t n = 0;
      for (int u = u0; u < units; u += step) {
        const Run r = take(u);
        if (lane == 0) {
          for (int g = g0; g < g1; ++g, ++n) {
            const uint32_t s = n % kStages, at = base + s * kStage;
            waits.wait_lane(&C.empty[s], (n / kStages & 1) ^ 1);
            mbar_arrive_expect_tx(&C.full[s], gather ? 2 * kPart : 2 * kPart + kX);
#pragma unroll
            for (int q = 0; q < 4; ++q)      // with the gated activation 64 rows of the gate's and of the others in turn
              tma_weight(&weight, g * kGroup, Gate ? (q & 1) * (p.n / 2) + r.col * kRows + (q >> 1) * 64 : r.col * kTile + q * 64, r.expert,
                         at + kX + q * 64 * kGroup, &C.full[s]);
            if (!gather) tma_load_2d(&rows, g * kGroup, static_cast<uint32_t>(r.row), stages + s * kStage, &C.full[s]);
          }
        }
        __syncwarp();
      }
    } else if (warp < kMma + 2) {
      constexpr uint32_t idesc = umma_idesc_e4m3_f32(kRows, kTile / 2);
      const uint32_t h = warp - kMma;
      uint32_t n = 0;
      for (int u = u0; u < units; u += step)
        for (int g = g0; g < g1; ++g, ++n) {
          const uint32_t s = n % kStages, b = 2 * (n & 1) + h;
          waits.wait_warp(&C.full[s], n / kStages & 1, &C.d_empty[b], (n >> 1 & 1) ^ 1);
          if (gather) {
            waits.wait_warp(&C.gathered[s], n / kStages & 1);
            fence_proxy_async_smem();
          }
          tc_fence_after();
          if (elect_one_sync()) {
            const uint64_t x = umma_desc_sw128(base + s * kStage), w = umma_desc_sw128(base + s * kStage + kX + h * kPart);
#pragma unroll
            for (int i = 0; i < 4; ++i) umma_f8(C.tmem + b * (kTile / 2), x + i * 2, w + i * 2, idesc, i > 0);
            umma_commit(&C.d_full[b]);
            umma_commit(&C.empty[s]);
          }
          __syncwarp();
        }
    } else if (warp == kFinder) {
      if constexpr (Runs) {
        int expert = 0;
        for (int u = u0; u < units; u += step, ++nth) {
          const Run r = division.unit_after(u, expert);
          const uint32_t slot = nth % kRuns;
          waits.wait(&C.taken[slot], (nth / kRuns & 1) ^ 1);
          if (waits.stopped()) break;
          if (lane == 0) {
            C.runs[slot] = r;
            mbar_arrive(&C.found[slot]);
          }
        }
      }
    } else {
      const int t = threadIdx.x - 32 * kFirstLoader, chunk = t & 7, r0 = t >> 3;
      constexpr int kEach = kRows / (kLoaders / 8);           // rows of a thread, sixteen apart
      uint32_t n = 0;
      for (int u = u0; u < units; u += step) {
        const Run r = take(u);
        // Rows past the unit's are left as they are, nobody reads what comes of them. (One row for all of them would be asked for by
        // every CTA at once: 174 us instead of 113 for 2048 tokens through 256 experts' up projection.)
        auto row = [&](int i) { return i < r.rows ? source_row(p, r.row + i) : 0; };
        const float* xs = p.xs + static_cast<int64_t>(row(t)) * p.groups;
        const int block = t == 0 ? (Gate ? r.col : 2 * r.col) : Gate ? r.col + p.blocks / 2 : min(2 * r.col + 1, p.blocks - 1);
        const float* ws = p.ws + (static_cast<int64_t>(r.expert) * p.blocks + block) * p.groups;
        uint32_t src[kEach];                 // rows of x, in pieces of 16 bytes
        if (gather) {
#pragma unroll
          for (int i = 0; i < kEach; ++i) src[i] = static_cast<uint32_t>(row(r0 + kLoaders / 8 * i)) * static_cast<uint32_t>(p.k / 16);
        }
        for (int g = g0; g < g1; ++g, ++n) {
          const uint32_t s = n % kStages, slot = n % kScales;
          waits.wait(&C.s_empty[slot], (n / kScales & 1) ^ 1);
          if (t < r.rows) cp_async4(smem_u32(&C.x_scale[slot][t]), xs + g);
          if (t < 2) cp_async4(smem_u32(&C.w_scale[slot][t]), ws + g);
          cp_async_arrive_noinc(&C.s_full[slot]);
          if (gather) {
            waits.wait(&C.empty[s], (n / kStages & 1) ^ 1);
            const int k = g * kGroup + chunk * 16;
            const uint32_t dst = base + s * kStage + r0 * 128 + ((chunk ^ (r0 & 7)) << 4), bytes = k < p.k ? 16 : 0;
            const uint8_t* x = p.x + (bytes ? k : 0);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
              if (r0 + kLoaders / 8 * i < r.rows) cp_async16_or_zero(dst + i * (kLoaders / 8 * 128), x + static_cast<uint64_t>(src[i]) * 16, bytes);
            cp_async_arrive_noinc(&C.gathered[s]);
          }
        }
      }
      cp_async_commit();
      cp_async_wait<0>();                    // of a launch that gave up, too
    }
    if (Split && u0 < units) {               // as the readers do
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    reg_inc<kRegsReader>();
    const int quarter = warp & 3, half = (warp - kFirstReader) >> 2;
    const uint32_t staging = base + kStages * kStage + (warp - kFirstReader) * kStaging;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    // The residual of a unit is brought to where its results will lie while the groups are summed.
    const bool bring = !Gate && !Runs && !Split && !Plain && p.residual != nullptr && p.vec;
    uint32_t n = 0, brought = 0;
    for (int u = u0; u < units; u += step) {
      const Run r = take(u);
      const int in = quarter * 32, mine = max(0, min(32, r.rows - in));   // rows of this warp
      const int64_t row0 = static_cast<int64_t>(r.row) + in;
      const bool here = bring && mine > 0 && r.col * kTile + half * 128 < p.n;
      if (here && lane == 0) {
        const int col = r.col * kTile + half * 128, boxes = col + 64 < p.n ? 2 : 1;
        uint8_t* to = stages + kStages * kStage + (warp - kFirstReader) * kStaging;
        uint64_t* bar = &C.r_full[warp - kFirstReader];
        bulk_wait_read<0>();                 // the results of the unit before
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(bar, boxes * kBox);
        for (int i = 0; i < boxes; ++i) tma_load_2d(&residual, col + i * 64, static_cast<uint32_t>(row0), to + i * kBox, bar);
      }
      __syncwarp();
      float2 acc[2][32] = {};
      // The sums of group n are in the buffer, and its scales in shared memory.
      auto ready = [&](uint32_t n) {
        waits.wait(&C.s_full[n % kScales], n / kScales & 1, &C.d_full[2 * (n & 1) + half], n >> 1 & 1);
        tc_fence_after();
      };
      auto release = [&](uint32_t n) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&C.d_empty[2 * (n & 1) + half]);
          mbar_arrive(&C.s_empty[n % kScales]);
        }
      };
      auto buffer = [&](uint32_t n) { return C.tmem + (2 * (n & 1) + half) * (kTile / 2) + lanes; };
      auto add = [&](const uint32_t (&v)[32], float scale, float2* to) {
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i] = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), make_float2(scale, scale), to[i]);
      };
      if (mine > 0) {
        // 32 columns at a time, the next ones on their way while these are added
        uint32_t v0[32], v1[32];
        ready(n);
        tmem_ld32(buffer(n), v0);
        for (int g = g0; g < g1; ++g, ++n) {
          const uint32_t d = buffer(n), slot = n % kScales;
          const float x = C.x_scale[slot][quarter * 32 + lane], sa = x * C.w_scale[slot][Gate ? 0 : half], sb = Gate ? x * C.w_scale[slot][1] : sa;
          tmem_ld_wait();
          tmem_ld32(d + 32, v1);
          add(v0, sa, acc[0]);
          tmem_ld_wait();
          tmem_ld32(d + 64, v0);
          add(v1, sa, acc[0] + 16);
          tmem_ld_wait();
          tmem_ld32(d + 96, v1);
          add(v0, sb, acc[1]);
          tmem_ld_wait();
          release(n);                        // read out: the next product may have the buffer
          if (g + 1 < g1) {
            ready(n + 1);
            tmem_ld32(buffer(n + 1), v0);
          }
          add(v1, sb, acc[1] + 16);
        }
      } else {
        for (int g = g0; g < g1; ++g, ++n) {
          waits.wait(&C.d_full[2 * (n & 1) + half], n >> 1 & 1);
          release(n);
        }
      }
      bool writes = true;
      uint32_t to = staging;
      if constexpr (Split) {
        // One unit to a cluster; a CTA finishes 64 or 32 of its rows. The others' sums of them come into its ring, which then is free, [CTA][row], and
        // its own of other rows lie behind that until they are fetched; pieces of 16 bytes at places that spread over the banks.
        const int each = kRows / split, owner = in / each, row = in % each + lane;
        const uint32_t block = each * kTile * 4, come = base, go = base + (split - 1) * block, place = row * kTile * 4 + half * 512;
        named_bar_sync(6, kReaders * 32);    // both halves of this CTA have their sums
        cluster_arrive();
        if (owner != rank) {
          const uint32_t at = go + (owner - (owner > rank)) * block + place;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float2 a = acc[c >> 4][c % 16 * 2], b = acc[c >> 4][c % 16 * 2 + 1];
            const uint32_t w[4] = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)};
            st_shared_128(at + ((c ^ (lane & 7)) << 4), w);
          }
          fence_proxy_async_smem();
        }
        cluster_wait();
        named_bar_sync(6, kReaders * 32);
        if (threadIdx.x == 32 * kFirstReader) {
          mbar_arrive_expect_tx(&C.joined, (split - 1) * block);
          for (int c = 0; c < split; ++c)
            if (c != rank) bulk_to_cta(map_to_cta(come + (rank - (rank > c)) * block, c), go + (c - (c > rank)) * block, block, map_to_cta(smem_u32(&C.joined), c));
        }
        waits.wait_sent(&C.joined, 0);
        writes = owner == rank;
        to = base + kStages * kStage + (kReaders - 1 - half * (each / 32) - in % each / 32) * kStaging;     // the last pieces, of those that write
        if (writes) {
          for (int q = 0; q < split - 1; ++q) {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const uint4 w = ld_shared_128(come + q * block + place + ((c ^ (lane & 7)) << 4));
              float2 &a = acc[c >> 4][c % 16 * 2], &b = acc[c >> 4][c % 16 * 2 + 1];
              a.x += __uint_as_float(w.x); a.y += __uint_as_float(w.y); b.x += __uint_as_float(w.z); b.y += __uint_as_float(w.w);
            }
          }
        }
      }
      if (!writes) continue;
      if constexpr (Gate) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          acc[0][i].x = gated_sums(acc[0][i].x, acc[1][i].x);
          acc[0][i].y = gated_sums(acc[0][i].y, acc[1][i].y);
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
        const int col = r.col * kTile + half * 128;
        if (here) waits.wait(&C.r_full[warp - kFirstReader], brought++ & 1);
        if (col < p.n) write_out<Plain>(p, &out, to, lane, row0, mine, col, here, acc);
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
    if (Split && u0 < units) cluster_sync_all();              // what this CTA sent has been fetched
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (C.stop) settle();
  if (warp == kMma) tmem_dealloc(C.tmem, 512);
}

template <bool Gate, bool Runs, bool Split, bool Plain>
int launch(const Product& p, const CUtensorMap& weight, const CUtensorMap& x, const CUtensorMap& out, const CUtensorMap& residual, int split, int clusters, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(many_kernel<Gate, Runs, Split, Plain>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(static_cast<unsigned>(Split ? clusters * split : kSms));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = kSmem;
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = Split ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&c, many_kernel<Gate, Runs, Split, Plain>, weight, x, out, residual, p, split));
}

template <bool Gate, bool Plain>
int launch_as(const Product& p, const CUtensorMap& weight, const CUtensorMap& x, const CUtensorMap& out, const CUtensorMap& residual, int split, int clusters,
              cudaStream_t stream) {
  if (p.offsets) return launch<Gate, true, false, Plain>(p, weight, x, out, residual, 1, 0, stream);
  if (split > 1) return launch<Gate, false, true, Plain>(p, weight, x, out, residual, split, clusters, stream);
  return launch<Gate, false, false, Plain>(p, weight, x, out, residual, 1, 0, stream);
}

}  // namespace

namespace lin {
int launch_many(const Product& p, const CUtensorMap& weight, const CUtensorMap& x, const CUtensorMap& out, const CUtensorMap& residual, int split, int clusters, cudaStream_t stream) {
  if (p.codes) return launch_as<true, true>(p, weight, x, out, residual, split, clusters, stream);
  if (p.vec && !p.fp32 && !p.residual) return launch_as<false, true>(p, weight, x, out, residual, split, clusters, stream);
  return launch_as<false, false>(p, weight, x, out, residual, split, clusters, stream);
}
}  // namespace lin
}  // namespace mono
