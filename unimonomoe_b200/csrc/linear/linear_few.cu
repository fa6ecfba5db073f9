// Block-FP8 products for few rows: D^T = W X^T, with 128 rows of the weight as the rows of the tensor-core product and up to Tile
// rows of x as its columns, so that the weight is read once and nothing of the product is padding beyond 16 rows of x.
//
//   y[i, n] = sum_g sx[i, g] sw[n / 128, g] sum_{k in g} qx[i, k] qw[n, k]
//
// The sum over a group of 128 is made by the tensor core (e4m3, fp32 sums in tensor memory), the scales are applied to it in
// registers: a thread has one row of the weight and some rows of x. A stage of the ring has two pieces of the weight, [128 rows x 128]
// each: two groups, or with the gated activation the gate's rows and the other half's; waiting costs each role some 150 cycles a
// time, more than a piece of few rows takes to multiply. Twelve warps, one CTA to an SM:
//   0     requests the weight
//   1     issues the products
//   2, 3  bring the rows of x and the scales, by cp.async with the 128-byte swizzle written by hand: rows may lie anywhere (tokens). Rows in 16
//         bits are quantised by them and the readers at the start, in every CTA: for so few that takes less than a launch before this one
//   4-11  read the sums, four warps for the 128 rows, twice for the halves of the rows of x
// The groups of K may be divided among the CTAs of a cluster. Each then hands its sums to the CTA that finishes the row, by stores into its
// shared memory that its barrier counts, and they are added in the order of the CTAs: the result does not depend on timing. Without
// that a CTA goes from unit to unit, and the weight's requests run ahead across them.
//
// Bound by latency where there is one unit to a CTA: a launch, a division, the first bytes of the weight, its stages, the join and the results follow
// one another. In a graph 1 row of 2048 to 5120 columns takes 5.4 us (by one CTA for each unit, eight stages one after another, 1.2 more), 61 rows of 4096 to 2048, in 8 bits, 7.7;
// bound by memory where experts are many: the gated up projection of 24 tokens through 256 experts reads 275 MB in 46.7 us, 5.9 TB/s, the down projection
// of 64 tokens 233 MB in 41.5. A tile is as wide as the rows ask for: of 16 a stage takes 360 ns, of 64 600, and the room for its
// rows of x is room that the ring loses. The sums' way out by bf16 and tensor stores, as in the kernel of many rows, made 201 us of 184 where runs are of 60 rows.
#include "linear.cuh"
#include "../pair_sm100.cuh"

namespace mono {
namespace {

using namespace lin;

constexpr int kThreads = 384, kLoaders = 64, kReaders = 256, kRows = 128, kPiece = kRows * kGroup;
constexpr int kScales = 8;                   // stages whose scales are on their way or in use
constexpr int kSplit = 8;                    // CTAs of a cluster at most

template <int Tile, bool Gate>
struct Shape {
  static constexpr int Halves = Gate ? 2 : 1;
  static constexpr int Groups = few_groups(Gate);       // of K in a stage
  static constexpr int Pieces = Halves * Groups;              // of the weight in a stage
  static constexpr int Stage = Pieces * kPiece + Groups * Tile * kGroup;
  static constexpr int Add = Halves * (Tile + kSplit) * kRows * 4;    // bytes of a unit's sums
  static constexpr int Room = 206 * 1024 - Add;               // of stages
  static constexpr int Stages = Room / Stage < 8 ? Room / Stage : 8;
  static constexpr int Cols = Pieces * Tile;                  // of a stage's sums in tensor memory
  static constexpr int Used = Cols * Stages, Tmem = Used <= 128 ? 128 : Used <= 256 ? 256 : 512;
  static constexpr int Mine = Tile / 2;                       // rows of x of a thread
  static_assert(Used <= 512 && Stages >= 3, "columns of tensor memory");
};

template <int Tile, bool Gate>
struct Control {
  using S = Shape<Tile, Gate>;
  uint64_t full[8], done[8], read[8], s_full[kScales], s_empty[kScales], joined;
  uint32_t tmem, stop;
  int sums[32];
  Run found;
  alignas(16) float scale[kScales][S::Pieces][Tile];          // of a stage: those of a row of x times the weight's
  int first[MONO_LIN_MAX_EXPERTS + 1];
};

template <int Tile, bool Gate>
constexpr int smem_bytes() {
  return Shape<Tile, Gate>::Stages * Shape<Tile, Gate>::Stage + Shape<Tile, Gate>::Add + static_cast<int>(sizeof(Control<Tile, Gate>)) + 1024;
}

__device__ __forceinline__ int cluster_id() {
  int id;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(id));
  return id;
}
// A store into the shared memory of a CTA of the cluster, which that one's barrier counts.
__device__ __forceinline__ void st_counted(uint32_t addr, float v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(addr), "f"(v), "r"(bar) : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "columns at a time");
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(t) : "memory");
  else if constexpr (N == 16)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(t) : "memory");
  else tmem_ld32(t, v);
}
__device__ __forceinline__ void tma_weight(const CUtensorMap* m, int k, int row, int expert, uint32_t dst, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(k), "r"(row), "r"(expert), "r"(smem_u32(bar)) : "memory");
}
// Rows [lo, hi) of a unit, whose sums lie in this CTA's shared memory, those of CTA c of the cluster at [c][half][row - lo] of rows
// of 128: a lane has four columns, a warp two rows at a time.
template <bool Gate, bool Split>
__device__ __forceinline__ void finish(const Product& p, const Run& r, const float* sums, int split, int each, int lo, int hi, int w, int lane) {
  constexpr int kHalves = Gate ? 2 : 1, kWarps = kReaders / 32, kAtOnce = 2;
  const float* mine = sums + lane * 4;
#pragma unroll 1
  for (int first = lo + w; first < hi; first += kWarps * kAtOnce) {
    float4 v[kAtOnce][kHalves];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int i = min(first + q * kWarps, hi - 1);
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const float* at = mine + (h * each + i - lo) * kRows;
        v[q][h] = *reinterpret_cast<const float4*>(at);
        if constexpr (Split) {
#pragma unroll 1
          for (int c = 1; c < split; ++c) {
            at += kHalves * each * kRows;
            const float4 t = *reinterpret_cast<const float4*>(at);
            v[q][h].x += t.x; v[q][h].y += t.y; v[q][h].z += t.z; v[q][h].w += t.w;
          }
        }
      }
    }
    if constexpr (Gate) {
      uint32_t m[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        float4 &a = v[q][0], &b = v[q][1];
        a = make_float4(gated_sums(a.x, b.x), gated_sums(a.y, b.y), gated_sums(a.z, b.z), gated_sums(a.w, b.w));
        m[q] = __reduce_max_sync(0xFFFFFFFFu, max(max(magnitude(a.x), magnitude(a.y)), max(magnitude(a.z), magnitude(a.w))));
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int i = first + q * kWarps;
        const GroupScale gs(m[q]);
        if (i < hi) {
          const int64_t row = static_cast<int64_t>(r.row) + i;
          const float4 a = v[q][0];
          *reinterpret_cast<uint32_t*>(p.codes + row * (p.n / 2) + r.col * kRows + lane * 4) =
              pack_e4m3x4(a.x * gs.inverse, a.y * gs.inverse, a.z * gs.inverse, a.w * gs.inverse);
          if (lane == 0) p.scales[row * (p.n / 2 / kGroup) + r.col] = gs.scale;
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int i = first + q * kWarps;
        if (i < hi) store4(p, static_cast<int64_t>(r.row) + i, r.col * kRows + lane * 4, v[q][0]);
      }
    }
  }
}

// Rows in 16 bits of this CTA's groups, which all find room in the ring: codes into the stages' rows of x, scales times the weight's. By all warps
// but the first two: eight lanes share a group, 16 values each; the next one's values are on their way while one is quantised, the first ones' while
// the CTA sets itself up.
constexpr int kTeams = (kThreads - 64) / 8;
struct Piece {
  uint4 a, b;
  float weight;                              // its scale, for the lanes that write the product of both
};
template <bool Gate>
__device__ __forceinline__ Piece fetch_piece(const Product& p, const Run& r, int g0, int items, int i) {
  const int lane8 = threadIdx.x & 7, in = static_cast<uint32_t>(i) / static_cast<uint32_t>(r.rows), g = g0 + in, k = g * kGroup + lane8 * 16;
  const bool have = i < items && k < p.k;
  const uint4* src = reinterpret_cast<const uint4*>(p.raw + (i - in * r.rows) * p.raw_stride + k);
  Piece x;
  x.a = have ? __ldg(src) : make_uint4(0, 0, 0, 0);
  x.b = have ? __ldg(src + 1) : make_uint4(0, 0, 0, 0);
  // behind the last group sums and scales are zero
  x.weight = i < items && g < p.groups && lane8 < (Gate ? 2 : 1) ? __ldg(p.ws + (static_cast<int64_t>(r.col) + lane8 * (p.blocks / 2)) * p.groups + g) : 0.0f;
  return x;
}
template <int Tile, bool Gate>
__device__ __forceinline__ void quantise_rows(const Product& p, Control<Tile, Gate>& C, const Run& r, uint32_t base, int t0, int t1, Piece next) {
  using S = Shape<Tile, Gate>;
  const int lane8 = threadIdx.x & 7, g0 = t0 * S::Groups, items = (t1 - t0) * S::Groups * r.rows;
  for (int i = (threadIdx.x - 64) >> 3; __any_sync(0xFFFFFFFFu, i < items); i += kTeams) {
    float2 v[8];
    unpack16(next.a, next.b, v);
    const float weight = next.weight;
    next = fetch_piece<Gate>(p, r, g0, items, i + kTeams);
    const int g = static_cast<uint32_t>(i) / static_cast<uint32_t>(r.rows), row = i - g * r.rows, s = g / S::Groups, j = g - s * S::Groups;   // group and row, stage and group of it
    const GroupScale scale(top_of_group(v));
    if (i < items) {
      const uint4 c = codes16(v, scale.inverse);
      const uint32_t words[4] = {c.x, c.y, c.z, c.w};
      st_shared_128(base + s * S::Stage + S::Pieces * kPiece + (j * Tile + row) * 128 + ((lane8 ^ (row & 7)) << 4), words);
      if (lane8 < S::Halves) C.scale[s][Gate ? lane8 : j][row] = g0 + g < p.groups ? scale.scale * weight : 0.0f;
    }
  }
  fence_proxy_async_smem();                  // the tensor core reads what was stored here
  named_bar_sync(3, kThreads - 64);
}

template <int Tile, bool Gate>
__global__ void __launch_bounds__(kThreads, 1) few_kernel(const __grid_constant__ CUtensorMap weight, const __grid_constant__ Product p, const int split) {
  using S = Shape<Tile, Gate>;
  extern __shared__ uint8_t raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* sums = reinterpret_cast<float*>(stages + S::Stages * S::Stage);
  const uint32_t base = smem_u32(stages);
  Control<Tile, Gate>& C = *reinterpret_cast<Control<Tile, Gate>*>(stages + S::Stages * S::Stage + S::Add);
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const int rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const Waits waits{&C.stop, p.status};
  // With K divided a cluster has one unit.
  const int step = split > 1 ? 1 << 30 : static_cast<int>(gridDim.x), u0 = split > 1 ? cluster_id() : static_cast<int>(blockIdx.x);
  const uint32_t steps = (p.groups + S::Groups - 1) / S::Groups;
  const int t0 = steps * rank / split, t1 = steps * (rank + 1) / split;       // stages of this CTA
  // Stage s gets the pieces of step t of unit r; the n-th use of the ring.
  auto request = [&](const Run& r, int t, uint32_t s) {
    const uint32_t at = base + s * S::Stage;
    mbar_arrive_expect_tx(&C.full[s], S::Pieces * kPiece);
#pragma unroll
    for (int i = 0; i < S::Groups; ++i) tma_weight(&weight, (t * S::Groups + i) * kGroup, r.col * kRows, r.expert, at + i * kPiece, &C.full[s]);
    if constexpr (Gate) tma_weight(&weight, t * kGroup, p.n / 2 + r.col * kRows, r.expert, at + kPiece, &C.full[s]);
  };

  if (p.offsets && static_cast<int>(threadIdx.x) <= p.experts) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.offsets + threadIdx.x));

  // The first requests come before the other barriers are made; what other CTAs have to wait for comes before them.
  if (warp == 0) {
    if (lane < S::Stages) mbar_init(&C.full[lane], 1 + kLoaders);
    if (lane == 0) {
      tma_prefetch_desc(&weight);
      mbar_init(&C.joined, 1);
    }
    mbar_init_fence();
    __syncwarp();
  }
  // What is to be seen by the others are barriers, which their fence has released.
  if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  auto other_barriers = [&]() {
    if (warp == 0) {
      if (lane < S::Stages) {
        mbar_init(&C.done[lane], 1);
        mbar_init(&C.read[lane], kReaders / 32);
      }
      if (lane < kScales) {
        mbar_init(&C.s_full[lane], kLoaders);
        mbar_init(&C.s_empty[lane], kReaders / 32);
      }
      if (lane == 0) C.stop = 0;
      mbar_init_fence();
      __syncwarp();
    }
  };
  const Division<Tile> division(p, C.first);
  Run at_first{};                            // all warps'
  if (p.offsets) {
    other_barriers();                        // while the offsets are on their way
    const int tile = u0 / p.cols;
    Division<Tile>::fill(p, C.first, C.sums, kThreads, tile, &C.found);
    at_first = C.found;
    at_first.col = u0 - tile * p.cols;
  }
  const int units = division.units();
  if (!p.offsets && u0 < units) at_first = division.unit(u0);
  int expert = at_first.expert;
  auto unit = [&](int u) { return u == u0 ? at_first : division.unit_after(u, expert); };
  const int early = u0 < units ? min(t1 - t0, S::Stages) : 0;
  if (threadIdx.x == 0)
    for (int i = 0; i < early; ++i) request(at_first, t0 + i, i);
  __syncwarp();
  if (!p.offsets) other_barriers();
  const bool in_16 = Tile >= MONO_LIN_FEW_ROWS && Tile < 2 * MONO_LIN_FEW_ROWS && p.raw != nullptr;   // what takes_rows says yes to has this tile
  const bool quantise = in_16 && warp >= 2 && u0 < units;
  Piece first_piece{};
  if (quantise) first_piece = fetch_piece<Gate>(p, at_first, t0 * S::Groups, (t1 - t0) * S::Groups * at_first.rows, (threadIdx.x - 64) >> 3);
  if (warp == 1) {
    tmem_alloc(&C.tmem, S::Tmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // the others run: their shared memory may be written

  if (quantise) quantise_rows<Tile, Gate>(p, C, at_first, base, t0, t1, first_piece);

  if (warp == 0) {
    uint32_t before = 0;                     // stages of the units before
    for (int u = u0; u < units; u += step, before += t1 - t0) {
      const int first = u == u0 ? early : 0;
      if (first == t1 - t0) continue;        // all of it is requested
      const Run r = unit(u);
      if (lane == 0)
        for (int t = t0 + first; t < t1; ++t) {
          const uint32_t n = before + t - t0, s = n % S::Stages;
          waits.wait_lane(&C.done[s], (n / S::Stages & 1) ^ 1);
          request(r, t, s);
        }
      __syncwarp();
    }
  } else if (warp == 1) {
    uint32_t n = 0;
    for (int u = u0; u < units; u += step) {
      const Run r = unit(u);
      const uint32_t idesc = umma_idesc_e4m3_f32(kRows, (r.rows + 15) / 16 * 16);
      for (int t = t0; t < t1; ++t, ++n) {
        const uint32_t s = n % S::Stages, phase = n / S::Stages & 1;
        waits.wait_warp(&C.read[s], phase ^ 1, &C.full[s], phase);
        fence_proxy_async_smem();            // rows of x were written by cp.async
        tc_fence_after();
        if (elect_one_sync()) {
          const uint32_t at = base + s * S::Stage, d = C.tmem + s * S::Cols;
#pragma unroll
          for (int j = 0; j < S::Pieces; ++j) {
            const uint64_t w = umma_desc_sw128(at + j * kPiece), x = umma_desc_sw128(at + S::Pieces * kPiece + (Gate ? 0 : j * Tile * kGroup));
#pragma unroll
            for (int i = 0; i < 4; ++i) umma_f8(d + j * Tile, w + i * 2, x + i * 2, idesc, i > 0);
          }
          umma_commit(&C.done[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 4 && in_16) {
    if (u0 < units)
      for (int n = 0; n < t1 - t0; ++n) {
        mbar_arrive(&C.full[n]);
        mbar_arrive(&C.s_full[n]);
      }
  } else if (warp < 4) {
    const int t_ = threadIdx.x - 64, chunk = t_ & 7, r0 = t_ >> 3;
    constexpr int kEach = Tile / 8;          // rows of a thread, eight apart
    static_assert(Tile <= kLoaders, "a thread has the scales of one row");
    uint32_t n = 0;
    for (int u = u0; u < units; u += step) {
      const Run r = unit(u);
      // rows past the unit's are left as they are: nobody reads what comes of them
      auto row = [&](int i) { return static_cast<int64_t>(i < r.rows ? source_row(p, r.row + i) : 0); };
      const uint8_t* src[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) src[i] = p.x + row(r0 + 8 * i) * p.k;
      // Scales: a row of x a thread, two stages ahead in registers. Behind the last group the sums are zero, and so are the scales:
      // the last ones may be infinite.
      const float* xs = p.xs + row(t_) * p.groups;
      const float *ws = p.ws + (static_cast<int64_t>(r.expert) * p.blocks + r.col) * p.groups, *ws2 = ws + static_cast<int64_t>(p.blocks / 2) * p.groups;
      if (u == u0) wait_for_launch_before();
      float x[2][S::Groups], wt[2][S::Pieces];
      auto fetch = [&](int t, int into) {
#pragma unroll
        for (int j = 0; j < S::Groups; ++j) {
          const int g = min(t * S::Groups + j, p.groups - 1);
          x[into][j] = ld_after(xs + g);
          wt[into][j] = __ldg(ws + g);
          if constexpr (Gate) wt[into][1] = __ldg(ws2 + g);
        }
      };
      fetch(t0, 0);
      fetch(t0 + 1, 1);
      for (int t = t0; t < t1; ++t, ++n) {
        const uint32_t s = n % S::Stages, slot = n % kScales;
        waits.wait(&C.done[s], (n / S::Stages & 1) ^ 1);
#pragma unroll
        for (int j = 0; j < S::Groups; ++j) {
          const int k = (t * S::Groups + j) * kGroup + chunk * 16;
          const uint32_t dst = base + s * S::Stage + S::Pieces * kPiece + (j * Tile + r0) * 128 + ((chunk ^ (r0 & 7)) << 4), bytes = k < p.k ? 16 : 0;
          const int at = bytes ? k : 0;
#pragma unroll
          for (int i = 0; i < kEach; ++i)
            if (r0 + 8 * i < r.rows) cp_async16_or_zero(dst + i * 1024, src[i] + at, bytes);
        }
        cp_async_arrive_noinc(&C.full[s]);
        waits.wait(&C.s_empty[slot], (n / kScales & 1) ^ 1);
        auto put = [&](int from) {
#pragma unroll
          for (int j = 0; j < S::Pieces; ++j)
            if (t_ < Tile) C.scale[slot][j][t_] = Gate || t * S::Groups + j < p.groups ? x[from][Gate ? 0 : j] * wt[from][j] : 0.0f;
          fetch(t + 2, from);
        };
        if ((t - t0) & 1) put(1); else put(0);
        mbar_arrive(&C.s_full[slot]);
      }
    }
    cp_async_commit();
    cp_async_wait<0>();                      // of a launch that gave up, too
  } else {
    wait_for_launch_before();
    const int quarter = warp & 3, half = (warp - 4) >> 2, w = warp - 4;
    constexpr int kCols = S::Pieces * S::Mine / 2;            // a stage's sums of a thread are read in two loads
    static_assert(kCols * 2 == S::Pieces * S::Mine && (S::Mine % kCols == 0), "of one piece of the weight each");
    const int i0 = half * S::Mine;                            // first row of x of this thread
    uint32_t n = 0;
    for (int u = u0; u < units; u += step) {
      const Run r = unit(u);
      float2 acc[S::Halves][S::Mine / 2] = {};
      const bool some = i0 < r.rows;
      for (int t = t0; t < t1; ++t, ++n) {
        const uint32_t s = n % S::Stages, ring = n % kScales;
        const float* scale = &C.scale[ring][0][i0];
        waits.wait(&C.s_full[ring], n / kScales & 1, &C.done[s], n / S::Stages & 1);
        tc_fence_after();
        if (some) {
          const uint32_t d = C.tmem + s * S::Cols + i0 + (static_cast<uint32_t>(quarter * 32) << 16);
          constexpr int kNext = S::Mine == kCols ? Tile : kCols;       // where the second load's columns lie
          uint32_t v[2][kCols];
          tmem_ld<kCols>(d, v[0]);
          tmem_ld<kCols>(d + kNext, v[1]);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&C.read[s]);                      // the next product may have the buffer
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            constexpr bool kSame = S::Mine != kCols;                   // both of one piece
            const int j = kSame ? 0 : q, c = kSame ? q * kCols : 0;
#pragma unroll
            for (int i = 0; i < kCols; i += 4) {
              const float4 sc = *reinterpret_cast<const float4*>(scale + j * Tile + c + i);
              float2& a0 = acc[Gate ? j : 0][(c + i) / 2];
              float2& a1 = acc[Gate ? j : 0][(c + i) / 2 + 1];
              a0 = fma2(make_float2(__uint_as_float(v[q][i]), __uint_as_float(v[q][i + 1])), make_float2(sc.x, sc.y), a0);
              a1 = fma2(make_float2(__uint_as_float(v[q][i + 2]), __uint_as_float(v[q][i + 3])), make_float2(sc.z, sc.w), a1);
            }
          }
          __syncwarp();
        } else if (lane == 0) {
          mbar_arrive(&C.read[s]);
        }
        if (lane == 0) mbar_arrive(&C.s_empty[ring]);
      }
      // The unit's sums are complete, for this CTA's groups: each row's go to the CTA that finishes it.
      if (split == 1) {
        float* at = sums + i0 * kRows + quarter * 32 + lane;
#pragma unroll
        for (int h = 0; h < S::Halves; ++h)
#pragma unroll
          for (int i = 0; i < S::Mine; ++i)
            if (i0 + i < r.rows) at[(h * r.rows + i) * kRows] = i & 1 ? acc[h][i / 2].y : acc[h][i / 2].x;
        named_bar_sync(2, kReaders);
        finish<Gate, false>(p, r, sums, 1, r.rows, 0, r.rows, w, lane);
        named_bar_sync(2, kReaders);         // all rows are read
      } else {
        // one unit to a cluster; each CTA finishes a share of its rows
        const int each = (r.rows + split - 1) / split, lo = each * rank, hi = min(lo + each, r.rows);
        if (threadIdx.x == 128) mbar_arrive_expect_tx(&C.joined, static_cast<uint32_t>(max(hi - lo, 0) * split * S::Halves * kRows * 4));
        int owner = i0 / each, in = i0 - owner * each;
#pragma unroll
        for (int i = 0; i < S::Mine; ++i) {
          if (i0 + i >= r.rows) break;
          const uint32_t to = map_to_cta(smem_u32(sums + (rank * S::Halves * each + in) * kRows + quarter * 32 + lane), owner);
          const uint32_t bar = map_to_cta(smem_u32(&C.joined), owner);
#pragma unroll
          for (int h = 0; h < S::Halves; ++h) st_counted(to + h * each * kRows * 4, i & 1 ? acc[h][i / 2].y : acc[h][i / 2].x, bar);
          if (++in == each) {
            in = 0;
            ++owner;
          }
        }
        if (!Gate && p.residual && lo + w < hi && r.col * kRows + lane * 4 < p.n)      // what the results will wait for
          asm volatile("prefetch.global.L1 [%0];" ::"l"(p.residual + (static_cast<int64_t>(r.row) + lo + w) * p.n + r.col * kRows + lane * 4));
        waits.wait_sent(&C.joined, 0);
        finish<Gate, true>(p, r, sums, split, each, lo, hi, w, lane);
      }
    }
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
int few_stages(int tile, bool gate) {
  if (gate) return tile == 16 ? Shape<16, true>::Stages : tile == 32 ? Shape<32, true>::Stages : Shape<64, true>::Stages;
  return tile == 16 ? Shape<16, false>::Stages : tile == 32 ? Shape<32, false>::Stages : Shape<64, false>::Stages;
}
int few_clusters(int split) {
  static int known[kSplit + 1] = {};
  if (split == 1) return kSms;
  if (known[split] == 0) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(static_cast<unsigned>(split));
    c.blockDim = dim3(kThreads);
    c.dynamicSmemBytes = smem_bytes<16, false>();
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = 1;
    int n = 0;
    cudaFuncSetAttribute(few_kernel<16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<16, false>());
    known[split] = cudaOccupancyMaxActiveClusters(&n, few_kernel<16, false>, &c) == cudaSuccess && n > 0 ? n : kSms / split;
  }
  return known[split];
}
int launch_few(const Product& p, const CUtensorMap& weight, int tile, int split, int64_t clusters, cudaStream_t stream) {
  if (p.codes)
    return tile == 16 ? launch<16, true>(p, weight, split, clusters, stream) : tile == 32 ? launch<32, true>(p, weight, split, clusters, stream)
                                                                                              : launch<64, true>(p, weight, split, clusters, stream);
  return tile == 16   ? launch<16, false>(p, weight, split, clusters, stream)
         : tile == 32 ? launch<32, false>(p, weight, split, clusters, stream)
                      : launch<64, false>(p, weight, split, clusters, stream);
}
}  // namespace lin
}  // namespace mono
