// Entries of the block-FP8 products: checks, tensor maps, and which kernel is launched.
#include <cmath>
#include "linear.cuh"

namespace mono {
namespace {

using namespace lin;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Through the runtime, so that the library loads on a machine without a driver.
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(sym);
  }
  return fn;
}

// Bytes [matrices][rows][k], boxes of `box_rows` rows x 128 with the 128-byte swizzle; what lies outside a matrix reads as zero.
bool map_bytes(CUtensorMap* m, const void* base, int rank, uint64_t k, uint64_t rows, uint64_t matrices, uint32_t box_rows) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {k, rows, matrices}, strides[2] = {k, k * rows};
  const cuuint32_t box[3] = {kGroup, box_rows, 1}, steps[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// bf16 or fp32 [rows][n], boxes of 32 rows x 128 bytes with the 128-byte swizzle.
bool map_rows(CUtensorMap* m, const void* base, bool fp32, uint64_t n, uint64_t rows) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint32_t size = fp32 ? 4 : 2, box[2] = {128 / size, 32}, steps[2] = {1, 1};
  const cuuint64_t dims[2] = {n, rows}, strides[1] = {size * n};
  return fn(m, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// What things take, in ns, about: a launch; a stage of the kernel of few rows, a unit of it around its stages, joining the CTAs of a cluster, for each
// row of the tile too; a group of K of a tile of the kernel of many, a unit of it, joining its CTAs, each of them. What is chosen by them was timed in graphs against
// each kernel with each tile and split: 427 products, dense and of 8 to 256 experts, N from 256 to 9216, K from 512 to 7168, 1 to 2048 rows or 6000 tokens, routed evenly and
// not. It takes 2.0% more than the fastest of all these, on average (dense 1.5%, gated 1.2%, experts 2.3%; 40% at most, where routing is uneven); always the tile of 16, 32 or 64
// rows, or the kernel of many, each in its fastest split, 41%, 24%, 29%, 23%.
constexpr int64_t kStart = 2500, kJoin = 700, kJoinRow = 40, kManyGroup = 500, kManyUnit = 2000, kManyGate = 1200, kManyJoin = 1700, kManyPart = 1000;
struct Few {
  int tile;
  int64_t stage, unit;
};
constexpr Few kFew[3] = {{16, 360, 700}, {32, 420, 800}, {64, 620, 1400}};

struct Choice {
  int tile, split;                           // of the kernel of few rows; tile 0: the kernel of many
  int64_t clusters, cost;
};

// The kernel, tile (`only` this one, unless 0) and split with the shortest time by these figures. `likely(t)`: row tiles of t rows; `most(t)`: as
// many as there can be.
template <typename Likely, typename Most>
Choice choose(const Product& p, bool may_many, int only, Likely likely, Most most) {
  const bool gate = p.codes != nullptr;
  const int64_t few_cols = gate ? p.n / 2 / kGroup : div_up(p.n, kGroup), many_cols = gate ? p.n / 2 / kGroup : div_up(p.n, 2 * kGroup);
  const int64_t steps = div_up(p.groups, few_groups(gate));
  Choice best{0, 1, 0, INT64_MAX};
  if (may_many) {
    const int64_t tiles = likely(128) * many_cols;
    best.cost = kStart + div_up(tiles, kSms) * (p.groups * kManyGroup + kManyUnit + (gate ? kManyGate : 0));
    for (int split = 2; split <= 4 && split <= p.groups && !p.offsets; split *= 2) {
      const int64_t cost = kStart + div_up(p.groups, split) * kManyGroup + kManyUnit + (gate ? kManyGate : 0) + kManyJoin + split * kManyPart;
      if (tiles <= few_clusters(split) && cost < best.cost) best = {0, split, tiles, cost};
    }
  }
  for (const Few& f : kFew) {
    if (only && f.tile != only) continue;
    const int64_t units = likely(f.tile) * few_cols, all = most(f.tile) * few_cols;
    for (int split = 1; split <= 8 && split <= steps && (split == 1 || all * split <= kSms); ++split) {
      const int64_t cost = kStart + div_up(units, few_clusters(split)) * (div_up(steps, split) * f.stage + f.unit / split + (split > 1 ? kJoin + kJoinRow * f.tile : 0));
      if (cost < best.cost) best = {f.tile, split, split > 1 || all < kSms ? all : kSms, cost};
    }
  }
  return best;
}

// Of a dense product. Few rows are one row tile, whether they come in 8 bits or in 16: the results are the same bits. (Quantised in the launch, K of 2048
// and 5120 columns: 1 row 5.4 us, 16 rows 6.6; in a launch before it 6.5 and 7.0. From 17 rows on the launch before it is faster: 24 rows 8.6 and
// 7.4, 61 rows, K of 4096 and 2048 columns, 13.4 and 8.7.)
Choice dense(const Product& p) {
  const auto tiles = [&](int t) { return div_up(p.rows, t); };
  const bool few = p.rows <= MONO_LIN_FEW_ROWS;
  return choose(p, !few, few ? 16 : 0, tiles, tiles);
}

int run(Product& p, const uint8_t* weight, const Choice& c, cudaStream_t stream) {
  CUtensorMap w, x, out{}, residual{};
  if (!map_bytes(&w, weight, 3, p.k, p.n, p.experts, c.tile ? 128 : 64)) return MONO_LIN_DRIVER;
  const bool gate = p.codes != nullptr;
  if (c.tile) {
    p.cols = static_cast<int>(gate ? p.n / 2 / kGroup : div_up(p.n, kGroup));
    return launch_few(p, w, c.tile, c.split, c.clusters, stream);
  }
  if (!map_bytes(&x, p.x, 2, p.k, p.x_rows, 1, 128)) return MONO_LIN_DRIVER;
  p.cols = static_cast<int>(gate ? p.n / 2 / kGroup : div_up(p.n, 2 * kGroup));
  if (!gate && p.vec && !map_rows(&out, p.out, p.fp32, p.n, p.rows)) return MONO_LIN_DRIVER;
  if (p.residual && p.vec && !map_rows(&residual, p.residual, false, p.n, p.rows)) return MONO_LIN_DRIVER;
  return launch_many(p, w, x, out, residual, c.split, static_cast<int>(c.clusters), stream);
}

// What every product checks; fills in what follows from the sizes.
int check(Product& p, const uint8_t* weight) {
  if (p.n < 1 || p.k < 16 || p.k % 16 || p.n > (1 << 24) || p.k > (1 << 24) || p.rows < 0 || p.rows > INT32_MAX || p.x_rows < 0 || p.x_rows > INT32_MAX)
    return MONO_LIN_BAD_SIZE;
  if (p.codes && p.n % (2 * kGroup)) return MONO_LIN_BAD_SIZE;
  p.groups = (p.k + kGroup - 1) / kGroup;
  p.blocks = (p.n + kGroup - 1) / kGroup;
  if ((p.rows / 16 + p.experts + 1) * p.blocks > INT32_MAX) return MONO_LIN_BAD_SIZE;      // units are counted in 32 bits
  if (p.rows == 0) return 0;
  if ((!p.raw && (!p.x || !p.xs)) || !weight || !p.ws || !p.status || (p.out == nullptr) == (p.codes == nullptr) || (p.codes == nullptr) != (p.scales == nullptr)) return MONO_LIN_NULL;
  if ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(p.codes)) & 15) return MONO_LIN_ALIGNMENT;
  p.vec = p.n % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.residual)) & 15) == 0;
  return 0;
}

}  // namespace
}  // namespace mono

extern "C" int mono_lin_product(const uint8_t* codes, const float* scales, int64_t rows, const uint8_t* weight, const float* weight_scale, int n, int k,
                                void* out, int out_fp32, const void* residual, uint8_t* codes_out, float* scales_out, int after_quantize,
                                uint32_t* status, mono_lin_stream_t stream) {
  using namespace mono;
  Product p{};
  p.x = codes; p.xs = scales; p.ws = weight_scale;
  p.residual = static_cast<const __nv_bfloat16*>(residual);
  p.out = out; p.codes = codes_out; p.scales = scales_out; p.status = status;
  p.rows = p.x_rows = rows;
  p.n = n; p.k = k; p.experts = 1;
  p.fp32 = out_fp32;
  if (const int rc = check(p, weight)) return rc;
  if (rows == 0) return 0;
  const Choice c = dense(p);
  p.after = after_quantize && c.tile;        // the kernel of many rows is launched when that one has ended
  return run(p, weight, c, stream);
}

namespace mono {
namespace {
// Whether rows in 16 bits are taken: in one row tile, every CTA's groups of K in its ring.
bool takes_rows(const Product& p, Choice& c) {
  if (p.rows > MONO_LIN_FEW_ROWS) return false;
  const bool gate = p.codes != nullptr;
  c = dense(p);
  const int64_t units = gate ? p.n / 2 / kGroup : div_up(p.n, kGroup);
  return units <= c.clusters && div_up(div_up(p.groups, few_groups(gate)), c.split) <= few_stages(c.tile, gate);
}
}  // namespace
}  // namespace mono

extern "C" int mono_lin_takes_rows(int rows, int n, int k, int silu) {
  using namespace mono;
  if (rows < 1 || n < 1 || k < 16 || k % 16 || (silu && n % (2 * kGroup))) return 0;
  Product p{};
  uint8_t any;
  p.codes = silu ? &any : nullptr;
  p.rows = rows;
  p.n = n; p.k = k;
  p.groups = (k + kGroup - 1) / kGroup;
  Choice c;
  return takes_rows(p, c);
}

extern "C" int mono_lin_product_rows(const void* x, int64_t row_stride, int rows, const uint8_t* weight, const float* weight_scale, int n, int k, void* out,
                                     int out_fp32, const void* residual, uint8_t* codes_out, float* scales_out, uint32_t* status, mono_lin_stream_t stream) {
  using namespace mono;
  if (row_stride < 0) return MONO_LIN_BAD_SIZE;
  Product p{};
  p.raw = static_cast<const __nv_bfloat16*>(x);
  p.raw_stride = row_stride;
  p.ws = weight_scale;
  p.residual = static_cast<const __nv_bfloat16*>(residual);
  p.out = out; p.codes = codes_out; p.scales = scales_out; p.status = status;
  p.rows = p.x_rows = rows;
  p.n = n; p.k = k; p.experts = 1;
  p.fp32 = out_fp32;
  if (rows > 0 && !x) return MONO_LIN_NULL;
  if (const int rc = check(p, weight)) return rc;
  if (rows == 0) return 0;
  if (reinterpret_cast<uintptr_t>(x) & 15 || row_stride % 8) return MONO_LIN_ALIGNMENT;
  Choice c;
  if (!takes_rows(p, c)) return MONO_LIN_BAD_SIZE;
  return run(p, weight, c, stream);
}

extern "C" int mono_lin_experts(const uint8_t* codes, const float* scales, int64_t x_rows, const int32_t* tokens, const int32_t* offsets, int64_t rows,
                                int experts, const uint8_t* weight, const float* weight_scale, int n, int k, void* out, uint8_t* codes_out,
                                float* scales_out, uint32_t* status, mono_lin_stream_t stream) {
  using namespace mono;
  if (experts < 1 || experts > MONO_LIN_MAX_EXPERTS) return MONO_LIN_BAD_SIZE;
  Product p{};
  p.x = codes; p.xs = scales; p.ws = weight_scale;
  p.offsets = offsets; p.tokens = tokens;
  p.out = out; p.codes = codes_out; p.scales = scales_out; p.status = status;
  p.rows = rows; p.x_rows = x_rows;
  p.n = n; p.k = k; p.experts = experts;
  if (const int rc = check(p, weight)) return rc;
  if (rows == 0) return 0;
  if (!offsets) return MONO_LIN_NULL;
  if (!tokens && x_rows < rows) return MONO_LIN_BAD_SIZE;
  if (x_rows == 0) return MONO_LIN_BAD_SIZE;
  // the kernel of many rows counts gathered rows in 32 bits, 16 bytes at a time
  const bool may_many = !tokens || x_rows * (k / 16) <= UINT32_MAX;
  // experts that even routing reaches; each has a last tile that is half full
  const double reached = experts * (1.0 - exp(-static_cast<double>(rows) / experts));
  const Choice c = choose(
      p, may_many, 0,
      [&](int t) {
        const double n = static_cast<double>(rows) / t + 0.5 * reached;
        return static_cast<int64_t>(n > reached ? n : reached) + 1;
      },
      [&](int t) { return rows < experts ? rows : experts + rows / t; });
  return run(p, weight, c, stream);
}
