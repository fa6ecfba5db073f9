// Attention over the 4-bit cache for requests of many query rows: chunks and whole prompts.
//
// A CTA takes row blocks (all query heads of one KV head for some tokens) against tiles of 128 keys:
//   S = Q K^T and O += P V on tcgen05 (bf16, fp32 sums in tensor memory), the softmax between them in registers.
// Heads of 64 and 128: two Q tiles of 128 rows, which share the operands made of the codes; the scores of half a tile of keys are made
// while the other half's have their softmax. Heads of 256, whose O alone takes half of tensor memory: one Q tile, whose scores are
// made a tile of keys ahead.
// Nineteen warps, 27 for heads of 256, one CTA on an SM:
//   8 turn codes into operands (8 those of keys, 8 those of values for heads of 256): a block of 16 tokens each, s * c exact in bf16, into a ring of [128 keys x 128 dims] slots in the
//     128-byte-swizzled layout, keys for S with dims along K, values as they are (dims along N). A block's words are what a lane
//     stores as 16 bytes, eight dims in the order 0 4 1 5 2 6 3 7 in which masking leaves them; queries are stored in the same
//     order, and the output is put back from it.
//   1 lists the segments of the CTA's run, a few ahead of the others.
//   2 issue the products, one those of each Q tile (the second has nothing to do for heads of 256).
//   8 do the softmax, a thread to a row: four warps have one Q tile each, or every other tile of keys (the running maximum
//     then goes through shared memory). S is read twice, for the maximum and for the weights, instead of being kept in
//     128 registers. P goes back to tensor memory over S. O is only rescaled when a row's maximum has grown by more than 2^8 (by
//     the warps of that row themselves; sums are fp32, so nothing is lost by a maximum that is a little old).
// Where there are no more (request, KV head, row block) items than CTAs, each gets an equal number of CTAs; else, or where that leaves too much
// to the longest, all tiles are cut into equal runs, one to a CTA. Items that several CTAs have are joined in a fixed order, so results do
// not depend on timing.
// All waits are bounded.
//
// Bound by the tensor cores, 4 D operations for each pair of a query and a key it sees, and behind them by what surrounds them. Seven
// chunks of 350 to 700 tokens behind contexts to 4096 (32 query and 4 KV heads of 128): 245 to 250 us, 0.72 PFLOP/s; a prompt of 8192 (16 query and 2 KV
// heads of 256): 671 to 690 us, 0.80 to 0.82 PFLOP/s. Once the pipeline runs, a tile of 256 rows and 128 keys takes 2050 ns for heads of 128,
// where its products alone would take 1100: the softmax of each half tile takes 1850 cycles of the 2050 that pass between two, on two warps
// of each scheduler that exchange 64 x 32 exponentials a warp and wait for tensor memory. Replacing some of the exponentials by
// polynomials made it slower (243 -> 251 us for one pair in eight), as did keeping the scores in registers (247 -> 265 us), 16
// softmax warps (245 -> 261 us) and their 27 warps' registers (243 -> 263 us). Heads of 256 take 2100 ns for 128 rows and 128 keys:
// their operands, twice as many for each product, pass shared memory three times, 2560 cycles of its bandwidth in 4000.
#include <climits>
#include <type_traits>
#include "kv4_attention.cuh"
#include "kv4_tiles.cuh"
#include "../ptx_sm100.cuh"

namespace mono {
namespace {

using namespace kv4;

constexpr int kSoftmaxWarps = 8;
constexpr int kMmaWarp = 0, kMmaWarps = 2, kPlanWarp = 2, kFirstSoftmax = 3, kFirstFill = kFirstSoftmax + kSoftmaxWarps;
constexpr int kSegs = 4;                    // segments that the roles may be apart
constexpr int kRows = 128;                  // of a product's tile, as kKeys
constexpr int kPanel = kKeys * 128;         // bytes of [128 rows x 64 dims]
constexpr float kLow = -1e38f, kRoom = 8.0f;
constexpr int kHits = 16;                   // words of the rows that see values that are not numbers
// States that one CTA joins. 256 rows over 65536 tokens (4 KV heads of 128, 37 states): 208 us alone, 123 in two steps; four requests of 64 tokens over 16384
// (5 to 7 states) 111, with 6 here 126; 32 tokens (10 states) 137 alone, 114.
constexpr int kJoinAlone = 8;
// In tiles: what joining the states of s CTAs takes, and what runs that begin and end inside items cost beyond parts of one item. One request
// of 200, 400, 800 tokens (32 query and 4 KV heads of 128) takes 21, 23, 32 us in parts of items, 40, 42, 62 in equal runs; one of 3000, with
// more items than CTAs, or of 1600, whose last item is many times its first, 72 us in equal runs. With kCut 4 a chunk of 256 tokens over 4096 goes
// to runs, 70 us instead of 58; with 14 one of 64 over 4096 to parts, 71 instead of
// 63, one of 24 too, 58 instead of 68 (both with 2 + 1.5 t for joining; with 2 + t two of 64 over 2000 take 52 instead of 64).
constexpr int kCut = 8;
__device__ __forceinline__ int join_cost(int s) {
  int t = s;
  if (s > kJoinAlone)
    for (t = 2; t * t < 4 * s;) ++t;        // two steps of sqrt(s)
  return s == 1 ? 0 : 2 + t;
}
constexpr uint64_t kWaitNs = 2000000000ull;

template <int D>
struct Shape {
  static constexpr int NG = D / kGroup;
  static constexpr int Panels = D == 64 ? 1 : 2;        // of a slot
  static constexpr int Slot = Panels * kPanel;
  static constexpr int PerTile = NG / Panels;           // slots of a tile's keys, or of its values
  static constexpr bool Twin = D <= 128;                // two Q tiles (their outputs and scores fill 512 columns); else one, and the softmax warps take turns at the keys
  static constexpr int Rows = Twin ? 2 * kRows : kRows; // of a row block
  // Keys and values are filled in by eight warps each, else by the same eight. Heads of 256 (prompt of 8192): 640 us, else 686; heads of 128
  // (chunks of 700) 263 us, else 243: they do not wait for operands, and 27 warps leave 72 registers.
  static constexpr bool Split = !Twin;
  static constexpr int FillWarps = Split ? 16 : 8, Threads = (kFirstFill + FillWarps) * 32;
  static constexpr int Slots = D == 64 ? 8 : 5;
  static constexpr int Q = (Twin ? 2 : 1) * NG * kPanel;
  static constexpr int Sub = Twin ? 64 : 128;           // keys of a score buffer
  static constexpr int Cols = Twin ? D : D / 2;         // output columns of a thread
  static constexpr int Part = Rows * (D + 2);           // floats of a CTA's state: output, maximum and sum
  static constexpr int HitWords = kHits / NG;           // for each group of dims
  static_assert(HitWords * 32 >= Rows, "a bit for each token of a row block");
};

// Tiles [first, first + count) of keys for a row block: all query heads of a KV head for some tokens of a request.
struct Segment {
  int request, head, q_row, rows;           // first query row; query rows of the block
  int place, begin, end;                    // place of the first token; [begin, end): keys that any row sees
  int first, count;
  int c0, c1;                               // the CTAs that share the item: more than one where count is not all of it
  int whole, more;
};

struct Control {
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  uint64_t full[8], empty[8];               // ring slots
  uint64_t q_full, q_empty;
  uint64_t s_full[4], p_full[4];            // score buffers: 2 Q tile + half of the tile of keys, or tile of keys modulo 2
  uint64_t o_done[2], o_all, o_free;        // a buffer's products with values (for each Q tile), a segment's; the segment's output has been read
  uint32_t tmem, abort, last;
  int found;
  long long found_at;
  long long wsum[32];
  int witems[32], wlongest[32];
  Segment seg[kSegs];
  uint32_t hit[kSegs][kHits];               // for each group of dims, the segment's tokens that see a value there which is not a number
  float top[kRows], sum[2][kRows];          // running maxima; the sums of the two sets of warps
};

template <int D>
constexpr int smem_bytes() { return Shape<D>::Q + Shape<D>::Slots * Shape<D>::Slot + static_cast<int>(sizeof(Control)); }

__device__ __forceinline__ Item item_of(const AttnArgs& a, const Request& r, int rows) {
  return {r.len - r.n, r.n * a.group > a.split_rows ? r.n : 0, r.len, rows / a.group, a.window};
}

// The segments of a CTA's run, one after another: tiles [t0, t1) of an item.
template <int Rows>
struct Walk {
  int b, head, rb, blocks, tiles, t0, t1;
  int64_t at, u, u1, i0;                    // in units of the whole launch
  Request r;
  Item it;
  __device__ __forceinline__ void load(const AttnArgs& a) {
    r = request_of(a, b, false);
    it = item_of(a, r, Rows);
    blocks = it.blocks();
  }
  // The part of item (b, head, rb), which begins at `at`, that lies behind u: its tiles come behind its own kOwn units.
  __device__ __forceinline__ void open() {
    tiles = it.tiles(rb);
    i0 = at + kOwn;
    t0 = static_cast<int>(max(u - i0, static_cast<int64_t>(0)));
    t1 = static_cast<int>(min(static_cast<int64_t>(tiles), u1 - i0));   // t1 <= t0: the run ends before its tiles
  }
  __device__ __forceinline__ bool next(const AttnArgs& a) {   // false behind the run's end
    u = i0 + t1;
    if (u >= u1) return false;
    at = i0 + tiles;
    if (++rb == blocks) {
      rb = 0;
      if (++head == a.hk) {
        head = 0;
        do { ++b; load(a); } while (blocks == 0 && b + 1 < a.batch);
      }
    }
    open();
    return t1 > t0;
  }
};

// ---- waits
// Phase `parity` of a barrier. One that does not come is reported, and from then on no such wait waits: every role runs through its
// loop, whatever is in memory, and the launch ends. The segment list alone is always waited for, so that all roles run
// through the same loops; nobody who keeps it waiting waits for anything else then.
// The clock is only read once in 64 polls: reading it takes longer than most waits.
template <bool Always = false>
__device__ __forceinline__ bool gave_up(uint32_t polls, uint64_t& since, Control& C, const AttnArgs& a) {
  if ((polls & 63u) != 0u) return false;
  volatile uint32_t* stop = &C.abort;
  if (!Always && *stop) return true;
  const uint64_t now = globaltimer_ns();
  if (since == 0) since = now;
  if (now - since <= (Always ? 8 : 1) * kWaitNs) return false;
  report(a.status, kWaitTimeout, blockIdx.x);
  *stop = 1u;
  return true;
}
template <bool Always = false>
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, Control& C, const AttnArgs& a) {
  uint64_t since = 0;
  for (uint32_t polls = 1; !mbar_try_wait(bar, parity) && !gave_up<Always>(polls, since, C, a); ++polls) {}
  __syncwarp();
}

// The same with a result that is the same for the whole warp in a way that the compiler sees, so that the code after it stays in
// uniform control flow: the warp that issues the products, whose descriptors and addresses then stay in uniform registers.
// (Moved there for each instruction, they took longer to issue than the tensor cores to work: 135 cycles instead of 64.)
template <bool Always = false>
__device__ __forceinline__ void wait_warp(uint64_t* bar, uint32_t parity, Control& C, const AttnArgs& a) {
  uint64_t since = 0;
  for (uint32_t polls = 1; !__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity)); ++polls)
    if (__any_sync(0xFFFFFFFFu, gave_up<Always>(polls, since, C, a))) break;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xFFFFFFFFu, x, 0); }

// Reads the segments in order.
struct Reader {
  uint32_t n = 0;
  __device__ __forceinline__ Segment& take(Control& C, const AttnArgs& a) {
    wait<true>(&C.seg_full[n % kSegs], (n / kSegs) & 1, C, a);
    return C.seg[n % kSegs];
  }
  __device__ __forceinline__ void done(Control& C) {    // this warp has no more use for it
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&C.seg_empty[n % kSegs]);
    ++n;
  }
};

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t x, uint32_t y, uint32_t z) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y), *reinterpret_cast<const __nv_bfloat162*>(&z));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t x, uint32_t y) {
  const __nv_bfloat162 r = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// A scale in both halves, and -24 times it (exact: five bits by two).
struct Scale {
  uint32_t s, n;
  __device__ __forceinline__ Scale(uint32_t word, int gi) {
    s = gi & 1 ? __byte_perm(word, word, 0x3232) : __byte_perm(word, word, 0x1010);
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&s), __float2bfloat162_rn(-24.0f));
    n = *reinterpret_cast<const uint32_t*>(&r);
  }
};
// Eight codes of a word times their scale, dims 0 4 1 5 2 6 3 7: a code c + 8 as the top four bits of the mantissa under the
// exponent of 16 is 24 + c, and (24 + c) s - 24 s is exact in one fused multiply-add.
// (Mask and exponent come in registers: with both as immediates masking is two instructions.)
struct Codes { uint32_t mask, magic; };
__device__ __forceinline__ Codes codes() {
  Codes c;
  asm volatile("mov.b32 %0, 0x00780078;" : "=r"(c.mask));
  asm volatile("mov.b32 %0, 0x41804180;" : "=r"(c.magic));
  return c;
}
__device__ __forceinline__ uint4 values8(uint32_t w, const Scale& s, const Codes& c) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(i ? w >> (4 * i - 3) : w << 3), "r"(c.mask), "r"(c.magic));   // (w & mask) | magic
    v[i] = fma_bf16x2(y, s.s, s.n);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void sts128(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// B operand with N along the rows of 128 bytes: 64 dims, then the next panel; 8 keys to 1024 bytes along K.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t at) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((at & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kPanel >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_bf16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
               "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int count) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

constexpr uint32_t kSCol = 0, kOCol = 256;

// ---- the warps that fill the ring
// A lane's words and scales of a block of 16 tokens: of its keys (tokens g, g + 8), or of its values (2t, 2t+1, 2t+8, 2t+9).
// 16 bytes that nobody else on this SM reads: not kept in what shared memory leaves of L1.
__device__ __forceinline__ uint4 ldg_once(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <int D, bool VALUE>
struct Raw {
  static constexpr int NG = D / kGroup, Tok = VALUE ? 4 : 2, SW = (NG + 1) / 2;
  uint4 code[NG];
  uint32_t scale[Tok][SW];

  // The block at p; null: one before or behind all keys, or without a page, read as zeros.
  __device__ __forceinline__ void load(const uint8_t* p, int g, int t, int lane) {
    if (p == nullptr) {
#pragma unroll
      for (int i = 0; i < NG; ++i) code[i] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
#pragma unroll
      for (int i = 0; i < Tok; ++i)
#pragma unroll
        for (int k = 0; k < SW; ++k) scale[i][k] = 0;
      return;
    }
    const uint8_t* c = p + (VALUE ? 8 * D : 0) + lane * 16;
#pragma unroll
    for (int i = 0; i < NG; ++i) code[i] = ldg_once(c + i * 512);
#pragma unroll
    for (int i = 0; i < Tok; ++i) {
      const int tok = VALUE ? 2 * t + (i & 1) + 8 * (i >> 1) : g + 8 * i;
      const uint8_t* sc = p + 16 * D + tok * 4 * NG + (VALUE ? 2 * NG : 0);
      if constexpr (NG == 1) {
        scale[i][0] = __ldg(reinterpret_cast<const uint16_t*>(sc));
      } else if constexpr (NG == 2) {
        scale[i][0] = __ldg(reinterpret_cast<const uint32_t*>(sc));
      } else {
        const uint2 y = __ldg(reinterpret_cast<const uint2*>(sc));
        scale[i][0] = y.x;
        scale[i][1] = y.y;
      }
    }
  }
  // The groups of the next slot in the place of this one's: one slot's code for all of them, which the instruction cache holds.
  __device__ __forceinline__ void next_slot() {
    if constexpr (D == 256) {
#pragma unroll
      for (int i = 0; i < Tok; ++i) scale[i][0] = scale[i][1];
      if constexpr (VALUE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { code[i].x = code[i].z; code[i].y = code[i].w; }
      } else {
        code[0] = code[1];
        code[2] = code[3];
      }
    }
  }
  // Keys: word k (0, 1) of group gi of token g + 8 h. Values: the word of group gi of the u-th token.
  __device__ __forceinline__ uint32_t key_word(int h, int gi, int k) const {
    const int w = h * 2 * NG + 2 * gi + k;
    const uint4& c = code[w >> 2];
    return (w & 3) == 0 ? c.x : (w & 3) == 1 ? c.y : (w & 3) == 2 ? c.z : c.w;
  }
  __device__ __forceinline__ uint32_t value_word(int u, int gi) const {
    const int w = u * NG + gi;
    const uint4& c = code[w >> 2];
    return (w & 3) == 0 ? c.x : (w & 3) == 1 ? c.y : (w & 3) == 2 ? c.z : c.w;
  }
};

// Marks the tokens of a row block that see the key `at` places behind its first token (before it where negative).
__device__ __noinline__ void seen_by(uint32_t* hit, int words, int at, int window) {
  const int to = window > 0 ? at + window : INT_MAX;
  for (int i = 0; i < words; ++i) {
    const int lo = min(max(at - 32 * i, 0), 32), hi = min(max(to - 32 * i, 0), 32);
    if (lo < hi) atomicOr(hit + i, (0xFFFFFFFFu >> (32 - (hi - lo))) << lo);
  }
}

// `warp`: which of the eight blocks of 16 tokens of a tile. A ring is in the order in which the products take it:
// K0 V0 K1 V1 .., or with scores a tile ahead K0 K1 V0 K2 V1 .. V(last). What is stored is loaded again at once, for the tile after.
template <int D, bool KEYS, bool VALUES>
__device__ __forceinline__ void fill_role(const AttnArgs& a, uint8_t* smem, Control& C, int warp, int lane) {
  using S = Shape<D>;
  constexpr int NG = S::NG;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t q_at = smem_u32(smem), ring = q_at + S::Q;
  const int page_shift = a.shift - 4;                   // blocks of a page
  // where a lane stores: the two pieces of a key's row (tokens 8 further on 1024 bytes further), values of tokens 2t and 2t + 1
  const uint32_t k_off = (warp * 16 + g) * 128 + (((2 * t) ^ g) << 4), k_flip = 16;   // 2t and 2t + 1 differ in the lowest bit
  const uint32_t v_off0 = (warp * 16 + 2 * t) * 128 + ((g ^ (2 * t)) << 4), v_off1 = (warp * 16 + 2 * t + 1) * 128 + ((g ^ (2 * t + 1)) << 4);
  const Codes code = codes();
  struct Nothing {};
  uint32_t slot = 0, round = 0;                         // ring position
  Reader reader;
  auto filled = [&]() {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&C.full[slot]);
    if (++slot == S::Slots) { slot = 0; ++round; }
  };
  auto skip = [&]() {                                   // a tile of the other kind
    slot += S::PerTile;
    if (slot >= S::Slots) { slot -= S::Slots; ++round; }
  };
  for (;;) {
    const Segment& w = reader.take(C, a);
    const uint32_t seg = reader.n;
    const int first = w.first, count = w.count, begin = w.begin, end = w.end, more = w.more, request = w.request, place = w.place;
    if (count == 0) break;
    const int64_t head_at = static_cast<int64_t>(w.head) << page_shift, page_blocks = static_cast<int64_t>(a.hk) << page_shift;

    // page of this warp's block of tile `lane` of each 32 tiles; none for a block that no row sees, whose entry may be gone
    int pages = 0;
    auto seen = [&](int blk) { return blk * 16 < end && blk * 16 + 16 > begin; };
    auto block = [&](int j) -> const uint8_t* {
      if ((j & 31) == 0) {
        const int blk = (first + j + lane) * (kKeys / 16) + warp;
        pages = seen(blk) ? page_of(a, request, blk >> page_shift) : 0;
      }
      const int blk = (first + j) * (kKeys / 16) + warp, pg = __shfl_sync(0xFFFFFFFFu, pages, j & 31);
      return pg >= 0 && seen(blk) ? a.cache + (pg * page_blocks + head_at + (blk & ((1 << page_shift) - 1))) * block_bytes(D) : nullptr;
    };
    std::conditional_t<KEYS, Raw<D, false>, Nothing> k;
    std::conditional_t<VALUES, Raw<D, true>, Nothing> v;
    const uint8_t* at = block(0);                       // block whose values are loaded next
    if constexpr (KEYS) k.load(at, g, t, lane);
    if constexpr (VALUES) v.load(at, g, t, lane);

    // queries, in the order of the operands
    wait(&C.q_empty, (seg & 1) ^ 1, C, a);
    {
      constexpr int Lanes = D / 8, Step = 32 / Lanes, N = S::Rows / S::FillWarps / Step, Each = kRows / S::FillWarps;
      const int part = (warp + (KEYS ? 0 : 8)) * Each;  // rows of each Q tile
      const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
      const int col = lane % Lanes, rows = w.rows;
      const bool twin = rows > kRows;
#pragma unroll 1
      for (int i0 = 0; i0 < N; i0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = part + (i0 + i) * Step / Each * kRows + (i0 + i) * Step % Each + lane / Lanes;
          x[i] = make_uint4(0, 0, 0, 0);
          if (row < rows)
            {
              const int tok = by_group(a, row);
              x[i] = __ldg(reinterpret_cast<const uint4*>(a.q + (w.q_row + tok) * a.q_ts + (w.head * a.group + row - tok * a.group) * a.q_hs + 8 * col));
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = part + (i0 + i) * Step % Each + lane / Lanes, tile = (i0 + i) * Step / Each;
          if (tile == 0 || twin)
            sts128(q_at + (tile * NG + (col >> 3)) * kPanel + row * 128 + (((col & 7) ^ (row & 7)) << 4),
                   make_uint4(__byte_perm(x[i].x, x[i].z, 0x5410) ^ flip, __byte_perm(x[i].x, x[i].z, 0x7632) ^ flip,
                              __byte_perm(x[i].y, x[i].w, 0x5410) ^ flip, __byte_perm(x[i].y, x[i].w, 0x7632) ^ flip));
        }
      }
    }
    reader.done(C);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&C.q_full);

    auto store_keys = [&]() {
      if constexpr (KEYS) {
#pragma unroll 1
      for (int s = 0; s < S::PerTile; ++s) {
        const uint32_t base = ring + slot * S::Slot + k_off;
        wait(&C.empty[slot], (round & 1) ^ 1, C, a);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int p = 0; p < S::Panels; ++p) {
            const Scale sc(k.scale[h][0], p);
#pragma unroll
            for (int i = 0; i < 2; ++i) sts128((base ^ (i * k_flip)) + p * kPanel + h * 1024, values8(k.key_word(h, p, i), sc, code));
          }
        filled();
        k.next_slot();
      }
      }
    };
    auto store_values = [&](int j) {
      if constexpr (VALUES) {
      // behind the sequence there may be anything; a group that is not a number must not reach the rows that do not see it
      const int key0 = (first + j) * kKeys + warp * 16;
      if (key0 + 16 > end) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (key0 + 2 * t + (u & 1) + 8 * (u >> 1) >= end)
#pragma unroll
            for (int i = 0; i < Raw<D, true>::SW; ++i) v.scale[u][i] = 0;
      }
      uint32_t sum = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < Raw<D, true>::SW; ++i) sum = add_bf16x2(sum, v.scale[u][i]);
      if (__any_sync(0xFFFFFFFFu, (sum & 0x7FFFu) > 0x7F80u || (sum & 0x7FFF0000u) > 0x7F800000u)) {
        // in the segment's own list: the one before may still be read, and the one before that, where a single tile lies between
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            uint32_t& x = v.scale[u][gi >> 1];
            if ((x >> (gi & 1) * 16 & 0x7FFFu) > 0x7F80u) {
              x &= gi & 1 ? 0x0000FFFFu : 0xFFFF0000u;
              if (g == 0) seen_by(C.hit[seg % kSegs] + gi * S::HitWords, S::HitWords, key0 + 2 * t + (u & 1) + 8 * (u >> 1) - place, a.window);
            }
          }
        __syncwarp();
      }
#pragma unroll 1
      for (int s = 0; s < S::PerTile; ++s) {
        const uint32_t base = ring + slot * S::Slot;
        wait(&C.empty[slot], (round & 1) ^ 1, C, a);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int p = 0; p < S::Panels; ++p)
            sts128(base + (u & 1 ? v_off1 : v_off0) + p * kPanel + (u >> 1) * 1024, values8(v.value_word(u, p), Scale(v.scale[u][0], p), code));
        filled();
        v.next_slot();
      }
      }
    };
    if constexpr (S::Split) {
      for (int j = 0; j < count; ++j) {
        const uint8_t* next = j + 1 < count ? block(j + 1) : nullptr;
        if constexpr (KEYS) {
          store_keys();
          if (j > 0) skip();
          if (j + 1 == count) skip();
          else k.load(next, g, t, lane);
        } else {
          if (j == 0) skip();
          if (j + 1 < count) skip();
          store_values(j);
          if (j + 1 < count) v.load(next, g, t, lane);
        }
      }
    } else {
      store_keys();
      if (count > 1) {
        at = block(1);
        k.load(at, g, t, lane);
      }
      for (int j = 0; j < count; ++j) {
        store_values(j);
        if (j + 1 < count) {
          v.load(at, g, t, lane);
          store_keys();
          if (j + 2 < count) {
            at = block(j + 2);
            k.load(at, g, t, lane);
          }
        }
      }
    }
    if (!more) break;
  }
}

// ---- the warps that issue the products: each its Q tile's, or the first one all of them
template <int D>
__device__ __forceinline__ void mma_role(const AttnArgs& a, uint8_t* smem, Control& C, int tile) {
  using S = Shape<D>;
  const uint32_t q_at = smem_u32(smem), ring = q_at + S::Q, tmem = uniform(C.tmem);
  constexpr uint32_t qk = umma_idesc_bf16_f32(kRows, S::Sub), pv = umma_idesc_bf16_f32(kRows, S::Panels * 64) | (1u << 16);
  uint32_t slot = 0, round = 0;                         // ring position
  Reader reader;
  // Everything between two waits is issued in one go by one lane: what the warp does beside issuing keeps the tensor cores waiting.
  auto advance = [&]() {
    if (++slot == S::Slots) { slot = 0; ++round; }
  };
  auto filled = [&]() { wait_warp(&C.full[slot], round & 1, C, a); };
  // Q tile `tile` against the keys from `key` on of the slot `at` (the s-th of a tile's keys), into the score buffers from `buf` on
  auto scores = [&](int tile, int buf, int s, uint32_t at, int key) {
    const uint64_t dq = umma_desc_sw128(q_at + (tile * S::NG + s * S::Panels) * kPanel), dk = umma_desc_sw128(ring + at * S::Slot + key * 128);
    const uint32_t d = tmem + kSCol + buf * S::Sub;
#pragma unroll
    for (int p = 0; p < S::Panels; ++p)
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_bf16(d, dq + (p * kPanel + k * 32) / 16, dk + (p * kPanel + k * 32) / 16, qk, (s | p | k) != 0);
  };
  // weights of buffer `buf` times the values from `key` on of the slot `at` (the s-th of a tile's values), onto the output of Q tile `tile`
  auto values = [&](int tile, int buf, int s, uint32_t at, int key, bool add) {
    const uint64_t dv = desc_mn_sw128(ring + at * S::Slot + key * 128);
    const uint32_t d = tmem + kOCol + tile * kRows + s * S::Panels * 64, p = tmem + kSCol + buf * S::Sub;
#pragma unroll
    for (int k = 0; k < S::Sub / 16; ++k) umma_bf16_ts(d, p + k * 8, dv + k * 2048 / 16, pv, add || k != 0);
  };
  uint32_t n = 0;                                       // tiles of keys so far (of this warp's Q tile)
  for (;;) {
    const uint32_t seg = reader.n;
    wait_warp<true>(&C.seg_full[seg % kSegs], (seg / kSegs) & 1, C, a);
    const Segment& w = C.seg[seg % kSegs];
    const int count = uniform(w.count), more = uniform(w.more);
    const bool mine = tile == 0 || uniform(w.rows) > kRows;    // else only the ring's slots are handed on
    if (count == 0) break;
    reader.done(C);
    wait_warp(&C.q_full, seg & 1, C, a);
    if constexpr (S::Twin) {
      filled();
      tc_fence_after();
      if (elect_one_sync()) {
        if (mine)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            scores(tile, 2 * tile + half, 0, slot, half * S::Sub);
            umma_commit(&C.s_full[2 * tile + half]);
          }
        umma_commit(&C.empty[slot]);
        if (count == 1) umma_commit(&C.q_empty);
      }
      __syncwarp();
      advance();
#pragma unroll 1
      for (int j = 0; j < count; ++j) {
        const uint32_t v = slot;
        const bool next = j + 1 < count;
        filled();
        advance();
        const uint32_t k = slot;
        if (next) {
          filled();
          advance();
        }
        if (j == 0) wait_warp(&C.o_free, (seg & 1) ^ 1, C, a);
        // half a tile: its products with the values, then the scores of the next tile's half into its buffer
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int b = 2 * tile + half;
          if (mine) wait_warp(&C.p_full[b], n & 1, C, a);
          tc_fence_after();
          if (elect_one_sync()) {
            if (mine) {
              values(tile, b, 0, v, half * S::Sub, j > 0 || half > 0);
              umma_commit(&C.o_done[tile]);
            }
            if (half) umma_commit(&C.empty[v]);
            if (next) {
              if (mine) {
                scores(tile, b, 0, k, half * S::Sub);
                umma_commit(&C.s_full[b]);
              }
              if (half) {
                umma_commit(&C.empty[k]);
                if (j + 2 == count) umma_commit(&C.q_empty);
              }
            }
          }
          __syncwarp();
        }
        n += mine;
      }
    } else {
      // scores of a tile, its keys in PerTile slots
      auto next_scores = [&](uint32_t tile, bool last) {
#pragma unroll 1
        for (int s = 0; s < S::PerTile; ++s) {
          filled();
          tc_fence_after();
          if (elect_one_sync()) {
            scores(0, tile & 1, s, slot, 0);
            umma_commit(&C.empty[slot]);
            if (s + 1 == S::PerTile) {
              umma_commit(&C.s_full[tile & 1]);
              if (last) umma_commit(&C.q_empty);
            }
          }
          __syncwarp();
          advance();
        }
      };
      next_scores(n, count == 1);
#pragma unroll 1
      for (int j = 0; j < count; ++j, ++n) {
        if (j + 1 < count) next_scores(n + 1, j + 2 == count);
        if (j == 0) wait_warp(&C.o_free, (seg & 1) ^ 1, C, a);
        wait_warp(&C.p_full[n & 1], (n >> 1) & 1, C, a);
#pragma unroll 1
        for (int s = 0; s < S::PerTile; ++s) {
          filled();
          tc_fence_after();
          if (elect_one_sync()) {
            values(0, n & 1, s, slot, 0, j > 0);
            umma_commit(&C.empty[slot]);
            if (s + 1 == S::PerTile) umma_commit(&C.o_done[0]);
          }
          __syncwarp();
          advance();
        }
      }
    }
    if (elect_one_sync()) umma_commit(&C.o_all);
    __syncwarp();
    if (!more) {
      wait_warp(&C.o_all, seg & 1, C, a);        // nothing is in flight when tensor memory is given back
      break;
    }
  }
}

// ---- the eight warps of the softmax
template <int D>
__device__ __forceinline__ void softmax_role(const AttnArgs& a, Control& C, int warp, int quarter, int lane) {
  using S = Shape<D>;
  const int set = warp >> 2;                            // which four warps; `quarter`: their lanes of tensor memory
  const int row = (S::Twin ? set * kRows : 0) + quarter * 32 + lane, tile_row = quarter * 32 + lane;
  const int col0 = S::Twin ? 0 : set * S::Cols;         // output columns of this thread, in the epilogue
  const uint32_t lanes = C.tmem + (static_cast<uint32_t>(quarter * 32) << 16), scores0 = lanes + kSCol + set * kKeys;   // its first buffer, or its only one
  const uint32_t output = lanes + kOCol + set * kRows;  // of its Q tile, or its half of the only one
  const float scale = fmaxf(fabsf(a.scale_log2), 1e-37f);     // the queries carry its sign; not 0, for -inf times it stays -inf
  uint32_t n = 0, mine = 0;                             // tiles of keys so far; uses of this set's buffers
  Reader reader;
  for (;;) {
    const Segment& w = reader.take(C, a);
    const int first = w.first, count = w.count, more = w.more;
    if (count == 0) break;
    const bool real = row < w.rows, idle = S::Twin && set == 1 && w.rows <= kRows;
    const int tok = by_group(a, row), place = w.place + tok, hi = real ? place + 1 : 0, lo = a.window > 0 ? place + 1 - a.window : 0;
    // every row of the block sees all of [clear_lo, clear_hi)
    const int clear_hi = w.place + 1, clear_lo = a.window > 0 ? w.place + by_group(a, w.rows - 1) + 1 - a.window : 0;
    float m = kLow, l = 0.0f;
    // halves of tiles of keys; or, where the sets take turns, every other tile: the first or the second of the segment first
    const int steps = idle ? 0 : S::Twin ? 2 * count : count;
    for (int j = S::Twin ? 0 : (n ^ set) & 1; j < steps; j += S::Twin ? 1 : 2, ++mine) {
      const int key0 = first * kKeys + j * S::Sub, buf = S::Twin ? 2 * set + (j & 1) : set;
      const uint32_t scores = scores0 + (S::Twin ? (j & 1) * S::Sub : 0);
      wait(&C.s_full[buf], (S::Twin ? mine >> 1 : mine) & 1, C, a);
      tc_fence_after();
      const bool mask = key0 < clear_lo || key0 + S::Sub > clear_hi;
      const int from = lo - key0, to = hi - key0;
      if (mask) {                           // written back, so that what follows needs no masks
#pragma unroll 1
        for (int c = 0; c < S::Sub; c += 16) {
          uint32_t s[16];
          tmem_ld16(scores + c, s);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < from || c + i >= to) s[i] = 0xFF800000u;
          tmem_st16(scores + c, s);
        }
        tmem_st_wait();
      }
      uint32_t r0[16], r1[16];              // 16 columns in work, 16 on their way
      float *s0 = reinterpret_cast<float*>(r0), *s1 = reinterpret_cast<float*>(r1);
      float x = -INFINITY, y = -INFINITY;
      auto most = [&](const float* s) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          x = fmaxf(x, fmaxf(s[i], s[i + 1]));
          y = fmaxf(y, fmaxf(s[i + 2], s[i + 3]));
        }
      };
      tmem_ld16(scores, r0);
#pragma unroll 1
      for (int c = 0; c < S::Sub; c += 32) {
        tmem_ld_wait();
        tmem_ld16(scores + c + 16, r1);
        most(s0);
        tmem_ld_wait();
        tmem_ld16(scores + ((c + 32) & (S::Sub - 1)), r0);   // after the last the first again
        most(s1);
      }
      x = fmaxf(x, y) * scale;
      float before = m;                     // the maximum that O stands at
      if constexpr (!S::Twin) {
        if (j > 0) {
          named_bar_sync(1 + (set ^ 1) * 4 + quarter, 64);
          before = C.top[tile_row];
        }
      }
      float now = before;
      const bool grow = __any_sync(0xFFFFFFFFu, x > before + kRoom);
      if (grow) now = fmaxf(before, x);
      if constexpr (!S::Twin) {
        C.top[tile_row] = now;
        if (j + 1 < count) bar_arrive(1 + set * 4 + quarter, 64);
      }
      l *= ex2(m - now);
      m = now;
      if (grow && j > 0) {
        // the products of the buffer before have to be in O; no others are missing, for this one's scores came after them
        if constexpr (S::Twin) wait(&C.o_done[set], (mine - 1) & 1, C, a);
        else wait(&C.o_done[0], (n + j - 1) & 1, C, a);
        tc_fence_after();
        tmem_ld_wait();
        const float by = ex2(before - now);
#pragma unroll 1
        for (int i = 0; i < D; i += 16) {
          uint32_t o[16];
          tmem_ld16(lanes + kOCol + (S::Twin ? set * kRows : 0) + i, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
          tmem_st16(lanes + kOCol + (S::Twin ? set * kRows : 0) + i, o);
        }
      }
      float2 sum = make_float2(0.0f, 0.0f);
      auto weigh = [&](const float* s, uint32_t to) {
        uint32_t p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float2 e = fma2(make_float2(s[2 * i], s[2 * i + 1]), make_float2(scale, scale), make_float2(-m, -m));
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum = add2(sum, e);
          p[i] = pack_bf16x2(e.x, e.y);
        }
        tmem_st8(to, p);                    // over scores that have been read: 8 columns of weights to 16
      };
#pragma unroll 1
      for (int c = 0; c < S::Sub; c += 32) {
        tmem_ld_wait();
        tmem_ld16(scores + c + 16, r1);
        weigh(s0, scores + c / 2);
        tmem_ld_wait();
        if (c + 32 < S::Sub) tmem_ld16(scores + c + 32, r0);
        weigh(s1, scores + c / 2 + 8);
      }
      l += sum.x + sum.y;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&C.p_full[buf]);
    }
    n += count;
    if constexpr (!S::Twin) {               // the sets' sums, at the last maximum
      named_bar_sync(9, 256);
      const float last = C.top[tile_row];
      C.sum[set][tile_row] = l * ex2(m - last);
      m = last;
      named_bar_sync(9, 256);
      l = C.sum[0][tile_row] + C.sum[1][tile_row];
    }
    wait(&C.o_all, reader.n & 1, C, a);
    tc_fence_after();
    // groups that are not numbers and that this row sees
    uint32_t nans = 0;
#pragma unroll
    for (int gi = 0; gi < S::NG; ++gi)
      nans |= (*static_cast<volatile uint32_t*>(&C.hit[reader.n % kSegs][gi * S::HitWords + (tok >> 5)]) >> (tok & 31) & 1u) << gi;
    const bool whole = w.whole;
    const int c0 = w.c0, c1 = w.c1;
    float* part = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (static_cast<int>(blockIdx.x) == c0 ? 1 : 0)) * S::Part;
    auto write_out = [&](int rw, int d, const float (&x)[8], float inv) {       // eight dims, in the order of the operands
      const int in = by_group(a, rw), tk = w.q_row + in, hd = w.head * a.group + rw - in * a.group;
      float y[8] = {x[0] * inv, x[2] * inv, x[4] * inv, x[6] * inv, x[1] * inv, x[3] * inv, x[5] * inv, x[7] * inv};
      *reinterpret_cast<uint4*>(a.out + (static_cast<int64_t>(tk) * a.hq + hd) * D + d) = pack_bf16x8(y);
    };
    auto inverse = [](float sum) { return sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum; };
    auto write_lse = [&](int rw, float mx, float sum) {
      const int in = by_group(a, rw), tk = w.q_row + in, hd = w.head * a.group + rw - in * a.group;
      a.lse[static_cast<int64_t>(tk) * a.hq + hd] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
    };
    const float inv = inverse(l);
    if (!idle) {
      __nv_bfloat16* to = a.out + (static_cast<int64_t>(w.q_row + tok) * a.hq + w.head * a.group + row - tok * a.group) * D + col0;
#pragma unroll 1
      for (int i = 0; i < S::Cols; i += 16) {
        uint32_t o[16];
        tmem_ld16(output + i, o);
        tmem_ld_wait();
        if (real) {
          const float nan = nans >> ((col0 + i) >> 6) & 1u ? __uint_as_float(0x7FC00000u) : 0.0f;
          if (whole) {
#pragma unroll
            for (int k = 0; k < 16; k += 8) {
              float x[8];
#pragma unroll
              for (int c = 0; c < 8; ++c) x[c] = fmaf(__uint_as_float(o[k + c]), inv, nan);
              const float y[8] = {x[0], x[2], x[4], x[6], x[1], x[3], x[5], x[7]};
              *reinterpret_cast<uint4*>(to + i + k) = pack_bf16x8(y);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 16; k += 4)
              __stcg(reinterpret_cast<float4*>(part + row * D + col0 + i + k), make_float4(__uint_as_float(o[k]) + nan, __uint_as_float(o[k + 1]) + nan,
                                                                                           __uint_as_float(o[k + 2]) + nan, __uint_as_float(o[k + 3]) + nan));
          }
        }
      }
    }
    tc_fence_before();
    mbar_arrive(&C.o_free);
    if (whole) {
      if (real && col0 == 0 && a.lse) write_lse(row, m, l);
    } else {
      if (real && col0 == 0) __stcg(reinterpret_cast<float2*>(part + S::Rows * D + 2 * row), make_float2(m, l));
      // Whoever comes last joins. Where more than kJoinAlone CTAs have the item, first the last of each `group` of them joins the group's
      // states into the one of its first CTA, then the last group's last CTA those of the groups.
      const int all = c1 - c0 + 1;
      int group = all;
      if (all > kJoinAlone)
        for (group = 1; group * group < all;) ++group;
      const int groups = (all + group - 1) / group;
      int first = c0 + (static_cast<int>(blockIdx.x) - c0) / group * group, n = min(group, c1 + 1 - first), step = 1;
      bool final = groups == 1;
      uint32_t* counter = a.counters + MONO_ATTN_SMS + 2 * first + (first == c0 ? 1 : 0);
      for (;;) {
        __threadfence();
        named_bar_sync(9, 256);
        if (warp == 0 && lane == 0) {
          const uint32_t before = atomicAdd(counter, 1u);
          C.last = before == static_cast<uint32_t>(n - 1);
          if (C.last) *counter = 0;
          __threadfence();
        }
        named_bar_sync(9, 256);
        if (!C.last) break;
        auto state = [&](int i) {
          const int c = first + i * step;
          return a.partial + (static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * S::Part;
        };
        for (int idx = warp * 32 + lane; idx < w.rows * (D / 8); idx += 256) {
          const int rw = idx / (D / 8), d = idx % (D / 8) * 8;
          float mx = kLow, sum = 0.0f, x[8] = {};
          for (int i = 0; i < n; ++i) {
            const float* from = state(i);
            const float2 ms = __ldcg(reinterpret_cast<const float2*>(from + S::Rows * D + 2 * rw));
            const float4 p0 = __ldcg(reinterpret_cast<const float4*>(from + rw * D + d)), p1 = __ldcg(reinterpret_cast<const float4*>(from + rw * D + d + 4));
            const float to = fmaxf(mx, ms.x), old = ex2(mx - to), by = ex2(ms.x - to);
            mx = to;
            sum = fmaf(ms.y, by, sum * old);
            x[0] = fmaf(p0.x, by, x[0] * old); x[1] = fmaf(p0.y, by, x[1] * old);
            x[2] = fmaf(p0.z, by, x[2] * old); x[3] = fmaf(p0.w, by, x[3] * old);
            x[4] = fmaf(p1.x, by, x[4] * old); x[5] = fmaf(p1.y, by, x[5] * old);
            x[6] = fmaf(p1.z, by, x[6] * old); x[7] = fmaf(p1.w, by, x[7] * old);
          }
          if (final) {
            write_out(rw, d, x, inverse(sum));
            if (d == 0 && a.lse) write_lse(rw, mx, sum);
          } else {                          // nobody else reads these eight
            __stcg(reinterpret_cast<float4*>(state(0) + rw * D + d), make_float4(x[0], x[1], x[2], x[3]));
            __stcg(reinterpret_cast<float4*>(state(0) + rw * D + d + 4), make_float4(x[4], x[5], x[6], x[7]));
          }
        }
        if (final) break;
        named_bar_sync(9, 256);             // all have read the maxima and sums that are written now
        for (int rw = warp * 32 + lane; rw < w.rows; rw += 256) {
          float mx = kLow, sum = 0.0f;
          for (int i = 0; i < n; ++i) {
            const float2 ms = __ldcg(reinterpret_cast<const float2*>(state(i) + S::Rows * D + 2 * rw));
            const float to = fmaxf(mx, ms.x);
            sum = fmaf(ms.y, ex2(ms.x - to), sum * ex2(mx - to));
            mx = to;
          }
          __stcg(reinterpret_cast<float2*>(state(0) + S::Rows * D + 2 * rw), make_float2(mx, sum));
        }
        first = c0;
        step = group;
        n = groups;
        final = true;
        counter = a.counters + c0;
      }
    }
    reader.done(C);
    if (!more) break;
  }
}

// ---- the warp that lists the segments
template <int Rows>
__device__ __forceinline__ void plan_role(const AttnArgs& a, Control& C, int share, int64_t per, int64_t u0, int64_t u1, int lane) {
  Walk<Rows> w;
  w.b = C.found;
  w.load(a);
  auto publish = [&](uint32_t n, const Walk<Rows>& v, int c0, int c1, bool more) {
    if (lane < kHits) C.hit[n % kSegs][lane] = 0;
    __syncwarp();
    if (lane == 0) {
      const int tok = v.rb * v.it.tb;
      C.seg[n % kSegs] = {v.b, v.head, v.r.first + tok, min(v.it.tb, v.it.n - tok) * a.group, v.it.place0 + tok, v.it.begin(v.rb), v.it.seen(v.rb),
                          v.it.first_tile(v.rb) + v.t0, max(v.t1 - v.t0, 0), c0, c1, v.t1 - v.t0 == v.tiles, more};
      mbar_arrive(&C.seg_full[n % kSegs]);
    }
  };
  if (share) {                              // this CTA's part of item u0
    const int item = static_cast<int>(u0 - C.found_at);
    w.head = item / w.blocks;
    w.rb = item - w.head * w.blocks;
    w.tiles = w.it.tiles(w.rb);
    const int parts = min(share, w.tiles), c0 = static_cast<int>(u0) * share, part = static_cast<int>(blockIdx.x) - c0;
    w.t0 = part < parts ? w.tiles * part / parts : 0;
    w.t1 = part < parts ? w.tiles * (part + 1) / parts : 0;
    publish(0, w, c0, c0 + parts - 1, false);
    return;
  }
  w.u = u0;
  w.u1 = u1;
  {  // the head and row block that u0 lies in: the lanes bisect together, 32 places at a time
    const int64_t each = tiles_before(w.it, w.blocks), off = u0 - C.found_at;
    w.head = static_cast<int>(off / each);
    const int64_t rest = off - w.head * each;
    int low = 0, high = w.blocks;           // tiles_before(low) <= rest < tiles_before(high)
    while (high - low > 1) {
      const int step = (high - low + 31) / 32, at = min(low + lane * step, high);
      const bool below = at < high && tiles_before(w.it, at) <= rest;
      const int k = 31 - __clz(static_cast<int>(__ballot_sync(0xFFFFFFFFu, below)));    // lane 0's place is always below
      high = min(low + (k + 1) * step, high);
      low += k * step;
    }
    w.rb = low;
    w.at = C.found_at + w.head * each + tiles_before(w.it, low);
  }
  w.open();
  for (uint32_t n = 0;; ++n) {
    wait<true>(&C.seg_empty[n % kSegs], ((n / kSegs) & 1) ^ 1, C, a);
    const Walk<Rows> v = w;
    const bool more = w.t1 > w.t0 && w.next(a);   // else: a run of nothing but an item's own units
    publish(n, v, static_cast<int>(v.i0 / per), static_cast<int>((v.i0 + v.tiles - 1) / per), more);
    if (!more) break;
  }
}

template <int D>
__global__ __launch_bounds__(Shape<D>::Threads, 1) void prompt_kernel(const AttnArgs a) {
  using S = Shape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Control& C = *reinterpret_cast<Control*>(smem + S::Q + S::Slots * S::Slot);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // this CTA's run of all tiles
  const int chunk = (a.batch + S::Threads - 1) / S::Threads;
  long long mine = 0;
  int mine_items = 0, longest = 0;
  for (int b = tid * chunk; b < min((tid + 1) * chunk, a.batch); ++b) {
    const Item it = item_of(a, request_of(a, b, blockIdx.x == 0), S::Rows);
    const int blocks = it.blocks();
    mine += tiles_before(it, blocks) * a.hk;
    mine_items += blocks * a.hk;
    if (blocks) longest = max(longest, max(it.tiles(blocks - 1), it.tiles(max(blocks - 2, 0))));
  }
  long long upto = mine;
  int upto_items = mine_items;
  longest = __reduce_max_sync(0xFFFFFFFFu, longest);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long x = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    const int y = __shfl_up_sync(0xFFFFFFFFu, upto_items, d);
    if (lane >= d) { upto += x; upto_items += y; }
  }
  if (lane == 31) { C.wsum[warp] = upto; C.witems[warp] = upto_items; C.wlongest[warp] = longest; }
  __syncthreads();
  long long total = 0;
  int items = 0;
  for (int i = 0; i < S::Threads / 32; ++i) {
    if (i < warp) { upto += C.wsum[i]; upto_items += C.witems[i]; }
    total += C.wsum[i];
    items += C.witems[i];
    longest = max(longest, C.wlongest[i]);
  }
  const int ctas = static_cast<int>(gridDim.x);
  const long long per = (total + ctas - 1) / ctas;
  // CTAs for each item, by what the longest item then takes (0: equal runs)
  int share = 0;
  if (items > 0 && items <= ctas) {
    uint32_t best = 0xFFFFFFFFu;
    for (int s = 1 + lane; s <= min(ctas / items, longest); s += 32) best = min(best, static_cast<uint32_t>((longest + s - 1) / s + join_cost(s)) << 8 | s);
    best = __reduce_min_sync(0xFFFFFFFFu, best);
    if ((best >> 8) <= per + kCut) share = best & 255;
  }
  // where this CTA begins: its run of all tiles, or its item
  const long long u0 = share ? blockIdx.x / share : blockIdx.x * per, u1 = share ? items : min(u0 + per, total);
  if (u0 >= u1) return;                     // the whole CTA, before anything is allocated
  const long long before = share ? upto_items - mine_items : upto - mine, behind = share ? upto_items : upto;
  if (before <= u0 && u0 < behind) {
    long long at = before;
    int b = tid * chunk;
    if (chunk > 1)
      for (;; ++b) {
        const Item it = item_of(a, request_of(a, b, false), S::Rows);
        const long long cost = (share ? it.blocks() : tiles_before(it, it.blocks())) * a.hk;
        if (at + cost > u0) break;
        at += cost;
      }
    C.found = b;
    C.found_at = at;
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&C.tmem, 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    constexpr int issuers = S::Twin ? kMmaWarps : 1;
    for (int i = 0; i < S::Slots; ++i) { mbar_init(&C.full[i], 8); mbar_init(&C.empty[i], issuers); }
    for (int i = 0; i < kSegs; ++i) { mbar_init(&C.seg_full[i], 1); mbar_init(&C.seg_empty[i], kSoftmaxWarps + S::FillWarps + issuers); }
    mbar_init(&C.q_full, S::FillWarps);
    mbar_init(&C.q_empty, issuers);
    for (int i = 0; i < 4; ++i) { mbar_init(&C.s_full[i], 1); mbar_init(&C.p_full[i], kSoftmaxWarps * 16); }
    mbar_init(&C.o_done[0], 1);
    mbar_init(&C.o_done[1], 1);
    mbar_init(&C.o_all, issuers);
    mbar_init(&C.o_free, kSoftmaxWarps * 32);
    mbar_init_fence();
    C.abort = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp >= kFirstFill + 8) { if constexpr (S::Split) fill_role<D, false, true>(a, smem, C, warp - kFirstFill - 8, lane); }
  else if (warp >= kFirstFill) fill_role<D, true, !S::Split>(a, smem, C, warp - kFirstFill, lane);
  else if (warp >= kFirstSoftmax) softmax_role<D>(a, C, warp - kFirstSoftmax, warp & 3, lane);
  else if (warp < kMmaWarp + kMmaWarps) { if (S::Twin || warp == kMmaWarp) mma_role<D>(a, smem, C, S::Twin ? uniform(warp - kMmaWarp) : 0); }
  else plan_role<S::Rows>(a, C, share, per, u0, u1, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (C.abort) {                            // products may be in flight that nobody has waited for; they take microseconds
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000) __nanosleep(10000);
  }
  if (warp == kMmaWarp) tmem_dealloc(C.tmem, 512);
}

template <int D>
int launch(const AttnArgs& a, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(prompt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<D>());
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  prompt_kernel<D><<<MONO_ATTN_SMS, Shape<D>::Threads, smem_bytes<D>(), stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

static_assert(smem_bytes<256>() <= 232448 && smem_bytes<128>() <= 232448, "shared memory of an SM");

}  // namespace

namespace kv4 {
size_t prompt_partial_floats() { return static_cast<size_t>(MONO_ATTN_SMS) * 2 * (Shape<128>::Part > Shape<256>::Part ? Shape<128>::Part : Shape<256>::Part); }
int prompt(const AttnArgs& a, int head_dim, cudaStream_t stream) {
  return head_dim == 64 ? launch<64>(a, stream) : head_dim == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}
}  // namespace kv4
}  // namespace mono
