// Attention over the 4-bit cache for requests of few query rows: one token, or a few guessed ahead. The rows of all query heads
// that share a KV head are taken together, in blocks of 8 or 16.
//
// What bounds it is the cache, read once: 17/16 bytes for each key and value dim of a token. With 32 query and 4 KV heads of 128, 64
// sequences of 4096 to 8192 tokens take 63.5 us, 3.4 TB/s, two of 131072 take 45.9 us. Each 65536 tokens more in both add 13.5 us, 5.3 TB/s
// (a copy has 6.55): what lies between is the launch, the division of the work, the first copies' way and the join, some 13.8 us,
// which is also what one token after 777 others takes. A CTA-wide product of 64 or more
// rows on tcgen05 would be nearly all padding here, so the products go through mma.sync with the keys (and the dims of the
// values) as its 16 rows and the query rows as its 8 columns, and what is made cheap is the way of a code into an operand:
//  * A key's code c + 8 is left where it is and masked out of its word: as the low bits of an fp16 it is the subnormal
//    (c + 8) 2^-24, four bits higher 2^-20. Half an instruction for a value; no conversion, no subtraction. The 16 goes into the
//    query, the 8 is taken off the sum over a group: its accumulator starts at -8 sum(q). The sum is of 64 products of one size,
//    so little is lost by it.
//  * A value's code gets the exponent of 128 in the same instruction that masks it, and a packed subtraction leaves c itself.
//    Taking 8 sum(p) off at the end instead would be cheaper, but a dim in which the token with nearly all of the weight
//    has the code 0 would then be left with that token's rounding.
//  * Scales meet the sums, not the values: a group's part of q.k is multiplied by the key's scale as fp32, a row's weight by
//    the value's scale before it is rounded. Weights are bf16, whose exponents hold any product of the two: fp16 would round
//    them eight times finer and lose those below 2^-31 of the largest, which a dim of that kind shows too.
//  * The maximum is only moved when a weight would pass 2^8: one vote per step instead of a reduction.
//
// The work is all (request, KV head, row block) items, in steps of 256 tokens. Where there are fewer items than CTAs each gets an equal
// number of CTAs, which share its steps evenly; else, or where that leaves too much to the longest item, all steps are cut
// into equal runs, one to a CTA (kOwn steps more for an item's own cost), whatever items they lie in. An item that several CTAs
// have is joined by whoever of them finishes last, in the order of its tokens, so the result does not depend on which one that
// is. Each warp has every eighth pair of blocks, its own ring of copies in flight, and its own softmax state; the copies of a
// CTA's next item are on their way while the states of one are joined.
#include "kv4_attention.cuh"

namespace mono {
namespace {

using namespace kv4;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 32 * kWarps;          // tokens of one step of a CTA
// In steps: what an item costs beside them in a run; what joining costs. With kJoin 12 one sequence of 1500 to 3000 tokens is not divided
// and takes 21 us instead of 13; with 6 sixteen of 1000 to 2000 (heads of 256) take 23 us, with 3 or less 17; one of 777 takes 15.1 with 3, 14.6 with 2.
constexpr int kOwn = 1, kJoin = 2;
constexpr float kLow = -1e38f;              // below every score
constexpr float kRoom = 8.0f;               // log2 of what a weight may grow to before the maximum is moved

// 16 bytes, of which the first `bytes` are read and the others zeros.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1,
                                         float c2, float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma16816_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// c + 8 in the low four bits of both halves, to c as bf16.
// (mask and exponent in registers: with both as immediates it is two instructions)
__device__ __forceinline__ uint32_t signed_code(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(magic));   // (x & mask) | magic
  const uint32_t off = 0x43084308u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&y), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float half_lo(uint32_t x) { return __half2float(__ushort_as_half(static_cast<unsigned short>(x & 0xFFFFu))); }
__device__ __forceinline__ float half_hi(uint32_t x) { return __half2float(__ushort_as_half(static_cast<unsigned short>(x >> 16))); }

template <int D, int NT>
struct Shape {
  static constexpr int NG = D / kGroup;
  static constexpr int Rows = 8 * NT;                   // query rows of an item
  static constexpr int Block = block_bytes(D);
  static constexpr int Stage = 2 * Block;               // a pair of blocks
  static constexpr int Stages = D == 64 ? 3 : 2;
  static constexpr int Ring = Stages * Stage;           // of a warp
  static constexpr int Part = Rows * (D + 2);           // floats of a warp's or a CTA's state: output, maximum, sum
  static constexpr int State = (Part * 4 + 15) / 16 * 16;
  static constexpr int Smem = kWarps * (Ring + State);
  // 16 warps on an SM where their registers allow it, 8 of up to 255 registers where not
  static constexpr int PerSm = D == 64 || (D == 128 && NT == 1) ? 2 : 1;
  static constexpr int Ctas = MONO_ATTN_SMS * PerSm;
};

// Steps of one item of a request; 0 if the request is not this kernel's.
template <int Rows>
__device__ __forceinline__ void cost_of(const AttnArgs& a, const Request& r, int& items, int& steps, int& lo) {
  const int rows = r.n * a.group;
  items = rows == 0 || rows > a.split_rows ? 0 : a.hk * ((rows + Rows - 1) / Rows);
  lo = a.window > 0 ? max(r.len - r.n + 1 - a.window, 0) & ~(kTokens - 1) : 0;
  steps = max(1, (r.len - lo + kStep - 1) / kStep);
}

// Tokens [k0, k1) of an item: a block of `rows` query rows of a KV head.
struct Part {
  int b, head, rb, rows, k0, k1;
  int i0, i1, u, e;                          // steps of the item, and of this part
  int c0, c1;                                // the CTAs that share the item
  int first, place0, len;                    // of the request: its first query row, the place of it, the length
};

template <int D, int NT>
__global__ __launch_bounds__(kThreads, Shape<D, NT>::PerSm) void decode_kernel(const AttnArgs a) {
  using S = Shape<D, NT>;
  constexpr int NG = S::NG;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_sum[kWarps][3];
  __shared__ int s_found[2];
  __shared__ int s_last;
  __shared__ Part s_part;                    // the part whose states are joined
  __shared__ float s_weight[S::Rows][32], s_old[S::Rows], s_sums[S::Rows], s_top[S::Rows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint32_t mask4, magic;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask4));
  asm volatile("mov.b32 %0, 0x43004300;" : "=r"(magic));
  uint8_t* ring = smem + warp * S::Ring;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  float* states = reinterpret_cast<float*>(smem + kWarps * S::Ring);

  // All steps, all items and the longest item; the sums before each thread's requests.
  const int chunk = (a.batch + kThreads - 1) / kThreads;
  // Sums of steps stay at the largest integer: more than a launch could do in seconds, and reported (2^31 steps are 34 TB of a cache of heads of 64).
  auto add = [](int x, int y) { return static_cast<int>(min(static_cast<uint32_t>(x) + static_cast<uint32_t>(y), 0x7FFFFFFFu)); };
  int mine = 0, mine_items = 0, longest = 0;
  for (int b = tid * chunk; b < min((tid + 1) * chunk, a.batch); ++b) {
    int items, steps, lo;
    cost_of<S::Rows>(a, request_of(a, b, blockIdx.x == 0), items, steps, lo);
    mine = add(mine, static_cast<int>(min(static_cast<int64_t>(items) * (steps + kOwn), static_cast<int64_t>(INT32_MAX))));
    mine_items += items;
    if (items) longest = max(longest, steps);
  }
  int upto = mine, upto_items = mine_items;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xFFFFFFFFu, upto, d), y = __shfl_up_sync(0xFFFFFFFFu, upto_items, d);
    longest = max(longest, __shfl_xor_sync(0xFFFFFFFFu, longest, d));
    if (lane >= d) { upto = add(upto, x); upto_items += y; }
  }
  if (lane == 31) { s_sum[warp][0] = upto; s_sum[warp][1] = upto_items; s_sum[warp][2] = longest; }
  __syncthreads();
  int total = 0, all_items = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) { upto = add(upto, s_sum[w][0]); upto_items += s_sum[w][1]; }
    total = add(total, s_sum[w][0]);
    all_items += s_sum[w][1];
    longest = max(longest, s_sum[w][2]);
  }
  if (total == INT32_MAX) {
    if (blockIdx.x == 0 && tid == 0) report(a.status, kTooLong, 0);
    return;
  }
  const int ctas = static_cast<int>(gridDim.x), per = (total + ctas - 1) / ctas;
  // CTAs for each item (0: equal runs), from what the slowest CTA then has
  int share = 0;
  if (all_items > 0 && all_items <= ctas) {
    const int most = min(ctas / all_items, longest), split = (longest + most - 1) / most + kJoin;
    share = split < longest ? most : 1;
    if (min(split, longest) > per + kJoin) share = 0;
  }
  // where this CTA begins: its run [u0, u1) of all steps, or its item and its part of that
  const int u0 = share ? static_cast<int>(blockIdx.x) / share : static_cast<int>(blockIdx.x) * per, u1 = share ? all_items : min(u0 + per, total);
  if (u0 >= u1) return;
  const int before = share ? upto_items - mine_items : upto - mine, behind = share ? upto_items : upto;
  if (before <= u0 && u0 < behind) {
    int at = before, b = tid * chunk;
    if (chunk > 1)
      for (;; ++b) {
        int items, steps, lo;
        cost_of<S::Rows>(a, request_of(a, b, false), items, steps, lo);
        const int cost = share ? items : items * (steps + kOwn);
        if (at + cost > u0) break;
        at += cost;
      }
    s_found[0] = b;
    s_found[1] = at;
  }
  __syncthreads();

  // the parts of the run, one after another, and the copies of a part's first blocks
  int walk_b = s_found[0], walk_at = s_found[1], walk_u = u0;   // request, where its items begin, where the next part begins
  Part p;
  int count, pages, later, wstage = 0, rstage = 0;              // this warp's pairs of blocks; pages of 32 blocks and the 32 after
  const int page_shift = a.shift - 4, in_page = (1 << page_shift) - 1;
  const int page_bytes = (a.hk << page_shift) * S::Block;
  // the 32 blocks that this warp's pairs i0 .. i0 + 15 are: lane 2 i + h has block h of pair i
  auto pages_of = [&](int i0) {
    const int blk = (p.k0 >> 4) + 2 * (warp + kWarps * (i0 + (lane >> 1))) + (lane & 1);
    return blk * 16 < p.k1 ? page_of(a, p.b, blk >> page_shift) : 0;
  };
  auto issue = [&](int i) {
    if (i < count) {
      if ((i & 15) == 0 && i > 0) {
        pages = later;
        if (i + 16 < count) later = pages_of(i + 16);
      }
      const int blk = (p.k0 >> 4) + 2 * (warp + kWarps * i);
      const uint8_t* head_at = a.cache + static_cast<int64_t>(p.head << page_shift) * S::Block + lane * 16;
      const uint32_t to = ring_at + wstage * S::Stage + lane * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pg = __shfl_sync(0xFFFFFFFFu, pages, (i & 15) * 2 + h);
        if (h == 0 || (blk + 1) * 16 < p.k1) {
          const uint32_t bytes = pg < 0 ? 0 : 16;                 // no page: zeros
          const uint8_t* src = head_at + static_cast<int64_t>(max(pg, 0)) * page_bytes + ((blk + h) & in_page) * S::Block;
#pragma unroll
          for (int j = 0; j < (S::Block + 511) / 512; ++j)
            if ((j + 1) * 512 <= S::Block || lane < (S::Block - j * 512) / 16) cp16(to + h * S::Block + j * 512, src + j * 512, bytes);
        }
      }
      if (++wstage == S::Stages) wstage = 0;
    }
    cp_commit();
  };
  auto begin = [&]() {                       // false behind the last part
    for (;;) {
      if (walk_u >= u1) return false;
      Request r = request_of(a, walk_b, false);
      int items, steps, lo;
      cost_of<S::Rows>(a, r, items, steps, lo);
      while (!share && walk_u >= walk_at + items * (steps + kOwn)) {
        walk_at += items * (steps + kOwn);
        r = request_of(a, ++walk_b, false);
        cost_of<S::Rows>(a, r, items, steps, lo);
      }
      int item;
      if (share) {
        item = u0 - walk_at;
        const int parts = min(share, steps), part = static_cast<int>(blockIdx.x) - u0 * share;
        walk_u = u1;                         // the only one
        if (part >= parts) return false;
        p.i0 = 0;
        p.i1 = steps;
        p.u = steps * part / parts;
        p.e = steps * (part + 1) / parts;
        p.c0 = u0 * share;
        p.c1 = p.c0 + parts - 1;
      } else {
        item = (walk_u - walk_at) / (steps + kOwn);
        p.i0 = walk_at + item * (steps + kOwn) + kOwn;   // an item's own steps come first, and belong to nobody
        p.i1 = p.i0 + steps;
        p.u = max(walk_u, p.i0);
        p.e = min(p.i1, u1);
        p.c0 = p.i0 / per;
        p.c1 = (p.i1 - 1) / per;
        walk_u = p.e;
        if (p.u >= p.e) {                    // the run ends before the item's tokens
          walk_u = u1;
          return false;
        }
      }
      p.b = walk_b;
      const int row_blocks = items / a.hk;
      p.head = item / row_blocks;
      p.rb = item - p.head * row_blocks;
      p.rows = min(S::Rows, r.n * a.group - p.rb * S::Rows);
      p.first = r.first;
      p.place0 = r.len - r.n;
      p.len = r.len;
      const int tok_last = by_group(a, p.rb * S::Rows + p.rows - 1), seen = min(r.len, max(p.place0 + tok_last + 1, 0));
      p.k0 = lo + (p.u - p.i0) * kStep;
      p.k1 = min(lo + (p.e - p.i0) * kStep, seen);
      const int pairs = p.k1 > p.k0 ? (p.k1 - p.k0 + 31) / 32 : 0;
      count = pairs > warp ? (pairs - warp + kWarps - 1) / kWarps : 0;
      pages = count > 0 ? pages_of(0) : 0;
      later = count > 16 ? pages_of(16) : 0;
#pragma unroll
      for (int i = 0; i < S::Stages - 1; ++i) issue(i);
      return true;
    }
  };

  bool more = begin();
  while (more) {
    const int here = count;
    if (tid == 0) s_part = p;                // read behind a barrier, when p is the next one already
    // every row sees all of [clear_lo, clear_hi)
    const int tok_first = by_group(a, p.rb * S::Rows), tok_last = by_group(a, p.rb * S::Rows + p.rows - 1);
    const int clear_hi = max(p.place0 + tok_first + 1, 0), clear_lo = a.window > 0 ? max(p.place0 + tok_last + 1 - a.window, 0) : 0;
    const int k0 = p.k0, k1 = p.k1;

    // query: B operand, row n = g of each tile; scaled by a power of two to an fp16 with its largest value near 2^14
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;   // the query carries the scale's sign
    uint32_t qf[NT][4 * NG][2];
    float fac[NT][2], room[NT][2], qs[NT][NG][2];
    int hi_r[NT][2], lo_r[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = p.rb * S::Rows + nt * 8 + g, tok = by_group(a, row);
      const bool real = nt * 8 + g < p.rows;
      float x[NG][2][8];
      uint32_t top = 0;
      if (real) {
        const __nv_bfloat16* qp = a.q + (p.first + tok) * a.q_ts + (p.head * a.group + row - tok * a.group) * a.q_hs;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint4 raw = __ldg(reinterpret_cast<const uint4*>(qp + 64 * gi + 16 * t + 8 * w));
            raw = make_uint4(raw.x ^ flip, raw.y ^ flip, raw.z ^ flip, raw.w ^ flip);
            unpack_bf16x8(raw, x[gi][w]);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[gi][w][j]) & 0x7FFFFFFFu);
          }
      } else {
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int j = 0; j < 16; ++j) x[gi][j >> 3][j & 7] = 0.0f;
      }
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int ex = min(max(static_cast<int>(top >> 23) - 127, -100), 100);
      const float up = __uint_as_float(static_cast<uint32_t>(14 - ex + 127) << 23);
      // not 0 (a scale of 0, a row of zeros), for -inf times it stays -inf: below 1e-37 it makes no weight differ from 1
      const float f = fmaxf(fabsf(a.scale_log2) * __uint_as_float(static_cast<uint32_t>(24 - 14 + ex + 127) << 23), 1e-37f);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const uint32_t b0 = pack_f16(x[gi][w][2 * st] * up, x[gi][w][4 + 2 * st] * up);
            const uint32_t b1 = pack_f16(x[gi][w][1 + 2 * st] * (up * 0.0625f), x[gi][w][5 + 2 * st] * (up * 0.0625f));
            qf[nt][gi * 4 + w * 2 + st][0] = b0;
            qf[nt][gi * 4 + w * 2 + st][1] = b1;
            sum += half_lo(b0) + half_hi(b0) + 16.0f * (half_lo(b1) + half_hi(b1));
          }
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
        sum *= -8.0f * 0x1p-24f;
        qs[nt][gi][0] = __shfl_sync(0xFFFFFFFFu, sum, 8 * t);
        qs[nt][gi][1] = __shfl_sync(0xFFFFFFFFu, sum, 8 * t + 4);
      }
      fac[nt][0] = __shfl_sync(0xFFFFFFFFu, f, 8 * t);
      fac[nt][1] = __shfl_sync(0xFFFFFFFFu, f, 8 * t + 4);
      room[nt][0] = kRoom / fac[nt][0];
      room[nt][1] = kRoom / fac[nt][1];
#pragma unroll
      for (int c = 0; c < 2; ++c) {          // what row 2t + c of the tile sees: [lo_r, hi_r)
        const int rr = nt * 8 + 2 * t + c, place = p.place0 + by_group(a, p.rb * S::Rows + rr);
        hi_r[nt][c] = rr < p.rows ? min(place + 1, p.len) : 0;
        lo_r[nt][c] = a.window > 0 ? place + 1 - a.window : 0;
      }
    }

    // running maximum of the unscaled scores, and what it takes off the scaled ones (nothing before there is one)
    float o[NT][4 * NG][4], l[NT][2], m[NT][2], off[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.0f;
      l[nt][0] = l[nt][1] = 0.0f;
      m[nt][0] = m[nt][1] = kLow;
      off[nt][0] = off[nt][1] = 0.0f;
    }

    for (int i = 0; i < here; ++i) {
      __syncwarp();                          // all lanes are done with the stage that is written now
      issue(i + S::Stages - 1);
      cp_wait<S::Stages - 1>();
      __syncwarp();
      const uint8_t* stage = ring + rstage * S::Stage;
      if (++rstage == S::Stages) rstage = 0;
      const int key0 = k0 + 32 * (warp + kWarps * i);
      const bool mask = key0 < clear_lo || key0 + 32 > clear_hi || key0 + 32 > k1;

      float s[2][NT][4];
      uint32_t vs[2][2][(NG + 1) / 2];       // value scales of tokens g and g + 8
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* blk = stage + h * S::Block;
        uint32_t kw[2][2 * NG], ks[2][(NG + 1) / 2];
        if constexpr (D == 64) {
          const uint4 x = *reinterpret_cast<const uint4*>(blk + lane * 16);
          kw[0][0] = x.x; kw[0][1] = x.y; kw[1][0] = x.z; kw[1][1] = x.w;
        } else {
#pragma unroll
          for (int j = 0; j < 2 * NG / 4; ++j)
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
              const uint4 x = *reinterpret_cast<const uint4*>(blk + (rr * (2 * NG / 4) + j) * 512 + lane * 16);
              kw[rr][4 * j] = x.x; kw[rr][4 * j + 1] = x.y; kw[rr][4 * j + 2] = x.z; kw[rr][4 * j + 3] = x.w;
            }
        }
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const uint8_t* sc = blk + 16 * D + (g + 8 * rr) * 4 * NG;
          if constexpr (NG == 1) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(sc);
            ks[rr][0] = x & 0xFFFFu;
            vs[h][rr][0] = x >> 16;
          } else if constexpr (NG == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(sc);
            ks[rr][0] = x.x;
            vs[h][rr][0] = x.y;
          } else {
            const uint4 x = *reinterpret_cast<const uint4*>(sc);
            ks[rr][0] = x.x; ks[rr][1] = x.y;
            vs[h][rr][0] = x.z; vs[h][rr][1] = x.w;
          }
        }
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          float acc[NT][4];
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              const uint32_t x0 = kw[0][2 * gi + w] >> (8 * st), x1 = kw[1][2 * gi + w] >> (8 * st);
              const uint32_t a0 = x0 & 0x000F000Fu, a1 = x1 & 0x000F000Fu, a2 = x0 & 0x00F000F0u, a3 = x1 & 0x00F000F0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t b0 = qf[nt][gi * 4 + w * 2 + st][0], b1 = qf[nt][gi * 4 + w * 2 + st][1];
                if (w == 0 && st == 0)
                  mma16816(acc[nt], a0, a1, a2, a3, b0, b1, qs[nt][gi][0], qs[nt][gi][1], qs[nt][gi][0], qs[nt][gi][1]);
                else
                  mma16816(acc[nt], a0, a1, a2, a3, b0, b1, acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
              }
            }
          float f[2];
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) f[rr] = __uint_as_float(gi & 1 ? ks[rr][gi >> 1] & 0xFFFF0000u : ks[rr][gi >> 1] << 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[h][nt][c] = gi == 0 ? acc[nt][c] * f[c >> 1] : fmaf(acc[nt][c], f[c >> 1], s[h][nt][c]);
        }
      }
      if (mask) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int key = key0 + 16 * h + g + 8 * (c >> 1);
              if (key < lo_r[nt][c & 1] || key >= min(hi_r[nt][c & 1], k1)) s[h][nt][c] = -INFINITY;
            }
        // Behind the last key there may be anything, and a value that is not a number must not reach the rows that do not see it (0
        // times it is not 0): its scale becomes 0, and the output of the rows that see it what it would have become.
        uint32_t bad = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            const bool behind = key0 + 16 * h + g + 8 * rr >= k1;
#pragma unroll
            for (int j = 0; j < (NG + 1) / 2; ++j) {
              if (behind) vs[h][rr][j] = 0;
              if ((vs[h][rr][j] & 0x7FFFu) > 0x7F80u) bad |= 1u << ((h * 2 + rr) * 4 + 2 * j);
              if ((vs[h][rr][j] & 0x7FFF0000u) > 0x7F800000u) bad |= 2u << ((h * 2 + rr) * 4 + 2 * j);
            }
          }
        if (__any_sync(0xFFFFFFFFu, bad != 0)) {
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            uint32_t rows_hit = 0;           // bit 2 nt + c: row 2t + c of the tile sees a group gi that is not a number
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int rr = 0; rr < 2; ++rr)
                if (bad >> ((h * 2 + rr) * 4 + gi) & 1u) {
                  vs[h][rr][gi >> 1] &= gi & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                      const int key = key0 + 16 * h + g + 8 * rr;
                      if (key >= lo_r[nt][c] && key < hi_r[nt][c]) rows_hit |= 1u << (2 * nt + c);
                    }
                }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) rows_hit |= __shfl_xor_sync(0xFFFFFFFFu, rows_hit, d);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                if (rows_hit >> (2 * nt + c) & 1u)
#pragma unroll
                  for (int j = 0; j < 4; ++j) o[nt][4 * gi + j][c] = o[nt][4 * gi + j][c + 2] = __uint_as_float(0x7FC00000u);
          }
        }
      }
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          grow |= fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2])) > m[nt][c] + room[nt][c];
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2]));
            x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
            const float to = fmaxf(m[nt][c], x), by = ex2((m[nt][c] - to) * fac[nt][c]);
            m[nt][c] = to;
            off[nt][c] = to > kLow ? -to * fac[nt][c] : 0.0f;
            l[nt][c] *= by;
#pragma unroll
            for (int j = 0; j < 4 * NG; ++j) {
              o[nt][j][c] *= by;
              o[nt][j][c + 2] *= by;
            }
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* blk = stage + h * S::Block + 8 * D;
        float pr[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            pr[nt][c] = ex2(fmaf(s[h][nt][c], fac[nt][c & 1], off[nt][c & 1]));
            l[nt][c & 1] += pr[nt][c];
          }
        uint32_t vw[4][NG];
        if constexpr (D == 64) {
          const uint4 x = *reinterpret_cast<const uint4*>(blk + lane * 16);
          vw[0][0] = x.x; vw[1][0] = x.y; vw[2][0] = x.z; vw[3][0] = x.w;
        } else if constexpr (D == 128) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 x = *reinterpret_cast<const uint4*>(blk + j * 512 + lane * 16);
            vw[2 * j][0] = x.x; vw[2 * j][1] = x.y; vw[2 * j + 1][0] = x.z; vw[2 * j + 1][1] = x.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 x = *reinterpret_cast<const uint4*>(blk + j * 512 + lane * 16);
            vw[j][0] = x.x; vw[j][1] = x.y; vw[j][2] = x.z; vw[j][3] = x.w;
          }
        }
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          float f[2];
#pragma unroll
          for (int rr = 0; rr < 2; ++rr)
            f[rr] = __uint_as_float(gi & 1 ? vs[h][rr][gi >> 1] & 0xFFFF0000u : vs[h][rr][gi >> 1] << 16);
          uint32_t pb[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = pr[nt][c] * f[c >> 1];
            pb[nt][0] = transpose8(pack_bf16x2(w[0], w[1]));
            pb[nt][1] = transpose8(pack_bf16x2(w[2], w[3]));
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = __byte_perm(vw[0][gi], vw[1][gi], half ? 0x7632 : 0x5410);
            const uint32_t y = __byte_perm(vw[2][gi], vw[3][gi], half ? 0x7632 : 0x5410);
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              const uint32_t a0 = signed_code(x >> (8 * st), mask4, magic), a1 = signed_code(x >> (8 * st + 4), mask4, magic);
              const uint32_t a2 = signed_code(y >> (8 * st), mask4, magic), a3 = signed_code(y >> (8 * st + 4), mask4, magic);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816_bf16(o[nt][gi * 4 + half * 2 + st], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            }
          }
        }
      }
    }
    __syncwarp();                            // the ring is free
    more = begin();                          // the next part's copies, while this one's states are joined

    float* part = states + warp * (S::State / 4);
    float* ml = part + S::Rows * D;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
        x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
        x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
        const int row = nt * 8 + 2 * t + c;
        if (g == 0) {
          ml[2 * row] = m[nt][c] > kLow ? m[nt][c] * fac[nt][c] : kLow;
          ml[2 * row + 1] = x;
        }
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(part + row * D + 64 * gi + 8 * g + 2 * j) = make_float2(o[nt][gi * 4 + j][c], o[nt][gi * 4 + j][c + 2]);
      }
    __syncthreads();

    const Part& q = s_part;
    const bool whole = q.u == q.i0 && q.e == q.i1;
    const int c0 = q.c0, c1 = q.c1, rows = q.rows;
    float* mine_at = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (static_cast<int>(blockIdx.x) == c0 ? 1 : 0)) * S::Part;
    auto finish = [&](int row, int d, float4 x, float mx, float sum) {
      const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;   // a sum that is not a number stays one
      const int rr = q.rb * S::Rows + row, in = by_group(a, rr), tok = q.first + in, hd = q.head * a.group + rr - in * a.group;
      *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(tok) * a.hq + hd) * D + d) =
          make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
      if (d == 0 && a.lse) a.lse[static_cast<int64_t>(tok) * a.hq + hd] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
    };
    constexpr int Wf = S::State / 4, Work = S::Rows * D / 4, PerThread = (Work + kThreads - 1) / kThreads;
    const int work = rows * (D / 4);
    for (int idx = tid; idx < work; idx += kThreads) {
      const int row = idx / (D / 4), d = idx % (D / 4) * 4;
      float mx = kLow, sum = 0.0f;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, states[w * Wf + S::Rows * D + 2 * row]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float by = ex2(states[w * Wf + S::Rows * D + 2 * row] - mx);
        const float4 y = *reinterpret_cast<const float4*>(states + w * Wf + row * D + d);
        sum = fmaf(states[w * Wf + S::Rows * D + 2 * row + 1], by, sum);
        x.x = fmaf(y.x, by, x.x); x.y = fmaf(y.y, by, x.y); x.z = fmaf(y.z, by, x.z); x.w = fmaf(y.w, by, x.w);
      }
      if (whole) {
        finish(row, d, x, mx, sum);
      } else {
        __stcg(reinterpret_cast<float4*>(mine_at + row * D + d), x);
        if (d == 0) __stcg(reinterpret_cast<float2*>(mine_at + S::Rows * D + 2 * row), make_float2(mx, sum));
      }
    }
    __syncthreads();                         // the states may be written again; and the CTA's part is complete
    if (!whole) {
      if (tid == 0) {
        __threadfence();
        const uint32_t before = atomicAdd(a.counters + c0, 1u);
        s_last = before == static_cast<uint32_t>(c1 - c0);
        if (s_last) a.counters[c0] = 0;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        // 32 CTAs at a time: their weights, a lane to a CTA, then their outputs, whose loads do not wait for one another
        const int n = c1 - c0 + 1;
        auto from = [&](int i) { return a.partial + (static_cast<int64_t>(c0 + i) * 2 + (i == 0 ? 1 : 0)) * S::Part; };
        float4 x[PerThread];
#pragma unroll
        for (int k = 0; k < PerThread; ++k) x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = 0; i0 < n; i0 += 32) {
          for (int row = warp; row < rows; row += kWarps) {
            const float2 ms = i0 + lane < n ? __ldcg(reinterpret_cast<const float2*>(from(i0 + lane) + S::Rows * D + 2 * row)) : make_float2(kLow, 0.0f);
            const float top = i0 ? s_top[row] : kLow;
            float mx = fmaxf(ms.x, top);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
            const float by = ex2(ms.x - mx), old = ex2(top - mx);
            float sum = ms.y * by;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
            s_weight[row][lane] = by;
            if (lane == 0) {
              s_sums[row] = i0 ? fmaf(s_sums[row], old, sum) : sum;
              s_old[row] = old;
              s_top[row] = mx;
            }
          }
          __syncthreads();
          const int m = min(32, n - i0);
#pragma unroll
          for (int k = 0; k < PerThread; ++k) {
            const int idx = tid + k * kThreads, row = idx / (D / 4), d = idx % (D / 4) * 4;
            if (idx < work) {
              if (i0) {
                const float old = s_old[row];
                x[k].x *= old; x[k].y *= old; x[k].z *= old; x[k].w *= old;
              }
#pragma unroll 8
              for (int i = 0; i < m; ++i) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(from(i0 + i) + row * D + d));
                const float by = s_weight[row][i];
                x[k].x = fmaf(y.x, by, x[k].x); x[k].y = fmaf(y.y, by, x[k].y);
                x[k].z = fmaf(y.z, by, x[k].z); x[k].w = fmaf(y.w, by, x[k].w);
              }
            }
          }
          __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < PerThread; ++k) {
          const int idx = tid + k * kThreads, row = idx / (D / 4), d = idx % (D / 4) * 4;
          if (idx < work) finish(row, d, x[k], s_top[row], s_sums[row]);
        }
        __syncthreads();
      }
    }
  }
  cp_wait<0>();
}

template <int D, int NT>
int launch(const AttnArgs& a, cudaStream_t stream) {
  using S = Shape<D, NT>;
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::Smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) ready[dev] = true;
  }
  decode_kernel<D, NT><<<S::Ctas, kThreads, S::Smem, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

namespace kv4 {
size_t decode_partial_floats() { return static_cast<size_t>(MONO_ATTN_COUNTERS) * 2 * 16 * (128 + 2); }   // 16 rows of 128 dims, or 8 of 256
// Rows of an item: 8 or 16. 64 sequences to 8192, 4 KV heads of 128: 8 rows in items of 8 64.2 us, of 16 83.0; 16 rows 88.7 and 86.7; 32 rows
// 157.8 and 141.3. Heads of 64: 42 and 57; 58 and 59; 99 and 90. Heads of 256 have no registers for 16.
int decode(const AttnArgs& a, int head_dim, int rows, cudaStream_t stream) {
  if (head_dim == 256) return launch<256, 1>(a, stream);
  if (head_dim == 128) return rows <= 8 ? launch<128, 1>(a, stream) : launch<128, 2>(a, stream);
  return rows <= 8 ? launch<64, 1>(a, stream) : launch<64, 2>(a, stream);
}
}  // namespace kv4
}  // namespace mono
