// How many tiles of keys the row blocks of a request have, for the division of the work of kv4_prompt.cu among its CTAs.
#pragma once
#include <cstdint>

namespace mono {
namespace kv4 {

constexpr int kKeys = 128;                  // of a tile
// What an item costs beside its tiles, in tiles: loading its queries, filling and draining the pipeline, writing its output.
// It counts where work is divided, for the first blocks of a prompt are many and short.
constexpr int kOwn = 2;

// sum of floor((a i + b) / m), i < n (by Euclid's algorithm on a and m). n below 2^24 (the outputs of a row block take 16 KB or more), a up to 256,
// b below 2^31: a n + b fits 32 bits once both are below m, 128. The sum does not: one prompt of 750 000 tokens in blocks of one has 2^31 tiles.
__device__ inline int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  uint64_t sum = 0;
  while (n > 0) {
    const uint32_t qa = a / m, qb = b / m;
    sum += qa * (static_cast<uint64_t>(n) * (n - 1) / 2) + static_cast<uint64_t>(qb) * n;
    a -= qa * m;
    b -= qb * m;
    const uint32_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y - n * m;
    const uint32_t t = m;
    m = a;
    a = t;
  }
  return static_cast<int64_t>(sum);
}

// The row blocks of a request: `tb` tokens each, all query heads of a KV head.
struct Item {
  int place0, n, len, tb, window;
  __device__ __forceinline__ int blocks() const { return (n + tb - 1) / tb; }
  __device__ __forceinline__ int begin(int rb) const { return window > 0 ? max(place0 + rb * tb + 1 - window, 0) : 0; }
  __device__ __forceinline__ int first_tile(int rb) const { return begin(rb) / kKeys; }
  __device__ __forceinline__ int seen(int rb) const { return min(len, max(place0 + min((rb + 1) * tb, n), 0)); }
  // tiles of row block rb, at least one
  __device__ __forceinline__ int tiles(int rb) const { return max(1, (seen(rb) + kKeys - 1) / kKeys - first_tile(rb)); }
};

// Tiles, and kOwn for each block, of the row blocks before rb: the ends of what they see less its beginnings, each a sum of floors; counted one by
// one only where the first queries have no place in the sequence.
__device__ __noinline__ int64_t tiles_before(const Item& it, int rb) {
  int64_t sum = static_cast<int64_t>(rb) * kOwn;
  if (it.place0 < 0) {
    for (int i = 0; i < rb; ++i) sum += it.tiles(i);
    return sum;
  }
  const int full = min(rb, it.n / it.tb);                // blocks of tb tokens; a shorter one is the last
  sum += floor_sum(full, kKeys, it.tb, it.place0 + it.tb + kKeys - 1);
  if (it.window > 0) {
    const int begin = it.place0 + 1 - it.window;         // of the first row; blocks with a negative one begin at 0
    const int skip = begin < 0 ? min((-begin + it.tb - 1) / it.tb, full) : 0;
    sum -= floor_sum(full - skip, kKeys, it.tb, max(begin + skip * it.tb, 0));
  }
  if (rb > full) sum += it.tiles(full);
  return sum;
}

}  // namespace kv4
}  // namespace mono
