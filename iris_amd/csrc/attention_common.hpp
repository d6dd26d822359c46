// What the attention kernels share: the paged cache's addresses, the keys that rows see, the parts of a split axis.
#pragma once

#include "heads_common.hpp"

namespace iris_amd {

// Division by the launch's page size for dividends below 2^31: with s = ceil(log2 d), m = ceil(2^(31 + s) / d) < 2^32 + 1 and
// m d - 2^(31 + s) < 2^s, so that floor(n m / 2^(31 + s)) = floor(n / d) for n < 2^31.
struct PageDiv {
  uint32_t d, shift;
  uint64_t m;
};
__host__ __device__ inline PageDiv make_page_div(uint32_t d) {
  PageDiv p{d, 31, 0};
  while ((1ull << (p.shift - 31)) < d) ++p.shift;
  p.m = ((1ull << p.shift) + d - 1) / d;
  return p;
}
__host__ __device__ inline uint32_t page_div(uint32_t n, const PageDiv& p) { return (uint32_t)(((uint64_t)n * p.m) >> p.shift); }

struct AttentionKArgs {
  iris_attention_args a;
  PageDiv page;
  float scale_log2;   // scale * log2(e): scores are exponents of two
  int group;          // query heads to a key head
  int splits;         // parts of a unit's keys (prompts)
  int grid_units;     // workgroups that share the work (decode)
  float* slots;       // partial results, `slot_elems` floats each
  int32_t* counters;  // arrivals at split units; zero between launches
};

// The keys that the queries at positions first .. last see, as tiles of BT keys: `front` tiles that hold the first tokens (sinks),
// then tiles from `start` on; `count` in all.
struct KeyTiles {
  int front, start, count;
  int lo;  // the first key inside the window of the first query
  __device__ inline int tile(int j) const { return j < front ? j : start + j - front; }
};
template <int BT>
__device__ inline KeyTiles key_tiles(const iris_attention_args& a, int first, int last) {
  KeyTiles k{0, 0, 0, 0};
  if (last < 0) return k;
  const int end = last / BT + 1;
  if (a.window > 0) {
    k.lo = max(0, max(first, 0) - a.window + 1);
    const int sinks = min(a.sinks, k.lo);
    k.start = k.lo / BT;
    k.front = min((sinks + BT - 1) / BT, k.start);
  }
  k.count = k.front + end - k.start;
  return k;
}
// Does the query at position `at` see key `key`?  (window 0: all up to its own)
__device__ inline bool sees(const iris_attention_args& a, int at, int key) {
  return key <= at && (a.window <= 0 || at - key < a.window || key < a.sinks);
}

// Word i of an array that no kernel writes while this one runs, by a scalar load (i is the wave's).
__device__ inline int scalar_at(const int32_t* p, int64_t i) { return ((const __attribute__((address_space(4))) int32_t*)p)[i]; }

}  // namespace iris_amd
