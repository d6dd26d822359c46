// A paged cache in 8 bits: keys and values of new tokens into it, and cached tokens out of it.
//
// Writing.  With M the largest code, a block of tokens of a head gets the smallest scale s = 2^e >= 2^-100 with max |x| <= M s over its
// finite new elements, or keeps a larger one that its earlier tokens have; codes are x / s to nearest.  Earlier tokens' codes are rounded again
// only where the scale grew, by a power of two, which moves their exponents and costs places only where they become subnormal.
// One pass over the data: one wave (blocks of more than 16 tokens: four) takes one block of one head, of K or of V, 16 bytes a lane, and holds it
// in registers until the maximum is known.  Blocks are found from the slots alone: a token begins one where the last
// token before it that has a slot has none there.  bf16, 8 heads of 128, four prompts of up to 4096 tokens (50 MB): 12 us from cold caches, 18 behind 512 MB of
// dirty lines, 10.6 where the last-level cache holds some of it (four sets of operands in turn); a copy of 4 GiB takes 10.8 for as many bytes, at 4.58
// TB/s on the same card.  64 single tokens of one head in 2.9 us, a chain of slots, heads and scales, and stores.
//
// Reading.  A wave takes rows of one head of K or V, 16 bytes of them a lane; requests are found by bisection of their starts.  16 contexts of
// up to 16384 tokens, 2 heads of 128 (160 MB, of which 53 are codes): 36 us from cold caches, 45 behind dirty lines, 27.4 where the codes are in the
// last-level cache; one of 1999 in 3.5.
#include <initializer_list>
#include <type_traits>

#include "cache_codes.hpp"

namespace iris_amd {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_DIM = 256;
constexpr int NARROW = 8192;      // bytes of a block that a wave takes alone
constexpr int MOST_UNITS = 2048;  // waves that look for blocks, at most where that leaves them 32 tokens each
constexpr int FAR = 512;          // tokens in front of a wave's own, but for the last 64, that are looked at at once for one with a slot

// ---- writing -------------------------------------------------------------------

struct WriteKArgs {
  iris_write_cache_args a;
  PageDiv page, block;
  int span;       // tokens whose blocks a wave (or four) looks after
  int64_t units;  // waves (or workgroups) with something to do
};

// Magnitudes of type DT as whole numbers grow as they do; from INF on they are not finite.
template <int DT>
struct Magnitude {
  static constexpr bool F32 = DT == IRIS_DTYPE_F32;
  static constexpr uint32_t INF = F32 ? 0x7F800000u : DT == IRIS_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  static constexpr uint32_t NOT_A_NUMBER = F32 ? 0x7FFFFFFFu : 0x7FFF7FFFu;  // (one, or two)
  // the larger of `most` (two of them, 16 bits) and w's
  static __device__ inline uint32_t larger(uint32_t most, uint32_t w) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    if constexpr (F32)
      return max(most, w & 0x7FFFFFFFu);
    else
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most), __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu)));
  }
  static __device__ inline uint32_t only(uint32_t most) { return F32 ? most : max(most & 0xFFFFu, most >> 16); }
  static __device__ inline float number(uint32_t most) {
    return F32 ? __builtin_bit_cast(float, most) : from16<F32 ? IRIS_DTYPE_BF16 : DT>((unsigned short)most);
  }
  // w with what is not finite replaced
  static __device__ inline uint32_t replaced(uint32_t w, uint32_t by) {
    if constexpr (F32) return (w & 0x7FFFFFFFu) >= INF ? by : w;
    const uint32_t lo = (w & 0x7FFFu) >= INF ? by & 0xFFFFu : w & 0xFFFFu;
    const uint32_t hi = ((w >> 16) & 0x7FFFu) >= INF ? by & 0xFFFF0000u : w & 0xFFFF0000u;
    return lo | hi;
  }
};

// The codes of a lane's 16 bytes: eight, or of fp32 four.
template <int DT>
struct LaneCodes {
  static constexpr int ELEMS = DT == IRIS_DTYPE_F32 ? 4 : 8, WORDS = ELEMS / 4;
  uint32_t w[WORDS];
  __device__ inline void load(const IRIS_GLOBAL char* p) {
    if constexpr (WORDS == 1) {
      w[0] = *(const IRIS_GLOBAL uint32_t*)p;
    } else {
      const u32x2 x = *(const IRIS_GLOBAL u32x2*)p;
      w[0] = x[0], w[1] = x[1];
    }
  }
  __device__ inline void store(IRIS_GLOBAL char* p) const {
    if constexpr (WORDS == 1)
      *(IRIS_GLOBAL uint32_t*)p = w[0];
    else
      *(IRIS_GLOBAL u32x2*)p = u32x2{w[0], w[1]};
  }
  template <int CT>
  __device__ inline void encode(u32x4 x, float scale) {
    if constexpr (WORDS == 1) {
      const f32x4 f = __builtin_bit_cast(f32x4, x);
      w[0] = encode2_f32<CT, true>(encode2_f32<CT, false>(0, f[0], f[1], scale), f[2], f[3], scale);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) w[i] = encode2<CT, DT, true>(encode2<CT, DT, false>(0, x[2 * i], scale), x[2 * i + 1], scale);
    }
  }
  template <int CT>
  __device__ inline u32x4 decode(float scale) const {
    if constexpr (WORDS == 1)
      return __builtin_bit_cast(u32x4, decode4_f32<CT>(w[0], scale));
    else
      return u32x4{decode2<CT, DT, false>(w[0], scale), decode2<CT, DT, true>(w[0], scale), decode2<CT, DT, false>(w[1], scale),
                   decode2<CT, DT, true>(w[1], scale)};
  }
};

// LANES lanes hold a row, WIDE waves share a block, and each holds HOLD rows of it; MORE: blocks may have more, which are read twice.
template <int DT, int CT, int LANES, int WIDE, int HOLD, bool MORE>
__global__ __launch_bounds__(WIDE > 1 ? WIDE * 64 : THREADS) void write_kernel(WriteKArgs g) {
  using M = Magnitude<DT>;
  using Codes8 = LaneCodes<DT>;
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2, PASS = 64 / LANES, HELD = HOLD / PASS, BATCH = 4;
  __shared__ uint32_t wave_most[2][WIDE];
  const iris_write_cache_args& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part_of = WIDE > 1 ? wave : 0;
  const int64_t unit = WIDE > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * WAVES + wave;
  if (unit >= g.units) return;  // (with WIDE waves all of a workgroup's)
  // values and keys change fastest, then heads
  const bool values = unit & 1;
  const int64_t chunk = unit / 2 / a.heads;
  const int head = (int)(unit / 2 - chunk * a.heads);
  const IRIS_GLOBAL int64_t* slots = (const IRIS_GLOBAL int64_t*)a.slots;
  const IRIS_GLOBAL char* from = (const IRIS_GLOBAL char*)(values ? a.v : a.k);
  const int64_t stride_t = values ? a.stride_vt : a.stride_kt, stride_h = values ? a.stride_vh : a.stride_kh;
  IRIS_GLOBAL char* const to = (IRIS_GLOBAL char*)(values ? a.v_cache : a.k_cache);
  const int64_t to_page = values ? a.stride_vc_page : a.stride_kc_page, to_row = values ? a.stride_vc_row : a.stride_kc_row;
  const int64_t to_head = values ? a.stride_vc_head : a.stride_kc_head;
  IRIS_GLOBAL uint8_t* const scales = (IRIS_GLOBAL uint8_t*)(values ? a.v_scales : a.k_scales);
  const int64_t scale_page = values ? a.stride_vs_page : a.stride_ks_page, scale_block = values ? a.stride_vs_block : a.stride_ks_block;
  const int64_t scale_head = values ? a.stride_vs_head : a.stride_ks_head;

  // The chunk's tokens that begin a block.  Lanes behind the chunk hold the slots that its last block may go on with.
  const int64_t first = chunk * g.span;
  int64_t slot = -1, before = -1;
  if (first + lane < a.tokens) {
    slot = slots[first + lane];
    if (first + lane > 0) before = slots[first + lane - 1];
  }
  auto have = [&](int64_t s) { return s >= 0 && s < a.num_slots; };
  const bool inside = have(slot), beside = have(before);
  // The last slot in front of a token: its neighbour's, or where that one is skipped another's, for the block may have begun there, and two
  // waves that both took it to begin with them would race on its scale and its older codes.  (us with / without: 64 single tokens, every
  // other one padding, 3.0 / 2.7; prompts of up to 4096, each padded to the longest, 27.9 / 22.8; without padding the same
  // but for fp32 heads of 256 in blocks of 256, 21.0 / 20.2.)
  int last = beside ? (int)before : -1;
  if (__any(inside && !beside && lane < g.span)) {
    const uint64_t held = __ballot(inside);
    int in_front = -1;  // of the chunk
    if (__builtin_amdgcn_readlane((int)!beside, __builtin_ctzll(held))) {
      // (the nearest first; padding in front of a chunk may be long)
      const int64_t close = first > lane ? slots[first - 1 - lane] : -1;
      const uint64_t near = __ballot(have(close));
      if (near) in_front = __builtin_amdgcn_readlane((int)close, __builtin_ctzll(near));
      for (int64_t at = first - 64; in_front < 0 && at > 0; at -= FAR) {
        int64_t far[FAR / 64];
#pragma unroll
        for (int i = 0; i < FAR / 64; ++i) far[i] = at > i * 64 + lane ? slots[at - 1 - i * 64 - lane] : -1;
#pragma unroll
        for (int i = 0; i < FAR / 64; ++i) {
          const uint64_t any = __ballot(have(far[i]));
          if (in_front < 0 && any) in_front = __builtin_amdgcn_readlane((int)far[i], __builtin_ctzll(any));
        }
      }
    }
    const uint64_t below = held & ((1ull << lane) - 1);
    const int nearest = __shfl((int)slot, below ? 63 - __builtin_clzll(below) : 0);
    if (!beside) last = below ? nearest : in_front;
  }
  const bool goes_on = inside && last >= 0 && page_div((uint32_t)last, g.block) == page_div((uint32_t)slot, g.block);
  const bool in_order = goes_on && beside && slot == before + 1;
  if (lane < g.span && (slot >= a.num_slots || (goes_on && !in_order))) report(a.status, IRIS_STATUS_BAD_INDEX);
  const uint64_t in_a_row = __ballot(in_order);
  int parity = 0;
  for (uint64_t begins = __ballot(inside && !goes_on && lane < g.span); begins; begins &= begins - 1) {
    const int at = __builtin_ctzll(begins);
    const int64_t token = first + at;
    const uint32_t slot0 = __builtin_amdgcn_readlane((int)slot, at);
    const uint32_t page = page_div(slot0, g.page), row_in_page = slot0 - page * g.page.d;
    const uint32_t block = page_div(row_in_page, g.block);  // of the page
    const int older = (int)(row_in_page - block * g.block.d);
    IRIS_GLOBAL uint8_t* const scale_at = scales + page * scale_page + block * scale_block + head * scale_head;
    int old = 0;
    if (older) old = *scale_at;
    // the block's new tokens, those whose slots the lanes hold first
    const uint64_t breaks = ~(in_a_row >> at) & ~1ull;  // (bits past the lanes' are breaks)
    int rows = breaks ? __builtin_ctzll(breaks) : 64;
    if (rows == 64 - at) {
      for (int most = (int)min((int64_t)g.block.d - older, a.tokens - token); rows < most;) {
        const int i = rows + lane;
        const uint64_t others = ~__ballot(i < most && slots[token + min(i, most - 1)] == (int64_t)slot0 + i);
        const int n = others ? __builtin_ctzll(others) : 64;
        rows += n;
        if (n < 64) break;
      }
    }

    const int row = part_of * PASS + lane / LANES, part = lane % LANES;  // (of the first pass)
    const bool live = part * Codes8::ELEMS < a.head_dim;
    const IRIS_GLOBAL char* const source = from + ((token + row) * stride_t + head * stride_h) * ES + part * 16;
    IRIS_GLOBAL char* const target = to + page * to_page + (int64_t)row_in_page * to_row + head * to_head + part * Codes8::ELEMS;
    u32x4 held[HELD];
    uint32_t most = 0;
    auto mine = [&](int i) { return live && i * (WIDE * PASS) + row < rows; };
    auto load = [&](int i) { return mine(i) ? *(const IRIS_GLOBAL u32x4*)(source + (int64_t)i * (WIDE * PASS) * stride_t * ES) : u32x4{0, 0, 0, 0}; };
    auto measure = [&](u32x4 v) {
#pragma unroll
      for (int w = 0; w < 4; ++w) most = M::larger(most, v[w]);
    };
    auto replace = [&](u32x4 v, uint32_t by) {
#pragma unroll
      for (int w = 0; w < 4; ++w) v[w] = M::replaced(v[w], by);
      return v;
    };
    // The largest of the block's, as a number; all waves that share it agree.
    auto over_block = [&](uint32_t x) {
      uint32_t all = __builtin_bit_cast(uint32_t, over_lanes<64>(M::number(M::only(x)), Larger{}));
      if constexpr (WIDE > 1) {
        if (lane == 0) wave_most[parity][wave] = all;
        __syncthreads();  // (the other half is read before the next one's barrier, this one written behind it)
#pragma unroll
        for (int w = 0; w < WIDE; ++w) all = max(all, wave_most[parity][w]);
        parity ^= 1;
      }
      return all;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = load(i);
#pragma unroll
    for (int i = 0; i < HELD; ++i) measure(held[i]);
    // f(passes that are not held, one at a time), BATCH of their loads in flight
    auto rest = [&](auto f) {
      if constexpr (!MORE) return;
      for (int i0 = HELD; i0 * (WIDE * PASS) < rows; i0 += BATCH) {
        u32x4 v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) v[i] = load(i0 + i);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) f(i0 + i, v[i]);
      }
    };
    rest([&](int, u32x4 v) { measure(v); });
    // what is not finite counts for nothing here, and is no number as a code
    const bool odd = __any(M::only(most) >= M::INF);
    if (odd) {
      most = 0;
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        measure(replace(held[i], 0));
        held[i] = replace(held[i], M::NOT_A_NUMBER);
      }
      rest([&](int, u32x4 v) { measure(replace(v, 0)); });
    }
    old = __builtin_amdgcn_readfirstlane(old);  // (read by all waves that share the block, before one of them writes it)
    const uint32_t largest = over_block(most);
    // largest = 1.m * 2^(x - 127) and M = 1.75 * 2^(TOP - 1)
    int need = (int)(largest >> 23) - (Codes<CT>::TOP - 1) + ((largest & 0x7FFFFFu) > 0x600000u);
    need = __builtin_amdgcn_readfirstlane(max(need, SCALE_LEAST));
    const int now = older ? max(need, old) : need;
    const float scale = scale_of(min(now, 254));
    Codes8 y;
    auto write = [&](int i, u32x4 v) {
      if (!mine(i)) return;
      y.template encode<CT>(v, scale);
      y.store(target + (int64_t)(i * (WIDE * PASS) + row) * to_row);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) write(i, held[i]);
    rest([&](int i, u32x4 v) { write(i, odd ? replace(v, M::NOT_A_NUMBER) : v); });
    if (now == old && older) continue;
    if (lane == 0 && part_of == 0) *scale_at = (uint8_t)now;
    if (older) {
      const float shrink = scale_of(max(old - now + SCALE_ONE, 1));
      IRIS_GLOBAL char* const there = target - (int64_t)older * to_row;
      for (int r = row; r < older && live; r += WIDE * PASS) {
        y.load(there + (int64_t)r * to_row);
#pragma unroll
        for (int w = 0; w < Codes8::WORDS; ++w) {
          const f32x4 f = decode4_f32<CT>(y.w[w], shrink);
          y.w[w] = encode2_f32<CT, true>(encode2_f32<CT, false>(0, f[0], f[1], 1.f), f[2], f[3], 1.f);
        }
        y.store(there + (int64_t)r * to_row);
      }
    }
  }
}

// ---- reading -------------------------------------------------------------------

struct ReadKArgs {
  iris_read_cache_args a;
  PageDiv page, block;
  int64_t units;
};
constexpr int STARTS = 2048;  // requests whose starts a workgroup holds; with more they are looked up in memory

// LANES lanes hold a row; a wave takes PASSES times 64 / LANES rows.
template <int DT, int CT, int LANES, int PASSES>
__global__ __launch_bounds__(THREADS) void read_kernel(ReadKArgs g) {
  using Codes8 = LaneCodes<DT>;
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2, PASS = 64 / LANES;
  __shared__ int32_t starts[STARTS + 1];
  const iris_read_cache_args& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool held = a.requests <= STARTS;
  if (held) {
    for (int i = threadIdx.x; i <= a.requests; i += THREADS) starts[i] = a.starts[i];
    __syncthreads();
  }
  const int64_t unit = (int64_t)blockIdx.x * WAVES + wave;
  if (unit >= g.units) return;
  const bool values = unit & 1;
  const int64_t chunk = unit / 2 / a.heads;
  const int head = (int)(unit / 2 - chunk * a.heads);
  auto start = [&](int r) { return held ? starts[r] : a.starts[r]; };
  const int row = lane / LANES, part = lane % LANES;
  const bool live = part * Codes8::ELEMS < a.head_dim;
  const IRIS_GLOBAL char* const cache = (const IRIS_GLOBAL char*)(values ? a.v_cache : a.k_cache) + head * (values ? a.stride_vc_head : a.stride_kc_head) +
                                        part * Codes8::ELEMS;
  const uint8_t* const scales = (values ? a.v_scales : a.k_scales) + head * (values ? a.stride_vs_head : a.stride_ks_head);
  const int64_t from_page = values ? a.stride_vc_page : a.stride_kc_page, from_row = values ? a.stride_vc_row : a.stride_kc_row;
  const int64_t scale_page = values ? a.stride_vs_page : a.stride_ks_page, scale_block = values ? a.stride_vs_block : a.stride_ks_block;
  IRIS_GLOBAL char* const out = (IRIS_GLOBAL char*)(values ? a.v_out : a.k_out) + head * (values ? a.stride_vh : a.stride_kh) * ES + part * 16;
  const int64_t out_row = (values ? a.stride_vt : a.stride_kt) * ES;

  const int64_t first = chunk * (PASSES * PASS);
  // the last request that does not start behind the wave's first row, and from there for each row
  int lo = 0;
  for (int hi = a.requests; hi - lo > 1;) {
    const int mid = lo + (hi - lo) / 2;
    if (start(mid) <= first)
      lo = mid;
    else
      hi = mid;
  }
  int request[PASSES], position[PASSES], page[PASSES];
  bool mine[PASSES], there[PASSES];
  int ends = start(lo + 1), begins = start(lo);
  int64_t length = a.lengths[lo];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int64_t token = first + i * PASS + row;
    if (token >= ends && lo + 1 < a.requests) {
      // (of a wave's rows in a middle request; bisection again, for there may be many that have none)
      for (int hi = a.requests; hi - lo > 1;) {
        const int mid = lo + (hi - lo) / 2;
        if (start(mid) <= token)
          lo = mid;
        else
          hi = mid;
      }
      begins = start(lo);
      ends = start(lo + 1);
      length = a.lengths[lo];
    }
    request[i] = lo;
    mine[i] = token < a.tokens && begins <= token && token < ends;
    const int64_t at = length - ends + token;
    there[i] = mine[i] && at >= 0 && at < (int64_t)a.table_width * a.page_size;
    position[i] = there[i] ? (int)at : 0;
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    page[i] = -1;
    if (there[i]) page[i] = a.block_table[request[i] * a.stride_table + page_div((uint32_t)position[i], g.page)];
  }
  Codes8 codes[PASSES];
  uint32_t byte[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    there[i] = there[i] && (uint32_t)page[i] < (uint32_t)a.num_pages;
    byte[i] = SCALE_NAN;
    if (there[i] && live) {
      const int in_page = position[i] - (int)(page_div((uint32_t)position[i], g.page) * g.page.d);
      codes[i].load(cache + page[i] * from_page + in_page * from_row);
      byte[i] = scale_byte(scales + page[i] * scale_page + page_div((uint32_t)in_page, g.block) * scale_block);
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (!mine[i] || !live) continue;
    if (!there[i] && part == 0) report(a.status, IRIS_STATUS_BAD_INDEX);
    if (byte[i] == SCALE_NAN) {
#pragma unroll
      for (int w = 0; w < Codes8::WORDS; ++w) codes[i].w[w] = NAN_CODES;
      byte[i] = SCALE_ONE;
    }
    const u32x4 y = codes[i].template decode<CT>(scale_of((int)byte[i]));
    IRIS_GLOBAL u32x4* const to = (IRIS_GLOBAL u32x4*)(out + (first + i * PASS + row) * out_row);
    // (many rows pass the caches by, so that these keep codes from pass to pass: 160 MB, a third of them codes, 27.4 us for 39.8)
    if constexpr (PASSES > 2)
      __builtin_nontemporal_store(y, to);
    else
      *to = y;
  }
}

// ---- launches ------------------------------------------------------------------

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool sixteens(std::initializer_list<int64_t> strides, int64_t per) {
  for (const int64_t s : strides)
    if (s % per) return false;
  return true;
}

// What both calls take.
template <class Args>
bool sizes_ok(const Args& a) {
  return (a.dtype == IRIS_DTYPE_F32 || a.dtype == IRIS_DTYPE_F16 || a.dtype == IRIS_DTYPE_BF16) &&
         (a.code == IRIS_DTYPE_E4M3 || a.code == IRIS_DTYPE_E5M2) && a.tokens >= 0 && a.heads >= 0 && a.head_dim > 0 && a.head_dim <= MAX_DIM &&
         a.head_dim % 16 == 0 && a.page_size > 0 && a.page_size <= MAX_CODES_PAGE && a.block > 0 && a.block % 16 == 0 && a.page_size % a.block == 0;
}
// (a cache without a slot has no memory)
template <class Args>
bool memory_ok(const Args& a, const void* k, const void* v, bool any_slot) {
  const int64_t vec = 16 / dtype_size(a.dtype);
  if (!k || !v || (any_slot && (!a.k_cache || !a.v_cache || !a.k_scales || !a.v_scales))) return false;
  for (const void* p : {k, v, (const void*)a.k_cache, (const void*)a.v_cache})
    if (!aligned16(p)) return false;
  return sixteens({a.stride_kt, a.stride_kh, a.stride_vt, a.stride_vh}, vec) &&
         sixteens({a.stride_kc_page, a.stride_kc_row, a.stride_kc_head, a.stride_vc_page, a.stride_vc_row, a.stride_vc_head}, 16);
}

// f(type, code, lanes a row)
template <class Args, class F>
hipError_t with_types(const Args& a, F f) {
  using std::integral_constant;
  auto lanes = [&](auto dt, auto ct) {
    constexpr int ELEMS = LaneCodes<dt.value>::ELEMS;
    if (a.head_dim <= 64) return f(dt, ct, integral_constant<int, 64 / ELEMS>{});
    if (a.head_dim <= 128) return f(dt, ct, integral_constant<int, 128 / ELEMS>{});
    return f(dt, ct, integral_constant<int, 256 / ELEMS>{});
  };
  auto codes = [&](auto dt) {
    return a.code == IRIS_DTYPE_E4M3 ? lanes(dt, integral_constant<int, IRIS_DTYPE_E4M3>{}) : lanes(dt, integral_constant<int, IRIS_DTYPE_E5M2>{});
  };
  if (a.dtype == IRIS_DTYPE_F32) return codes(integral_constant<int, IRIS_DTYPE_F32>{});
  if (a.dtype == IRIS_DTYPE_F16) return codes(integral_constant<int, IRIS_DTYPE_F16>{});
  return codes(integral_constant<int, IRIS_DTYPE_BF16>{});
}

}  // namespace
}  // namespace iris_amd

extern "C" int iris_write_quantized_cache_launch(const iris_write_cache_args* args, void* stream) {
  using namespace iris_amd;
  if (!args) return hipErrorInvalidValue;
  const iris_write_cache_args& a = *args;
  if (!sizes_ok(a) || a.num_slots < 0 || a.num_slots > INT32_MAX) return hipErrorInvalidValue;
  if (a.tokens == 0 || a.heads == 0) return hipSuccess;
  if (!a.slots || !memory_ok(a, a.k, a.v, a.num_slots > 0)) return hipErrorInvalidValue;
  WriteKArgs g{};
  g.a = a;
  g.page = make_page_div((uint32_t)a.page_size);
  g.block = make_page_div((uint32_t)a.block);
  // A wave takes a short block alone, four share one of up to 128 tokens, sixteen a longer one.  (us with one / four, bf16: 32 tokens of 64
  // elements 7.0 / 10.0, of 128 10.1 / 10.9; with four / sixteen: 64 tokens of 128 9.7 / 35, 128 10.4 / 25, 256 of 256 34 / 21, fp32 50 / 20.)
  const int64_t row = (a.head_dim <= 64 ? 64 : a.head_dim <= 128 ? 128 : 256) * dtype_size(a.dtype);  // as lanes hold it
  const int wide = a.block <= 32 && a.block * row <= NARROW ? 1 : a.block <= 128 ? 4 : 16;
  // Units without a block cost their start, those with several take them one after another.  (us with 8192 / 2048 / 1024 units at most: prompts of
  // up to 8192 tokens, one head, 5.8 / 4.7 / 5.4; 500 tokens in blocks of 64 5.4 / 3.4 / 3.1; 256 single tokens of 8 heads 3.9 / 4.0 / 4.8.
  // That is in blocks of 16.  Of longer blocks waves that share one take as many in turn, whatever a block gets: the same single tokens in blocks of 64
  // 8.9 us, of 128 11.0, of 256 41, where only one of sixteen waves has a token.)
  g.span = 1;
  auto units = [&] { return ((int64_t)a.tokens + g.span - 1) / g.span * a.heads * 2; };
  while (g.span < (wide == 16 ? 64 : 32) && units() > MOST_UNITS / wide) g.span *= 2;
  g.units = units();
  const int64_t groups = wide > 1 ? g.units : (g.units + WAVES - 1) / WAVES;
  if (groups > INT32_MAX) return hipErrorInvalidValue;
  return with_types(a, [&](auto dt, auto ct, auto lanes) {
    constexpr int DT = dt.value, CT = ct.value, LANES = lanes.value;
    void (*kernel)(WriteKArgs) = nullptr;
    if constexpr (16 * LANES * 16 <= NARROW)
      if (wide == 1) kernel = write_kernel<DT, CT, LANES, 1, 16, false>;
    if constexpr (32 * LANES * 16 <= NARROW)
      if (wide == 1 && a.block == 32) kernel = write_kernel<DT, CT, LANES, 1, 32, false>;
    if (wide == 4) kernel = a.block <= 64 ? write_kernel<DT, CT, LANES, 4, 16, false> : write_kernel<DT, CT, LANES, 4, 32, false>;
    if (wide == 16) kernel = a.block <= 256 ? write_kernel<DT, CT, LANES, 16, 16, false> : write_kernel<DT, CT, LANES, 16, 8, true>;
    return launch(kernel, dim3((unsigned)groups), wide > 1 ? wide * 64 : THREADS, 0, stream, g);
  });
}

extern "C" int iris_read_quantized_cache_launch(const iris_read_cache_args* args, void* stream) {
  using namespace iris_amd;
  if (!args) return hipErrorInvalidValue;
  const iris_read_cache_args& a = *args;
  if (!sizes_ok(a) || a.requests < 0 || a.table_width < 0 || a.num_pages < 0) return hipErrorInvalidValue;
  if (a.tokens == 0 || a.heads == 0 || a.requests == 0) return hipSuccess;
  if (!a.lengths || !a.starts || (a.table_width && !a.block_table) || a.stride_table < a.table_width || !memory_ok(a, a.k_out, a.v_out, a.num_pages > 0))
    return hipErrorInvalidValue;
  if ((int64_t)a.table_width * a.page_size > INT32_MAX) return hipErrorInvalidValue;
  ReadKArgs g{};
  g.a = a;
  g.page = make_page_div((uint32_t)a.page_size);
  g.block = make_page_div((uint32_t)a.block);
  return with_types(a, [&](auto dt, auto ct, auto lanes) {
    constexpr int DT = dt.value, CT = ct.value, LANES = lanes.value, PASS = 64 / LANES;
    auto units = [&](int passes) { return ((int64_t)a.tokens + passes * PASS - 1) / (passes * PASS) * a.heads * 2; };
    auto run = [&](auto passes) {
      g.units = units(passes.value);
      const int64_t groups = (g.units + WAVES - 1) / WAVES;
      if (groups > INT32_MAX) return (hipError_t)hipErrorInvalidValue;
      return launch(read_kernel<DT, CT, LANES, passes.value>, dim3((unsigned)groups), THREADS, 0, stream, g);
    };
    using std::integral_constant;
    return units(8) >= 16 * (int64_t)current_cu_count() ? run(integral_constant<int, 8>{}) : run(integral_constant<int, 2>{});
  });
}
