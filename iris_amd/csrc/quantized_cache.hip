// A paged cache in 8 bits: keys and values of new tokens into it, and cached tokens out of it.
//
// Writing.  With M the largest code, a block of tokens of a head gets the smallest scale s = 2^e >= 2^-100 with max |x| <= M s over its
// finite new elements, or keeps a larger one that its earlier tokens have; codes are x / s to nearest.  Earlier tokens' codes are rounded again
// only where the scale grew, by a power of two, which moves their exponents and costs places only where they become subnormal.
// One pass: a wave takes one block of one head (of K or of V), sixteen elements a lane, holds it in registers until the
// maximum is known, which is an exchange within the wave, and nothing else is shared.  Blocks are found from the slots alone: a token
// begins one where the token before it has no slot there.
//
// Reading.  A wave takes rows of one head of K or V, sixteen elements a lane; requests are found by bisection of their starts.
#include <initializer_list>
#include <type_traits>

#include "cache_codes.hpp"

namespace iris_amd {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_DIM = 256;

// ---- writing -------------------------------------------------------------------

struct WriteKArgs {
  iris_write_cache_args a;
  PageDiv page, block;
  int span;       // tokens whose blocks a wave looks after
  int64_t units;  // waves with something to do
};

// Sixteen elements of type DT as they lie in memory.
template <int DT>
struct Sixteen {
  static constexpr bool F32 = DT == IRIS_DTYPE_F32;
  static constexpr int QUADS = F32 ? 4 : 2;
  u32x4 x[QUADS];
  __device__ inline void load(const IRIS_GLOBAL char* p) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) x[i] = *(const IRIS_GLOBAL u32x4*)(p + i * 16);
  }
  __device__ inline void clear() {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) x[i] = u32x4{0, 0, 0, 0};
  }
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

template <int DT, int CT>
__device__ inline u32x4 encode16(const Sixteen<DT>& v, float scale) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = 0;
    if constexpr (DT == IRIS_DTYPE_F32) {
      const f32x4 f = __builtin_bit_cast(f32x4, v.x[i]);
      w = encode2_f32<CT, false>(w, f[0], f[1], scale);
      w = encode2_f32<CT, true>(w, f[2], f[3], scale);
    } else {
      w = encode2<CT, DT, false>(w, v.x[i / 2][2 * (i & 1)], scale);
      w = encode2<CT, DT, true>(w, v.x[i / 2][2 * (i & 1) + 1], scale);
    }
    y[i] = w;
  }
  return y;
}

// LANES lanes hold a row.
template <int DT, int CT, int LANES>
__global__ __launch_bounds__(THREADS) void write_kernel(WriteKArgs g) {
  using M = Magnitude<DT>;
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2, PASS = 64 / LANES;
  constexpr int HOLD = DT == IRIS_DTYPE_F32 ? 4 : 8;  // passes of rows that stay in registers; more are read twice
  const iris_write_cache_args& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * WAVES + wave;
  if (unit >= g.units) return;
  // values and keys change fastest, then heads
  const bool values = unit & 1;
  const int chunk = (int)(unit / 2 / a.heads), head = (int)(unit / 2 - (int64_t)chunk * a.heads);
  const IRIS_GLOBAL int64_t* slots = (const IRIS_GLOBAL int64_t*)a.slots;
  const IRIS_GLOBAL char* from = (const IRIS_GLOBAL char*)(values ? a.v : a.k);
  const int64_t stride_t = values ? a.stride_vt : a.stride_kt, stride_h = values ? a.stride_vh : a.stride_kh;
  IRIS_GLOBAL char* const to = (IRIS_GLOBAL char*)(values ? a.v_cache : a.k_cache);
  const int64_t to_page = values ? a.stride_vc_page : a.stride_kc_page, to_row = values ? a.stride_vc_row : a.stride_kc_row;
  const int64_t to_head = values ? a.stride_vc_head : a.stride_kc_head;
  IRIS_GLOBAL uint8_t* const scales = (IRIS_GLOBAL uint8_t*)(values ? a.v_scales : a.k_scales);
  const int64_t scale_page = values ? a.stride_vs_page : a.stride_ks_page, scale_block = values ? a.stride_vs_block : a.stride_ks_block;
  const int64_t scale_head = values ? a.stride_vs_head : a.stride_ks_head;

  // the chunk's tokens that begin a block
  const int first = chunk * g.span;
  int64_t slot = -1, before = -1;
  if (lane < g.span && first + lane < a.tokens) {
    slot = slots[first + lane];
    if (first + lane > 0) before = slots[first + lane - 1];
  }
  const bool inside = slot >= 0 && slot < a.num_slots;
  const bool goes_on = inside && before >= 0 && before < a.num_slots && page_div((uint32_t)before, g.block) == page_div((uint32_t)slot, g.block);
  if (slot >= a.num_slots || (goes_on && slot != before + 1)) report(a.status, IRIS_STATUS_BAD_INDEX);
  for (uint64_t begins = __ballot(inside && !goes_on); begins; begins &= begins - 1) {
    const int at = __builtin_ctzll(begins), token = first + at;
    const uint32_t slot0 = __builtin_amdgcn_readlane((int)slot, at);
    const uint32_t page = page_div(slot0, g.page), row_in_page = slot0 - page * g.page.d;
    const uint32_t block = page_div(row_in_page, g.block);  // of the page
    const int older = (int)(row_in_page - block * g.block.d);
    // the block's new tokens
    int rows = 0;
    for (int most = min((int)g.block.d - older, a.tokens - token); rows < most;) {
      const int i = rows + lane;
      const uint64_t others = ~__ballot(i < most && slots[token + min(i, most - 1)] == (int64_t)slot0 + i);
      const int n = others ? __builtin_ctzll(others) : 64;
      rows += n;
      if (n < 64) break;
    }
    IRIS_GLOBAL uint8_t* const scale_at = scales + page * scale_page + block * scale_block + head * scale_head;
    int old = 0;
    if (older) old = *scale_at;

    const int row = lane / LANES, part = lane % LANES;
    const bool live = part * 16 < a.head_dim;
    const IRIS_GLOBAL char* const source = from + ((int64_t)(token + row) * stride_t + head * stride_h + part * 16) * ES;
    IRIS_GLOBAL char* const target = to + page * to_page + (int64_t)row_in_page * to_row + head * to_head + part * 16;
    Sixteen<DT> held[HOLD];
    uint32_t most = 0;
    auto load = [&](Sixteen<DT>& v, int i) {
      v.clear();
      if (live && i * PASS + row < rows) v.load(source + (int64_t)i * PASS * stride_t * ES);
    };
    auto measure = [&](const Sixteen<DT>& v) {
#pragma unroll
      for (int q = 0; q < Sixteen<DT>::QUADS; ++q)
#pragma unroll
        for (int w = 0; w < 4; ++w) most = M::larger(most, v.x[q][w]);
    };
    auto replace = [&](Sixteen<DT>& v, uint32_t by) {
#pragma unroll
      for (int q = 0; q < Sixteen<DT>::QUADS; ++q)
#pragma unroll
        for (int w = 0; w < 4; ++w) v.x[q][w] = M::replaced(v.x[q][w], by);
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (i * PASS < rows) load(held[i], i);
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (i * PASS < rows) measure(held[i]);
    for (int i = HOLD; i * PASS < rows; ++i) {
      Sixteen<DT> v;
      load(v, i);
      measure(v);
    }
    // what is not finite counts for nothing here, and is no number as a code
    const bool odd = __any(M::only(most) >= M::INF);
    if (odd) {
      most = 0;
      for (int i = 0; i * PASS < rows; ++i) {
        Sixteen<DT> v;
        load(v, i);
        replace(v, 0);
        measure(v);
      }
#pragma unroll
      for (int i = 0; i < HOLD; ++i)
        if (i * PASS < rows) replace(held[i], M::NOT_A_NUMBER);
    }
    const uint32_t largest = __builtin_bit_cast(uint32_t, over_lanes<64>(M::number(M::only(most)), Larger{}));
    // largest = 1.m * 2^(x - 127) and M = 1.75 * 2^(TOP - 1)
    int need = (int)(largest >> 23) - (Codes<CT>::TOP - 1) + ((largest & 0x7FFFFFu) > 0x600000u);
    need = __builtin_amdgcn_readfirstlane(max(need, SCALE_LEAST));
    old = __builtin_amdgcn_readfirstlane(old);
    const int now = older ? max(need, old) : need;
    const float scale = scale_of(min(now, 254));
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (live && i * PASS + row < rows) *(IRIS_GLOBAL u32x4*)(target + (int64_t)(i * PASS + row) * to_row) = encode16<DT, CT>(held[i], scale);
    for (int i = HOLD; i * PASS < rows; ++i) {
      Sixteen<DT> v;
      load(v, i);
      if (odd) replace(v, M::NOT_A_NUMBER);
      if (live && i * PASS + row < rows) *(IRIS_GLOBAL u32x4*)(target + (int64_t)(i * PASS + row) * to_row) = encode16<DT, CT>(v, scale);
    }
    if (now == old && older) continue;
    if (lane == 0) *scale_at = (uint8_t)now;
    if (older) {
      const float shrink = scale_of(max(old - now + SCALE_ONE, 1));
      IRIS_GLOBAL char* const there = target - (int64_t)older * to_row;
      for (int r = row; r < older; r += PASS) {
        if (!live) break;
        IRIS_GLOBAL char* const p = there + (int64_t)r * to_row;
        u32x4 y = *(const IRIS_GLOBAL u32x4*)p;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const f32x4 f = decode4_f32<CT>(y[w], shrink);
          uint32_t c = encode2_f32<CT, false>(0, f[0], f[1], 1.f);
          y[w] = encode2_f32<CT, true>(c, f[2], f[3], 1.f);
        }
        *(IRIS_GLOBAL u32x4*)p = y;
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
  const bool live = part * 16 < a.head_dim;

  int64_t token[PASSES];
  int request[PASSES], position[PASSES], page[PASSES];
  bool mine[PASSES], there[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    token[i] = chunk * (PASSES * PASS) + i * PASS + row;
    // the last request that does not start behind it
    int lo = 0;
    for (int hi = a.requests; hi - lo > 1;) {
      const int mid = (lo + hi) / 2;
      if (start(mid) <= token[i])
        lo = mid;
      else
        hi = mid;
    }
    request[i] = lo;
    mine[i] = token[i] < a.tokens && start(lo) <= token[i] && token[i] < start(lo + 1);
    position[i] = 0;
    there[i] = false;
    if (mine[i]) {
      const int64_t at = (int64_t)a.lengths[lo] - start(lo + 1) + token[i];
      there[i] = at >= 0 && at < (int64_t)a.table_width * a.page_size;
      position[i] = there[i] ? (int)at : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    page[i] = 0;
    if (there[i]) page[i] = a.block_table[request[i] * a.stride_table + page_div((uint32_t)position[i], g.page)];
    there[i] = there[i] && (uint32_t)page[i] < (uint32_t)a.num_pages;
    if (mine[i] && !there[i]) report(a.status, IRIS_STATUS_BAD_INDEX);
  }
  u32x4 codes[PASSES];
  uint32_t byte[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    codes[i] = u32x4{NAN_CODES, NAN_CODES, NAN_CODES, NAN_CODES};
    byte[i] = SCALE_ONE;
    if (there[i] && live) {
      const int in_page = position[i] - (int)(page_div((uint32_t)position[i], g.page) * g.page.d);
      const int block = (int)page_div((uint32_t)in_page, g.block);
      const int64_t at = values ? page[i] * a.stride_vc_page + in_page * a.stride_vc_row + head * a.stride_vc_head
                                : page[i] * a.stride_kc_page + in_page * a.stride_kc_row + head * a.stride_kc_head;
      const int64_t scale_at = values ? page[i] * a.stride_vs_page + block * a.stride_vs_block + head * a.stride_vs_head
                                      : page[i] * a.stride_ks_page + block * a.stride_ks_block + head * a.stride_ks_head;
      codes[i] = *(const IRIS_GLOBAL u32x4*)((const IRIS_GLOBAL char*)(values ? a.v_cache : a.k_cache) + at + part * 16);
      byte[i] = scale_byte((values ? a.v_scales : a.k_scales) + scale_at);
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (!mine[i] || !live) continue;
    IRIS_GLOBAL char* out = values ? (IRIS_GLOBAL char*)a.v_out + (token[i] * a.stride_vt + head * a.stride_vh + part * 16) * ES
                                   : (IRIS_GLOBAL char*)a.k_out + (token[i] * a.stride_kt + head * a.stride_kh + part * 16) * ES;
    if (byte[i] == SCALE_NAN) codes[i] = u32x4{NAN_CODES, NAN_CODES, NAN_CODES, NAN_CODES}, byte[i] = SCALE_ONE;
    const float scale = scale_of((int)byte[i]);
    if constexpr (DT == IRIS_DTYPE_F32) {
#pragma unroll
      for (int w = 0; w < 4; ++w) *(IRIS_GLOBAL f32x4*)(out + w * 16) = decode4_f32<CT>(codes[i][w], scale);
    } else {
      u32x4 y[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        y[w / 2][2 * (w & 1)] = decode2<CT, DT, false>(codes[i][w], scale);
        y[w / 2][2 * (w & 1) + 1] = decode2<CT, DT, true>(codes[i][w], scale);
      }
      *(IRIS_GLOBAL u32x4*)out = y[0];
      *(IRIS_GLOBAL u32x4*)(out + 16) = y[1];
    }
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
    if (a.head_dim <= 64) return f(dt, ct, integral_constant<int, 4>{});
    if (a.head_dim <= 128) return f(dt, ct, integral_constant<int, 8>{});
    return f(dt, ct, integral_constant<int, 16>{});
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
  // Waves without a block cost their start only, waves with several take them one after another.
  g.span = 1;
  auto units = [&] { return ((int64_t)a.tokens + g.span - 1) / g.span * a.heads * 2; };
  while (g.span < 64 && units() > 16384) g.span *= 2;
  g.units = units();
  const int64_t groups = (g.units + WAVES - 1) / WAVES;
  if (groups > INT32_MAX) return hipErrorInvalidValue;
  return with_types(a, [&](auto dt, auto ct, auto lanes) {
    return launch(write_kernel<dt.value, ct.value, lanes.value>, dim3((unsigned)groups), THREADS, 0, stream, g);
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
    return units(4) >= 8 * 4 * (int64_t)current_cu_count() ? run(integral_constant<int, 4>{}) : run(integral_constant<int, 1>{});
  });
}
