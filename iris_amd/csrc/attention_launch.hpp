// A call of attention: checked, planned from the sizes that the host has, and launched as the kernel that the plan names.  CT: the codes of
// the cache (or 0: it is of the heads' own type); a source file instantiates these for each.
#pragma once

#include <type_traits>

#include "attention_rows.hpp"
#include "attention_tiles.hpp"

namespace iris_amd {
namespace calls {

constexpr int64_t COUNTERS = 4096;      // arrival counters, one a split unit, at the workspace's start
constexpr int64_t ROW_SLOTS = 4096;     // partial results of 16 rows that a full workspace holds
constexpr int MAX_HEAD_DIM = 256;

inline int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Floats of a partial result of 16 rows.
inline int64_t row_slot(int dim) { return rows::ROWS * (padded_dim(dim) + 4); }

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int CT>
hipError_t check(const iris_attention_args& a, const iris_cache_scales* s) {
  if (a.dtype != IRIS_DTYPE_F32 && a.dtype != IRIS_DTYPE_F16 && a.dtype != IRIS_DTYPE_BF16) return hipErrorInvalidValue;
  if (a.requests < 0 || a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0 || a.page_size <= 0 || a.table_width < 0 || a.num_pages < 0 ||
      a.window < 0 || a.sinks < 0 || !(a.scale > 0.f) || !(a.scale < INFINITY))
    return hipErrorInvalidValue;
  const int es = dtype_size(a.dtype), vec = 16 / es;
  const int cache_vec = CT ? 16 : vec;  // elements of the cache in 16 bytes
  if (a.head_dim <= 0 || a.head_dim > MAX_HEAD_DIM || a.head_dim % cache_vec) return hipErrorInvalidValue;
  if constexpr (CT != 0)
    if (s->block <= 0 || s->block % 16 || a.page_size % s->block || a.page_size > MAX_CODES_PAGE) return hipErrorInvalidValue;
  if (a.tokens == 0 || a.q_heads == 0) return hipSuccess;
  if (a.k_heads == 0 || a.q_heads % a.k_heads || a.requests == 0 || a.table_width == 0 || a.num_pages == 0) return hipErrorInvalidValue;
  if (!a.query_starts && a.requests != a.tokens) return hipErrorInvalidValue;
  if constexpr (CT != 0) {
    if (!s->k_scales || !s->v_scales) return hipErrorInvalidValue;
    for (const int64_t step : {a.stride_kc_page / 16, a.stride_vc_page / 16, s->stride_ks_page, s->stride_vs_page, s->stride_ks_block, s->stride_vs_block})
      if (step < 0 || step > UINT32_MAX) return hipErrorInvalidValue;
  }
  if (!a.q || !a.k_cache || !a.v_cache || !a.block_table || !a.lengths || !a.out || a.stride_table < a.table_width) return hipErrorInvalidValue;
  if ((int64_t)a.table_width * a.page_size > INT32_MAX) return hipErrorInvalidValue;
  for (const void* p : {a.q, a.k_cache, a.v_cache, (const void*)a.out, (const void*)a.workspace})
    if (!aligned16(p)) return hipErrorInvalidValue;
  for (const int64_t step : {a.stride_qt, a.stride_qh, a.stride_ot, a.stride_oh})
    if (step % vec) return hipErrorInvalidValue;
  for (const int64_t step : {a.stride_kc_page, a.stride_kc_row, a.stride_kc_head, a.stride_vc_page, a.stride_vc_row, a.stride_vc_head})
    if (step % cache_vec) return hipErrorInvalidValue;
  return hipSuccess;
}

template <int CT, class F>
hipError_t with_types(const iris_attention_args& a, F f) {
  using std::integral_constant;
  auto paged = [&](auto dt, auto dp) {
    if constexpr (CT != 0)
      return f(dt, dp, std::true_type{});
    else
      return a.page_size % 16 == 0 ? f(dt, dp, std::true_type{}) : f(dt, dp, std::false_type{});
  };
  auto dims = [&](auto dt) {
    switch (padded_dim(a.head_dim)) {
      case 64: return paged(dt, integral_constant<int, 64>{});
      case 128: return paged(dt, integral_constant<int, 128>{});
      default: return paged(dt, integral_constant<int, 256>{});
    }
  };
  if (a.dtype == IRIS_DTYPE_F32) return dims(integral_constant<int, IRIS_DTYPE_F32>{});
  if (a.dtype == IRIS_DTYPE_F16) return dims(integral_constant<int, IRIS_DTYPE_F16>{});
  return dims(integral_constant<int, IRIS_DTYPE_BF16>{});
}

// What a launch does.
struct Plan {
  int kernel = IRIS_ATTENTION_NOTHING;
  int64_t workgroups = 0;
  int64_t splits = 1;   // parts of a unit's keys (prompts)
  int by_length = 0;    // (AttentionKArgs)
  int dealt = 0;        // (QuantizedKArgs)
  int64_t parted = 0;   // floats behind the workspace's counters that parts are left in; 0: no unit is split
};

template <int DT, int DP, bool PG, int CT>
hipError_t make_plan(const iris_attention_args& a, int cus, Plan* p) {
  using C = rows::Cfg<DT, DP, CT>;
  const int group = a.q_heads / a.k_heads;
  const int64_t slots = a.workspace && a.workspace_elems > COUNTERS ? (a.workspace_elems - COUNTERS) / C::SLOT : 0;
  // the most keys that a row may see
  const int64_t room = (int64_t)a.table_width * a.page_size;
  const int64_t most_keys = a.window > 0 && (int64_t)a.window + a.sinks < room ? (int64_t)a.window + a.sinks : room;
  if (!a.query_starts) {
    p->kernel = IRIS_ATTENTION_DECODE;
    const int64_t units = (int64_t)a.requests * a.k_heads * ((group + rows::ROWS - 1) / rows::ROWS);
    const int64_t line = units * ((most_keys + C::BT - 1) / C::BT + 2 + rows::REST);  // at most
    if (line > INT32_MAX) return hipErrorInvalidValue;
    int64_t grid = line;
    // As many workgroups as have 64 KiB of keys and values in flight a CU; more only leave more parts to join (us at 1 / 2 / 3 a CU:
    // heads of 128, 64 requests of up to 8192 keys 20.6 / 22.1 / 23.1, 16 of up to 131072 119 / 120 / 123; heads of 64, 128
    // requests that see 1028 keys 24.3 / 19.6 / 20.1).
    constexpr int per_cu = 2 * C::BT * DP * C::CS <= 32 * 1024 ? 2 : 1;
    if (grid > per_cu * cus) grid = per_cu * cus;
    if (grid > rows::LATER) grid = rows::LATER;
    // A workgroup may leave a part of its run's first unit and one of its last, in two slots of its own.  Where the slots are for no more
    // workgroups than there are units, nothing is split and a unit is a workgroup's.
    const bool split = slots / 2 >= (units < grid ? units + 1 : grid);
    if (split && grid > slots / 2) grid = slots / 2;
    p->workgroups = grid;
    if (split) p->parted = 2 * grid * C::SLOT;
    return hipSuccess;
  }
  const int64_t few_tiles = (int64_t)a.tokens * group / rows::ROWS + a.requests, few_units = few_tiles * a.k_heads;  // of 16 rows
  if constexpr (DT != IRIS_DTYPE_F32 && PG) {
    // Tiles of 128 rows read keys once for all of them, tiles of 16 fill the chip with fewer rows and end sooner.  us in tiles of 128 /
    // of 16, bf16, 8 + 1 heads of 128 unless stated.  By rows a request: 64 requests behind up to 4096 tokens, 19 rows each
    // 41 / 37, 27 each 41 / 46, 42 each 42 / 49.  By 16-row units and the most keys a row may see: 102 x 200 11.3 / 7.7,
    // 93 x 2004 20.5 / 17.2, 201 x 400 16.4 / 10.9, 460 x 500 17.1 / 13.4, 57 x 8001 31 / 26; 501 x 1000 20.2 / 20.5,
    // 188 x 4113 29 / 39, 268 x 2001 (4 + 4 heads) 27 / 37, 55 x 46398 79 / 86; 537 x 180 12.6 / 14.1.  Over a cache in 8 bits the line
    // lies there too: 64 requests behind up to 4096, up to 6 tokens each 37 / 31, 10 each 38 / 39, 16 each 40 / 41; one prompt of 300 tokens
    // 14.4 / 9.5, 700 20.4 / 14.8, 1000 21.2 / 19.3; 8 of up to 60 behind 4000 25.3 / 18.1, 4 of up to 300 behind 2000 22.8 / 29.8.
    const bool few_rows = (int64_t)a.tokens * group <= 24 * (int64_t)a.requests ||
                          (few_units <= 2 * cus && few_units * most_keys <= (int64_t)1536 * cus);
    const int64_t row_tiles = (int64_t)a.tokens * group / tiles::ROWS + a.requests;
    // (a page's rows are addressed with 32 bits)
    const int64_t reach = (int64_t)a.page_size * C::CS * (a.stride_kc_row > a.stride_vc_row ? a.stride_kc_row : a.stride_vc_row) + 512;
    if (!few_rows && row_tiles * a.k_heads <= INT32_MAX / 64 && reach <= INT32_MAX && a.stride_kc_row >= 0 && a.stride_vc_row >= 0) {
      constexpr int64_t SLOT = tiles::Cfg<DT, DP>::SLOT;
      p->kernel = IRIS_ATTENTION_PROMPT_TILES;
      const int64_t units = row_tiles * a.k_heads, places = tiles::waves_a_simd(DP) * cus;
      // Where places are left, several take a row tile, of four tiles of keys each or more.  (One prompt of 1000 tokens, us in one part / of
      // four / of two key tiles: 28 / 20 / 26; of 2000: 49 / 34 / 34.)
      if (2 * units <= places && units <= rows::LATER) {
        p->splits = places / units;
        const int64_t room_for = slots * C::SLOT / (SLOT * units);
        if (p->splits > most_keys / (4 * tiles::BT)) p->splits = most_keys / (4 * tiles::BT);
        if (p->splits > tiles::MOST_PARTS) p->splits = tiles::MOST_PARTS;
        if (p->splits > room_for) p->splits = room_for;
        if (p->splits < 1) p->splits = 1;
      }
      // Which starts first matters where places are taken twice: a CU's, or with a window (whose rows are nearly alike) all of them.  (us in the
      // requests' order / by length: window of 1024, 642 row tiles on 768 places 44.4 / 46.3; no window, 381 on 512 99.7 / 97.)
      if (p->splits == 1 && a.requests <= 64 && units > (a.window > 0 ? places : cus)) p->by_length = cus > a.k_heads ? cus / a.k_heads : 1;
      // Where row tiles fill the places, how the empty ones among them are spread matters; where they do not, as they are is up to 3 us less.
      p->dealt = p->splits == 1 && !p->by_length && units >= places;
      p->workgroups = units * p->splits;
      if (p->splits > 1) p->parted = units * p->splits * SLOT;
      return hipSuccess;
    }
  }
  // (8 prompts of up to 4 tokens behind up to 4096, us in one part / as many as make one / two workgroups a CU: 65 / 15 / 16; fp32, a
  // prompt of 500: 25 / 19 / 19; more a CU the same)
  p->kernel = IRIS_ATTENTION_PROMPT_ROWS;
  if (few_units < 2 * cus && few_units <= rows::LATER) {
    p->splits = 2 * cus / few_units;
    if (p->splits > most_keys / (2 * C::BT)) p->splits = most_keys / (2 * C::BT);
    if (p->splits > slots / few_units) p->splits = slots / few_units;
    if (p->splits > rows::FLAT) p->splits = rows::FLAT;
    if (p->splits < 1) p->splits = 1;
  }
  if (few_tiles * p->splits > INT32_MAX || a.k_heads > 65535) return hipErrorInvalidValue;
  p->workgroups = few_units * p->splits;
  if (p->splits > 1) p->parted = few_units * p->splits * C::SLOT;
  return hipSuccess;
}

template <int CT>
using Kernel = void (*)(KArgs<CT>);
template <int DT, int DP, bool PG, int CT>
Kernel<CT> kernel_of(int kernel, bool lse) {
  if (kernel == IRIS_ATTENTION_DECODE) return rows::decode_kernel<DT, DP, PG, CT>;
  if constexpr (DT != IRIS_DTYPE_F32 && PG)
    if (kernel == IRIS_ATTENTION_PROMPT_TILES) return lse ? tiles::prompt_tiles_kernel<DT, DP, true, CT> : tiles::prompt_tiles_kernel<DT, DP, false, CT>;
  return rows::prompt_rows_kernel<DT, DP, PG, CT>;
}

template <int CT>
int launch_call(const iris_attention_args& a, const iris_cache_scales* s, void* stream) {
  const hipError_t bad = check<CT>(a, s);
  if (bad != hipSuccess) return bad;
  if (a.tokens == 0 || a.q_heads == 0) return hipSuccess;

  KArgs<CT> g{};
  g.a = a;
  if constexpr (CT != 0) {
    g.s = *s;
    g.k_page16 = (uint32_t)(a.stride_kc_page / 16), g.v_page16 = (uint32_t)(a.stride_vc_page / 16);
    g.ks_page = (uint32_t)s->stride_ks_page, g.vs_page = (uint32_t)s->stride_vs_page;
    g.ks_block = (uint32_t)s->stride_ks_block, g.vs_block = (uint32_t)s->stride_vs_block;
    g.block16 = make_block16((uint32_t)s->block);
  }
  g.page = make_page_div((uint32_t)a.page_size);
  g.scale_log2 = a.scale * 1.4426950408889634f;
  g.group = a.q_heads / a.k_heads;
  return with_types<CT>(a, [&](auto dt, auto dp, auto pg) {
    constexpr int DT = dt.value, DP = dp.value;
    constexpr bool PG = pg.value;
    Plan p;
    const hipError_t refused = make_plan<DT, DP, PG, CT>(a, current_cu_count(), &p);
    if (refused != hipSuccess) return refused;
    g.splits = (int)p.splits;
    g.by_length = p.by_length;
    if constexpr (CT != 0) g.dealt = p.dealt;
    g.grid_units = (int)p.workgroups;
    if (p.parted) {
      g.counters = (int32_t*)a.workspace;
      g.slots = a.workspace + COUNTERS;
    }
    static_assert(tiles::WAVES == rows::WAVES, "one size of workgroups");
    const unsigned heads = p.kernel == IRIS_ATTENTION_PROMPT_ROWS ? a.k_heads : 1;
    return launch(kernel_of<DT, DP, PG, CT>(p.kernel, a.lse), dim3((unsigned)(p.workgroups / heads), heads), rows::WAVES * 64, 0, stream, g);
  });
}

template <int CT>
int plan_call(const iris_attention_args& a, const iris_cache_scales* s, int32_t num_cus, iris_attention_plan_info* plan) {
  const hipError_t bad = check<CT>(a, s);
  if (bad != hipSuccess) return bad;
  *plan = iris_attention_plan_info{0, 0, IRIS_ATTENTION_NOTHING, 1};
  if (a.tokens == 0 || a.q_heads == 0) return hipSuccess;
  return with_types<CT>(a, [&](auto dt, auto dp, auto pg) {
    Plan p;
    const hipError_t refused = make_plan<dt.value, dp.value, pg.value, CT>(a, num_cus ? num_cus : current_cu_count(), &p);
    if (refused == hipSuccess) *plan = iris_attention_plan_info{p.parted ? COUNTERS + p.parted : 0, p.workgroups, p.kernel, (int32_t)p.splits};
    return refused;
  });
}

// The work that the workgroups at a place take, by its number in its own order (kernels that take it by lengths: as if they did not).
template <int CT>
int item_call(const iris_attention_args& a, const iris_cache_scales* s, int32_t num_cus, int64_t place, int64_t* item) {
  const hipError_t bad = check<CT>(a, s);
  if (bad != hipSuccess) return bad;
  if (a.tokens == 0 || a.q_heads == 0) return hipErrorInvalidValue;
  return with_types<CT>(a, [&](auto dt, auto dp, auto pg) {
    Plan p;
    const hipError_t refused = make_plan<dt.value, dp.value, pg.value, CT>(a, num_cus ? num_cus : current_cu_count(), &p);
    if (refused != hipSuccess) return refused;
    const int64_t places = p.kernel == IRIS_ATTENTION_DECODE ? p.workgroups : p.workgroups / a.k_heads;
    if (place < 0 || place >= places) return hipErrorInvalidValue;
    *item = CT != 0 && p.dealt ? dealt((int)place, (int)places) : place;
    return hipSuccess;
  });
}

template <int CT>
int info_call(const iris_attention_args& a, const iris_cache_scales* s, int* n_regs, int* n_spills) {
  const hipError_t bad = check<CT>(a, s);
  if (bad != hipSuccess) return bad;
  if (a.tokens == 0 || a.q_heads == 0) return hipErrorInvalidValue;
  return with_types<CT>(a, [&](auto dt, auto dp, auto pg) {
    Plan p;
    hipError_t err = make_plan<dt.value, dp.value, pg.value, CT>(a, current_cu_count(), &p);
    if (err != hipSuccess) return err;
    hipFuncAttributes at;
    err = hipFuncGetAttributes(&at, (const void*)kernel_of<dt.value, dp.value, pg.value, CT>(p.kernel, a.lse));
    if (err != hipSuccess) return err;
    *n_regs = at.numRegs;
    *n_spills = (int)at.localSizeBytes;
    return hipSuccess;
  });
}

// What a source file instantiates for its codes.
#define IRIS_ATTENTION_CALLS(extern_, CT)                                                                                                \
  extern_ template int launch_call<CT>(const iris_attention_args&, const iris_cache_scales*, void*);                                     \
  extern_ template int plan_call<CT>(const iris_attention_args&, const iris_cache_scales*, int32_t, iris_attention_plan_info*);          \
  extern_ template int item_call<CT>(const iris_attention_args&, const iris_cache_scales*, int32_t, int64_t, int64_t*);                  \
  extern_ template int info_call<CT>(const iris_attention_args&, const iris_cache_scales*, int*, int*);

}  // namespace calls
}  // namespace iris_amd
