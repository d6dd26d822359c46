// iris_attention_launch: checks a call, plans it from the sizes that the host has, and launches the kernel that the plan names.
#include <type_traits>

#include "attention_rows.hpp"
#include "attention_tiles.hpp"

namespace iris_amd {
namespace {

constexpr int64_t COUNTERS = 4096;      // arrival counters, one a split unit, at the workspace's start
constexpr int64_t ROW_SLOTS = 4096;     // partial results of 16 rows that a full workspace holds
constexpr int MAX_HEAD_DIM = 256;

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Floats of a partial result of 16 rows.
int64_t row_slot(int dim) { return rows::ROWS * (padded_dim(dim) + 4); }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

hipError_t check(const iris_attention_args& a) {
  if (a.dtype != IRIS_DTYPE_F32 && a.dtype != IRIS_DTYPE_F16 && a.dtype != IRIS_DTYPE_BF16) return hipErrorInvalidValue;
  if (a.requests < 0 || a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0 || a.page_size <= 0 || a.table_width < 0 || a.num_pages < 0 ||
      a.window < 0 || a.sinks < 0 || !(a.scale > 0.f) || !(a.scale < INFINITY))
    return hipErrorInvalidValue;
  const int es = dtype_size(a.dtype), vec = 16 / es;
  if (a.head_dim <= 0 || a.head_dim > MAX_HEAD_DIM || a.head_dim % vec) return hipErrorInvalidValue;
  if (a.tokens == 0 || a.q_heads == 0) return hipSuccess;
  if (a.k_heads == 0 || a.q_heads % a.k_heads || a.requests == 0 || a.table_width == 0 || a.num_pages == 0) return hipErrorInvalidValue;
  if (!a.query_starts && a.requests != a.tokens) return hipErrorInvalidValue;
  if (!a.q || !a.k_cache || !a.v_cache || !a.block_table || !a.lengths || !a.out || a.stride_table < a.table_width) return hipErrorInvalidValue;
  if ((int64_t)a.table_width * a.page_size > INT32_MAX) return hipErrorInvalidValue;
  for (const void* p : {a.q, a.k_cache, a.v_cache, (const void*)a.out, (const void*)a.workspace})
    if (!aligned16(p)) return hipErrorInvalidValue;
  for (const int64_t s : {a.stride_qt, a.stride_qh, a.stride_ot, a.stride_oh, a.stride_kc_page, a.stride_kc_row, a.stride_kc_head, a.stride_vc_page,
                          a.stride_vc_row, a.stride_vc_head})
    if (s % vec) return hipErrorInvalidValue;
  return hipSuccess;
}

template <class F>
hipError_t with_types(const iris_attention_args& a, F f) {
  using std::integral_constant;
  auto paged = [&](auto dt, auto dp) {
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
  int64_t parted = 0;   // floats behind the workspace's counters that parts are left in; 0: no unit is split
};

template <int DT, int DP, bool PG>
hipError_t make_plan(const iris_attention_args& a, int cus, Plan* p) {
  using C = rows::Cfg<DT, DP>;
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
    constexpr int per_cu = 2 * C::BT * DP * C::ES <= 32 * 1024 ? 2 : 1;
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
    // 188 x 4113 29 / 39, 268 x 2001 (4 + 4 heads) 27 / 37, 55 x 46398 79 / 86; 537 x 180 12.6 / 14.1.
    const bool few_rows = (int64_t)a.tokens * group <= 24 * (int64_t)a.requests ||
                          (few_units <= 2 * cus && few_units * most_keys <= (int64_t)1536 * cus);
    const int64_t row_tiles = (int64_t)a.tokens * group / tiles::ROWS + a.requests;
    // (a page's rows are addressed with 32 bits)
    const int64_t reach = (int64_t)a.page_size * 2 * (a.stride_kc_row > a.stride_vc_row ? a.stride_kc_row : a.stride_vc_row) + 512;
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

using Kernel = void (*)(AttentionKArgs);
template <int DT, int DP, bool PG>
Kernel kernel_of(int kernel, bool lse) {
  if (kernel == IRIS_ATTENTION_DECODE) return rows::decode_kernel<DT, DP, PG>;
  if constexpr (DT != IRIS_DTYPE_F32 && PG)
    if (kernel == IRIS_ATTENTION_PROMPT_TILES) return lse ? tiles::prompt_tiles_kernel<DT, DP, true> : tiles::prompt_tiles_kernel<DT, DP, false>;
  return rows::prompt_rows_kernel<DT, DP, PG>;
}

}  // namespace
}  // namespace iris_amd

extern "C" int64_t iris_attention_workspace_elems(int32_t head_dim) {
  using namespace iris_amd;
  if (head_dim <= 0 || head_dim > MAX_HEAD_DIM) return 0;
  return COUNTERS + ROW_SLOTS * row_slot(head_dim);
}

extern "C" int iris_attention_launch(const iris_attention_args* args, void* stream) {
  using namespace iris_amd;
  if (!args) return hipErrorInvalidValue;
  const iris_attention_args& a = *args;
  const hipError_t bad = check(a);
  if (bad != hipSuccess) return bad;
  if (a.tokens == 0 || a.q_heads == 0) return hipSuccess;

  AttentionKArgs g{};
  g.a = a;
  g.page = make_page_div((uint32_t)a.page_size);
  g.scale_log2 = a.scale * 1.4426950408889634f;
  g.group = a.q_heads / a.k_heads;
  return with_types(a, [&](auto dt, auto dp, auto pg) {
    constexpr int DT = dt.value, DP = dp.value;
    constexpr bool PG = pg.value;
    Plan p;
    const hipError_t refused = make_plan<DT, DP, PG>(a, current_cu_count(), &p);
    if (refused != hipSuccess) return refused;
    g.splits = (int)p.splits;
    g.by_length = p.by_length;
    g.grid_units = (int)p.workgroups;
    if (p.parted) {
      g.counters = (int32_t*)a.workspace;
      g.slots = a.workspace + COUNTERS;
    }
    static_assert(tiles::WAVES == rows::WAVES, "one size of workgroups");
    const unsigned heads = p.kernel == IRIS_ATTENTION_PROMPT_ROWS ? a.k_heads : 1;
    return launch(kernel_of<DT, DP, PG>(p.kernel, a.lse), dim3((unsigned)(p.workgroups / heads), heads), rows::WAVES * 64, 0, stream, g);
  });
}

extern "C" int iris_attention_plan(const iris_attention_args* args, int32_t num_cus, iris_attention_plan_info* plan) {
  using namespace iris_amd;
  if (!args || !plan || num_cus < 0) return hipErrorInvalidValue;
  const iris_attention_args& a = *args;
  const hipError_t bad = check(a);
  if (bad != hipSuccess) return bad;
  *plan = iris_attention_plan_info{0, 0, IRIS_ATTENTION_NOTHING, 1};
  if (a.tokens == 0 || a.q_heads == 0) return hipSuccess;
  return with_types(a, [&](auto dt, auto dp, auto pg) {
    Plan p;
    const hipError_t refused = make_plan<dt.value, dp.value, pg.value>(a, num_cus ? num_cus : current_cu_count(), &p);
    if (refused == hipSuccess) *plan = iris_attention_plan_info{p.parted ? COUNTERS + p.parted : 0, p.workgroups, p.kernel, (int32_t)p.splits};
    return refused;
  });
}

extern "C" int iris_attention_kernel_info(const iris_attention_args* args, int* n_regs, int* n_spills) {
  using namespace iris_amd;
  if (!args || !n_regs || !n_spills) return hipErrorInvalidValue;
  const iris_attention_args& a = *args;
  const hipError_t bad = check(a);
  if (bad != hipSuccess) return bad;
  if (a.tokens == 0 || a.q_heads == 0) return hipErrorInvalidValue;
  return with_types(a, [&](auto dt, auto dp, auto pg) {
    Plan p;
    hipError_t err = make_plan<dt.value, dp.value, pg.value>(a, current_cu_count(), &p);
    if (err != hipSuccess) return err;
    hipFuncAttributes at;
    err = hipFuncGetAttributes(&at, (const void*)kernel_of<dt.value, dp.value, pg.value>(p.kernel, a.lse));
    if (err != hipSuccess) return err;
    *n_regs = at.numRegs;
    *n_spills = (int)at.localSizeBytes;
    return hipSuccess;
  });
}
