// Attention of up to 16 query rows of one key head at a time: single tokens (the heads that share a key head are the
// rows), and prompts of few rows or of types and head sizes that the tiles of attention_tiles.hpp are not built for.
//
// Bound by reading the keys and values once.  So nothing passes through LDS: a wave takes KS keys a step, whose loads
// are the matrix instructions' operands as they lie in memory, and each of a workgroup's four waves its own steps.
//   scores   S^T[key, row] = K Q^T: a lane loads 16 bytes of the key of its own row of the 16 x 16 tile; the elements of a
//            head are summed in whatever order the loads bring them, the queries' the same.
//   weights  one running maximum and sum a row (online softmax).  A lane holds four keys of one row in S^T, so a row's
//            maximum is an exchange between four lanes, and the factor that rescales the sums is the lane's own.
//   output   O^T[d, row] += V^T P^T: P^T's operand layout wants for each row eight keys a lane, and which keys is free: it is
//            given the ones whose weights the lane holds.  A lane loads those keys' values, d contiguous, and pairs
//            of keys meet in a register by one byte permute each (16-bit types; none for fp32).
// At the end the four waves' maxima, sums and outputs meet in LDS; the parts of a split unit meet in the workspace.
//
// Single tokens, heads of 128: 606 MB of keys and values in 116 us, 5.2 TB/s, where a copy of 4 GB runs at 4.9; 56 MB in 20.2 us,
// of which 10 are a chain of latencies, as is all of one request's 9.9 (1999 keys, 4 MB): launch 2.4, lengths and the cut of
// the line 1.5, table, keys and values 2.3 a step, the waves' meeting 1, hand-over 0.8, join 2.2.
#pragma once

#include "attention_common.hpp"

namespace iris_amd {
namespace rows {

constexpr int WAVES = 4, ROWS = 16;
// Parts that meet at once, how many do where there are more, and fans at most.  (One request, 8 rows of 128, us where 16 / 24 / 48 meet at
// once: 2500 keys, 20 parts 13.4 / 12.3 / 12.3; 6000 keys, 47 parts 13.6 / 14.0 / 16.4.)
constexpr int FLAT = 24, FAN = 16, MEET = 64;
constexpr int REST = 2;                           // tiles that cost as much as beginning and ending a unit does (64 requests of up to
                                                  // 8192 keys, us at 1 / 2 / 4: 21.3 / 20.7 / 22.0)
constexpr int LATER = 1024, TOP = 2048;           // counters of fans but the first (by their first workgroup), and of a unit's fans

template <int DT, int DP>
struct Cfg {
  static constexpr bool F32 = DT == IRIS_DTYPE_F32;
  static constexpr int ES = F32 ? 4 : 2;
  static constexpr int SUBS = F32 ? 1 : 2;           // 16-key tiles of S^T a step
  static constexpr int KS = 16 * SUBS;               // keys a wave takes a step
  static constexpr int BT = KS * WAVES;              // keys a workgroup takes a step
  static constexpr int KC = DP * ES / 64;            // 16-byte pieces of a key that a lane loads
  static constexpr int VE = DP / 16;                 // elements of a value that a lane loads
  static constexpr int VB = VE * ES;                 // their bytes: 8, 16, 32 or 64
  static constexpr int VW = VB / 4;                  // their words
  static constexpr int SLOT = ROWS * (DP + 4);       // floats of a partial result
  // Weights are 2^(score - maximum + LIFT): fp16 ones of keys far below the maximum stay normal numbers (to 2^-28 of the largest
  // weight), and the sum, lifted alike, takes it out again.
  static constexpr float LIFT = DT == IRIS_DTYPE_F16 ? 14.f : 0.f;
};

template <int DT>
__device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == IRIS_DTYPE_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == IRIS_DTYPE_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
}

// A run of a unit's key tiles, [j0, j1) of the `tiles` that its rows see.
struct Piece {
  int request, head;   // key head
  int row0, rows;      // the unit's first row of the request's rows (token-major, then head), and how many it has
  int token0;          // the request's first token
  int length, first;   // keys, and the position of the request's first query
  KeyTiles tiles;
  int j0, j1;
  // a split unit: the parts' slots are first_slot and, for part i, later_slot + i * slot_step
  int parts, part, first_slot, later_slot, slot_step, counter;
};
__device__ inline int slot_of(const Piece& p, int part) { return part ? p.later_slot + part * p.slot_step : p.first_slot; }

template <int DT, int DP>
struct alignas(16) Lds {
  float o[WAVES][ROWS][DP + 4];
  f32x4 ml[WAVES][ROWS];  // maximum, sums
  int last;
};

// Writes eight (fewer at the head's end) elements of an output row.
template <int DT>
__device__ inline void store_out(const iris_attention_args& a, int64_t at, int d, const float (&v)[8]) {
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
  IRIS_GLOBAL char* p = (IRIS_GLOBAL char*)a.out + (at + d) * ES;
  if constexpr (DT == IRIS_DTYPE_F32) {
    *(IRIS_GLOBAL f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
    if (d + 4 < a.head_dim) *(IRIS_GLOBAL f32x4*)(p + 16) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    *(IRIS_GLOBAL u32x4*)p = u32x4{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
  }
}

// PG: page sizes are multiples of 16, so that 16 keys lie in one page (its number is the wave's); otherwise each lane
// looks its keys' pages up.
// ONE: all of a unit's rows stand at one position (single tokens).
template <int DT, int DP, bool PG, bool ONE>
struct Unit {
  using C = Cfg<DT, DP>;
  const AttentionKArgs& g;
  const iris_attention_args& a;
  Lds<DT, DP>& lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;  // the lane's row, and which of its four shares of a key or of the keys
  bool bad_page;

  __device__ inline Unit(const AttentionKArgs& g, Lds<DT, DP>& lds) : g(g), a(g.a), lds(lds) {}

  // The table's entries for a step's keys (for the wave, or for each of the lane's keys), and the keys and values themselves.
  struct Pages {
    int k[C::SUBS], v[C::SUBS][4];
  };
  struct Step {
    u32x4 k[C::SUBS][C::KC];
    uint32_t v[C::SUBS][4][C::VW];
  };
  __device__ inline int step_base(const Piece& p, int j) { return p.tiles.tile(j) * C::BT + wave * C::KS; }

  // The state of the lane's row.  l: the sum of the weights as they are multiplied; lse_l: as they are, for the logarithm.
  struct Row {
    u32x4 q[C::KC];
    f32x4 o[C::VE];
    float m, l, lse_l;
    int at;                // the row's position
    int first_at, last_at; // of the unit's rows
  };

  // Does some row of the unit see one of the keys first .. last?  (Positions of a unit's rows are neighbours.)
  __device__ inline bool some_see(const Row& row, int first, int last) {
    return first <= row.last_at && (a.window <= 0 || row.first_at - last < a.window || first < a.sinks);
  }
  // Steps of a tile that no row sees a key of (the wave's share of the last keys, of the window's edge, behind the first
  // tokens) are left out: their loads all go to one key, the request's first or (where its page is none) the cache's.
  __device__ inline bool seen(const Piece& p, const Row& row, int j) {
    const int base = step_base(p, j);
    return some_see(row, base, base + C::KS - 1);
  }
  __device__ inline void look_up(const Piece& p, int j, int last, Pages& pages) {
    const int base = step_base(p, j);
    const int64_t row = (int64_t)p.request * a.stride_table;
#pragma unroll
    for (int s = 0; s < C::SUBS; ++s) {
      const int first_key = base + 16 * s;
      if constexpr (PG) {
        pages.k[s] = scalar_at(a.block_table, row + page_div((uint32_t)min(first_key, last), g.page));
      } else {
        pages.k[s] = a.block_table[row + page_div((uint32_t)min(first_key + n, last), g.page)];
#pragma unroll
        for (int r = 0; r < 4; ++r) pages.v[s][r] = a.block_table[row + page_div((uint32_t)min(first_key + quad * 4 + r, last), g.page)];
      }
    }
  }
  // A table's entry for the keys first .. last.  One that is no page of the cache is none of the rows' business where they see none of
  // its keys (pages behind a window may be gone): then, as otherwise, what is read for it is the first page's.
  __device__ inline int64_t checked(int page, const Row& row, int first, int last) {
    if ((uint32_t)page < (uint32_t)a.num_pages) return page;
    bad_page |= some_see(row, first, last);
    return 0;
  }
  __device__ inline int in_page(int key) { return key - (int)(page_div((uint32_t)key, g.page) * g.page.d); }

  // Keys past `last` are read as that one, and hidden later.
  __device__ inline void load(const Piece& p, const Row& row, int j, int last, const Pages& pages, Step& x) {
    const int base = step_base(p, j);
#pragma unroll
    for (int s = 0; s < C::SUBS; ++s) {
      const int first_key = base + 16 * s, own = min(first_key + n, last);
      const int64_t page = PG ? checked(pages.k[s], row, first_key, first_key + 15) : checked(pages.k[s], row, first_key + n, first_key + n);
      const IRIS_GLOBAL char* kp = (const IRIS_GLOBAL char*)a.k_cache +
                                   (page * a.stride_kc_page + (int64_t)in_page(own) * a.stride_kc_row + (int64_t)p.head * a.stride_kc_head) * C::ES + quad * 16;
#pragma unroll
      for (int c = 0; c < C::KC; ++c) {
        x.k[s][c] = u32x4{0, 0, 0, 0};
        if ((c * 64 + quad * 16) / C::ES < a.head_dim) x.k[s][c] = *(const IRIS_GLOBAL u32x4*)(kp + c * 64);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int own_key = first_key + quad * 4 + r, key = min(own_key, last);
        const int64_t vpage = PG ? page : checked(pages.v[s][r], row, own_key, own_key);
        const IRIS_GLOBAL char* vp = (const IRIS_GLOBAL char*)a.v_cache +
                                     (vpage * a.stride_vc_page + (int64_t)in_page(key) * a.stride_vc_row + (int64_t)p.head * a.stride_vc_head) * C::ES + n * C::VB;
#pragma unroll
        for (int w = 0; w < C::VW; ++w) x.v[s][r][w] = 0;
        if constexpr (C::VB == 8) {
          if (n * C::VE < a.head_dim) {
            const u32x2 y = *(const IRIS_GLOBAL u32x2*)vp;
            x.v[s][r][0] = y[0], x.v[s][r][1] = y[1];
          }
        } else {
#pragma unroll
          for (int w = 0; w < C::VW; w += 4)
            if (n * C::VE + w * 4 / C::ES < a.head_dim) {
              const u32x4 y = *(const IRIS_GLOBAL u32x4*)(vp + w * 4);
#pragma unroll
              for (int i = 0; i < 4; ++i) x.v[s][r][w + i] = y[i];
            }
        }
      }
    }
  }

  __device__ inline void compute(const Piece& p, int j, Step& x, Row& row) {
    const int base = step_base(p, j);
    auto& v = x.v;
    f32x4 s[C::SUBS];
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < C::KC; ++c) s[u] = mfma<DT>(x.k[u][c], row.q[c], s[u]);
    }
    // Some of the step's keys may be hidden from some of the rows?  (the last keys; the window's edge)
    const bool edge = base + C::KS - 1 > row.first_at || (a.window > 0 && row.last_at - base >= a.window && base + C::KS > a.sinks);
    bool poisoned = false;  // a value that some row must not see is not a finite number
    if (edge) {
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = base + 16 * u + quad * 4 + r;
          if (!sees(a, row.at, key)) s[u][r] = -INFINITY;
          // hidden from every row: no product may see it either, whatever it is
          const bool any = ONE ? sees(a, p.first, key) : key <= row.last_at && (a.window <= 0 || row.first_at - key < a.window || key < a.sinks);
#pragma unroll
          for (int w = 0; w < C::VW; ++w) {
            if (!any) v[u][r][w] = 0;
            if (!ONE) poisoned |= not_finite(v[u][r][w]);
          }
        }
      if (!ONE) poisoned = __any(poisoned);
    }
    // the running maximum (less LIFT) and sum
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[u][r]);
    top = over_32(over_16(top * g.scale_log2 - C::LIFT, Larger{}), Larger{});
    const float m_new = fmaxf(row.m, top);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float shrink = __builtin_amdgcn_exp2f(row.m - ref);
    row.m = m_new;
    row.l *= shrink;
    row.lse_l *= shrink;
#pragma unroll
    for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[u][r] = __builtin_amdgcn_exp2f(s[u][r] * g.scale_log2 - ref);
    u32x4 weights;  // in the operand's type: for fp32 themselves
    if constexpr (C::F32) {
      weights = __builtin_bit_cast(u32x4, s[0]);
      row.l += (s[0][0] + s[0][1]) + (s[0][2] + s[0][3]);
      row.lse_l = row.l;
    } else {
      weights = u32x4{pack2<DT>(s[0][0], s[0][1]), pack2<DT>(s[0][2], s[0][3]), pack2<DT>(s[1][0], s[1][1]), pack2<DT>(s[1][2], s[1][3])};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        row.l = add_weights<DT>(weights[e], row.l);
        row.lse_l += s[0][e] + s[1][e];
      }
    }
#pragma unroll
    for (int e = 0; e < C::VE; ++e) row.o[e] *= shrink;
    if (!poisoned) {
      add_values(weights, v, row.o);
    } else {
      // (0 times it would still be NaN: each row's keys apart, with what it does not see taken out)
      for (int y = 0; y < ROWS; ++y) {
        const int at_y = __shfl(row.at, y, 64);
        uint32_t vy[C::SUBS][4][C::VW];
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool seen = sees(a, at_y, base + 16 * u + quad * 4 + r);
#pragma unroll
            for (int w = 0; w < C::VW; ++w) vy[u][r][w] = seen ? v[u][r][w] : 0;
          }
        f32x4 one[C::VE];
#pragma unroll
        for (int e = 0; e < C::VE; ++e) one[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        add_values(weights, vy, one);
#pragma unroll
        for (int e = 0; e < C::VE; ++e)
          if (n == y) row.o[e] += one[e];
      }
    }
  }

  __device__ inline void run(const Piece& p) {
    bad_page = false;
    Row row;
    // the lane's row: its query, and its position
    const bool have_row = n < p.rows;
    const int index = p.row0 + (have_row ? n : 0);
    const int token = ONE ? 0 : (int)((uint32_t)index / (uint32_t)g.group);
    const int head = p.head * g.group + index - token * g.group;
    row.at = have_row ? p.first + token : -1;
    row.first_at = ONE ? p.first : p.first + p.row0 / g.group;
    row.last_at = ONE ? p.first : p.first + (p.row0 + p.rows - 1) / g.group;
    Pages pages;
    Step x;
        {
      const IRIS_GLOBAL char* qp =
          (const IRIS_GLOBAL char*)a.q + ((int64_t)(p.token0 + token) * a.stride_qt + (int64_t)head * a.stride_qh) * C::ES + quad * 16;
#pragma unroll
      for (int c = 0; c < C::KC; ++c) {
        row.q[c] = u32x4{0, 0, 0, 0};
        if (have_row && (c * 64 + quad * 16) / C::ES < a.head_dim) row.q[c] = *(const IRIS_GLOBAL u32x4*)(qp + c * 64);
      }
    }
#pragma unroll
    for (int e = 0; e < C::VE; ++e) row.o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    row.m = -INFINITY;
    row.l = row.lse_l = 0.f;

    // A step's pages are looked up while the step before it is worked on.  (Its keys and values as well, in registers of their own,
    // took 116 us where this takes 119 for 606 MB, and the same for everything shorter, with half as much code again.)
    int last = 0;
    auto prepare = [&](int j) {
      last = seen(p, row, j) ? p.length - 1 : 0;
      look_up(p, j, last, pages);
    };
    if (p.j0 < p.j1) prepare(p.j0);
    int j = p.j0;
    for (; j < p.j1; ++j) {
      load(p, row, j, last, pages, x);
      if (j + 1 < p.j1) prepare(j + 1);
      if (seen(p, row, j)) compute(p, j, x, row);
    }
    row.l = over_32(over_16(row.l, Sum{}), Sum{});
    row.lse_l = over_32(over_16(row.lse_l, Sum{}), Sum{});
    finish(p, row.m, row.l, row.lse_l, row.o);
  }

  static __device__ inline bool not_finite(uint32_t w) {
    if constexpr (DT == IRIS_DTYPE_F32) return (w & 0x7F800000u) == 0x7F800000u;
    constexpr uint32_t E = DT == IRIS_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
    return (w & E) == E || ((w >> 16) & E) == E;
  }

  // O^T += V^T P^T
  __device__ inline void add_values(u32x4 w, const uint32_t (&v)[C::SUBS][4][C::VW], f32x4 (&o)[C::VE]) {
    if constexpr (C::F32) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < C::VE; ++e)
          o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, v[0][r][e]), __builtin_bit_cast(f32x4, w)[r], o[e], 0, 0, 0);
    } else {
      // The weights are in 16 bits, as the matrix instruction takes both its operands: off by half a last place of the values' own
      // type, which the output is rounded to as well.  (Errors against 64 bits 0.0015 to 0.0016 of the output where fp32 weights
      // have 0.0014 to 0.0015, fp16 4.9e-5 for 4.5e-5; a second product for the rest of each weight would double these instructions.)
#pragma unroll
      for (int e = 0; e < C::VE; ++e) {
        u32x4 t;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            t[2 * u + h] = __builtin_amdgcn_perm(v[u][2 * h + 1][e / 2], v[u][2 * h][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
        o[e] = mfma<DT>(t, w, o[e]);
      }
    }
  }

  // The waves' shares meet; the unit's result is written, or its part handed over.
  __device__ inline void finish(const Piece& p, float m, float l, float lse_l, const f32x4 (&o)[C::VE]) {
    if (__any(bad_page)) {
      if (lane == 0) report(a.status, IRIS_STATUS_BAD_INDEX);
      l = lse_l = __builtin_nanf("");
    }
    __syncthreads();  // (the last unit's shares have been read)
    if (quad == 0) lds.ml[wave][n] = f32x4{m, l, lse_l, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < C::VE; e += 4) {
        const f32x4 x = {o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
        *(f32x4*)&lds.o[wave][n][(quad * 4 + r) * C::VE + e] = x;
      }
    __syncthreads();
    // sixteen lanes a row
    const int row = threadIdx.x / 16, part = threadIdx.x % 16;
    float top = -INFINITY, sum = 0.f, lse_sum = 0.f, weight[WAVES];
    f32x4 ml[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      ml[w] = lds.ml[w][row];
      top = fmaxf(top, ml[w][0]);
    }
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      weight[w] = __builtin_amdgcn_exp2f(ml[w][0] - (top == -INFINITY ? 0.f : top));
      sum += weight[w] * ml[w][1];
      lse_sum += weight[w] * ml[w][2];
    }
    if (p.parts > 1) {
      if (row < p.rows) {
        float* slot = g.slots + (int64_t)slot_of(p, p.part) * C::SLOT;
#pragma unroll
        for (int d = part * 4; d < DP; d += 64) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < WAVES; ++w) x += weight[w] * *(const f32x4*)&lds.o[w][row][d];
          store16_any<AUX_SC1>((IRIS_GLOBAL char*)(slot + row * DP + d), __builtin_bit_cast(u32x4, x));
        }
        if (part == 0)
          store16_any<AUX_SC1>((IRIS_GLOBAL char*)(slot + ROWS * DP + 4 * row), __builtin_bit_cast(u32x4, f32x4{top, sum, lse_sum, 0.f}));
      }
      // Up to FLAT parts meet at once; more meet FAN by FAN, and then what they left in their first ones' slots.
      const int fan = p.parts <= FLAT ? p.parts : FAN, mine = p.part / fan * fan, members = min(fan, p.parts - mine);
      if (members > 1) {
        if (!last_to_arrive(mine ? LATER + p.counter + mine : p.counter, members)) return;
        join(p, mine, 1, members, fan == p.parts);
      }
      if (fan == p.parts) return;
      const int fans = (p.parts + fan - 1) / fan;
      if (last_to_arrive(TOP + p.counter, fans)) join(p, 0, fan, fans, true);
      return;
    }
    if (row >= p.rows) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const Target t = target(p, row);
    if (part == 0 && a.lse) a.lse[t.token * a.stride_lse + t.head] = lse_sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(lse_sum)) * 0.6931471805599453f;
#pragma unroll
    for (int d = part * 8; d < DP; d += 128)
      if (d < a.head_dim) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = 0.f;
#pragma unroll
          for (int w = 0; w < WAVES; ++w) x[e] += weight[w] * lds.o[w][row][d + e];
          x[e] *= inv;
        }
        store_out<DT>(a, t.token * a.stride_ot + t.head * a.stride_oh, d, x);
      }
  }

  struct Target {
    int64_t token, head;
  };
  __device__ inline Target target(const Piece& p, int row) {
    const int r = p.row0 + row, token = ONE ? 0 : (int)((uint32_t)r / (uint32_t)g.group);
    return {p.token0 + token, p.head * g.group + r - token * g.group};
  }

  // Counts this workgroup at counter `index`, once its stores have reached the agent's coherence point; true for the last of `all`,
  // which takes the counter back to zero.
  __device__ inline bool last_to_arrive(int index, int all) {
    IRIS_WAIT_VMCNT(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      IRIS_GLOBAL int32_t* count = (IRIS_GLOBAL int32_t*)(g.counters + index);
      lds.last = arrive(count, false, false) == all - 1;
      if (lds.last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return lds.last;
  }

  // Adds the parts first, first + step, ... (`count` of them, no more than MEET): into the output, or back into the first one's slot.
  // LANES lanes hold a row, and the first `count` of them (of LANES twice or four times in turn) its parts' maxima and sums, from
  // which every part's weight follows at once; where there are few rows, sets of lanes take every so many-th part's output
  // and add up in LDS.  Fixed orders all the way.  Heads of 256 load 16 bytes and 16 parts at once (two requests of up to 16602 keys,
  // 16 rows: 32.7 us, 37.6 with 8); for shorter ones that costs the rest of the kernel as much as it gives (606 MB in heads of 128
  // 121 us for 118.5, one request of 1999 keys 11.0 for 10.3).
  __device__ inline void join(const Piece& p, int first, int step, int count, bool whole) {
    constexpr int LANES = DP / 4, GROUPS = WAVES * 64 / LANES, AT_ONCE = DP == 256 ? FAN : 8, HOLD = (MEET + LANES - 1) / LANES;
    int abreast = 1;  // rows that are worked on at once
    while (abreast < p.rows && abreast < GROUPS) abreast *= 2;
    const int sets = GROUPS / abreast, group = threadIdx.x / LANES, set = group / abreast, in_row = threadIdx.x % LANES, d = in_row * 4;
    float* const flat = &lds.o[0][0][0];         // sets' sums
    float* const weights = flat + GROUPS * DP;   // the groups' weights of the parts
    // What other workgroups have written through, 16 bytes at float `at` of part i.  (The parts of a launch lie within 31 bits: at most
    // two a workgroup or 24 a unit of 512.)
    auto load_slot = [&](int i, int at) {
      const int64_t word = (int64_t)slot_of(p, first + i * step) * C::SLOT + at;
      if constexpr (DP == 256) {
        const __amdgpu_buffer_rsrc_t slots = tile_rsrc((const IRIS_GLOBAL char*)g.slots, 0x7FFFFFFF);
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(slots, (int)word * 4, 0, AUX_SC1));
      } else {
        const IRIS_GLOBAL uint64_t* at16 = (const IRIS_GLOBAL uint64_t*)(g.slots + word);
        const u32x2 lo = __builtin_bit_cast(u32x2, __hip_atomic_load(at16, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        const u32x2 hi = __builtin_bit_cast(u32x2, __hip_atomic_load(at16 + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        return __builtin_bit_cast(f32x4, u32x4{lo[0], lo[1], hi[0], hi[1]});
      }
    };
    auto row_of = [&](int row0) { return min(row0 + group % abreast, p.rows - 1); };  // (groups without a row repeat the last)
    f32x4 ml[HOLD], next_ml[HOLD];
    auto fetch_ml = [&](int row0) {
#pragma unroll
      for (int i = 0; i < HOLD; ++i) {
        next_ml[i] = f32x4{-INFINITY, 0.f, 0.f, 0.f};
        if (i * LANES + in_row < count) next_ml[i] = load_slot(i * LANES + in_row, ROWS * DP + 4 * row_of(row0));
      }
    };
    fetch_ml(0);
    for (int row0 = 0; row0 < p.rows; row0 += abreast) {
      const int row = row0 + group % abreast, used = row_of(row0);
#pragma unroll
      for (int i = 0; i < HOLD; ++i) ml[i] = next_ml[i];
      f32x4 y[AT_ONCE];
      auto fetch = [&](int i0) {
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
          if (i0 + i * sets < count) y[i] = load_slot(i0 + i * sets, used * DP + d);
      };
      fetch(set);
      if (row0 + abreast < p.rows) fetch_ml(row0 + abreast);
      float top = -INFINITY, sum = 0.f, lse_sum = 0.f;
#pragma unroll
      for (int i = 0; i < HOLD; ++i) top = fmaxf(top, ml[i][0]);
      top = over_lanes<LANES>(top, Larger{});
      __syncthreads();  // (what LDS held has been read)
#pragma unroll
      for (int i = 0; i < HOLD; ++i) {
        const float w = __builtin_amdgcn_exp2f(ml[i][0] - (top == -INFINITY ? 0.f : top));
        sum += w * ml[i][1];
        lse_sum += w * ml[i][2];
        if (i * LANES + in_row < MEET) weights[group * MEET + i * LANES + in_row] = w;
      }
      sum = over_lanes<LANES>(sum, Sum{});
      lse_sum = over_lanes<LANES>(lse_sum, Sum{});
      __syncthreads();
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      for (int i0 = set; i0 < count; i0 += sets * AT_ONCE) {
        if (i0 > set) fetch(i0);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
          if (i0 + i * sets < count) x += y[i] * weights[group * MEET + i0 + i * sets];
      }
      if (sets > 1) {
        *(f32x4*)(flat + group * DP + d) = x;
        __syncthreads();
        if (set == 0) {
          x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < GROUPS; ++i)
            if (i < sets) x += *(const f32x4*)(flat + (group + i * abreast) * DP + d);
        }
      }
      if (set > 0 || row >= p.rows) continue;
      if (!whole) {
        char* slot = (char*)(g.slots + (int64_t)slot_of(p, first) * C::SLOT);
        store16_any<AUX_SC1>((IRIS_GLOBAL char*)slot + (row * DP + d) * 4, __builtin_bit_cast(u32x4, x));
        if (d == 0) store16_any<AUX_SC1>((IRIS_GLOBAL char*)slot + (ROWS * DP + 4 * row) * 4, __builtin_bit_cast(u32x4, f32x4{top, sum, lse_sum, 0.f}));
        continue;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const Target t = target(p, row);
      if (d == 0 && a.lse) a.lse[t.token * a.stride_lse + t.head] = lse_sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(lse_sum)) * 0.6931471805599453f;
      if (d >= a.head_dim) continue;
      IRIS_GLOBAL char* out = (IRIS_GLOBAL char*)a.out + (t.token * a.stride_ot + t.head * a.stride_oh + d) * C::ES;
      x *= inv;
      if constexpr (C::F32)
        *(IRIS_GLOBAL f32x4*)out = x;
      else
        *(IRIS_GLOBAL u32x2*)out = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
    }
  }
};

// Rows that see nothing: zeros.
template <int DT>
__device__ inline void clear_row(const iris_attention_args& a, int64_t token, int head) {
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
  for (int d = (threadIdx.x & 63) * (16 / ES); d < a.head_dim; d += 64 * (16 / ES))
    *(IRIS_GLOBAL u32x4*)((IRIS_GLOBAL char*)a.out + (token * a.stride_ot + head * a.stride_oh + d) * ES) = u32x4{0, 0, 0, 0};
  if (a.lse && (threadIdx.x & 63) == 0) a.lse[token * a.stride_lse + head] = -INFINITY;
}

// A request's keys: never more than its table row has pages for.
__device__ inline int keys_of(const AttentionKArgs& g, int request) {
  const int64_t room = (int64_t)g.a.table_width * g.page.d;
  const int length = max(g.a.lengths[request], 0);
  if (length > room) {
    report(g.a.status, IRIS_STATUS_BAD_INDEX);
    return (int)room;
  }
  return length;
}

// Single tokens.  All units (request, key head, rows of 16) lie in one line, each as long as its key tiles and REST more for what a
// unit costs beside them, and the workgroups cut the line into equal runs: requests of any lengths load every workgroup
// alike.  A run's first and last unit may be shared with the workgroups beside it.
template <int DT, int DP, bool PG>
__global__ __launch_bounds__(WAVES * 64, DP == 256 ? 1 : 2) void decode_kernel(AttentionKArgs g) {
  using C = Cfg<DT, DP>;
  __shared__ Lds<DT, DP> lds;
  __shared__ int wave_sum[WAVES];
  __shared__ int found_request, found_before, found_length;
  touch_args<sizeof(AttentionKArgs)>();
  const iris_attention_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row_tiles = (g.group + ROWS - 1) / ROWS, units = a.k_heads * row_tiles;
  constexpr int STEP = WAVES * 64;

  // what a unit of `length` keys takes of the line
  auto span_of = [&](int length) { return length > 0 ? key_tiles<C::BT>(a, length - 1, length - 1).count + REST : 0; };
  // The line's length, and the request in which this workgroup's run begins: sums over the requests, STEP of them at a time, once
  // where they are no more than that.  (The launcher has seen to it that the line is no longer than 31 bits count.)
  int length = 0, own = 0, sum = 0;  // keys and span of the lane's request, and spans up to it in the wave
  auto add_up = [&](int base) {
    const int r = base + tid;
    length = r < a.requests ? keys_of(g, r) : 0;
    own = span_of(length);
    sum = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(sum, d, 64);
      if (lane >= d) sum += x;
    }
    __syncthreads();
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int chunk = 0;
    for (int w = 0; w < WAVES; ++w) chunk += wave_sum[w];
    return chunk;
  };
  int total = 0;
  for (int base = 0; base < a.requests; base += STEP) total += add_up(base);
  const uint32_t all = (uint32_t)total * units, groups = min(all, (uint32_t)g.grid_units);
  if (blockIdx.x < groups) {
    // runs of `each`, the first `longer` of them one longer
    const uint32_t each = all / groups, longer = all - each * groups;
    const uint32_t begin = blockIdx.x * each + min(blockIdx.x, longer), end = begin + each + (blockIdx.x < longer);
    auto group_at = [&](uint32_t x) { return x < longer * (each + 1) ? x / (each + 1) : longer + (x - longer * (each + 1)) / each; };
    int before = 0;  // spans of earlier chunks
    for (int base = 0; base < a.requests; base += STEP) {
      const int chunk = a.requests > STEP ? add_up(base) : total;
      int ahead = before;
      for (int w = 0; w < wave; ++w) ahead += wave_sum[w];
      const uint32_t lo = (uint32_t)(ahead + sum - own) * units, hi = (uint32_t)(ahead + sum) * units;
      if (lo <= begin && begin < hi) {
        found_request = base + tid;
        found_before = ahead + sum - own;
        found_length = length;
      }
      before += chunk;
      if ((uint32_t)before * units > begin) break;
    }
    __syncthreads();
    int request = __builtin_amdgcn_readfirstlane(found_request), next_length = __builtin_amdgcn_readfirstlane(found_length);
    uint32_t base = (uint32_t)__builtin_amdgcn_readfirstlane(found_before) * units;  // the request's place in the line

    Unit<DT, DP, PG, true> unit(g, lds);
    for (uint32_t at = begin; at < end; ++request) {
      Piece p;
      p.request = request;
      p.length = next_length;
      p.first = p.length - 1;
      p.tiles = key_tiles<C::BT>(a, p.first, p.first);
      const uint32_t span = p.length > 0 ? p.tiles.count + REST : 0, request_end = base + span * units;
      while (at < end && at < request_end) {
        const uint32_t u = (at - base) / span, unit_begin = base + u * span, tiles_begin = unit_begin + REST, unit_end = unit_begin + span;
        const uint32_t from = max(at, tiles_begin), to = min(end, unit_end);
        at = unit_end;
        if (from >= to) continue;  // (the run ends in what stands before the tiles)
        p.head = row_tiles == 1 ? u : u / row_tiles;
        p.row0 = (u - p.head * row_tiles) * ROWS;
        p.rows = min(ROWS, g.group - p.row0);
        p.token0 = request;
        p.parts = 1;
        p.j0 = from - tiles_begin;
        p.j1 = to - tiles_begin;
        if (g.slots) {
          // the workgroups of the first and the last tile
          const int first = tiles_begin >= begin ? (int)blockIdx.x : group_at(tiles_begin);
          const int last = unit_end <= end ? (int)blockIdx.x : group_at(unit_end - 1);
          p.parts = last - first + 1;
          p.part = (int)blockIdx.x - first;
          p.first_slot = 2 * first + 1;
          p.later_slot = 2 * first;
          p.slot_step = 2;
          p.counter = first;
        } else {  // nothing is split: a unit is its first tile's workgroup's
          if (p.j0) continue;
          p.j1 = p.tiles.count;
        }
        unit.run(p);
      }
      base = request_end;
      if (at < end) next_length = min(max(scalar_at(a.lengths, request + 1), 0), (int)(a.table_width * g.page.d));
    }
  }
  // idle requests
  for (int64_t r = blockIdx.x * WAVES + wave; r < a.requests; r += (int64_t)gridDim.x * WAVES)
    if (a.lengths[r] <= 0)
      for (int h = 0; h < a.q_heads; ++h) clear_row<DT>(a, r, h);
}

// Prompts: a workgroup for 16 rows of a request and key head, and a share of the keys they see.  Row tile x of the grid is the
// (x - bound)-th of the last request whose bound, floor(query_starts * group / 16) + request, is not past x: bounds leave each
// request room for its row tiles without a sum over the requests.
template <int DT, int DP, bool PG>
__global__ __launch_bounds__(WAVES * 64, DP == 256 ? 1 : 2) void prompt_rows_kernel(AttentionKArgs g) {
  using C = Cfg<DT, DP>;
  __shared__ Lds<DT, DP> lds;
  const iris_attention_args& a = g.a;
  const int x = blockIdx.x / g.splits, split = blockIdx.x - x * g.splits;
  auto bound = [&](int r) { return (int)((int64_t)scalar_at(a.query_starts, r) * g.group / ROWS) + r; };
  int lo = 0, hi = a.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (bound(mid) <= x)
      lo = mid;
    else
      hi = mid;
  }
  Piece p;
  p.request = lo;
  p.token0 = scalar_at(a.query_starts, lo);
  const int tokens = min(scalar_at(a.query_starts, lo + 1), a.tokens) - p.token0;
  p.row0 = (x - bound(lo)) * ROWS;
  if (p.row0 < 0 || p.token0 < 0 || tokens <= 0 || p.row0 >= (int64_t)tokens * g.group) return;
  p.rows = min((int64_t)ROWS, (int64_t)tokens * g.group - p.row0);
  p.head = blockIdx.y;
  p.length = __builtin_amdgcn_readfirstlane(keys_of(g, lo));
  p.first = p.length - tokens;
  p.tiles = key_tiles<C::BT>(a, p.first + p.row0 / g.group, p.first + (p.row0 + p.rows - 1) / g.group);
  p.parts = max(min(g.splits, p.tiles.count), 1);
  p.part = split;
  if (split >= p.parts) return;
  p.j0 = (int)((int64_t)p.tiles.count * split / p.parts);
  p.j1 = (int)((int64_t)p.tiles.count * (split + 1) / p.parts);
  const int index = blockIdx.y * (gridDim.x / g.splits) + x;
  p.first_slot = index * g.splits;
  p.later_slot = p.first_slot;
  p.slot_step = 1;
  p.counter = index;
  Unit<DT, DP, PG, false> unit(g, lds);
  unit.run(p);
}

}  // namespace rows
}  // namespace iris_amd
