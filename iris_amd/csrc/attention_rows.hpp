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
#pragma once

#include "attention_common.hpp"

namespace iris_amd {
namespace rows {

constexpr int WAVES = 4, ROWS = 16;

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
  float m[WAVES][ROWS], l[WAVES][ROWS], lse_l[WAVES][ROWS];
  int last;
};

// One row's maximum (sum) over the four lanes that hold its keys.
__device__ inline float max_of_row(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}

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

  __device__ inline int64_t page_at(const Piece& p, int key, bool uniform) {
    const int64_t at = (int64_t)p.request * a.stride_table + page_div((uint32_t)key, g.page);
    int page = uniform ? scalar_at(a.block_table, at) : a.block_table[at];
    if ((uint32_t)page >= (uint32_t)a.num_pages) {
      bad_page = true;
      page = 0;
    }
    return page;
  }
  // byte offset of key `key` (below the request's length) in a cache
  struct Where {
    int64_t k, v;
  };
  __device__ inline Where where(const Piece& p, int64_t page, int key) {
    const int in_page = key - (int)(page_div((uint32_t)key, g.page) * g.page.d);
    return {(page * a.stride_kc_page + (int64_t)in_page * a.stride_kc_row + (int64_t)p.head * a.stride_kc_head) * C::ES,
            (page * a.stride_vc_page + (int64_t)in_page * a.stride_vc_row + (int64_t)p.head * a.stride_vc_head) * C::ES};
  }

  __device__ inline void run(const Piece& p) {
    bad_page = false;
    // the lane's row: its query, and its position
    const int row = p.row0 + n;
    const bool have_row = n < p.rows;
    const int token = ONE ? 0 : (int)((uint32_t)(have_row ? row : p.row0) / (uint32_t)g.group);
    const int head = p.head * g.group + (have_row ? row : p.row0) - token * g.group;
    const int at = have_row ? p.first + token : -1;
    const int first_at = ONE ? p.first : p.first + p.row0 / g.group;
    const int last_at = ONE ? p.first : p.first + (p.row0 + p.rows - 1) / g.group;
    u32x4 q[C::KC];
    {
      const IRIS_GLOBAL char* qp =
          (const IRIS_GLOBAL char*)a.q + ((int64_t)(p.token0 + token) * a.stride_qt + (int64_t)head * a.stride_qh) * C::ES + quad * 16;
#pragma unroll
      for (int c = 0; c < C::KC; ++c) {
        q[c] = u32x4{0, 0, 0, 0};
        if (have_row && (c * 64 + quad * 16) / C::ES < a.head_dim) q[c] = *(const IRIS_GLOBAL u32x4*)(qp + c * 64);
      }
    }
    f32x4 o[C::VE];
#pragma unroll
    for (int e = 0; e < C::VE; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    // l: the sum of the weights as they are multiplied; lse_l: as they are, for the logarithm
    float m = -INFINITY, l = 0.f, lse_l = 0.f;

    for (int j = p.j0; j < p.j1; ++j) {
      const int base = p.tiles.tile(j) * C::BT + wave * C::KS;
      if (base > last_at) continue;
      const int last_key = p.length - 1;
      u32x4 k[C::SUBS][C::KC];
      uint32_t v[C::SUBS][4][C::VW];
#pragma unroll
      for (int s = 0; s < C::SUBS; ++s) {
        const int first_key = base + 16 * s, own = min(first_key + n, last_key);
        const int64_t page = page_at(p, PG ? min(first_key, last_key) : own, PG);
        const IRIS_GLOBAL char* kp = (const IRIS_GLOBAL char*)a.k_cache + where(p, page, own).k + quad * 16;
#pragma unroll
        for (int c = 0; c < C::KC; ++c) {
          k[s][c] = u32x4{0, 0, 0, 0};
          if ((c * 64 + quad * 16) / C::ES < a.head_dim) k[s][c] = *(const IRIS_GLOBAL u32x4*)(kp + c * 64);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = min(first_key + quad * 4 + r, last_key);
          const int64_t vpage = PG ? page : page_at(p, key, false);
          const IRIS_GLOBAL char* vp = (const IRIS_GLOBAL char*)a.v_cache + where(p, vpage, key).v + n * C::VB;
#pragma unroll
          for (int w = 0; w < C::VW; ++w) v[s][r][w] = 0;
          if constexpr (C::VB == 8) {
            if (n * C::VE < a.head_dim) {
              const u32x2 x = *(const IRIS_GLOBAL u32x2*)vp;
              v[s][r][0] = x[0], v[s][r][1] = x[1];
            }
          } else {
#pragma unroll
            for (int w = 0; w < C::VW; w += 4)
              if (n * C::VE + w * 4 / C::ES < a.head_dim) {
                const u32x4 x = *(const IRIS_GLOBAL u32x4*)(vp + w * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[s][r][w + i] = x[i];
              }
          }
        }
      }
      f32x4 s[C::SUBS];
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u) {
        s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C::KC; ++c) s[u] = mfma<DT>(k[u][c], q[c], s[u]);
      }
      // Some of the step's keys may be hidden from some of the rows?  (the last keys; the window's edge)
      const bool edge = base + C::KS - 1 > first_at || (a.window > 0 && last_at - base >= a.window && base + C::KS > a.sinks);
      bool poisoned = false;  // a value that some row must not see is not a finite number
      if (edge) {
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = base + 16 * u + quad * 4 + r;
            if (!sees(a, at, key)) s[u][r] = -INFINITY;
            // hidden from every row: no product may see it either, whatever it is
            const bool any = ONE ? sees(a, p.first, key) : key <= last_at && (a.window <= 0 || first_at - key < a.window || key < a.sinks);
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
      top = max_of_row(top * g.scale_log2 - C::LIFT);
      const float m_new = fmaxf(m, top);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float shrink = __builtin_amdgcn_exp2f(m - ref);
      m = m_new;
      l *= shrink;
      lse_l *= shrink;
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[u][r] = __builtin_amdgcn_exp2f(s[u][r] * g.scale_log2 - ref);
      u32x4 weights;  // in the operand's type: for fp32 themselves
      if constexpr (C::F32) {
        weights = __builtin_bit_cast(u32x4, s[0]);
        l += (s[0][0] + s[0][1]) + (s[0][2] + s[0][3]);
        lse_l = l;
      } else {
        weights = u32x4{pack2<DT>(s[0][0], s[0][1]), pack2<DT>(s[0][2], s[0][3]), pack2<DT>(s[1][0], s[1][1]), pack2<DT>(s[1][2], s[1][3])};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          l = add_weights<DT>(weights[e], l);
          lse_l += s[0][e] + s[1][e];
        }
      }
#pragma unroll
      for (int e = 0; e < C::VE; ++e) o[e] *= shrink;
      if (!poisoned) {
        add_values(weights, v, o);
      } else {
        // (0 times it would still be NaN: each row's keys apart, with what it does not see taken out)
        for (int x = 0; x < ROWS; ++x) {
          const int at_x = __shfl(at, x, 64);
          uint32_t vx[C::SUBS][4][C::VW];
#pragma unroll
          for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool seen = sees(a, at_x, base + 16 * u + quad * 4 + r);
#pragma unroll
              for (int w = 0; w < C::VW; ++w) vx[u][r][w] = seen ? v[u][r][w] : 0;
            }
          f32x4 one[C::VE];
#pragma unroll
          for (int e = 0; e < C::VE; ++e) one[e] = f32x4{0.f, 0.f, 0.f, 0.f};
          add_values(weights, vx, one);
#pragma unroll
          for (int e = 0; e < C::VE; ++e)
            if (n == x) o[e] += one[e];
        }
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    lse_l += __shfl_xor(lse_l, 16, 64);
    lse_l += __shfl_xor(lse_l, 32, 64);
    finish(p, m, l, lse_l, o);
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
      // (the weights are in 16 bits, as the matrix instruction takes them: off by half a last place of the values' own type)
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
    if (quad == 0) {
      lds.m[wave][n] = m;
      lds.l[wave][n] = l;
      lds.lse_l[wave][n] = lse_l;
    }
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
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds.m[w][row]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      weight[w] = __builtin_amdgcn_exp2f(lds.m[w][row] - (top == -INFINITY ? 0.f : top));
      sum += weight[w] * lds.l[w][row];
      lse_sum += weight[w] * lds.lse_l[w][row];
    }
    if (p.parts > 1) {
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
      // the stores have reached the agent's coherence point before the arrival is counted
      IRIS_WAIT_VMCNT(0);
      __syncthreads();
      if (threadIdx.x == 0) {
        IRIS_GLOBAL int32_t* count = (IRIS_GLOBAL int32_t*)(g.counters + p.counter);
        lds.last = arrive(count, false, false) == p.parts - 1;
        if (lds.last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (lds.last) join(p, row, part);
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

  // The last part to arrive adds all parts, in their order.
  __device__ inline void join(const Piece& p, int row, int part) {
    if (row >= p.rows) return;
    auto buffer = [&](int i) { return tile_rsrc((const IRIS_GLOBAL char*)(g.slots + (int64_t)slot_of(p, i) * C::SLOT), C::SLOT * 4); };
    float top = -INFINITY, sum = 0.f, lse_sum = 0.f;
    constexpr int NV = (DP + 63) / 64;
    f32x4 x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < p.parts; ++i) {
      const __amdgpu_buffer_rsrc_t rs = buffer(__builtin_amdgcn_readfirstlane(i));
      const f32x4 ml = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (ROWS * DP + 4 * row) * 4, 0, AUX_SC1));
      u32x4 y[NV];
#pragma unroll
      for (int d = 0; d < NV; ++d) y[d] = __builtin_amdgcn_raw_buffer_load_b128(rs, (row * DP + d * 64 + part * 4) * 4, 0, AUX_SC1);
      const float mi = ml[0];
      const float t = fmaxf(top, mi), ref = t == -INFINITY ? 0.f : t;
      const float old = __builtin_amdgcn_exp2f(top - ref), now = __builtin_amdgcn_exp2f(mi - ref);
      top = t;
      sum = sum * old + ml[1] * now;
      lse_sum = lse_sum * old + ml[2] * now;
#pragma unroll
      for (int d = 0; d < NV; ++d) x[d] = x[d] * old + __builtin_bit_cast(f32x4, y[d]) * now;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const Target t = target(p, row);
    if (part == 0 && a.lse) a.lse[t.token * a.stride_lse + t.head] = lse_sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(lse_sum)) * 0.6931471805599453f;
#pragma unroll
    for (int d = 0; d < NV; ++d) {
      const int at = d * 64 + part * 4;
      if (at >= a.head_dim) continue;
      IRIS_GLOBAL char* out = (IRIS_GLOBAL char*)a.out + (t.token * a.stride_ot + t.head * a.stride_oh + at) * C::ES;
      x[d] *= inv;
      if constexpr (C::F32)
        *(IRIS_GLOBAL f32x4*)out = x[d];
      else
        *(IRIS_GLOBAL u32x2*)out = u32x2{pack2<DT>(x[d][0], x[d][1]), pack2<DT>(x[d][2], x[d][3])};
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

// Single tokens.  All units' key tiles lie in one line (request, key head, rows of 16, tile), which the workgroups cut into
// equal runs: requests of any lengths load every workgroup alike.  A run's first and last unit may be shared with
// the workgroups beside it.
template <int DT, int DP, bool PG>
__global__ __launch_bounds__(WAVES * 64, DP == 256 ? 1 : 2) void decode_kernel(AttentionKArgs g) {
  using C = Cfg<DT, DP>;
  __shared__ Lds<DT, DP> lds;
  __shared__ int wave_sum[WAVES];
  __shared__ int found_request, found_before;
  const iris_attention_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row_tiles = (g.group + ROWS - 1) / ROWS, units = a.k_heads * row_tiles;
  constexpr int STEP = WAVES * 64;

  auto tiles_of = [&](int request) {
    const int length = keys_of(g, request);
    return key_tiles<C::BT>(a, length - 1, length - 1).count;
  };
  // idle requests
  for (int64_t r = blockIdx.x * WAVES + wave; r < a.requests; r += (int64_t)gridDim.x * WAVES)
    if (keys_of(g, (int)r) == 0)
      for (int h = 0; h < a.q_heads; ++h) clear_row<DT>(a, r, h);

  // all tiles, then the request in which this workgroup's run begins
  int64_t total = 0;
  int mine = 0;
  for (int r = tid; r < a.requests; r += STEP) mine += tiles_of(r);
  for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d, 64);
  if (lane == 0) wave_sum[wave] = mine;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) total += wave_sum[w];
  const int64_t all = total * units;
  if (all == 0) return;
  const int64_t groups = all < g.grid_units ? all : g.grid_units;
  if (blockIdx.x >= groups) return;
  const int64_t begin = all * blockIdx.x / groups, end = all * (blockIdx.x + 1) / groups;
  int before = 0;
  for (int base = 0; base < a.requests; base += STEP) {
    __syncthreads();
    const int r = base + tid, own = r < a.requests ? tiles_of(r) : 0;
    int sum = own;
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(sum, d, 64);
      if (lane >= d) sum += x;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int ahead = before, chunk = 0;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) ahead += wave_sum[w];
      chunk += wave_sum[w];
    }
    const int64_t lo = (int64_t)(ahead + sum - own) * units, hi = (int64_t)(ahead + sum) * units;
    if (lo <= begin && begin < hi) {
      found_request = r;
      found_before = ahead + sum - own;
    }
    before += chunk;
    if ((int64_t)before * units > begin) break;
  }
  __syncthreads();
  int request = __builtin_amdgcn_readfirstlane(found_request);
  int64_t base = (int64_t)__builtin_amdgcn_readfirstlane(found_before) * units;  // the request's first tile in the line

  Unit<DT, DP, PG, true> unit(g, lds);
  for (int64_t at = begin; at < end;) {
    Piece p;
    p.request = request;
    p.length = __builtin_amdgcn_readfirstlane(keys_of(g, request));
    p.first = p.length - 1;
    p.tiles = key_tiles<C::BT>(a, p.first, p.first);
    const int64_t request_end = base + (int64_t)p.tiles.count * units;
    if (at >= request_end) {  // (idle requests have no tiles)
      base = request_end;
      ++request;
      continue;
    }
    const int u = (int)((at - base) / p.tiles.count);
    const int64_t unit_begin = base + (int64_t)u * p.tiles.count, unit_end = unit_begin + p.tiles.count;
    p.head = u / row_tiles;
    p.row0 = (u - p.head * row_tiles) * ROWS;
    p.rows = min(ROWS, g.group - p.row0);
    p.token0 = request;
    if (!g.slots) {  // nothing is split: a unit is its first tile's workgroup's
      at = unit_end;
      if (at - p.tiles.count < begin) continue;
      p.j0 = 0;
      p.j1 = p.tiles.count;
      p.parts = 1;
      unit.run(p);
      continue;
    }
    p.j0 = (int)(at - unit_begin);
    p.j1 = (int)((end < unit_end ? end : unit_end) - unit_begin);
    // the workgroups that hold the unit's first and last tile
    const int first = (int)(((unit_begin + 1) * groups - 1) / all), last = (int)((unit_end * groups - 1) / all);
    p.parts = last - first + 1;
    p.part = (int)blockIdx.x - first;
    p.first_slot = 2 * first + 1;
    p.later_slot = 2 * first;
    p.slot_step = 2;
    p.counter = first;
    unit.run(p);
    at = unit_begin + p.j1;
  }
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
  p.parts = g.splits;
  p.part = split;
  p.j0 = (int)((int64_t)p.tiles.count * split / g.splits);
  p.j1 = (int)((int64_t)p.tiles.count * (split + 1) / g.splits);
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
