// Attention of prompts in 16 bits: 128 query rows of one key head a workgroup, keys and values through LDS.
//
// Rows are (token, query head of the key head) pairs, token-major, so that heads that share keys share their tiles.  Four waves
// take 32 rows each and walk the keys in tiles of 64:
//   scores   S^T[key, row] = K Q^T on 32 x 32 x 16 matrix instructions; the queries stay in registers.
//   weights  one pass with a running reference and sum a row (online softmax).  A lane holds half of a row's keys of the tile
//            and only one row, so a maximum is one exchange and a rescaling factor the lane's own; and the reference need not be the
//            maximum, only near enough that weights and sums stay in range, so almost no tile looks for the one or needs the other.
//   output   O^T[d, row] += V^T P^T: the lane's weights are P^T's operand as they are, four consecutive keys at a time, and
//            V^T's comes out of LDS transposed (ds_read_b64_tr_b16: four keys of sixteen columns).
// Tiles go from the pages to LDS by LDS-DMA, 16 bytes a lane, two stages, with the 16-byte chunks of a row exchanged
// (XOR) so that neither read meets its own banks; keys past the end and columns past the head are read out of
// the buffer's range and arrive as zeros.
//
// bf16, heads of 128, four prompts of up to 8192 tokens (310 GFLOP): 327 to 335 us, 0.93 to 0.95 PFLOP/s, where a large matrix product runs at
// 1.19; fp16, heads of 64, a window of 1024 (25 GFLOP): 51 to 52 us, 0.48.  The matrix cores are busy for 0.41 of the time and
// vector instructions issue for 0.33, the one wave's beside the other's; the rest is LDS reads, barriers and
// power (zeros take an eighth less).  Tiles of 64 rows a wave, or a tile's scores taken ahead of the last one's values, took
// more registers than there are and 394 us and more.
// The waves take all the registers that so many a SIMD have, and spill: 15 to 21 words a lane for heads of 64, 21 to 26 for 128, of
// which the loop reads none (with log-sums one); 90 for heads of 256, whose loop reads eight, behind a wait that the next tile's
// loads are part of (0.59 PFLOP/s on prompts of 4096 and 2500 tokens, 8 + 2 heads, where heads of 128 have 0.48).
#pragma once

#include "attention_rows.hpp"

namespace iris_amd {
namespace tiles {

constexpr int WAVES = 4, ROWS = 128, WAVE_ROWS = 32, BT = 64;
constexpr int AHEAD = 4;  // operands in flight ahead of the matrix instructions (three, four or six: the same time)
// Parts of a row tile's keys: of no fewer than LEAST tiles (rows that see few keys are not cut as the longest are: 8 prompts of up to
// 32 tokens behind up to 4096, 40.5 us for 41.9), and no more than MOST_PARTS, for the last adds them up one by one (8 of up to
// 30 behind up to 8000, us at 4 / 8 / 16 / 31 parts: 51 / 35 / 31 / 53).
constexpr int LEAST = 2, MOST_PARTS = 16;
constexpr int SCHED_MFMA = 0x8, SCHED_DS_READ = 0x100;  // kinds of instructions of __builtin_amdgcn_sched_group_barrier

// As many as their registers let in.  (Heads of 64, a window of 1024: two 58 us, three 55, four 77, for they spill.)
constexpr int waves_a_simd(int dp) { return dp == 64 ? 3 : dp == 128 ? 2 : 1; }

template <int DT, int DP>
struct Cfg {
  static constexpr int ROW_BYTES = DP * 2;
  static constexpr int TILE_BYTES = BT * ROW_BYTES;
  static constexpr int CHUNKS = ROW_BYTES / 16;        // 16-byte chunks of a key
  static constexpr int DMA_ROWS = 1024 / ROW_BYTES;    // keys that one LDS-DMA instruction of a wave moves
  static constexpr int DMAS = 16 / DMA_ROWS;           // ... and how many move a wave's 16 keys of a tile
  static constexpr int KC = DP / 16;                   // matrix instructions over a head
  static constexpr int DTILES = DP / 32;               // 32-column tiles of the output
  static constexpr int SLOT = ROWS * DP + WAVES * 64 * 4;  // floats of a partial result
  // Weights are 2^(score - reference), and the reference is the maximum, less LIFT, of the first keys that the row sees; it stays
  // until a lane's 32 weights of a tile sum up to more than MOST.  fp16 ends at 65504 and loses places below 2^-14, so that LIFT
  // stands between.  bf16 has fp32's range, but so have its values: weights begin at 2^-16 at most and are not let past 1, so that
  // their products with values sum up to no more than those against the running maximum would.  (The same time as with a
  // reference at the maximum and sums of up to 2^60, where values of 3e20 and more could leave fp32's range.)
  static constexpr float LIFT = DT == IRIS_DTYPE_F16 ? 6.f : -16.f;
  static constexpr float MOST = DT == IRIS_DTYPE_F16 ? 32768.f : 1.f;
};

// The chunk of its row that lies at chunk position p (and the other way round: both are XORs).
template <int DP>
__device__ inline int swizzle_k(int row, int p) {
  return p ^ (DP == 64 ? (row >> 1) & 7 : row & 15);
}
template <int DP>
__device__ inline int swizzle_v(int row, int p) {
  return p ^ (DP == 64 ? 2 * ((row >> 1) & 3) : 2 * (row & 7));
}

template <int DT>
__device__ inline f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == IRIS_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Which of the keys base .. base + 31 the query at position `at` sees, as bits.
__device__ inline uint32_t visible(const iris_attention_args& a, int at, int base) {
  auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
  const uint32_t past = below(at + 1 - base);
  return a.window > 0 ? past & (~below(at - a.window + 1 - base) | below(a.sinks - base)) : past;
}

// The row tile that sees the k-th most keys, later rows before earlier ones: workgroups that start last are then the
// short ones.  (A prompt of 8192 tokens among others, 1153 row tiles of 1 to 128 key tiles on 512 places: 382 us in the requests'
// order, 336 by length; with a window, 796 row tiles of heads of 64 on 768, 54.8 and 52.3; heads of 256, a prompt of
// 6000, 320 and 279.)  Request r has tiles_r row tiles, and of those that see at least c
// key tiles the number is known in closed form; the largest c with more than k of them in all is found by bisection, the
// lanes adding up the requests.
__device__ inline bool nth_longest(const AttentionKArgs& g, int k, int* request, int* row_tile) {
  const iris_attention_args& a = g.a;
  const int lane = threadIdx.x & 63;
  struct Rows {
    int64_t rows;
    int first, tiles;
  };
  // the lane's request (at most 64 of them)
  Rows own{0, 0, 0};
  if (lane < a.requests) {
    const int begin = a.query_starts[lane], tokens = max(min(a.query_starts[lane + 1], a.tokens) - begin, 0);
    own.rows = (int64_t)tokens * g.group;
    own.first = (int)min((int64_t)max(a.lengths[lane], 0), (int64_t)a.table_width * g.page.d) - tokens;
    own.tiles = (int)((own.rows + ROWS - 1) / ROWS);
  }
  const int all = (int)(((int64_t)a.table_width * g.page.d + BT - 1) / BT), most = a.window > 0 ? min(all, a.window / BT + 1) : all;
  auto at_least = [&](int c) {  // its row tiles that see at least c key tiles (a window: `most` and more are one)
    if (c > most) return 0;
    const int64_t q = ((int64_t)(c - 1) * BT - own.first) * g.group;
    return c <= 0 || q <= 0 ? own.tiles : own.rows <= q ? 0 : own.tiles - (int)(q / ROWS);
  };
  auto sum_of = [&](int x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
    return __builtin_amdgcn_readfirstlane(x);
  };
  if (k >= sum_of(own.tiles)) return false;
  int lo = 0;
  for (int hi = most + 1; hi - lo > 1;) {
    const int mid = (lo + hi) / 2;
    if (sum_of(at_least(mid)) > k)
      lo = mid;
    else
      hi = mid;
  }
  const int more = at_least(lo + 1), exactly = at_least(lo) - more;
  k -= sum_of(more);  // the k-th of those with exactly lo, request by request
  int sum = exactly;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(sum, d, 64);
    if (lane >= d) sum += y;
  }
  const int at = __builtin_ctzll(__ballot(k < sum) | 1ull << 63);
  *request = at;
  *row_tile = __builtin_amdgcn_readlane(own.tiles - more - 1 - (k - (sum - exactly)), at);
  return true;
}

// LSE: the logarithms of the rows' sums are wanted.
template <int DT, int DP, bool LSE>
__global__ __launch_bounds__(WAVES * 64, waves_a_simd(DP)) __attribute__((amdgpu_waves_per_eu(waves_a_simd(DP), waves_a_simd(DP)))) void prompt_tiles_kernel(AttentionKArgs g) {
  using C = Cfg<DT, DP>;
  __shared__ __attribute__((aligned(1024))) char lds[2][2][C::TILE_BYTES];  // [stage][keys, values]
  const iris_attention_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, half = lane >> 5;

  // The workgroup's rows, and its share of their keys.  Key heads change fastest: with eight of them each XCD has one.
  const int item = blockIdx.x / a.k_heads, head = blockIdx.x - item * a.k_heads, x = item / g.splits, split = item - x * g.splits;
  int request, row_tile;
  if (g.by_length) {
    // Of those that take one place a CU every other batch is turned round: beside the longest runs the shortest of the next.  (One prompt
    // of 8192 tokens, 512 row tiles: 199 us without, 189 with.)
    const int batch = x / g.by_length, first_of = batch * g.by_length;
    const int k = batch % 2 ? first_of + min(g.by_length, (int)gridDim.x / a.k_heads - first_of) - 1 - (x - first_of) : x;
    if (!nth_longest(g, k, &request, &row_tile)) return;
  } else {
    // x counts row tiles with room for each request's, without a sum over the requests: request r's begin at bound(r).
    auto bound = [&](int r) { return (int)((int64_t)scalar_at(a.query_starts, r) * g.group / ROWS) + r; };
    request = 0;
    for (int hi = a.requests; hi - request > 1;) {
      const int mid = (request + hi) / 2;
      if (bound(mid) <= x)
        request = mid;
      else
        hi = mid;
    }
    row_tile = x - bound(request);
  }
  const int token0 = scalar_at(a.query_starts, request);
  const int tokens = min(scalar_at(a.query_starts, request + 1), a.tokens) - token0;
  const int row0 = row_tile * ROWS;
  if (row0 < 0 || token0 < 0 || tokens <= 0 || row0 >= (int64_t)tokens * g.group) return;
  const int num_rows = (int)min((int64_t)ROWS, (int64_t)tokens * g.group - row0);
  int length = max(scalar_at(a.lengths, request), 0);
  if ((int64_t)length > (int64_t)a.table_width * g.page.d) {
    if (tid == 0) report(a.status, IRIS_STATUS_BAD_INDEX);
    length = (int)(a.table_width * g.page.d);
  }
  const int first = length - tokens;  // position of the request's first query
  const int rows_first = first + row0 / g.group, rows_last = first + (row0 + num_rows - 1) / g.group;
  const KeyTiles list = key_tiles<BT>(a, rows_first, rows_last);
  // the workgroup's share of the tiles
  const int parts = max(min(g.splits, list.count / LEAST), 1);
  if (split >= parts) return;
  const int j0 = (int)((int64_t)list.count * split / parts), j1 = (int)((int64_t)list.count * (split + 1) / parts);

  // the lane's row
  const int wrow = wave * WAVE_ROWS;
  const bool have_row = wrow + n < num_rows;
  const int row = row0 + (have_row ? wrow + n : 0);
  const int token = (int)((uint32_t)row / (uint32_t)g.group), qhead = head * g.group + row - token * g.group;
  const int at = have_row ? first + token : -1;
  // positions of the wave's rows, from .. to (no row: an empty range)
  const int wave_first = first + (row0 + min(wrow, num_rows)) / g.group;
  const int wave_last = wrow < num_rows ? first + (row0 + min(wrow + WAVE_ROWS, num_rows) - 1) / g.group : -1;

  u32x4 q[C::KC];
  {
    const IRIS_GLOBAL char* qp = (const IRIS_GLOBAL char*)a.q + ((int64_t)(token0 + token) * a.stride_qt + (int64_t)qhead * a.stride_qh) * 2 + half * 16;
#pragma unroll
    for (int c = 0; c < C::KC; ++c) {
      q[c] = u32x4{0, 0, 0, 0};
      if (have_row && c * 16 + half * 8 < a.head_dim) q[c] = *(const IRIS_GLOBAL u32x4*)(qp + c * 32);
    }
  }

  // What a wave fetches: 16 keys of each tile, DMA_ROWS an instruction.  Offsets of the lane's chunk from the first of the 16.
  uint32_t k_off[C::DMAS], v_off[C::DMAS];
#pragma unroll
  for (int i = 0; i < C::DMAS; ++i) {
    const int r = i * C::DMA_ROWS + lane / C::CHUNKS, p = lane % C::CHUNKS;
    const int kc = swizzle_k<DP>(r, p), vc = swizzle_v<DP>(r, p);
    k_off[i] = kc * 8 < a.head_dim ? (uint32_t)(r * a.stride_kc_row * 2) + kc * 16 : DEAD_OFFSET;
    v_off[i] = vc * 8 < a.head_dim ? (uint32_t)(r * a.stride_vc_row * 2) + vc * 16 : DEAD_OFFSET;
  }
  bool bad_page = false;
  auto fetch_page = [&](int j) {  // the page of the wave's keys of list tile j
    const int key = list.tile(j) * BT + wave * 16;
    return key < length ? scalar_at(a.block_table, (int64_t)request * a.stride_table + page_div((uint32_t)key, g.page)) : 0;
  };
  auto fetch = [&](int j, int page, int stage) {
    const int key = list.tile(j) * BT + wave * 16;
    if ((uint32_t)page >= (uint32_t)a.num_pages) {
      // (of the rows' business only where one of them sees one of the 16 keys; pages behind a window may be gone)
      bad_page |= key <= rows_last && (key + 15 >= list.lo || key < a.sinks);
      page = 0;
    }
    const int in_page = key - (int)(page_div((uint32_t)key, g.page) * g.page.d);
    const int valid = length - key;  // of the 16 keys
    const __amdgpu_buffer_rsrc_t kr = tile_rsrc((const IRIS_GLOBAL char*)a.k_cache + ((int64_t)page * a.stride_kc_page + (int64_t)head * a.stride_kc_head) * 2, 0x7FFFFFFF);
    const __amdgpu_buffer_rsrc_t vr = tile_rsrc((const IRIS_GLOBAL char*)a.v_cache + ((int64_t)page * a.stride_vc_page + (int64_t)head * a.stride_vc_head) * 2, 0x7FFFFFFF);
    const int k_at = in_page * (int)(a.stride_kc_row * 2), v_at = in_page * (int)(a.stride_vc_row * 2);
    char* const to = &lds[stage][0][wave * 16 * C::ROW_BYTES];
    auto dma = [&](int i, uint32_t ko, uint32_t vo) {
      lds_dma16(kr, (IRIS_LDS void*)(to + i * 1024), ko, k_at);
      lds_dma16(vr, (IRIS_LDS void*)(to + C::TILE_BYTES + i * 1024), vo, v_at);
    };
    if (valid >= 16) {
#pragma unroll
      for (int i = 0; i < C::DMAS; ++i) dma(i, k_off[i], v_off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < C::DMAS; ++i) {
        const bool there = i * C::DMA_ROWS + lane / C::CHUNKS < valid;
        dma(i, there ? k_off[i] : DEAD_OFFSET, there ? v_off[i] : DEAD_OFFSET);
      }
    }
  };
  // where the lane reads: keys by row, values by groups of four keys
  int k_read[C::KC];
#pragma unroll
  for (int c = 0; c < C::KC; ++c) k_read[c] = n * C::ROW_BYTES + swizzle_k<DP>(n, 2 * c + half) * 16;
  const int v_row = half * 4 + ((lane & 15) >> 2);  // (and eight further on for the second four)
  int v_read[C::DTILES];
#pragma unroll
  for (int t = 0; t < C::DTILES; ++t) {
    const int column = t * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    v_read[t] = v_row * C::ROW_BYTES + swizzle_v<DP>(v_row, column / 8) * 16 + (column & 7) * 2;
  }
  // (both swizzles repeat after 16 rows)
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  auto read_v = [&](const char* base, int t, int group) {  // V^T's operand: 16 keys of 32 columns
    const IRIS_LDS char* p = (const IRIS_LDS char*)base + group * 16 * C::ROW_BYTES;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((IRIS_LDS s16x4*)(p + v_read[t]));
    // rows eight further on: for 128 columns the swizzle is the same, for 64 it is too ((row >> 1) & 3 repeats after 8)
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((IRIS_LDS s16x4*)(p + v_read[t] + 8 * C::ROW_BYTES));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x16 o[C::DTILES];
#pragma unroll
  for (int t = 0; t < C::DTILES; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  // l: the sum of the weights as they are multiplied; lse_l: as they are, for the logarithm
  float ref = have_row ? -INFINITY : 0.f, l = 0.f, lse_l = 0.f;
  bool poisoned = false;

  // Tiles are fetched a stage ahead by all waves; the last ones of a workgroup may lie past a wave's own last key.
  int page = 0;
  if (j0 < j1) {
    fetch(j0, fetch_page(j0), j0 & 1);
    if (j0 + 1 < j1) page = fetch_page(j0 + 1);
  }
  auto next_stage = [&](int j) {
    IRIS_WAIT_VMCNT(0);  // this wave's share of the tile has arrived; behind the barrier everyone's has
    const int base = list.tile(j) * BT;
    if (base + BT - 1 > rows_first || (a.window > 0 && rows_last - base >= a.window && base + BT > a.sinks)) {
      // some rows must not see some of the tile's values: is any among the wave's share of them not a finite number?
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 most = {0, 0};
#pragma unroll
      for (int i = 0; i < C::DMAS; ++i) {
        const u32x4 v = *(const IRIS_LDS u32x4*)((const IRIS_LDS char*)lds[j & 1][1] + wave * 16 * C::ROW_BYTES + i * 1024 + lane * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, v[w] & 0x7FFF7FFFu));
      }
      constexpr unsigned short INF = DT == IRIS_DTYPE_BF16 ? 0x7F80 : 0x7C00;
      poisoned |= most[0] >= INF || most[1] >= INF;
    }
    block_barrier_raw();
    if (j + 1 < j1) {
      fetch(j + 1, page, (j + 1) & 1);
      if (j + 2 < j1) page = fetch_page(j + 2);
    }
  };
  f32x16 s[2];
  u32x4 p[4];  // P^T's operands: 16 keys each
  float sum, exact;
  // The scores of list tile j.  Operands are read AHEAD matrix instructions before they are used; two sums in turn, so that
  // neither waits for its own last step.
  auto score = [&](int j) {
    const char* kt = lds[j & 1][0];
    u32x4 f[AHEAD];
    auto read_k = [&](int i) { return *(const IRIS_LDS u32x4*)((const IRIS_LDS char*)kt + (i & 1) * 32 * C::ROW_BYTES + k_read[i / 2]); };
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = read_k(i);
    __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < 2 * C::KC; ++i) {
      s[i & 1] = mfma<DT>(f[i % AHEAD], q[i / 2], s[i & 1]);
      __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 1, 0);
      if (i + AHEAD < 2 * C::KC) {
        f[i % AHEAD] = read_k(i + AHEAD);
        __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, 1, 0);
      }
    }
    // May some of the tile's keys be hidden from some of the wave's rows?
    const int base = list.tile(j) * BT;
    if (base + BT - 1 > wave_first || (a.window > 0 && wave_last - base >= a.window && base + BT > a.sinks)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // the keys that the row sees as bits, those of the lane from bit 0 on: two instructions a score
        const uint32_t mask = visible(a, at, base + 32 * u) >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t keep = (uint32_t)((int)(mask << (31 - (8 * (r / 4) + r % 4))) >> 31);
          const float score = s[u][r];  // (a bit_cast of a vector's element would read its first)
          s[u][r] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, score) & keep) | (~keep & 0xFF800000u));
        }
      }
    }
  };
  // The weights, against the reference as it stands.
  auto weigh = [&] {
    const float from = ref == -INFINITY ? 0.f : ref;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    exact = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][8 * i + e], g.scale_log2, -from));
        }
        // (in 16 bits for the product with the values, and summed as rounded: bf16 outputs are off by 0.0022 of themselves, fp16 by
        // 0.00026, where fp32 weights have 0.0017 and 0.00021; the rest of each weight would be half as many matrix instructions again)
        p[2 * u + i] = u32x4{pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7])};
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[e] = add_weights<DT>(p[2 * u + i][e], sums[e]);
        if (LSE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) exact += w[e];
        }
      }
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  };
  auto add_values = [&](int j) {
    l += sum;
    lse_l += exact;
    const char* vt = lds[j & 1][1];
    u32x4 f[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = read_v(vt, i % C::DTILES, i / C::DTILES);
    __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, 2 * AHEAD, 1);
#pragma unroll
    for (int i = 0; i < 4 * C::DTILES; ++i) {
      o[i % C::DTILES] = mfma<DT>(f[i % AHEAD], p[i / C::DTILES], o[i % C::DTILES]);
      __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 1, 1);
      if (i + AHEAD < 4 * C::DTILES) {
        f[i % AHEAD] = read_v(vt, (i + AHEAD) % C::DTILES, (i + AHEAD) / C::DTILES);
        __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, 2, 1);
      }
    }
  };
  int j = j0, own_end = j0;  // the tiles that hold keys of the wave's
  while (own_end < j1 && list.tile(own_end) * BT <= wave_last) ++own_end;
  for (;; ++j) {
    // The maximum is looked for only where there is no reference yet, or where the sum says that the reference is far too low: a
    // tile in hundreds, outside the loop that the others stay in (sums that are rescaled in it would be kept twice).
    for (; j < own_end; ++j) {
      next_stage(j);
      score(j);
      if (__any(ref == -INFINITY)) break;
      weigh();
      if (__any(sum > C::MOST)) break;
      add_values(j);
    }
    if (j >= own_end) break;
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    const float next = fmaxf(ref, over_32(top, Larger{}) * g.scale_log2 - C::LIFT);
    const float shrink = __builtin_amdgcn_exp2f(ref - (next == -INFINITY ? 0.f : next));
    ref = next;
    l *= shrink;
    lse_l *= shrink;
#pragma unroll
    for (int t = 0; t < C::DTILES; ++t) o[t] *= shrink;
    weigh();
    add_values(j);
  }
  for (; j < j1; ++j) next_stage(j);

  l = over_32(l, Sum{});
  lse_l = over_32(lse_l, Sum{});
  // what one wave found is every row's
  bool redo = __syncthreads_or(poisoned);
  float flags = __syncthreads_or(bad_page) ? __builtin_nanf("") : 0.f;
  if (parts > 1) {
    // The parts meet in the workspace, each in the order of its registers: the last to arrive has the rows of all in the same lanes.
    const int unit = x * a.k_heads + head;
    auto slot = [&](int part) { return (IRIS_GLOBAL char*)(g.slots + ((int64_t)unit * g.splits + part) * C::SLOT); };
    const uint32_t mine = (wave * 64 + lane) * 16;
#pragma unroll
    for (int t = 0; t < C::DTILES; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4 v = {o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]};
        store16_any<AUX_SC1>(slot(split) + (t * 4 + r / 4) * (WAVES * 1024) + mine, __builtin_bit_cast(u32x4, v));
      }
    const f32x4 tail = {ref, l, lse_l, redo ? 1.f : flags};
    store16_any<AUX_SC1>(slot(split) + C::DTILES * 4 * (WAVES * 1024) + mine, __builtin_bit_cast(u32x4, tail));
    IRIS_WAIT_VMCNT(0);
    __syncthreads();
    int last = 0;
    if (tid == 0) {
      IRIS_GLOBAL int32_t* count = (IRIS_GLOBAL int32_t*)(g.counters + unit);
      last = arrive(count, false, false) == parts - 1;
      if (last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!__syncthreads_or(last)) return;
#pragma unroll
    for (int t = 0; t < C::DTILES; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    ref = -INFINITY;
    l = lse_l = 0.f;
    bool bad = false, again = false;
    for (int part = 0; part < parts; ++part) {
      const __amdgpu_buffer_rsrc_t rs = tile_rsrc(slot(part), C::SLOT * 4);
      const f32x4 m = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)mine, C::DTILES * 4 * (WAVES * 1024), AUX_SC1));
      const float next = fmaxf(ref, m[0]), from = next == -INFINITY ? 0.f : next;
      const float old = __builtin_amdgcn_exp2f(ref - from), now = __builtin_amdgcn_exp2f(m[0] - from);
      ref = next;
      l = l * old + m[1] * now;
      lse_l = lse_l * old + m[2] * now;
      again |= m[3] == 1.f;
      bad |= __builtin_isnan(m[3]);
#pragma unroll
      for (int t = 0; t < C::DTILES; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const f32x4 v =
              __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)mine, (t * 4 + r / 4) * (WAVES * 1024), AUX_SC1));
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][r + i] = o[t][r + i] * old + v[i] * now;
        }
    }
    redo = __any(again);
    flags = __any(bad) ? __builtin_nanf("") : 0.f;
  }
  if (flags != 0.f && lane == 0) report(a.status, IRIS_STATUS_BAD_INDEX);

  // A weight of 0 times a value that is no number is NaN: then the rows are computed again by the kernel that takes hidden values out.
  if (redo) {
    static_assert(sizeof(rows::Lds<DT, DP>) <= sizeof(lds), "the tiles' room is given over");
    rows::Unit<DT, DP, true, false> unit(g, *(rows::Lds<DT, DP>*)lds);
#pragma unroll 1
    for (int r = 0; r < num_rows; r += rows::ROWS) {
      rows::Piece p{};
      p.request = request;
      p.head = head;
      p.row0 = row0 + r;
      p.rows = min(rows::ROWS, num_rows - r);
      p.token0 = token0;
      p.length = length;
      p.first = first;
      p.tiles = key_tiles<rows::Cfg<DT, DP>::BT>(a, first + p.row0 / g.group, first + (p.row0 + p.rows - 1) / g.group);
      p.j1 = p.tiles.count;
      p.parts = 1;
      unit.run(p);
    }
    return;
  }
  if (!have_row) return;
  // (a page outside the cache: every number of the rows is NaN)
  const float inv = flags != 0.f ? flags : l == 0.f ? 0.f : 1.f / l;
  const int64_t out_token = token0 + token;
  if (LSE && half == 0)
    a.lse[out_token * a.stride_lse + qhead] = flags != 0.f ? flags : lse_l == 0.f ? -INFINITY : (ref + __builtin_amdgcn_logf(lse_l)) * 0.6931471805599453f;
  IRIS_GLOBAL char* out = (IRIS_GLOBAL char*)a.out + (out_token * a.stride_ot + (int64_t)qhead * a.stride_oh) * 2;
#pragma unroll
  for (int t = 0; t < C::DTILES; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = t * 32 + 2 * r + 4 * half;
      if (d < a.head_dim)
        *(IRIS_GLOBAL u32x2*)(out + d * 2) = u32x2{pack2<DT>(o[t][r] * inv, o[t][r + 1] * inv), pack2<DT>(o[t][r + 2] * inv, o[t][r + 3] * inv)};
    }
}

}  // namespace tiles
}  // namespace iris_amd
