// Norms of query and key heads, their rotation by position, and the write of keys and values into a paged cache, in
// one pass; and the gradient.
//
// y = x r w with r = 1 / sqrt(mean(x^2) + eps); pairs of y turn by their position's angle:
// (z1, z2) = (y1 cos - y2 sin, y2 cos + y1 sin).  A pair is (i, i + R/2) or, interleaved, (2i, 2i + 1); elements from R on
// keep their places.  Everything between the load and the one rounding at the end is fp32.
//
// The gradient: g = dz turned back, dw = sum over rows of g x r, dx = r (g w - x r^2 mean(g w x)).
//
// The work is one read and one write of each head, so it is bound by memory: a head is held by the fewest lanes that
// load it eight elements each, as two runs of four of which one holds a pair's first and one its second elements, so
// that no rotation crosses lanes; the norm is the only exchange, within 16 lanes by DPP.  A lane keeps its angles for the heads of
// its token that it has.  bf16, heads of 128: 8191 tokens of 8 + 2 + 2 heads (54.6 MB) in 11.9 us, 4.6 TB/s, a copy of
// 4 GB runs at 4.9; the gradient of 8192 tokens of 32 + 8 heads (256 MB) in 55.6 us, 4.6 TB/s.  (Loads unpacked as they
// arrive and both weights in one workgroup took 208 registers and 105 us for the latter.)
#include <type_traits>

#include "heads_common.hpp"

namespace iris_amd {
namespace {

constexpr int THREADS = 256;
constexpr int BATCH = 4;  // heads whose loads a lane has in flight together

// Where a lane's V first and V second elements of a row lie.
template <int V>
struct Place {
  int first, second;
  int pair;   // index of the first angle, where the lane's elements turn
  bool live, turns;
};
template <int V>
__device__ inline Place<V> place(int item, int dim, int rotary, bool interleaved) {
  Place<V> p;
  p.live = item * 2 * V < dim;
  p.turns = item * 2 * V < rotary;
  const bool split = p.turns && !interleaved;
  p.first = split ? item * V : item * 2 * V;
  p.second = split ? rotary / 2 + item * V : item * 2 * V + V;
  p.pair = item * V;
  return p;
}

// Turns a lane's pairs by their angles (BACK: by the angles' negatives).
template <int V, bool BACK>
__device__ inline void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V], bool interleaved) {
  if (V > 1 && interleaved) {
    // pairs (a0, a1), (a2, a3), (b0, b1), (b2, b3)
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const int ca = e / 2, cb = V / 2 + e / 2;
      const float sa = BACK ? -s[ca] : s[ca], sb = BACK ? -s[cb] : s[cb];
      const float a0 = a[e], a1 = a[(e + 1) % V], b0 = b[e], b1 = b[(e + 1) % V];
      a[e] = a0 * c[ca] - a1 * sa;
      a[(e + 1) % V] = a1 * c[ca] + a0 * sa;
      b[e] = b0 * c[cb] - b1 * sb;
      b[(e + 1) % V] = b1 * c[cb] + b0 * sb;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float se = BACK ? -s[e] : s[e], x = a[e], y = b[e];
      a[e] = x * c[e] - y * se;
      b[e] = y * c[e] + x * se;
    }
  }
}

template <int V, int ITEMS>
struct Angles {
  float c[ITEMS][V], s[ITEMS][V];
};
// The angles of token t's position at a lane's pairs; a position outside the table is reported and gives NaN.
template <int V, int ITEMS, class Args>
__device__ inline void load_angles(const Args& a, int64_t t, const Place<V> (&at)[ITEMS], Angles<V, ITEMS>& g) {
  int64_t pos = 0;
  if (a.rotary_dim) pos = a.positions_64 ? ((const int64_t*)a.positions)[t] : ((const int32_t*)a.positions)[t];
  const bool inside = pos >= 0 && pos < a.max_positions;
  if (!inside && a.rotary_dim) report(a.status, IRIS_STATUS_BAD_INDEX);
  const int64_t row = inside ? pos : 0;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) g.c[i][e] = 1.f, g.s[i][e] = 0.f;
    if (at[i].turns) {
      Raw<IRIS_DTYPE_F32, V> c, s;
      c.load((const IRIS_GLOBAL char*)(a.cos + row * a.stride_cos + at[i].pair));
      s.load((const IRIS_GLOBAL char*)(a.sin + row * a.stride_sin + at[i].pair));
      c.get(g.c[i]);
      s.get(g.s[i]);
      if (!inside) {
#pragma unroll
        for (int e = 0; e < V; ++e) g.c[i][e] = g.s[i][e] = __builtin_nanf("");
      }
    }
  }
}

// A lane's elements of a head: in their own type, and as fp32.
template <int DT, int V, int ITEMS>
struct Packed {
  static constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
  Raw<DT, V> a[ITEMS], b[ITEMS];
  __device__ inline void load(const IRIS_GLOBAL char* p, const Place<V> (&at)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      a[i] = b[i] = Raw<DT, V>{};
      if (at[i].live) {
        a[i].load(p + at[i].first * ES);
        b[i].load(p + at[i].second * ES);
      }
    }
  }
  __device__ inline void store(IRIS_GLOBAL char* p, const Place<V> (&at)[ITEMS]) const {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (at[i].live) {
        a[i].store(p + at[i].first * ES);
        b[i].store(p + at[i].second * ES);
      }
  }
};
template <int V, int ITEMS>
struct Wide {
  float a[ITEMS][V], b[ITEMS][V];
  template <int DT>
  __device__ inline void get(const Packed<DT, V, ITEMS>& x) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) x.a[i].get(a[i]), x.b[i].get(b[i]);
  }
  template <int DT>
  __device__ inline void put(Packed<DT, V, ITEMS>& x) const {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) x.a[i].set(a[i]), x.b[i].set(b[i]);
  }
  // A weight vector at the lane's elements, in the heads' type DT or fp32.
  template <int DT>
  __device__ inline void load_weight(const void* w, bool fp32, const Place<V> (&at)[ITEMS]) {
    if (fp32) {
      Packed<IRIS_DTYPE_F32, V, ITEMS> x;
      x.load((const IRIS_GLOBAL char*)w, at);
      get(x);
    } else {
      Packed<DT, V, ITEMS> x;
      x.load((const IRIS_GLOBAL char*)w, at);
      get(x);
    }
  }
};

// The tokens and heads of one kind (queries, keys or values), as groups of lanes take them: `heads_each` heads of a token.
struct Kind {
  int heads, heads_each, parts, blocks;
  FastDiv div;  // by parts
};
Kind make_kind(int64_t tokens, int heads, int heads_each, int64_t per_block) {
  Kind k{};
  if (!heads) return k;
  k.heads = heads;
  k.heads_each = heads_each < heads ? heads_each : heads;
  k.parts = (heads + k.heads_each - 1) / k.heads_each;
  k.blocks = (int)((tokens * k.parts + per_block - 1) / per_block);
  k.div = make_fast_div((uint32_t)k.parts, (uint64_t)(k.blocks * per_block));
  return k;
}
__device__ inline int64_t token_of(const Kind& k, int64_t group) {
  return k.div.m || k.parts == 1 ? (int64_t)fast_div((uint32_t)group, k.div) : group / k.parts;
}

// LANES lanes hold a head, V elements twice and ITEMS times each.  The first kinds[0].blocks workgroups take queries, the next
// kinds[1].blocks keys, and (with a cache) the last values: a workgroup has one weight and one way.
struct ForwardArgs {
  iris_qk_norm_rope_args a;
  Kind kinds[3];
};
template <int DT, int V, int LANES, int ITEMS>
__global__ __launch_bounds__(THREADS) void qk_norm_rope_kernel(ForwardArgs args) {
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
  const iris_qk_norm_rope_args& a = args.a;
  int block = blockIdx.x, which = 0;
  if (block >= args.kinds[0].blocks) block -= args.kinds[0].blocks, which = 1;
  if (which == 1 && block >= args.kinds[1].blocks) block -= args.kinds[1].blocks, which = 2;
  Kind kind = args.kinds[0];
  if (which == 1) kind = args.kinds[1];
  if (which == 2) kind = args.kinds[2];
  const int64_t group = ((int64_t)block * THREADS + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t t = token_of(kind, group);
  if (t >= a.tokens) return;  // (all lanes of a group together)
  const int begin = (int)(group - t * kind.parts) * kind.heads_each, end = min(begin + kind.heads_each, kind.heads);

  Place<V> at[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) at[i] = place<V>(lane + i * LANES, a.head_dim, a.rotary_dim, a.interleaved);
  const IRIS_GLOBAL char* source = (const IRIS_GLOBAL char*)(which == 0 ? a.q : which == 1 ? a.k : a.v) +
                                   t * (which == 0 ? a.stride_qt : which == 1 ? a.stride_kt : a.stride_vt) * ES;
  const int64_t source_step = (which == 0 ? a.stride_qh : which == 1 ? a.stride_kh : a.stride_vh) * ES;
  Packed<DT, V, ITEMS> x[BATCH];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (h0 + u < end) x[u].load(source + (h0 + u) * source_step, at);
  };
  fetch(begin);
  Angles<V, ITEMS> angle;
  if (which < 2) load_angles(a, t, at, angle);
  const void* weight = which == 0 ? a.q_weight : which == 1 ? a.k_weight : nullptr;
  Wide<V, ITEMS> w;
  if (weight) w.template load_weight<DT>(weight, a.weight_fp32, at);
  // where the heads go: a tensor, and for keys and values the token's slot of the cache (none where it is negative)
  IRIS_GLOBAL char* out = which == 0 ? (IRIS_GLOBAL char*)a.q_out + t * a.stride_qot * ES
                          : which == 1 && a.k_out ? (IRIS_GLOBAL char*)a.k_out + t * a.stride_kot * ES
                                                  : nullptr;
  const int64_t out_step = (which == 0 ? a.stride_qoh : a.stride_koh) * ES;
  IRIS_GLOBAL char* cached = nullptr;
  int64_t cached_step = 0;
  if (which > 0 && a.slots) {
    const int64_t slot = a.slots[t];
    if (slot >= a.num_slots) report(a.status, IRIS_STATUS_BAD_INDEX);
    if (slot >= 0 && slot < a.num_slots) {
      const int64_t page = (uint32_t)slot / (uint32_t)a.page_size, row = (int)slot - (int)page * a.page_size;
      cached = which == 1 ? (IRIS_GLOBAL char*)a.k_cache + (page * a.stride_kc_page + row * a.stride_kc_row) * ES
                          : (IRIS_GLOBAL char*)a.v_cache + (page * a.stride_vc_page + row * a.stride_vc_row) * ES;
    }
    cached_step = (which == 1 ? a.stride_kc_head : a.stride_vc_head) * ES;
  }

  for (int h0 = begin; h0 < end; h0 += BATCH) {
    if (h0 > begin) fetch(h0);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int h = h0 + u;
      if (h >= end) break;
      if (which < 2) {
        Wide<V, ITEMS> y;
        y.get(x[u]);
        if (weight) {
          float square = 0.f;
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) square += y.a[i][e] * y.a[i][e] + y.b[i][e] * y.b[i][e];
          const float rs = rsqrtf(sum_lanes<LANES>(square) / (float)a.head_dim + a.eps);
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) y.a[i][e] *= rs * w.a[i][e], y.b[i][e] *= rs * w.b[i][e];
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (at[i].turns) turn<V, false>(y.a[i], y.b[i], angle.c[i], angle.s[i], a.interleaved);
        y.put(x[u]);
      }
      if (out) x[u].store(out + h * out_step, at);
      if (cached) x[u].store(cached + h * cached_step, at);
    }
  }
}

// The gradient.  The first kinds[0].blocks workgroups take queries, the others keys.  A group of lanes takes `heads_each` heads of a
// token, then those `blocks` workgroups further on, and keeps its share of the weight's gradient in registers; a workgroup
// adds its groups' shares in LDS in a fixed order and leaves one row of partial sums, which weight_gradient_kernel
// adds in a fixed order: the same inputs give the same bits.
struct BackwardArgs {
  iris_qk_norm_rope_backward_args a;
  Kind kinds[2];
};
template <int DT, int V, int LANES, int ITEMS>
__global__ __launch_bounds__(THREADS) void qk_norm_rope_backward_kernel(BackwardArgs args) {
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2, GROUPS = THREADS / LANES, PAIR = BATCH / 2;
  const iris_qk_norm_rope_backward_args& a = args.a;
  const bool keys = (int)blockIdx.x >= args.kinds[0].blocks;
  Kind kind = args.kinds[0];
  if (keys) kind = args.kinds[1];
  const int block = blockIdx.x - (keys ? args.kinds[0].blocks : 0);
  const int lane = threadIdx.x % LANES, in_block = threadIdx.x / LANES;
  Place<V> at[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) at[i] = place<V>(lane + i * LANES, a.head_dim, a.rotary_dim, a.interleaved);
  const void* weight = keys ? a.k_weight : a.q_weight;
  Wide<V, ITEMS> w, dw;
  if (weight) w.template load_weight<DT>(weight, a.weight_fp32, at);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) dw.a[i][e] = dw.b[i][e] = 0.f;

  const float inv_dim = 1.f / (float)a.head_dim;
  const int64_t xh = (keys ? a.stride_kh : a.stride_qh) * ES, zh = (keys ? a.stride_dkoh : a.stride_dqoh) * ES,
                dh = (keys ? a.stride_dkh : a.stride_dqh) * ES;
  const int64_t groups = (int64_t)a.tokens * kind.parts, step = (int64_t)kind.blocks * GROUPS;
  for (int64_t group = (int64_t)block * GROUPS + in_block; group < groups; group += step) {
    const int64_t t = token_of(kind, group);
    const int begin = (int)(group - t * kind.parts) * kind.heads_each, end = min(begin + kind.heads_each, kind.heads);
    const IRIS_GLOBAL char* xs = (const IRIS_GLOBAL char*)(keys ? a.k : a.q) + t * (keys ? a.stride_kt : a.stride_qt) * ES;
    const IRIS_GLOBAL char* zs = (const IRIS_GLOBAL char*)(keys ? a.dk_out : a.dq_out) + t * (keys ? a.stride_dkot : a.stride_dqot) * ES;
    IRIS_GLOBAL char* ds = (IRIS_GLOBAL char*)(keys ? a.dk : a.dq) + t * (keys ? a.stride_dkt : a.stride_dqt) * ES;
    Packed<DT, V, ITEMS> x[PAIR], z[PAIR];
    auto fetch = [&](int h0) {
#pragma unroll
      for (int u = 0; u < PAIR; ++u)
        if (h0 + u < end) {
          z[u].load(zs + (h0 + u) * zh, at);
          if (weight) x[u].load(xs + (h0 + u) * xh, at);
        }
    };
    fetch(begin);
    Angles<V, ITEMS> angle;
    load_angles(a, t, at, angle);
    for (int h0 = begin; h0 < end; h0 += PAIR) {
      if (h0 > begin) fetch(h0);
#pragma unroll
      for (int u = 0; u < PAIR; ++u) {
        if (h0 + u >= end) break;
        Wide<V, ITEMS> g;
        g.get(z[u]);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (at[i].turns) turn<V, true>(g.a[i], g.b[i], angle.c[i], angle.s[i], a.interleaved);
        if (weight) {
          Wide<V, ITEMS> y;
          y.get(x[u]);
          // dx is what is left of g w when its part along x is taken out: of heads of two elements very little.  Those are laid out as
          // single pairs, and single pairs (heads of any size whose sizes or addresses allow no runs of four) take it out in 64 bits.
          using Acc = std::conditional_t<V == 1, double, float>;
          Acc square = 0, along = 0;
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              square += (Acc)y.a[i][e] * y.a[i][e] + (Acc)y.b[i][e] * y.b[i][e];
              along += (Acc)g.a[i][e] * w.a[i][e] * y.a[i][e] + (Acc)g.b[i][e] * w.b[i][e] * y.b[i][e];
            }
          square = sum_lanes<LANES>(square);
          along = sum_lanes<LANES>(along);
          const float rs = rsqrtf((float)(square * inv_dim) + a.eps);
          const Acc back = along / (square + (Acc)a.head_dim * a.eps);
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              dw.a[i][e] += g.a[i][e] * y.a[i][e] * rs;
              dw.b[i][e] += g.b[i][e] * y.b[i][e] * rs;
              g.a[i][e] = rs * (float)((Acc)g.a[i][e] * w.a[i][e] - y.a[i][e] * back);
              g.b[i][e] = rs * (float)((Acc)g.b[i][e] * w.b[i][e] - y.b[i][e] * back);
            }
        }
        g.put(z[u]);
        z[u].store(ds + (h0 + u) * dh, at);
      }
    }
  }
  if (!(keys ? a.dk_weight : a.dq_weight)) return;
  // the groups' shares: rows of head_dim floats in LDS, added by column
  extern __shared__ float shares[];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (at[i].live)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        shares[in_block * a.head_dim + at[i].first + e] = dw.a[i][e];
        shares[in_block * a.head_dim + at[i].second + e] = dw.b[i][e];
      }
  __syncthreads();
  for (int c = threadIdx.x; c < a.head_dim; c += THREADS) {
    float sum = 0.f;
    for (int g = 0; g < GROUPS; ++g) sum += shares[g * a.head_dim + c];
    a.workspace[(int64_t)blockIdx.x * a.head_dim + c] = sum;
  }
}

// Adds the workgroups' partial sums, those of the queries' weight in the first `q_rows` rows and of the keys' in the next `k_rows`:
// 16 columns a workgroup, 64 lanes a column.
constexpr int SUM_THREADS = 1024;
struct SumArgs {
  const float* partials;
  int q_rows, k_rows, dim;
  float* dq_weight;
  float* dk_weight;
};
__global__ __launch_bounds__(SUM_THREADS) void weight_gradient_kernel(SumArgs a) {
  __shared__ float sums[SUM_THREADS / 16][17];
  const int c = threadIdx.x % 16, part = threadIdx.x / 16, column = blockIdx.x * 16 + c;
  const bool keys = blockIdx.y;
  float* out = keys ? a.dk_weight : a.dq_weight;
  if (!out) return;
  const int begin = keys ? a.q_rows : 0, end = keys ? a.q_rows + a.k_rows : a.q_rows;
  float sum = 0.f;
  if (column < a.dim) {
#pragma unroll 4
    for (int r = begin + part; r < end; r += SUM_THREADS / 16) sum += a.partials[(int64_t)r * a.dim + column];
  }
  sums[part][c] = sum;
  __syncthreads();
  for (int n = SUM_THREADS / 32; n > 0; n /= 2) {
    if (part < n) sums[part][c] += sums[part + n][c];
    __syncthreads();
  }
  if (part == 0 && column < a.dim) out[column] = sums[0][c];
}

bool known_dtype(int dt) { return dt == IRIS_DTYPE_F32 || dt == IRIS_DTYPE_F16 || dt == IRIS_DTYPE_BF16; }

bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p % bytes) == 0; }

// Lanes and elements: eight elements a lane in runs of four where sizes, strides and addresses allow loads of four,
// single pairs otherwise.
template <class F>
hipError_t with_layout(bool wide, int dim, F f) {
  using std::integral_constant;
  if (wide) {
    if (dim <= 64) return f(integral_constant<int, 4>{}, integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (dim <= 128) return f(integral_constant<int, 4>{}, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (dim <= 256) return f(integral_constant<int, 4>{}, integral_constant<int, 32>{}, integral_constant<int, 1>{});
    return f(integral_constant<int, 4>{}, integral_constant<int, 64>{}, integral_constant<int, 1>{});
  }
  return f(integral_constant<int, 1>{}, integral_constant<int, 64>{}, integral_constant<int, 4>{});
}
template <class F>
hipError_t with_dtype(int dt, F f) {
  using std::integral_constant;
  if (dt == IRIS_DTYPE_F32) return f(integral_constant<int, IRIS_DTYPE_F32>{});
  if (dt == IRIS_DTYPE_F16) return f(integral_constant<int, IRIS_DTYPE_F16>{});
  return f(integral_constant<int, IRIS_DTYPE_BF16>{});
}

constexpr int MAX_HEAD_DIM = 512;
constexpr int MOST_GROUPS = 4;  // workgroups a CU of the gradient; each costs a row of partial sums (8 a CU: 59 us where 4 take 56)

// Heads of a token that a group of lanes takes: they share the token's angles, up to four (eight gain nothing), as long as two
// workgroups a CU are left.  Forward, bf16 heads of 128, us at 1 / 2 / 4 / 8 heads: 500 tokens of 8 + 2 + 2 heads 3.6 / 3.9 / 4.3 / 6.0,
// 2000 of them 6.3 / 5.8 / 5.8 / 7.7, 8191 15.3 / 13.8 / 13.1 / 13.6, 2000 of 32 + 8 + 8 15.6 / 12.6 / 11.7 / 12.7.
int heads_each(int64_t tokens, int heads, int64_t per_block) {
  const int64_t enough = 2 * (int64_t)current_cu_count() * per_block;
  int each = 1;
  while (each < 4 && tokens * ((heads + 2 * each - 1) / (2 * each)) >= enough) each *= 2;
  return each;
}

}  // namespace
}  // namespace iris_amd

extern "C" int iris_qk_norm_rope_launch(const iris_qk_norm_rope_args* args, void* stream) {
  using namespace iris_amd;
  if (!args) return hipErrorInvalidValue;
  const iris_qk_norm_rope_args& a = *args;
  if (!known_dtype(a.dtype) || a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0 || a.head_dim <= 0 || a.head_dim % 2 || a.head_dim > MAX_HEAD_DIM ||
      a.rotary_dim < 0 || a.rotary_dim % 2 || a.rotary_dim > a.head_dim || (a.rotary_dim && (!a.cos || !a.sin || !a.positions || a.max_positions <= 0)))
    return hipErrorInvalidValue;
  if ((a.slots != nullptr) != (a.k_cache != nullptr) || (a.slots != nullptr) != (a.v_cache != nullptr) || (a.slots != nullptr) != (a.v != nullptr))
    return hipErrorInvalidValue;
  if (a.slots && (a.page_size <= 0 || a.num_slots < 0 || a.num_slots > INT32_MAX)) return hipErrorInvalidValue;
  if (a.tokens == 0 || a.q_heads + a.k_heads == 0) return hipSuccess;
  if ((a.q_heads && (!a.q || !a.q_out)) || (a.k_heads && (!a.k || (!a.k_out && !a.k_cache)))) return hipErrorInvalidValue;

  const int es = dtype_size(a.dtype), run = 4 * es, wes = a.weight_fp32 ? 4 : es;
  bool wide = a.head_dim % 8 == 0 && a.rotary_dim % 8 == 0;
  for (const void* p : {a.q, a.k, a.v, (const void*)a.q_out, (const void*)a.k_out, (const void*)a.k_cache, (const void*)a.v_cache})
    wide = wide && aligned(p, run);
  for (const int64_t s : {a.stride_qt, a.stride_qh, a.stride_kt, a.stride_kh, a.stride_vt, a.stride_vh, a.stride_qot, a.stride_qoh, a.stride_kot,
                          a.stride_koh, a.stride_kc_page, a.stride_kc_row, a.stride_kc_head, a.stride_vc_page, a.stride_vc_row, a.stride_vc_head})
    wide = wide && s % 4 == 0;
  wide = wide && aligned(a.cos, 16) && aligned(a.sin, 16) && a.stride_cos % 4 == 0 && a.stride_sin % 4 == 0 && aligned(a.q_weight, 4 * wes) &&
         aligned(a.k_weight, 4 * wes);

  return with_dtype(a.dtype, [&](auto dt) {
    return with_layout(wide, a.head_dim, [&](auto v, auto lanes, auto items) {
      const int64_t per_block = THREADS / lanes.value;
      const int each = heads_each(a.tokens, a.q_heads + (a.v ? 2 : 1) * a.k_heads, per_block);
      ForwardArgs f{a, {make_kind(a.tokens, a.q_heads, each, per_block), make_kind(a.tokens, a.k_heads, each, per_block),
                        make_kind(a.tokens, a.v ? a.k_heads : 0, each, per_block)}};
      const int64_t grid = (int64_t)f.kinds[0].blocks + f.kinds[1].blocks + f.kinds[2].blocks;
      if (grid > INT32_MAX) return hipErrorInvalidValue;
      return launch(qk_norm_rope_kernel<dt.value, v.value, lanes.value, items.value>, dim3((unsigned)grid), THREADS, 0, stream, f);
    });
  });
}

extern "C" int iris_qk_norm_rope_backward_launch(const iris_qk_norm_rope_backward_args* args, void* stream) {
  using namespace iris_amd;
  if (!args) return hipErrorInvalidValue;
  const iris_qk_norm_rope_backward_args& a = *args;
  if (!known_dtype(a.dtype) || a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0 || a.head_dim <= 0 || a.head_dim % 2 || a.head_dim > MAX_HEAD_DIM ||
      a.rotary_dim < 0 || a.rotary_dim % 2 || a.rotary_dim > a.head_dim || (a.rotary_dim && (!a.cos || !a.sin || !a.positions || a.max_positions <= 0)))
    return hipErrorInvalidValue;
  // a weight's gradient is asked for where there is a weight, and both need the workspace's rows
  if ((a.dq_weight && !a.q_weight) || (a.dk_weight && !a.k_weight)) return hipErrorInvalidValue;
  const bool weights = a.dq_weight || a.dk_weight;
  if (weights && (!a.workspace || a.workspace_elems < 2 * a.head_dim)) return hipErrorInvalidValue;
  const bool some = a.tokens && a.q_heads + a.k_heads;
  if (!some && !weights) return hipSuccess;
  if (some && ((a.q_heads && (!a.dq_out || !a.dq || (a.q_weight && !a.q))) || (a.k_heads && (!a.dk_out || !a.dk || (a.k_weight && !a.k)))))
    return hipErrorInvalidValue;

  const int es = dtype_size(a.dtype), run = 4 * es, wes = a.weight_fp32 ? 4 : es;
  bool wide = a.head_dim % 8 == 0 && a.rotary_dim % 8 == 0;
  for (const void* p : {a.q, a.k, a.dq_out, a.dk_out, (const void*)a.dq, (const void*)a.dk}) wide = wide && aligned(p, run);
  for (const int64_t s : {a.stride_qt, a.stride_qh, a.stride_kt, a.stride_kh, a.stride_dqot, a.stride_dqoh, a.stride_dkot, a.stride_dkoh, a.stride_dqt,
                          a.stride_dqh, a.stride_dkt, a.stride_dkh})
    wide = wide && s % 4 == 0;
  wide = wide && aligned(a.cos, 16) && aligned(a.sin, 16) && a.stride_cos % 4 == 0 && a.stride_sin % 4 == 0 && aligned(a.q_weight, 4 * wes) &&
         aligned(a.k_weight, 4 * wes);
  return with_dtype(a.dtype, [&](auto dt) {
    return with_layout(wide, a.head_dim, [&](auto v, auto lanes, auto items) {
      const int64_t per_block = THREADS / lanes.value;
      const int each = heads_each(a.tokens, a.q_heads + a.k_heads, per_block);
      BackwardArgs f{a, {make_kind(a.tokens, a.q_heads, each, per_block), make_kind(a.tokens, a.k_heads, each, per_block)}};
      // persistent workgroups, each with a row of the workspace; the kinds have their shares of them, one at least
      const int64_t room = weights ? a.workspace_elems / a.head_dim : INT32_MAX, most = room < MOST_GROUPS * current_cu_count() ? room : MOST_GROUPS * current_cu_count();
      const int64_t all = (int64_t)f.kinds[0].blocks + f.kinds[1].blocks;
      if (all > most) {
        int64_t q = most * f.kinds[0].blocks / all;
        if (f.kinds[0].blocks && q < 1) q = 1;
        if (f.kinds[1].blocks && q > most - 1) q = most - 1;
        if (q < f.kinds[0].blocks) f.kinds[0].blocks = (int)q;
        if (most - q < f.kinds[1].blocks) f.kinds[1].blocks = (int)(most - q);
      }
      const int q_blocks = f.kinds[0].blocks, k_blocks = f.kinds[1].blocks;
      const size_t lds = weights ? per_block * a.head_dim * sizeof(float) : 0;
      if (q_blocks + k_blocks) {
        const hipError_t err =
            launch(qk_norm_rope_backward_kernel<dt.value, v.value, lanes.value, items.value>, dim3(q_blocks + k_blocks), THREADS, lds, stream, f);
        if (err != hipSuccess) return err;
      }
      if (!weights) return hipSuccess;
      return launch(weight_gradient_kernel, dim3((a.head_dim + 15) / 16, 2), SUM_THREADS, 0, stream,
                    SumArgs{a.workspace, q_blocks, k_blocks, a.head_dim, a.dq_weight, a.dk_weight});
    });
  });
}
