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
// that no rotation crosses lanes; the norm is the only exchange.  A lane keeps its angles for the heads of its token.
#include <type_traits>

#include "heads_common.hpp"

namespace iris_amd {
namespace {

constexpr int THREADS = 256;
constexpr int BATCH = 4;  // heads whose loads a lane has in flight together

// Where a lane's V first and V second elements of a row lie.  ROT: the pairs that turn.
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
      load_elems<IRIS_DTYPE_F32, V>((const IRIS_GLOBAL char*)(a.cos + row * a.stride_cos + at[i].pair), g.c[i]);
      load_elems<IRIS_DTYPE_F32, V>((const IRIS_GLOBAL char*)(a.sin + row * a.stride_sin + at[i].pair), g.s[i]);
      if (!inside) {
#pragma unroll
        for (int e = 0; e < V; ++e) g.c[i][e] = g.s[i][e] = __builtin_nanf("");
      }
    }
  }
}

template <int DT, int V, int ITEMS>
struct Row {
  float a[ITEMS][V], b[ITEMS][V];
  __device__ inline void load(const IRIS_GLOBAL char* p, const Place<V> (&at)[ITEMS]) {
    constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) a[i][e] = b[i][e] = 0.f;
      if (at[i].live) {
        load_elems<DT, V>(p + at[i].first * ES, a[i]);
        load_elems<DT, V>(p + at[i].second * ES, b[i]);
      }
    }
  }
  __device__ inline void store(IRIS_GLOBAL char* p, const Place<V> (&at)[ITEMS]) const {
    constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (at[i].live) {
        store_elems<DT, V>(p + at[i].first * ES, a[i]);
        store_elems<DT, V>(p + at[i].second * ES, b[i]);
      }
  }
};

// A weight vector at a lane's elements; ones where there is none.
template <int DT, int V, int ITEMS>
__device__ inline void load_weight(const void* w, bool fp32, const Place<V> (&at)[ITEMS], Row<DT, V, ITEMS>& out) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) out.a[i][e] = out.b[i][e] = 1.f;
  if (!w) return;
  if (!fp32) {
    out.load((const IRIS_GLOBAL char*)w, at);
    return;
  }
  Row<IRIS_DTYPE_F32, V, ITEMS> wide;
  wide.load((const IRIS_GLOBAL char*)w, at);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) out.a[i][e] = wide.a[i][e], out.b[i][e] = wide.b[i][e];
}

template <int V, int ITEMS, class A, class B>
__device__ inline float dot_items(const A& x, const B& y) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) sum += x.a[i][e] * y.a[i][e] + x.b[i][e] * y.b[i][e];
  return sum;
}

// LANES lanes hold a row, V elements twice and ITEMS times each.  A group of lanes takes `heads_each` of a token's rows:
// query heads, key heads, and (with a cache) value heads, in this order.
template <int DT, int V, int LANES, int ITEMS>
__global__ __launch_bounds__(THREADS) void qk_norm_rope_kernel(iris_qk_norm_rope_args a, FastDiv parts, int heads_each) {
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2;
  const int64_t group = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t t = parts.m || parts.d == 1 ? (int64_t)fast_div((uint32_t)group, parts) : group / parts.d;
  if (t >= a.tokens) return;  // (all lanes of a group together)
  const int rows = a.q_heads + a.k_heads + (a.v ? a.k_heads : 0);
  const int begin = (int)(group - t * parts.d) * heads_each, end = min(begin + heads_each, rows);

  Place<V> at[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) at[i] = place<V>(lane + i * LANES, a.head_dim, a.rotary_dim, a.interleaved);
  // the slot of the token's keys and values; none where it is negative
  int64_t slot = -1;
  if (a.slots) {
    slot = a.slots[t];
    if (slot >= a.num_slots) {
      report(a.status, IRIS_STATUS_BAD_INDEX);
      slot = -1;
    }
  }
  const int page = slot < 0 ? 0 : (int)((uint32_t)slot / (uint32_t)a.page_size);
  const int in_page = slot < 0 ? 0 : (int)slot - page * a.page_size;

  auto source = [&](int r) -> const IRIS_GLOBAL char* {
    const char* base = (const char*)(r < a.q_heads ? a.q : r < a.q_heads + a.k_heads ? a.k : a.v);
    const int64_t off = r < a.q_heads                ? t * a.stride_qt + r * a.stride_qh
                        : r < a.q_heads + a.k_heads ? t * a.stride_kt + (r - a.q_heads) * a.stride_kh
                                                    : t * a.stride_vt + (r - a.q_heads - a.k_heads) * a.stride_vh;
    return (const IRIS_GLOBAL char*)(base + off * ES);
  };
  Row<DT, V, ITEMS> x[BATCH];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (r0 + u < end) x[u].load(source(r0 + u), at);
  };
  fetch(begin);
  Angles<V, ITEMS> angle;
  load_angles(a, t, at, angle);
  Row<DT, V, ITEMS> wq, wk;
  load_weight(a.q_weight, a.weight_fp32, at, wq);
  load_weight(a.k_weight, a.weight_fp32, at, wk);

  for (int r0 = begin; r0 < end; r0 += BATCH) {
    if (r0 > begin) fetch(r0);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int r = r0 + u;
      if (r >= end) break;
      const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + a.k_heads;
      if (!is_v) {
        const bool normed = (is_q ? a.q_weight : a.k_weight) != nullptr;
        if (normed) {
          const float rs = rsqrtf(sum_lanes<LANES>(dot_items<V, ITEMS>(x[u], x[u])) / (float)a.head_dim + a.eps);
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              x[u].a[i][e] *= rs * (is_q ? wq.a[i][e] : wk.a[i][e]);
              x[u].b[i][e] *= rs * (is_q ? wq.b[i][e] : wk.b[i][e]);
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (at[i].turns) turn<V, false>(x[u].a[i], x[u].b[i], angle.c[i], angle.s[i], a.interleaved);
      }
      if (is_q) {
        x[u].store((IRIS_GLOBAL char*)a.q_out + (t * a.stride_qot + r * a.stride_qoh) * ES, at);
      } else if (!is_v) {
        const int h = r - a.q_heads;
        if (a.k_out) x[u].store((IRIS_GLOBAL char*)a.k_out + (t * a.stride_kot + h * a.stride_koh) * ES, at);
        if (slot >= 0)
          x[u].store((IRIS_GLOBAL char*)a.k_cache + (page * a.stride_kc_page + in_page * a.stride_kc_row + h * a.stride_kc_head) * ES, at);
      } else if (slot >= 0) {
        const int h = r - a.q_heads - a.k_heads;
        x[u].store((IRIS_GLOBAL char*)a.v_cache + (page * a.stride_vc_page + in_page * a.stride_vc_row + h * a.stride_vc_head) * ES, at);
      }
    }
  }
}

// The gradient.  A group takes whole tokens, `step` groups apart, and keeps its share of the weights' gradients in
// registers; a workgroup adds its groups' shares in LDS in a fixed order and leaves one row of partial sums, which
// weight_gradient_kernel adds in a fixed order: the same inputs give the same bits.
template <int DT, int V, int LANES, int ITEMS>
__global__ __launch_bounds__(THREADS) void qk_norm_rope_backward_kernel(iris_qk_norm_rope_backward_args a) {
  constexpr int ES = DT == IRIS_DTYPE_F32 ? 4 : 2, GROUPS = THREADS / LANES;
  const int lane = threadIdx.x % LANES, in_block = threadIdx.x / LANES;
  Place<V> at[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) at[i] = place<V>(lane + i * LANES, a.head_dim, a.rotary_dim, a.interleaved);
  Row<DT, V, ITEMS> w[2], dw[2];
  load_weight(a.q_weight, a.weight_fp32, at, w[0]);
  load_weight(a.k_weight, a.weight_fp32, at, w[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) dw[k].a[i][e] = dw[k].b[i][e] = 0.f;

  const float inv_dim = 1.f / (float)a.head_dim;
  for (int64_t t = (int64_t)blockIdx.x * GROUPS + in_block; t < a.tokens; t += (int64_t)gridDim.x * GROUPS) {
    Angles<V, ITEMS> angle;
    load_angles(a, t, at, angle);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int heads = k ? a.k_heads : a.q_heads;
      const bool normed = (k ? a.k_weight : a.q_weight) != nullptr;
      const IRIS_GLOBAL char* xs = (const IRIS_GLOBAL char*)(k ? a.k : a.q) + t * (k ? a.stride_kt : a.stride_qt) * ES;
      const IRIS_GLOBAL char* zs = (const IRIS_GLOBAL char*)(k ? a.dk_out : a.dq_out) + t * (k ? a.stride_dkot : a.stride_dqot) * ES;
      IRIS_GLOBAL char* ds = (IRIS_GLOBAL char*)(k ? a.dk : a.dq) + t * (k ? a.stride_dkt : a.stride_dqt) * ES;
      const int64_t xh = (k ? a.stride_kh : a.stride_qh) * ES, zh = (k ? a.stride_dkoh : a.stride_dqoh) * ES,
                    dh = (k ? a.stride_dkh : a.stride_dqh) * ES;
      for (int h0 = 0; h0 < heads; h0 += BATCH) {
        Row<DT, V, ITEMS> x[BATCH], g[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (h0 + u < heads) {
            g[u].load(zs + (h0 + u) * zh, at);
            if (normed) x[u].load(xs + (h0 + u) * xh, at);
          }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (h0 + u >= heads) break;
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
            if (at[i].turns) turn<V, true>(g[u].a[i], g[u].b[i], angle.c[i], angle.s[i], a.interleaved);
          if (normed) {
            // dx is what is left of g w when its part along x is taken out: in short heads very little, so those (which single
            // pairs serve) take it out in 64 bits
            using Acc = std::conditional_t<V == 1, double, float>;
            Acc square = 0, along = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
              for (int e = 0; e < V; ++e) {
                square += (Acc)x[u].a[i][e] * x[u].a[i][e] + (Acc)x[u].b[i][e] * x[u].b[i][e];
                along += (Acc)g[u].a[i][e] * w[k].a[i][e] * x[u].a[i][e] + (Acc)g[u].b[i][e] * w[k].b[i][e] * x[u].b[i][e];
              }
            square = sum_lanes<LANES>(square);
            along = sum_lanes<LANES>(along);
            const float rs = rsqrtf((float)(square * inv_dim) + a.eps);
            const Acc back = along / (square + (Acc)a.head_dim * a.eps);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
              for (int e = 0; e < V; ++e) {
                dw[k].a[i][e] += g[u].a[i][e] * x[u].a[i][e] * rs;
                dw[k].b[i][e] += g[u].b[i][e] * x[u].b[i][e] * rs;
                g[u].a[i][e] = rs * (float)((Acc)g[u].a[i][e] * w[k].a[i][e] - x[u].a[i][e] * back);
                g[u].b[i][e] = rs * (float)((Acc)g[u].b[i][e] * w[k].b[i][e] - x[u].b[i][e] * back);
              }
          }
          g[u].store(ds + (h0 + u) * dh, at);
        }
      }
    }
  }
  if (!a.dq_weight && !a.dk_weight) return;
  // the groups' shares: rows of `width` floats in LDS, added by column
  extern __shared__ float shares[];
  const int width = 2 * a.head_dim;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (at[i].live)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          shares[in_block * width + k * a.head_dim + at[i].first + e] = dw[k].a[i][e];
          shares[in_block * width + k * a.head_dim + at[i].second + e] = dw[k].b[i][e];
        }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += THREADS) {
    float sum = 0.f;
    for (int g = 0; g < GROUPS; ++g) sum += shares[g * width + c];
    a.workspace[(int64_t)blockIdx.x * width + c] = sum;
  }
}

// Adds the workgroups' partial sums: 16 columns a workgroup, 16 lanes a column.
__global__ __launch_bounds__(THREADS) void weight_gradient_kernel(const float* partials, int rows, int dim, float* dq_weight, float* dk_weight) {
  __shared__ float sums[16][17];
  const int c = threadIdx.x % 16, part = threadIdx.x / 16, column = blockIdx.x * 16 + c, width = 2 * dim;
  float sum = 0.f;
  if (column < width)
    for (int r = part; r < rows; r += 16) sum += partials[(int64_t)r * width + column];
  sums[part][c] = sum;
  __syncthreads();
  if (part == 0 && column < width) {
    float all = 0.f;
    for (int p = 0; p < 16; ++p) all += sums[p][c];
    float* out = column < dim ? dq_weight : dk_weight;
    if (out) out[column < dim ? column : column - dim] = all;
  }
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

  const int rows = a.q_heads + a.k_heads + (a.v ? a.k_heads : 0);
  return with_dtype(a.dtype, [&](auto dt) {
    return with_layout(wide, a.head_dim, [&](auto v, auto lanes, auto items) {
      // All of a token's heads in one group share its angles; few tokens are spread over more groups.
      const int64_t per_block = THREADS / lanes.value, enough = (int64_t)4 * current_cu_count() * per_block;
      int heads_each = rows;
      while (heads_each > BATCH && (int64_t)a.tokens * ((rows + heads_each - 1) / heads_each) < enough) heads_each = (heads_each + 1) / 2;
      if ((int64_t)a.tokens * rows <= enough) heads_each = 1;
      const int parts = (rows + heads_each - 1) / heads_each;
      const int64_t groups = (int64_t)a.tokens * parts, grid = (groups + per_block - 1) / per_block;
      if (grid > INT32_MAX) return hipErrorInvalidValue;
      qk_norm_rope_kernel<dt.value, v.value, lanes.value, items.value>
          <<<(int)grid, THREADS, 0, (hipStream_t)stream>>>(a, make_fast_div((uint32_t)parts, (uint64_t)(grid * per_block)), heads_each);
      return hipGetLastError();
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
      int64_t grid = (a.tokens + per_block - 1) / per_block, most = 4 * (int64_t)current_cu_count();
      if (weights && a.workspace_elems / (2 * a.head_dim) < most) most = a.workspace_elems / (2 * a.head_dim);
      grid = grid < 1 ? 1 : grid > most ? most : grid;
      const size_t lds = weights ? per_block * 2 * a.head_dim * sizeof(float) : 0;
      qk_norm_rope_backward_kernel<dt.value, v.value, lanes.value, items.value><<<(int)grid, THREADS, lds, (hipStream_t)stream>>>(a);
      hipError_t err = hipGetLastError();
      if (err != hipSuccess || !weights) return err;
      weight_gradient_kernel<<<(2 * a.head_dim + 15) / 16, THREADS, 0, (hipStream_t)stream>>>(a.workspace, (int)grid, a.head_dim, a.dq_weight,
                                                                                              a.dk_weight);
      return hipGetLastError();
    });
  });
}
