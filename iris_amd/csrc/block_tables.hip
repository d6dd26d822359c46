// Block tables of a paged key-value cache, from request lengths: which pages a step takes from the ring of free
// pages and which it gives back, and position and slot of every new token.
//
// need_i = pages(c_i + n_i) - pages(c_i), pages(n) = ceil(n / P).  Everything follows from three prefix sums over the
// requests: of the pages needed (where each request's pages start in the ring), of the new tokens (query starts), and of
// the pages given back.  The sums are 12 bytes a request, so every workgroup computes all of them for itself in LDS
// and then takes its share of what is written (tokens, fresh table entries, returned pages), which a binary search in
// the sums maps back to its request: one launch, no workgroup waits for another.
#include "heads_common.hpp"

namespace iris_amd {
namespace {

constexpr int MAX_REQUESTS = 8192;  // three sums of them fit in LDS

struct Sums {
  int need, back, tokens;
};

// What request i asks for, before the ring's end is looked at.
struct Request {
  int cached, add, held, want;
  bool ended, fits;
};
__device__ inline Request request(const iris_block_tables_args& a, int i) {
  Request r;
  const int n = a.new_tokens[i];
  r.cached = max(a.cached[i], 0);
  r.ended = n < 0;
  r.add = max(n, 0);
  const int64_t want = ((int64_t)r.cached + r.add + a.page_size - 1) / a.page_size;
  r.held = (int)(((int64_t)r.cached + a.page_size - 1) / a.page_size);
  r.fits = !r.ended && want <= a.table_width;
  r.want = r.fits ? (int)want : r.held;
  if (r.ended) r.held = min(r.held, a.table_width);
  return r;
}

// The largest i < n with before[i] <= x, where before[0] == 0.
__device__ inline int owner(const int* before, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void block_tables_kernel(iris_block_tables_args a) {
  extern __shared__ int lds[];
  __shared__ Sums wave_sums[THREADS / 64];
  __shared__ int granted;  // pages taken by the requests that were served
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.requests;
  int* const need_before = lds;
  int* const back_before = lds + n;
  int* const tokens_before = lds + 2 * n;
  const int64_t taken = a.pool_state[0], returned = a.pool_state[1];
  const int64_t free64 = returned - taken;
  const int free_pages = (int)(free64 < 0 ? 0 : free64 > a.pool_size ? a.pool_size : free64);
  if (tid == 0) granted = 0;

  // exclusive prefix sums of the requests, THREADS of them at a time
  Sums carry{0, 0, 0};
  for (int base = 0; base < n; base += THREADS) {
    const int i = base + tid;
    Sums own{0, 0, 0};
    if (i < n) {
      const Request r = request(a, i);
      own.need = r.fits ? r.want - r.held : 0;
      own.back = r.ended ? r.held : 0;
      own.tokens = r.add;
    }
    Sums s = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(s.need, d, 64), y = __shfl_up(s.back, d, 64), z = __shfl_up(s.tokens, d, 64);
      if (lane >= d) {
        s.need += x;
        s.back += y;
        s.tokens += z;
      }
    }
    __syncthreads();  // (the last chunk's sums have been read)
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    Sums before = carry;
    for (int w = 0; w < THREADS / 64; ++w) {
      const Sums t = wave_sums[w];
      if (w < wave) {
        before.need += t.need;
        before.back += t.back;
        before.tokens += t.tokens;
      }
      carry.need += t.need;
      carry.back += t.back;
      carry.tokens += t.tokens;
    }
    if (i < n) {
      need_before[i] = before.need + s.need - own.need;
      back_before[i] = before.back + s.back - own.back;
      tokens_before[i] = before.tokens + s.tokens - own.tokens;
      // The requests that need pages are served while the ring lasts: a prefix of them, whose last sum is the number taken.
      if (own.need && before.need + s.need <= free_pages) atomicMax(&granted, before.need + s.need);
    }
  }
  __syncthreads();
  const int total = carry.tokens;
  const uint32_t ring = (uint32_t)a.pool_size;
  const uint32_t taken_at = (uint32_t)(taken % ring), returned_at = (uint32_t)(returned % ring);
  // served: does request i get what it needs
  auto served = [&](const Request& r, int i) { return r.fits && (r.want == r.held || need_before[i] + r.want - r.held <= free_pages); };
  auto page_of = [&](int nth) { return a.pool[(taken_at + (uint32_t)nth) % ring]; };

  const int gid = blockIdx.x * THREADS + tid, step = gridDim.x * THREADS;
  for (int i = gid; i < n; i += step) {
    const Request r = request(a, i);
    const bool ok = served(r, i);
    a.lengths[i] = r.ended ? 0 : ok ? r.cached + r.add : r.cached;
    a.query_starts[i] = tokens_before[i];
    if (!r.ended && !ok) report(a.status, IRIS_STATUS_NO_PAGES);
  }
  if (gid == 0) {
    a.query_starts[n] = total;
    a.pool_state_out[0] = taken + granted;
    a.pool_state_out[1] = returned + carry.back;
    if (total > a.max_tokens) report(a.status, IRIS_STATUS_NO_ROOM);
  }
  for (int t = gid; t < a.max_tokens; t += step) {
    int position = 0;
    int64_t slot = -1;
    if (t < total) {
      const int i = owner(tokens_before, n, t);
      const Request r = request(a, i);
      position = r.cached + t - tokens_before[i];
      const int j = position / a.page_size;
      if (served(r, i) && position >= 0 && j < a.table_width) {
        const int page = j < r.held ? a.block_table[(int64_t)i * a.stride_table + j] : page_of(need_before[i] + j - r.held);
        slot = (int64_t)page * a.page_size + position % a.page_size;
      }
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }
  // (a request that was not served has sums past `granted`, and needs nothing where it has not)
  for (int x = gid; x < granted; x += step) {
    const int i = owner(need_before, n, x);
    const Request r = request(a, i);
    a.block_table[(int64_t)i * a.stride_table + r.held + x - need_before[i]] = page_of(x);
  }
  for (int x = gid; x < carry.back; x += step) {
    const int i = owner(back_before, n, x);
    a.pool[(returned_at + (uint32_t)x) % ring] = a.block_table[(int64_t)i * a.stride_table + x - back_before[i]];
  }
}

}  // namespace
}  // namespace iris_amd

extern "C" int iris_block_tables_launch(const iris_block_tables_args* args, void* stream) {
  using namespace iris_amd;
  if (!args) return hipErrorInvalidValue;
  const iris_block_tables_args& a = *args;
  if (a.requests < 0 || a.requests > MAX_REQUESTS || a.max_tokens < 0 || a.page_size <= 0 || a.pool_size <= 0 || a.table_width < 0 ||
      a.stride_table < a.table_width || !a.pool || !a.pool_state || !a.pool_state_out || !a.query_starts ||
      (a.max_tokens && (!a.positions || !a.slots)) || (a.requests && (!a.cached || !a.new_tokens || !a.lengths)) ||
      (a.requests && a.table_width && !a.block_table) || (int64_t)a.requests * a.table_width > INT32_MAX)
    return hipErrorInvalidValue;
  const size_t lds = (size_t)a.requests * 3 * sizeof(int);
  const int threads = a.requests > 1024 ? 1024 : 256;
  // a workgroup repeats the sums, so it is given a few items a thread to write
  const int64_t items = (int64_t)a.max_tokens + a.requests;
  const int64_t groups = (items + 2 * threads - 1) / (2 * threads);
  const int cus = current_cu_count();
  const int grid = (int)(groups < 1 ? 1 : groups > cus ? cus : groups);
  if (threads == 1024) {
    if (lds > 64 * 1024) {
      const hipError_t err = hipFuncSetAttribute((const void*)block_tables_kernel<1024>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (err != hipSuccess) return err;
    }
    block_tables_kernel<1024><<<grid, 1024, lds, (hipStream_t)stream>>>(a);
  } else {
    block_tables_kernel<256><<<grid, 256, lds, (hipStream_t)stream>>>(a);
  }
  return hipGetLastError();
}
