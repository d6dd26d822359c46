// Block tables of a paged key-value cache, from request lengths: which pages a step takes from the ring of free
// pages and which it gives back, and position and slot of every new token.
//
// need_i = pages(c_i + n_i) - pages(c_i), pages(n) = ceil(n / P).  Everything follows from three prefix sums over the
// requests: of the pages needed (where each request's pages start in the ring), of the new tokens (query starts), and of
// the pages given back.  The sums are 12 bytes a request, so every workgroup computes all of them for itself in LDS
// and then takes its share of what is written (tokens, fresh table entries, returned pages), which a binary search in
// the sums maps back to its request: one launch, no workgroup waits for another.
//
// The bytes are nothing (64 requests: 2 KB); what it takes is a chain of latencies, launch, lengths, sums, ring, store, and
// the time is that of the launch's call: 64 requests 4.7 us, 1000 of which 24 bring prompts and 15 end 6.8.
#include "heads_common.hpp"

namespace iris_amd {
namespace {

constexpr int MAX_REQUESTS = 8192;  // three sums and the lengths of them fit in LDS
constexpr int THREADS = 1024;

struct Sums {
  int need, back, tokens;
};
__device__ inline Sums operator+(Sums a, Sums b) { return {a.need + b.need, a.back + b.back, a.tokens + b.tokens}; }

struct Args {
  iris_block_tables_args a;
  PageDiv page;
  int room;  // tokens that a table row has pages for
};

__device__ inline int pages(int tokens, const PageDiv& p) { return tokens > 0 ? (int)page_div((uint32_t)tokens - 1, p) + 1 : 0; }

// What a request asks for, before the ring's end is looked at.
struct Request {
  int cached, add;
  bool ended, fits;
};
__device__ inline Request request(const Args& g, int i) {
  Request r;
  const int n = g.a.new_tokens[i];
  r.cached = max(g.a.cached[i], 0);
  r.ended = n < 0;
  r.add = max(n, 0);
  r.fits = !r.ended && (int64_t)r.cached + r.add <= g.room;
  return r;
}

// Inclusive sum over the wave.  DPP: shifts within rows of 16, then the rows' and halves' last lanes to the next ones.
template <int CTRL, int ROWS>
__device__ inline int shifted(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ inline int wave_prefix(int x) {
  x += shifted<0x111, 0xF>(x);
  x += shifted<0x112, 0xF>(x);
  x += shifted<0x114, 0xF>(x);
  x += shifted<0x118, 0xF>(x);
  x += shifted<0x142, 0xA>(x);
  x += shifted<0x143, 0xC>(x);
  return x;
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

// ITEMS requests a thread, neighbours.
template <int ITEMS>
__global__ __launch_bounds__(THREADS) void block_tables_kernel(Args g) {
  extern __shared__ int lds[];
  __shared__ Sums wave_sums[THREADS / 64];
  __shared__ int granted;  // pages taken by the requests that were served
  const iris_block_tables_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x / 64, n = a.requests;
  int* const need_before = lds;
  int* const back_before = lds + n;
  int* const tokens_before = lds + 2 * n;
  int* const lengths = lds + 3 * n;  // tokens in the cache; of requests that are not served, the complement
  const int64_t taken = a.pool_state[0], returned = a.pool_state[1];
  const int64_t free64 = returned - taken;
  const int free_pages = (int)(free64 < 0 ? 0 : free64 > a.pool_size ? a.pool_size : free64);
  if (tid == 0) granted = 0;

  // exclusive prefix sums of the requests
  Request r[ITEMS];
  Sums own[ITEMS], mine{0, 0, 0};
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = tid * ITEMS + k;
    own[k] = Sums{0, 0, 0};
    if (i < n) {
      r[k] = request(g, i);
      const int held = pages(r[k].cached, g.page);
      if (r[k].fits) own[k].need = pages(r[k].cached + r[k].add, g.page) - held;
      if (r[k].ended) own[k].back = min(held, a.table_width);
      own[k].tokens = r[k].add;
    }
    mine = mine + own[k];
  }
  const Sums upto{wave_prefix(mine.need), wave_prefix(mine.back), wave_prefix(mine.tokens)};
  if (lane == 63) wave_sums[wave] = upto;
  __syncthreads();
  Sums before{upto.need - mine.need, upto.back - mine.back, upto.tokens - mine.tokens}, all{0, 0, 0};
  for (int w = 0; w < waves; ++w) {
    const Sums t = wave_sums[w];
    if (w < wave) before = before + t;
    all = all + t;
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = tid * ITEMS + k;
    if (i < n) {
      // The requests that need pages are served while the ring lasts: a prefix of them, whose last sum is the number taken.
      const int after = before.need + own[k].need;
      const bool served = r[k].fits && (!own[k].need || after <= free_pages);
      if (own[k].need && served) atomicMax(&granted, after);
      need_before[i] = before.need;
      back_before[i] = before.back;
      tokens_before[i] = before.tokens;
      lengths[i] = served || r[k].ended ? r[k].cached : ~r[k].cached;
      if (blockIdx.x == 0) {
        a.lengths[i] = r[k].ended ? 0 : served ? r[k].cached + r[k].add : r[k].cached;
        a.query_starts[i] = before.tokens;
        if (!r[k].ended && !served) report(a.status, IRIS_STATUS_NO_PAGES);
      }
    }
    before = before + own[k];
  }
  __syncthreads();
  const uint32_t ring = (uint32_t)a.pool_size;
  const uint32_t taken_at = (uint32_t)(taken % ring), returned_at = (uint32_t)(returned % ring);
  auto page_of = [&](int nth) { return a.pool[(taken_at + (uint32_t)nth) % ring]; };

  const int gid = blockIdx.x * blockDim.x + tid, step = gridDim.x * blockDim.x;
  if (gid == 0) {
    a.query_starts[n] = all.tokens;
    a.pool_state_out[0] = taken + granted;
    a.pool_state_out[1] = returned + all.back;
    if (all.tokens > a.max_tokens) report(a.status, IRIS_STATUS_NO_ROOM);
  }
  for (int t = gid; t < a.max_tokens; t += step) {
    int position = 0;
    int64_t slot = -1;
    if (t < all.tokens) {
      const int i = owner(tokens_before, n, t), length = lengths[i];
      position = (length < 0 ? ~length : length) + t - tokens_before[i];
      // (a sum past 31 bits, of lengths that are none, may leave a position that is none)
      if (length >= 0 && position >= 0 && position < g.room) {
        const int j = (int)page_div((uint32_t)position, g.page), held = pages(length, g.page);
        const int page = j < held ? a.block_table[(int64_t)i * a.stride_table + j] : page_of(need_before[i] + j - held);
        slot = (int64_t)page * a.page_size + (position - j * a.page_size);
      }
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }
  // (a request that was not served has sums past `granted`, and needs nothing where it has not)
  for (int x = gid; x < granted; x += step) {
    const int i = owner(need_before, n, x), j = pages(lengths[i], g.page) + x - need_before[i];
    if ((uint32_t)j < (uint32_t)a.table_width) a.block_table[(int64_t)i * a.stride_table + j] = page_of(x);
  }
  for (int x = gid; x < all.back; x += step) {
    const int i = owner(back_before, n, x), j = x - back_before[i];
    if ((uint32_t)j < (uint32_t)a.table_width) a.pool[(returned_at + (uint32_t)x) % ring] = a.block_table[(int64_t)i * a.stride_table + j];
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
  if ((int64_t)a.table_width * a.page_size > INT32_MAX) return hipErrorInvalidValue;
  const Args g{a, make_page_div((uint32_t)a.page_size), a.table_width * a.page_size};
  const size_t lds = (size_t)a.requests * 4 * sizeof(int);
  constexpr size_t FIXED_LDS = THREADS / 64 * sizeof(Sums) + sizeof(int);  // the waves' sums, and what is granted
  // Four waves where they hold the requests, so that a small step's sums meet sooner; sixteen beyond.  An item (token) a thread: a
  // workgroup repeats the sums, but what it writes it looks for in several dependent reads.
  const int threads = a.requests > 256 ? THREADS : 256;
  const int64_t groups = ((int64_t)a.max_tokens + threads - 1) / threads;
  const int cus = current_cu_count();
  const int grid = (int)(groups < 1 ? 1 : groups > cus ? cus : groups);
  if (a.requests > THREADS) {
    constexpr int ITEMS = MAX_REQUESTS / THREADS;
    if (lds + FIXED_LDS > 64 * 1024) {  // (4084 requests and more)
      const hipError_t err = hipFuncSetAttribute((const void*)block_tables_kernel<ITEMS>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (err != hipSuccess) return err;
    }
    return launch(block_tables_kernel<ITEMS>, dim3(grid), threads, lds, stream, g);
  }
  return launch(block_tables_kernel<1>, dim3(grid), threads, lds, stream, g);
}
