// Block tables and slots of one scheduler step (smaq_page_step).
//
// Request b holds c_b tokens in ceil(c_b / bs) pages and gets n_b more, so it
// takes ceil((c_b + n_b) / bs) - ceil(c_b / bs) pages off the front of the free
// list, in request order: the free list's index of its first page and the row of
// its first token are exclusive sums over the requests.
//
// One launch, and nothing to wait for: every workgroup forms both sums over all
// requests in its own LDS (8000 requests are 64 KB, read from L2), then takes
// its share of the tokens, of the taken pages and of the requests, and finds an
// item's request by bisection.  A token's page is either the request's last,
// partly filled one -- an entry of the table that this call does not write -- or
// one off the free list, so no token waits for a table entry.
//
// Latency bounds it: two passes over the lengths, a scan, a bisection.  256 requests of one
// token take 8 us, 1000 requests with 37000 tokens (0.6 MB written) 11.
#include <algorithm>

#include "smaq_common.h"

namespace smaq {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 8000;  // two sums each in 64 KB of LDS
constexpr uint32_t kMost = 0x7fffffff;  // lengths, sums and results stop here

struct PageArgs {
  const void *context, *fresh;
  int context_wide, fresh_wide;
  int requests;
  int* table;
  uint32_t width;
  const int* free_blocks;
  uint32_t n_free, bs, tokens;
  long long *slots, *positions;
  int *starts, *seq_lens, *status;
};

__device__ __forceinline__ uint32_t length_at(const void* p, int wide, int b) {
  if (!wide) return (uint32_t)max(((const int*)p)[b], 0);
  return (uint32_t)min(max(((const long long*)p)[b], 0ll), (long long)kMost);
}

__device__ __forceinline__ uint32_t add_to_most(uint32_t x, uint32_t y) { return min(x + y, kMost); }  // both up to kMost

__device__ __forceinline__ uint32_t pages_of(uint32_t n, uint32_t bs) { return n / bs + (n % bs != 0); }

// the last index i of the ascending s[0..n) with s[i] <= x (s[0] <= x)
__device__ __forceinline__ int last_at_most(const uint32_t* s, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void page_step_kernel(PageArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t* row0 = lds;                    // [requests + 1] first token of each request
  uint32_t* page0 = lds + a.requests + 1;  // [requests + 1] first taken page of each request
  __shared__ uint32_t part[2][kThreads / 64], placed_all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.requests;
  const uint32_t bs = a.bs;
  // each thread sums its run of requests, then a scan over the threads
  const int each = (n + kThreads - 1) / kThreads;
  const int b0 = min(n, tid * each), b1 = min(n, b0 + each);
  uint32_t sum_n = 0, sum_t = 0;
  for (int b = b0; b < b1; ++b) {
    const uint32_t c = length_at(a.context, a.context_wide, b), m = length_at(a.fresh, a.fresh_wide, b);
    sum_n = add_to_most(sum_n, m);
    sum_t = add_to_most(sum_t, pages_of(c + m, bs) - pages_of(c, bs));
  }
  uint32_t in_n = sum_n, in_t = sum_t, run_n = 0, run_t = 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = __shfl_up(in_n, o, 64), y = __shfl_up(in_t, o, 64);
    if (lane >= o) {
      in_n = add_to_most(in_n, x);
      in_t = add_to_most(in_t, y);
    }
  }
  const uint32_t up_n = __shfl_up(in_n, 1, 64), up_t = __shfl_up(in_t, 1, 64);
  if (lane) {
    run_n = up_n;
    run_t = up_t;
  }
  if (lane == 63) {
    part[0][wave] = in_n;
    part[1][wave] = in_t;
  }
  if (tid == 0) placed_all = 0;
  __syncthreads();
  uint32_t total_n = 0, total_t = 0, wave_n = 0, wave_t = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w == wave) {
      wave_n = total_n;
      wave_t = total_t;
    }
    total_n = add_to_most(total_n, part[0][w]);
    total_t = add_to_most(total_t, part[1][w]);
  }
  run_n = add_to_most(run_n, wave_n);
  run_t = add_to_most(run_t, wave_t);
  uint32_t placed = 0;  // tokens of this thread's requests that get a slot (workgroup 0 reports them)
  for (int b = b0; b < b1; ++b) {
    row0[b] = run_n;
    page0[b] = run_t;
    const uint32_t c = length_at(a.context, a.context_wide, b), m = length_at(a.fresh, a.fresh_wide, b);
    const uint32_t held = pages_of(c, bs), taken = pages_of(c + m, bs) - held;
    if (blockIdx.x == 0) {
      const uint32_t got = min(a.n_free > run_t ? a.n_free - run_t : 0u, taken);
      const uint64_t room = (uint64_t)min(a.width, held + got) * bs;
      const uint32_t rows = min(a.tokens > run_n ? a.tokens - run_n : 0u, m);
      uint32_t ok = room > c ? (uint32_t)min(room - c, (uint64_t)rows) : 0u;
      if (c % bs && c / bs < a.width && a.table[(int64_t)b * a.width + c / bs] < 0) ok -= min(ok, bs - c % bs);
      placed += ok;
    }
    run_n = add_to_most(run_n, m);
    run_t = add_to_most(run_t, taken);
  }
  if (tid == 0) {
    row0[n] = total_n;
    page0[n] = total_t;
  }
  if (blockIdx.x == 0 && placed) atomicAdd(&placed_all, placed);
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    a.status[0] = (int)total_t;
    a.status[1] = (int)(total_n - placed_all);
  }
  const uint32_t stride = gridDim.x * kThreads, first = blockIdx.x * kThreads + tid;
  for (uint32_t b = first; b <= (uint32_t)n; b += stride) {
    a.starts[b] = (int)row0[b];
    if (b < (uint32_t)n)
      a.seq_lens[b] = (int)min(length_at(a.context, a.context_wide, (int)b) + length_at(a.fresh, a.fresh_wide, (int)b), kMost);
  }
  // taken pages: entry e of the free list goes to its request's next column
  for (uint32_t e = first; e < total_t; e += stride) {
    const int b = last_at_most(page0, n, e);
    const uint64_t col = (uint64_t)pages_of(length_at(a.context, a.context_wide, b), bs) + (e - page0[b]);
    if (col < a.width) a.table[(int64_t)b * a.width + col] = e < a.n_free ? a.free_blocks[e] : -1;
  }
  for (uint32_t i = first; i < a.tokens; i += stride) {
    int64_t slot = -1;
    uint32_t pos = 0;
    if (i < total_n) {
      const int b = last_at_most(row0, n, i);
      const uint32_t c = length_at(a.context, a.context_wide, b);
      pos = c + (i - row0[b]);
      const uint32_t col = pos / bs, held = pages_of(c, bs);
      if (col < a.width) {
        const uint64_t e = (uint64_t)page0[b] + (col - held);
        const int blk = col < held ? a.table[(int64_t)b * a.width + col] : (e < a.n_free ? a.free_blocks[e] : -1);
        if (blk >= 0) slot = (int64_t)blk * bs + pos % bs;
      }
    }
    a.slots[i] = slot;
    a.positions[i] = pos;
  }
}

}  // namespace
}  // namespace smaq

extern "C" int smaq_page_step(const void* context_lens, int context_bytes, const void* new_lens, int new_bytes,
                              int requests, int* block_table, int max_blocks, const int* free_blocks,
                              long long n_free, int block_size, long long tokens, long long* slot_mapping,
                              long long* positions, int* query_start_loc, int* seq_lens, int* status, void* stream) {
  using namespace smaq;
  SMAQ_REQUIRE(requests >= 0 && requests <= kMaxRequests, "smaq_page_step: %d requests are not in 0..%d", requests,
               kMaxRequests);
  SMAQ_REQUIRE(block_size >= 1 && block_size <= 65536 && max_blocks >= 0 && n_free >= 0 && tokens >= 0 &&
                   n_free <= (long long)kMost && tokens <= (long long)kMost,
               "smaq_page_step: bad sizes (block_size %d, max_blocks %d, %lld free, %lld tokens)", block_size,
               max_blocks, n_free, tokens);
  SMAQ_REQUIRE((context_bytes == 4 || context_bytes == 8) && (new_bytes == 4 || new_bytes == 8),
               "smaq_page_step: lengths of %d and %d bytes", context_bytes, new_bytes);
  SMAQ_REQUIRE((!requests || (context_lens && new_lens && seq_lens)) && (!requests || !max_blocks || block_table) &&
                   (!n_free || free_blocks) && (!tokens || (slot_mapping && positions)) && query_start_loc && status,
               "smaq_page_step: null pointer");
  PageArgs a{context_lens, new_lens, context_bytes == 8, new_bytes == 8, requests, block_table, (uint32_t)max_blocks,
             free_blocks, (uint32_t)n_free, (uint32_t)block_size, (uint32_t)tokens, slot_mapping, positions,
             query_start_loc, seq_lens, status};
  // a token or request a thread, up to one workgroup a CU
  const int64_t groups = std::min<int64_t>((std::max<int64_t>(tokens, requests + 1) + kThreads - 1) / kThreads, 256);
  const size_t bytes = 2 * sizeof(int) * (size_t)(requests + 1);
  page_step_kernel<<<(unsigned)std::max<int64_t>(groups, 1), kThreads, bytes, (hipStream_t)stream>>>(a);
  return launch_status("smaq_page_step");
}
