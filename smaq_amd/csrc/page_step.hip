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
#include <algorithm>

#include "smaq_common.h"

namespace smaq {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 8000;  // two sums each in 64 KB of LDS
constexpr int64_t kIntMax = 0x7fffffff;

struct PageArgs {
  const void *context, *fresh;
  int context_wide, fresh_wide;
  int requests;
  int* table;
  int width;
  const int* free_blocks;
  int64_t n_free;
  int bs;
  int64_t tokens;
  long long *slots, *positions;
  int *starts, *seq_lens, *status;
};

__device__ __forceinline__ int64_t length_at(const void* p, int wide, int b) {
  const int64_t v = wide ? (int64_t)((const long long*)p)[b] : (int64_t)((const int*)p)[b];
  return min(max(v, (int64_t)0), kIntMax);
}

// the last index i of the ascending s[0..n) with s[i] <= x (s[0] <= x)
__device__ __forceinline__ int last_at_most(const int* s, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void page_step_kernel(PageArgs a) {
  extern __shared__ int lds[];
  int* row0 = lds;                    // [requests + 1] first token of each request
  int* page0 = lds + a.requests + 1;  // [requests + 1] first taken page of each request
  __shared__ int64_t part[2][kThreads / 64];
  __shared__ int64_t placed_all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.requests, bs = a.bs;
  // each thread sums its run of requests, then a scan over the threads
  const int each = (n + kThreads - 1) / kThreads;
  const int b0 = min(n, tid * each), b1 = min(n, b0 + each);
  int64_t sum_n = 0, sum_t = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t c = length_at(a.context, a.context_wide, b), m = length_at(a.fresh, a.fresh_wide, b);
    sum_n += m;
    sum_t += (c + m + bs - 1) / bs - (c + bs - 1) / bs;
  }
  int64_t in_n = sum_n, in_t = sum_t;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t x = __shfl_up(in_n, o, 64), y = __shfl_up(in_t, o, 64);
    if (lane >= o) { in_n += x; in_t += y; }
  }
  if (lane == 63) { part[0][wave] = in_n; part[1][wave] = in_t; }
  if (tid == 0) placed_all = 0;
  __syncthreads();
  int64_t run_n = in_n - sum_n, run_t = in_t - sum_t, total_n = 0, total_t = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) { run_n += part[0][w]; run_t += part[1][w]; }
    total_n += part[0][w];
    total_t += part[1][w];
  }
  int64_t placed = 0;  // tokens of this thread's requests that get a slot (workgroup 0 reports them)
  for (int b = b0; b < b1; ++b) {
    row0[b] = (int)min(run_n, kIntMax);
    page0[b] = (int)min(run_t, kIntMax);
    const int64_t c = length_at(a.context, a.context_wide, b), m = length_at(a.fresh, a.fresh_wide, b);
    const int64_t held = (c + bs - 1) / bs, taken = (c + m + bs - 1) / bs - held;
    if (blockIdx.x == 0) {
      const int64_t pages = min((int64_t)a.width, held + min(max(a.n_free - run_t, (int64_t)0), taken));
      const int64_t rows = min(max(a.tokens - run_n, (int64_t)0), m);
      int64_t ok = min(max(pages * bs - c, (int64_t)0), rows);
      if (c % bs && c / bs < a.width && a.table[(int64_t)b * a.width + c / bs] < 0) ok -= min(ok, bs - c % bs);
      placed += ok;
    }
    run_n += m;
    run_t += taken;
  }
  if (tid == 0) {
    row0[n] = (int)min(total_n, kIntMax);
    page0[n] = (int)min(total_t, kIntMax);
  }
  if (blockIdx.x == 0 && placed) atomicAdd((unsigned long long*)&placed_all, (unsigned long long)placed);
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    a.status[0] = (int)min(total_t, kIntMax);
    a.status[1] = (int)min(total_n - placed_all, kIntMax);
  }
  const int64_t stride = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + tid;
  for (int64_t b = first; b <= n; b += stride) {
    a.starts[b] = row0[b];
    if (b < n)
      a.seq_lens[b] = (int)min(length_at(a.context, a.context_wide, (int)b) + length_at(a.fresh, a.fresh_wide, (int)b),
                               kIntMax);
  }
  // taken pages: entry e of the free list goes to its request's next column
  for (int64_t e = first; e < min(total_t, kIntMax); e += stride) {
    const int b = last_at_most(page0, n, (int)e);
    const int64_t c = length_at(a.context, a.context_wide, b);
    const int64_t col = (c + bs - 1) / bs + (e - page0[b]);
    if (col < a.width) a.table[(int64_t)b * a.width + col] = e < a.n_free ? a.free_blocks[e] : -1;
  }
  for (int64_t i = first; i < a.tokens; i += stride) {
    int64_t slot = -1, pos = 0;
    if (i < min(total_n, kIntMax)) {
      const int b = last_at_most(row0, n, (int)i);
      const int64_t c = length_at(a.context, a.context_wide, b);
      pos = c + (i - row0[b]);
      const int64_t col = pos / bs, held = (c + bs - 1) / bs;
      if (col < a.width) {
        const int64_t e = page0[b] + (col - held);
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
                   n_free <= kIntMax && tokens <= kIntMax,
               "smaq_page_step: bad sizes (block_size %d, max_blocks %d, %lld free, %lld tokens)", block_size,
               max_blocks, n_free, tokens);
  SMAQ_REQUIRE((context_bytes == 4 || context_bytes == 8) && (new_bytes == 4 || new_bytes == 8),
               "smaq_page_step: lengths of %d and %d bytes", context_bytes, new_bytes);
  SMAQ_REQUIRE((!requests || (context_lens && new_lens && seq_lens)) && (!requests || !max_blocks || block_table) &&
                   (!n_free || free_blocks) && (!tokens || (slot_mapping && positions)) && query_start_loc && status,
               "smaq_page_step: null pointer");
  PageArgs a{context_lens, new_lens, context_bytes == 8, new_bytes == 8, requests, block_table, max_blocks,
             free_blocks, n_free, block_size, tokens, slot_mapping, positions, query_start_loc, seq_lens, status};
  // four tokens a thread while there are many; one workgroup each 256 otherwise
  const int64_t groups = std::min<int64_t>(std::max<int64_t>((tokens + kThreads - 1) / kThreads, (requests + 255) / 256 + 1), 256);
  const size_t bytes = 2 * sizeof(int) * (size_t)(requests + 1);
  page_step_kernel<<<(unsigned)std::max<int64_t>(groups, 1), kThreads, bytes, (hipStream_t)stream>>>(a);
  return launch_status("smaq_page_step");
}
