// Tables of one serving step from the request lengths (sm_100a).
//
// Request r has c_r tokens in its cache's semantic numbering, n_r new ones and
// o_r tokens removed by compression.  With start[r] = n_0 + .. + n_{r-1}, token
// t = start[r] + j sits at semantic position c_r + j (what RoPE takes) and at
// physical position c_r + j - o_r (where its K/V goes and what attention
// counts), P = 128 * blocks_per_page tokens to a scheduler page:
//     slot[t] = pages[r][phys / P] * P + phys % P
//     blocks[r][i] = pages[r][i / bpp] * bpp + i % bpp      (i * 128 < length)
//
// Bound: launch latency.  The data is some tens of KB (20 bytes a token, 4 a
// block), under a tenth of a microsecond of HBM time, so the whole step is one
// launch and no CTA waits for another: every token CTA repeats the prefix sum
// of the R new-token counts in shared memory (R loads that hit L2) instead of
// a scan kernel before it, and block CTAs need no prefix sum at all.  Larger
// steps only add CTAs.  Measured: 6 us alone for 4 requests or for 96 with 9,000
// new tokens and 16 blocks to a page, 3 us behind another kernel; the call from
// Python is bound by the host (19 us).
#include <algorithm>

#include "kvc_common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 8192;  // prefix sums of a CTA: 32 KB of shared memory

struct Ints {  // an int32 or int64 array
  const void* p;
  int bytes;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return bytes == 4 ? (int64_t)__ldg(static_cast<const int32_t*>(p) + i)
                      : __ldg(static_cast<const long long*>(p) + i);
  }
};

struct TablesArgs {
  Ints computed, scheduled, pages;
  const int64_t* offsets;  // or null
  int64_t page_stride;     // elements between rows of `pages`
  int page_width;
  int R, bpp, max_blocks;
  int64_t num_tokens;
  int32_t* query_start;
  int32_t* seq_lens;
  int64_t* positions;
  int64_t* slots;
  int32_t* request;
  int32_t* blocks;
  int32_t* error_flag;
  int token_ctas;
};

// new tokens of request r (a negative count is an error and counts as none)
__device__ __forceinline__ int new_tokens(const TablesArgs& a, int r) {
  const int64_t n = a.scheduled[r];
  if (n < 0 || n > INT32_MAX) {
    kvc::raise_flag(a.error_flag, KVC_DEV_TOKEN_RANGE);
    return 0;
  }
  return (int)n;
}

__device__ __forceinline__ int64_t physical_length(const TablesArgs& a, int r) {
  const int64_t n = a.computed[r] + new_tokens(a, r) - (a.offsets ? __ldg(a.offsets + r) : 0);
  if (n < 0 || n > INT32_MAX) {
    kvc::raise_flag(a.error_flag, KVC_DEV_TOKEN_RANGE);
    return 0;
  }
  return n;
}

__global__ void __launch_bounds__(kThreads) step_tables_kernel(const TablesArgs a) {
  kvc::pdl_wait();
  kvc::pdl_trigger();
  extern __shared__ int32_t start[];  // [R + 1] (token CTAs)
  __shared__ int64_t warp_total[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if ((int)blockIdx.x >= a.token_ctas) {
    // ---- block table: one entry per thread ----
    const int64_t i = (int64_t)(blockIdx.x - a.token_ctas) * kThreads + tid;
    if (i >= (int64_t)a.R * a.max_blocks) return;
    const int r = (int)(i / a.max_blocks), b = (int)(i % a.max_blocks);
    const int64_t len = physical_length(a, r);
    int64_t id = -1;
    if ((int64_t)b * kvc::kBlock < len) {
      const int page = b / a.bpp;
      if (page < a.page_width) id = a.pages[r * a.page_stride + page];
      id = id < 0 || id > INT32_MAX ? -1 : id * a.bpp + b % a.bpp;  // below 2^62
      if (id < 0 || id > INT32_MAX) {
        kvc::raise_flag(a.error_flag, KVC_DEV_BLOCK_RANGE);
        id = -1;
      }
    }
    a.blocks[i] = (int32_t)id;
    if (b == 0 && len > (int64_t)a.max_blocks * kvc::kBlock) kvc::raise_flag(a.error_flag, KVC_DEV_BLOCK_RANGE);
    return;
  }

  // ---- prefix sums of the new tokens ----
  // In 64 bits: counts may add up to more than an int32.  Starts past one are kept as INT32_MAX, which no token
  // reaches, so that they stay in order.
  int64_t carry = 0;
  for (int r0 = 0; r0 < a.R; r0 += kThreads) {
    const int r = r0 + tid;
    const int n = r < a.R ? new_tokens(a, r) : 0;
    int64_t v = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_total[warp] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const int64_t t = warp_total[w];
      if (w < warp) before += t;
      all += t;
    }
    if (r < a.R) start[r] = (int32_t)kvc::min64(carry + before + v - n, INT32_MAX);
    carry += all;
    __syncthreads();
  }
  if (tid == 0) start[a.R] = (int32_t)kvc::min64(carry, INT32_MAX);
  __syncthreads();
  const int64_t total = carry;
  if (blockIdx.x == 0) {
    for (int r = tid; r <= a.R; r += kThreads) a.query_start[r] = start[r];
    for (int r = tid; r < a.R; r += kThreads) a.seq_lens[r] = (int32_t)physical_length(a, r);
    if (tid == 0 && total > a.num_tokens) kvc::raise_flag(a.error_flag, KVC_DEV_TOKEN_RANGE);
  }

  // ---- one token per thread ----
  const int64_t page_tokens = (int64_t)kvc::kBlock * a.bpp;
  const int64_t last_page = INT64_MAX / page_tokens - 1;  // whose slots are within 64 bits
  for (int64_t t = (int64_t)blockIdx.x * kThreads + tid; t < a.num_tokens; t += (int64_t)a.token_ctas * kThreads) {
    if (t >= total) {  // padding of a captured step: no request, no slot
      a.positions[t] = 0;
      a.slots[t] = -1;
      a.request[t] = -1;
      continue;
    }
    int lo = 0, hi = a.R - 1;  // the last request that starts at or before t (empty requests start where the next does)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= t) lo = mid; else hi = mid - 1;
    }
    const int64_t pos = a.computed[lo] + (t - start[lo]);
    const int64_t phys = pos - (a.offsets ? __ldg(a.offsets + lo) : 0);
    int64_t slot = -1;
    const int64_t page = phys / page_tokens;
    if (phys < 0) {
      kvc::raise_flag(a.error_flag, KVC_DEV_TOKEN_RANGE);
    } else {
      const int64_t id = page < a.page_width ? a.pages[lo * a.page_stride + page] : -1;
      if (id < 0 || id > last_page) kvc::raise_flag(a.error_flag, KVC_DEV_BLOCK_RANGE);
      else slot = id * page_tokens + (phys - page * page_tokens);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
    a.request[t] = lo;
  }
}

struct Range {
  const void* p;
  int64_t bytes;
};

bool overlap(const Range& a, const Range& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}

}  // namespace

extern "C" int kvc_step_tables(const void* computed, int computed_bytes, const void* scheduled, int scheduled_bytes,
                               const int64_t* offsets, int num_requests, const void* page_table, int page_bytes,
                               int64_t page_stride, int page_width, int blocks_per_page, int64_t num_tokens,
                               int max_blocks, int32_t* query_start_loc, int32_t* seq_lens, int64_t* positions,
                               int64_t* slot_mapping, int32_t* request_indices, int32_t* block_table,
                               int32_t* error_flag, void* stream) {
  KVC_CHECK_ARG(computed && scheduled && page_table && query_start_loc && seq_lens, KVC_ENULL);
  KVC_CHECK_ARG(num_tokens == 0 || (positions && slot_mapping && request_indices), KVC_ENULL);
  KVC_CHECK_ARG(max_blocks == 0 || block_table, KVC_ENULL);
  KVC_CHECK_ARG(num_requests > 0 && num_tokens >= 0 && max_blocks >= 0 && page_width > 0 && blocks_per_page > 0 &&
                    page_stride >= 0 && num_tokens <= INT32_MAX,
                KVC_EINVAL);
  KVC_CHECK_ARG((computed_bytes == 4 || computed_bytes == 8) && (scheduled_bytes == 4 || scheduled_bytes == 8) &&
                    (page_bytes == 4 || page_bytes == 8),
                KVC_EINVAL);
  KVC_CHECK_ARG(num_requests <= kMaxRequests, KVC_EUNSUPPORTED);
  // CTAs read the inputs while others write tables: lengths of an earlier call, say, cannot be both
  const int64_t R = num_requests, N = num_tokens;
  const Range read[] = {{computed, R * computed_bytes},
                        {scheduled, R * scheduled_bytes},
                        {offsets, offsets ? 8 * R : 0},
                        {page_table, ((R - 1) * page_stride + page_width) * page_bytes}};
  const Range written[] = {{query_start_loc, 4 * (R + 1)}, {seq_lens, 4 * R},        {positions, 8 * N},
                           {slot_mapping, 8 * N},          {request_indices, 4 * N}, {block_table, 4 * R * max_blocks}};
  for (const Range& w : written) {
    for (const Range& r : read) KVC_CHECK_ARG(!overlap(w, r), KVC_EINVAL);
    for (const Range& o : written) KVC_CHECK_ARG(&o == &w || !overlap(w, o), KVC_EINVAL);
  }
  TablesArgs a{};
  a.computed = {computed, computed_bytes};
  a.scheduled = {scheduled, scheduled_bytes};
  a.pages = {page_table, page_bytes};
  a.offsets = offsets;
  a.page_stride = page_stride;
  a.page_width = page_width;
  a.R = num_requests;
  a.bpp = blocks_per_page;
  a.max_blocks = max_blocks;
  a.num_tokens = num_tokens;
  a.query_start = query_start_loc;
  a.seq_lens = seq_lens;
  a.positions = positions;
  a.slots = slot_mapping;
  a.request = request_indices;
  a.blocks = block_table;
  a.error_flag = error_flag;
  // one token per thread up to two CTAs per SM, then a stride: more CTAs would only repeat the prefix sums
  a.token_ctas = (int)std::max<int64_t>(1, std::min<int64_t>(2 * kvc::sm_count(), (num_tokens + kThreads - 1) / kThreads));
  const int64_t block_ctas = ((int64_t)num_requests * max_blocks + kThreads - 1) / kThreads;
  KVC_CHECK_ARG(block_ctas + a.token_ctas <= INT32_MAX, KVC_EINVAL);
  kvc::launch_dep(step_tables_kernel, dim3((unsigned)(a.token_ctas + block_ctas)), dim3(kThreads),
                  sizeof(int32_t) * (num_requests + 1), (cudaStream_t)stream, a);
  return kvc::launch_status();
}
