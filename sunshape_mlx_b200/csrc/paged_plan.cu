// Block tables and slot maps of ragged requests, built on the GPU from the
// requests' lengths, so that a serving loop never reads lengths back.
//
// plan: with P(x) = ceil(x / page_size), request b (len_b tokens held, q_b new
// ones) needs need_b = P(len_b + q_b) - P(len_b) pages. With the exclusive
// scan off_b of need, its i-th new page is
//   table[b][P(len_b) + i] = free[n_free - 1 - off_b - i]
// and the new token at position p of request b goes to slot
//   table[b][p / page_size] * page_size + p % page_size.
// Both are functions of the inputs alone: the lengths and the count of free
// pages are not updated in place but written to new arrays, so no CTA waits
// for another and a repeated call gives the same result.
//
// A launch writes a few KB to a MB, so latency is all: one launch, in which every
// CTA scans all requests' needs by itself (two ints each, read from L2) rather
// than wait for a first kernel's sums. 64 requests 4.0 us, 1500 requests with
// prompt chunks 7.2 us (graph replays), of which an empty kernel is 2.5; through the
// API 10 us either way.
#include "common.cuh"

namespace ss {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 16384;  // two ints of shared memory each

// Exclusive block scan of (a, b) over the CTA's threads; the totals are returned in ta, tb.
__device__ void scan2(int64_t& a, int64_t& b, int64_t& ta, int64_t& tb) {
  __shared__ int64_t wa[kPlanThreads / 32], wb[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t px = __shfl_up_sync(0xffffffffu, x, o), py = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) { x += px; y += py; }
  }
  __syncthreads();
  if (lane == 31) { wa[warp] = x; wb[warp] = y; }
  __syncthreads();
  int64_t ba = 0, bb = 0;
  ta = tb = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w == warp) { ba = ta; bb = tb; }
    ta += wa[w];
    tb += wb[w];
  }
  a = ba + x - a;
  b = bb + y - b;
}

// Largest i in [0, n) with v[i] <= x (v ascending, v[0] <= x).
__device__ __forceinline__ int upper(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

struct PlanParams {
  const int32_t *seq_lens, *q_lens;
  int n;
  int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* free_pages;
  int n_pages;
  const int32_t* n_free;
  int page;
  int64_t n_tokens;
  int32_t *cu_q, *positions, *requests, *new_lens, *new_free, *status;
  int64_t* slots;
};

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanParams p) {
  extern __shared__ int sm[];
  int* s_cu = sm;        // [n] first token of each request
  int* s_off = sm + p.n; // [n] first new page of each request
  const int tid = threadIdx.x;
  const int per = (p.n + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(p.n, tid * per), b1 = min(p.n, b0 + per);
  int64_t q = 0, need = 0;
  int bad = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = max(p.seq_lens[b], 0), nq = max(p.q_lens[b], 0);
    const int64_t want = ((int64_t)len + nq + p.page - 1) / p.page;
    if (want > p.width) bad |= 2;
    if ((int64_t)len + nq > 0x7fffffff) bad |= 4;
    q += nq;
    need += want - (len + (int64_t)p.page - 1) / p.page;
  }
  int64_t tq, tneed;
  scan2(q, need, tq, tneed);
  const int nfree = min(max(p.n_free[0], 0), p.n_pages);
  if (tneed > nfree) bad |= 1;
  if (tq > p.n_tokens) bad |= 4;
  bad = __syncthreads_or(bad & 1) | (__syncthreads_or(bad & 2) ? 2 : 0) |
        (__syncthreads_or(bad & 4) ? 4 : 0);
  // all or nothing: a step that does not fit changes nothing and maps no token
  if (!bad) {
    for (int b = b0; b < b1; ++b) {
      const int len = max(p.seq_lens[b], 0), nq = max(p.q_lens[b], 0);
      s_cu[b] = (int)q;
      s_off[b] = (int)need;
      q += nq;
      need += ((int64_t)len + nq + p.page - 1) / p.page - (len + (int64_t)p.page - 1) / p.page;
    }
  }
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * kPlanThreads, first = (int64_t)blockIdx.x * kPlanThreads + tid;
  for (int64_t b = first; b < p.n; b += step) {
    p.cu_q[b] = bad ? 0 : s_cu[b];
    p.new_lens[b] = max(p.seq_lens[b], 0) + (bad ? 0 : max(p.q_lens[b], 0));
  }
  if (first == 0) {
    p.cu_q[p.n] = bad ? 0 : (int)tq;
    p.new_free[0] = bad ? nfree : nfree - (int)tneed;
    p.status[0] = bad;
  }
  if (!bad) {
    for (int64_t e = first; e < tneed; e += step) {  // new table entries
      const int b = upper(s_off, p.n, (int)e);
      const int held = (int)(((int64_t)max(p.seq_lens[b], 0) + p.page - 1) / p.page);
      p.table[b * p.table_stride + held + (e - s_off[b])] = p.free_pages[nfree - 1 - e];
    }
  }
  for (int64_t t = first; t < p.n_tokens; t += step) {
    int pos = 0, req = -1;
    int64_t slot = -1;
    if (!bad && t < tq) {
      req = upper(s_cu, p.n, (int)t);
      const int len = max(p.seq_lens[req], 0);
      pos = len + (int)(t - s_cu[req]);
      const int j = pos / p.page, held = (int)(((int64_t)len + p.page - 1) / p.page);
      const int page = j < held ? p.table[req * p.table_stride + j]
                                : p.free_pages[nfree - 1 - (s_off[req] + j - held)];
      if (page >= 0 && page < p.n_pages) slot = (int64_t)page * p.page + pos % p.page;
    }
    p.positions[t] = pos;
    p.requests[t] = req;
    p.slots[t] = slot;
  }
}

struct ReleaseParams {
  const int32_t* seq_lens;
  const uint8_t* done;
  int n;
  int32_t* table;
  int64_t table_stride;
  int width;
  int32_t* free_pages;
  int n_pages;
  const int32_t* n_free;
  int page;
  int32_t *new_lens, *new_free, *status;
};

// Pages of finished requests go back on the stack, in the order of the requests and of their tables.
__global__ void __launch_bounds__(kPlanThreads) release_kernel(ReleaseParams p) {
  extern __shared__ int sm[];
  int* s_off = sm;
  const int tid = threadIdx.x;
  const int per = (p.n + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(p.n, tid * per), b1 = min(p.n, b0 + per);
  auto held = [&](int b) {
    return p.done[b] ? min(p.width, (int)(((int64_t)max(p.seq_lens[b], 0) + p.page - 1) / p.page)) : 0;
  };
  int64_t pages = 0, none = 0, total, t2;
  for (int b = b0; b < b1; ++b) pages += held(b);
  scan2(pages, none, total, t2);
  const int nfree = min(max(p.n_free[0], 0), p.n_pages);
  const bool bad = total > p.n_pages - nfree;  // more pages than are out: nothing changes
  if (!bad) {
    for (int b = b0; b < b1; ++b) {
      s_off[b] = (int)pages;
      pages += held(b);
    }
  }
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * kPlanThreads, first = (int64_t)blockIdx.x * kPlanThreads + tid;
  for (int64_t b = first; b < p.n; b += step)
    p.new_lens[b] = (p.done[b] && !bad) ? 0 : max(p.seq_lens[b], 0);
  if (first == 0) {
    p.new_free[0] = bad ? nfree : nfree + (int)total;
    p.status[0] = bad ? 8 : 0;
  }
  if (bad) return;
  for (int64_t e = first; e < total; e += step) {
    const int b = upper(s_off, p.n, (int)e);
    int32_t* at = p.table + b * p.table_stride + (e - s_off[b]);
    p.free_pages[nfree + e] = *at;
    *at = -1;
  }
}

int plan_grid(int64_t items) {
  const int64_t want = (items + kPlanThreads - 1) / kPlanThreads;
  return (int)(want < 1 ? 1 : want > sm_count() ? sm_count() : want);
}

}  // namespace
}  // namespace ss

using namespace ss;

extern "C" {

int ss_plan_step(const int32_t* seq_lens, const int32_t* q_lens, int n, int32_t* block_table,
                 int64_t table_stride, int width, const int32_t* free_pages, int n_pages,
                 const int32_t* n_free, int page_size, int64_t n_tokens, int32_t* cu_q,
                 int32_t* positions, int32_t* requests, int64_t* slots, int32_t* new_lens,
                 int32_t* new_free, int32_t* status, void* stream) {
  return c_entry([&]() -> int {
    SS_REQUIRE(seq_lens && q_lens && block_table && free_pages && n_free && cu_q && new_lens &&
                   new_free && status && (n_tokens == 0 || (positions && requests && slots)),
               "ss_plan_step: null pointer");
    SS_REQUIRE(n >= 1 && n <= kPlanMaxRequests, "ss_plan_step: 1 to 16384 requests");
    SS_REQUIRE(width >= 1 && table_stride >= width && n_pages >= 1, "ss_plan_step: bad table or pool");
    SS_REQUIRE(page_size >= 16 && page_size % 16 == 0, "ss_plan_step: page_size must be a multiple of 16");
    SS_REQUIRE(n_tokens >= 0 && n_tokens <= 0x7fffffff, "ss_plan_step: bad n_tokens");
    count_dispatch("ss_plan_step");
    PlanParams p{seq_lens, q_lens, n, block_table, table_stride, width, free_pages, n_pages, n_free,
                 page_size, n_tokens, cu_q, positions, requests, new_lens, new_free, status, slots};
    const size_t smem = (size_t)n * 8;
    if (smem > 48 * 1024)
      cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    plan_kernel<<<plan_grid(n_tokens > n ? n_tokens : n), kPlanThreads, smem, as_stream(stream)>>>(p);
    return check_launch("ss_plan_step");
  });
}

int ss_release_pages(const int32_t* seq_lens, const uint8_t* done, int n, int32_t* block_table,
                     int64_t table_stride, int width, int32_t* free_pages, int n_pages,
                     const int32_t* n_free, int page_size, int32_t* new_lens, int32_t* new_free,
                     int32_t* status, void* stream) {
  return c_entry([&]() -> int {
    SS_REQUIRE(seq_lens && done && block_table && free_pages && n_free && new_lens && new_free && status,
               "ss_release_pages: null pointer");
    SS_REQUIRE(n >= 1 && n <= kPlanMaxRequests, "ss_release_pages: 1 to 16384 requests");
    SS_REQUIRE(width >= 1 && table_stride >= width && n_pages >= 1, "ss_release_pages: bad table or pool");
    SS_REQUIRE(page_size >= 16 && page_size % 16 == 0, "ss_release_pages: page_size must be a multiple of 16");
    count_dispatch("ss_release_pages");
    ReleaseParams p{seq_lens, done, n, block_table, table_stride, width, free_pages, n_pages, n_free,
                    page_size, new_lens, new_free, status};
    const size_t smem = (size_t)n * 4;
    if (smem > 48 * 1024)
      cudaFuncSetAttribute(release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    release_kernel<<<plan_grid((int64_t)n * 8), kPlanThreads, smem, as_stream(stream)>>>(p);
    return check_launch("ss_release_pages");
  });
}

}  // extern "C"
