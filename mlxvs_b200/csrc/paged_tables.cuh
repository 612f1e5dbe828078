// Page tables and slot maps of one step, from the requests' lengths.
//
// A request that holds `past` tokens and gets `fresh` more owns the pages
// b0 = ceil(past / P) so far and needs b1 = min(ceil((past + fresh) / P), W);
// the free list's pages are handed out in request order, so page b0 + i of a
// request is free[off + i] with off the exclusive prefix sum of b1 - b0.
// Lengths or sums of 2^31 and more (which the caller rules out) give wrong tokens,
// but no place outside the table or the free list is read or written for them.
// Everything a token needs follows from (past, first token, off) of its
// request, so blocks share nothing: each one scans all requests (8 bytes a
// request, from L2) and keeps those that its own range of tokens meets.  One
// launch; the work is 16 bytes written per token.
//
// Bound: the latency of lengths -> sums -> pages -> slots, and for prompts the
// instructions of each token's search and division (issue slots 52 % busy).  64
// requests with a token each take 3.1 us; 1,000 requests with 665,693 new tokens
// 8.6 us (1.2 TB/s; the floor at the copy rate is 1.6 us, at a launch's latency 3).
#pragma once

#include "paged_common.cuh"

namespace mlxvs_b200 {

constexpr int TABLES_THREADS = 256;
constexpr int TABLES_TOKENS = 2048;  // tokens of one block
constexpr int TABLES_UNROLL = 4;     // tokens of one thread at a time

struct TablesParams {
  const int32_t *past, *fresh;
  int64_t requests;
  FastDiv page;
  const int32_t* free_pages;
  int64_t num_free;
  int32_t* table;
  int64_t width, num_tokens;
  int32_t *starts, *token_requests, *lengths;
  int64_t* slots;
  int32_t* used;
};

// Inclusive sums of three values over a block's threads; *total gets all.
__device__ __forceinline__ int3 block_scan3(int3 v, int3* warp_sums, int3* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(~0u, v.x, o), y = __shfl_up_sync(~0u, v.y, o),
              z = __shfl_up_sync(~0u, v.z, o);
    if (lane >= o) v.x += x, v.y += y, v.z += z;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int3 before = make_int3(0, 0, 0), all = make_int3(0, 0, 0);
#pragma unroll
  for (int w = 0; w < TABLES_THREADS / 32; ++w) {
    const int3 s = warp_sums[w];
    if (w < warp) before.x += s.x, before.y += s.y, before.z += s.z;
    all.x += s.x, all.y += s.y, all.z += s.z;
  }
  __syncthreads();
  *total = all;
  return make_int3(v.x + before.x, v.y + before.y, v.z + before.z);
}

// ITEMS: requests of one thread at a time.
template <int ITEMS>
__global__ void __launch_bounds__(TABLES_THREADS) paged_tables_kernel(const TablesParams p) {
  __shared__ int3 warp_sums[TABLES_THREADS / 32];
  __shared__ int4 met[TABLES_TOKENS];  // first token, past, request, page base
  __shared__ int lost_sum;
  const int t0 = (int)blockIdx.x * TABLES_TOKENS;
  const int t1 = min(t0 + TABLES_TOKENS, (int)p.num_tokens);
  const bool writer = blockIdx.x == 0;
  const int P = (int)p.page.d;
  const int width_tokens = (int)min((int64_t)INT32_MAX, p.width * P);
  if (threadIdx.x == 0) lost_sum = 0;
  __syncthreads();
  int2 base = make_int2(0, 0);  // tokens and pages of the requests before
  int count = 0;                // requests met so far
  for (int64_t r0 = 0; r0 < p.requests && (writer || base.x < t1);
       r0 += TABLES_THREADS * ITEMS) {
    // a few requests per thread, in order
    int past[ITEMS], fresh[ITEMS], need[ITEMS], b0[ITEMS];
    int3 mine = make_int3(0, 0, 0);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int64_t r = r0 + threadIdx.x * ITEMS + i;
      past[i] = fresh[i] = 0;
      if (r < p.requests) past[i] = max(p.past[r], 0), fresh[i] = max(p.fresh[r], 0);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      b0[i] = (int)p.page.div((uint32_t)past[i] + P - 1);
      const uint32_t end = min((uint32_t)past[i] + (uint32_t)fresh[i], (uint32_t)INT32_MAX);
      const int b1 = (int)min((int64_t)p.page.div(end + P - 1), p.width);
      need[i] = max(b1 - b0[i], 0);
      mine.x += fresh[i], mine.y += need[i];
    }
    int3 total;
    int3 sum = block_scan3(mine, warp_sums, &total);
    int start = base.x + sum.x - mine.x, off = base.y + sum.y - mine.y;
    const bool range_meets = base.x < t1 && base.x + total.x > t0;
    base.x += total.x, base.y += total.y;
    int at = count;
    uint32_t kept = 0;  // a bit for each request of the thread
    if (range_meets) {
      // some request of these may meet the block's tokens: keep those, in order
      int first = start;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        kept |= (uint32_t)(fresh[i] > 0 && first < t1 && first + fresh[i] > t0) << i;
        first += fresh[i];
      }
      const int meets = __popc(kept);
      sum = block_scan3(make_int3(meets, 0, 0), warp_sums, &total);
      at += sum.x - meets;
      count = min(count + total.x, TABLES_TOKENS);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int64_t r = r0 + threadIdx.x * ITEMS + i;
      if ((kept >> i & 1) && at < TABLES_TOKENS)
        met[at++] = make_int4(start, past[i], (int)r, off - b0[i]);
      if (writer && r < p.requests) {
        p.starts[r] = start;
        if (fresh[i] > 0) {
          // tokens that get no slot: past the table's width, past the end of
          // the free list, or in a begun page that the table does not hold
          const int64_t avail = max((int64_t)0, min((int64_t)need[i], p.num_free - off));
          const int64_t end = (int64_t)past[i] + fresh[i];
          const int64_t held = min(min(end, (b0[i] + avail) * P), (int64_t)width_tokens);
          int64_t lost = end - max(held, (int64_t)past[i]);
          const int begun = past[i] % P == 0 ? 0 : min(fresh[i], P - past[i] % P);
          if (begun > 0 && past[i] < width_tokens &&
              p.table[r * p.width + p.page.div(past[i])] < 0)
            lost += begun;
          if (lost > 0) atomicAdd(&lost_sum, (int)lost);
        }
      }
      start += fresh[i], off += need[i];
    }
  }
  __syncthreads();
  if (writer && threadIdx.x == 0) {
    p.starts[p.requests] = base.x;
    p.used[0] = base.y;
    p.used[1] = lost_sum;
  }
  for (int u0 = t0 + threadIdx.x; u0 < t1; u0 += TABLES_THREADS * TABLES_UNROLL) {
    int row[TABLES_UNROLL], length[TABLES_UNROLL], in[TABLES_UNROLL];
    int64_t entry[TABLES_UNROLL];  // of the table, to be filled (-1: none)
    int32_t page[TABLES_UNROLL];
#pragma unroll
    for (int u = 0; u < TABLES_UNROLL; ++u) {
      const int t = u0 + u * TABLES_THREADS;
      // the last request met that starts at or before t
      int lo = 0, hi = t < t1 ? count : 0;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (met[mid].x <= t) lo = mid + 1;
        else hi = mid;
      }
      row[u] = -1, length[u] = 0, page[u] = -1;
      if (t < t1 && t < base.x && lo > 0) {
        const int4 m = met[lo - 1];
        const uint32_t pos = (uint32_t)m.y + (uint32_t)t - (uint32_t)m.x;
        row[u] = m.z, length[u] = (int)min(pos, (uint32_t)INT32_MAX - 1) + 1;
        if (pos < (uint32_t)width_tokens) {
          const int b = (int)p.page.div(pos);
          in[u] = (int)pos - b * P;
          const bool fresh = b * P >= m.y;  // handed out in this step
          const int64_t place = (int64_t)m.z * p.width + b, listed = (int64_t)m.w + b;
          if (!fresh) page[u] = p.table[place];
          else if (listed >= 0 && listed < p.num_free) page[u] = p.free_pages[listed];
          entry[u] = fresh && in[u] == 0 ? place : -1;
        } else {
          in[u] = 0, entry[u] = -1;
        }
      } else {
        in[u] = 0, entry[u] = -1;
      }
    }
#pragma unroll
    for (int u = 0; u < TABLES_UNROLL; ++u) {
      const int t = u0 + u * TABLES_THREADS;
      if (t >= t1) break;
      if (entry[u] >= 0) p.table[entry[u]] = page[u];  // a new page's first token
      p.token_requests[t] = row[u];
      p.lengths[t] = length[u];
      p.slots[t] = page[u] >= 0 ? (int64_t)page[u] * P + in[u] : -1;
    }
  }
}

}  // namespace mlxvs_b200
