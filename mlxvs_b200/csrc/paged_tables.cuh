// Page tables and slot maps of one step, from the requests' lengths.
//
// A request that holds `past` tokens and gets `fresh` more owns the pages
// b0 = ceil(past / P) so far and needs b1 = min(ceil((past + fresh) / P), W);
// the free list's pages are handed out in request order, so page b0 + i of a
// request is free[off + i] with off the exclusive prefix sum of b1 - b0.
// Everything a token needs follows from (past, first token, off) of its
// request, so blocks share nothing: each one scans all requests (8 bytes a
// request, from L2) and keeps those that its own range of tokens meets.  One
// launch; the work is 16 bytes written per token.
#pragma once

#include "paged_common.cuh"

namespace mlxvs_b200 {

constexpr int TABLES_THREADS = 256;
constexpr int TABLES_TOKENS = 2048;  // tokens of one block

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
  for (int64_t r0 = 0; r0 < p.requests && (writer || base.x < t1); r0 += TABLES_THREADS) {
    const int64_t r = r0 + threadIdx.x;
    int past = 0, fresh = 0, need = 0, b0 = 0;
    if (r < p.requests) {
      past = max(p.past[r], 0);
      fresh = max(p.fresh[r], 0);
      b0 = (int)p.page.div((uint32_t)past + P - 1);
      const int b1 = min((int)p.page.div((uint32_t)past + fresh + P - 1), (int)p.width);
      need = max(b1 - b0, 0);
    }
    int3 total;
    int3 sum = block_scan3(make_int3(fresh, need, 0), warp_sums, &total);
    const int start = base.x + sum.x - fresh, off = base.y + sum.y - need;
    const bool range_meets = base.x < t1 && base.x + total.x > t0;
    base.x += total.x, base.y += total.y;
    if (range_meets) {
      // some request of these may meet the block's tokens: keep those, in order
      const int meets = fresh > 0 && start < t1 && start + fresh > t0;
      sum = block_scan3(make_int3(meets, 0, 0), warp_sums, &total);
      if (meets) met[count + sum.x - 1] = make_int4(start, past, (int)r, off - b0);
      count += total.x;
    }
    if (writer && r < p.requests) {
      p.starts[r] = start;
      if (fresh > 0) {
        // tokens that get no slot: past the table's width, past the end of
        // the free list, or in a begun page that the table does not hold
        const int64_t avail = max((int64_t)0, min((int64_t)need, p.num_free - off));
        const int end = past + fresh;
        const int64_t held = min(min((int64_t)end, (b0 + avail) * P), (int64_t)width_tokens);
        int64_t lost = end - max(held, (int64_t)min(past, end));
        const int begun = past % P == 0 ? 0 : min(fresh, P - past % P);
        if (begun > 0 && past < width_tokens &&
            p.table[r * p.width + p.page.div(past)] < 0)
          lost += begun;
        if (lost > 0) atomicAdd(&lost_sum, (int)lost);
      }
    }
  }
  __syncthreads();
  if (writer && threadIdx.x == 0) {
    p.starts[p.requests] = base.x;
    p.used[0] = base.y;
    p.used[1] = lost_sum;
  }
  for (int t = t0 + threadIdx.x; t < t1; t += TABLES_THREADS) {
    // the last request met that starts at or before t
    int lo = 0, hi = count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (met[mid].x <= t) lo = mid + 1;
      else hi = mid;
    }
    const int4 m = lo > 0 ? met[lo - 1] : make_int4(-1, 0, -1, 0);
    int length = 0;
    int64_t slot = -1;
    if (t < base.x && m.x >= 0) {
      const int pos = m.y + (t - m.x);
      length = pos + 1;
      if (pos < width_tokens) {
        const int b = (int)p.page.div(pos), in = pos - b * P;
        int32_t page;
        if (b * P >= m.y) {  // handed out in this step
          const int64_t i = (int64_t)m.w + b;
          page = i < p.num_free ? p.free_pages[i] : -1;
          if (in == 0) p.table[(int64_t)m.z * p.width + b] = page;
        } else {
          page = p.table[(int64_t)m.z * p.width + b];
        }
        if (page >= 0) slot = (int64_t)page * P + in;
      }
    }
    p.token_requests[t] = length > 0 ? m.z : -1;
    p.lengths[t] = length;
    p.slots[t] = slot;
  }
}

}  // namespace mlxvs_b200
