// Page selection: the n pages of its request that each new token and key
// head attends to.
//
// The score of a page is an estimate in 8 bits of the upper bound of q . key over
// its rows, summed over the query heads of the key head: with the page's bounds
// lo, hi and the parts q+ = max(q, 0), q- = min(q, 0),
//     q . key <= q+ . hi + q- . lo   for every key of the page.
// The query heads share one power of two that puts their largest magnitude in
// [64, 128); each is rounded to whole numbers of at most 127, the parts are
// summed over the heads and shifted right by ceil(log2 G), which leaves codes
// of at most 127: rounding to nearest and the shift can leave a score a little
// below the bound.  The dot products are whole numbers below 2^24
// (2 * 256 * 127 * 127 at the widest), the page's scale is a power of two, so
// a score is one exact float: it does not depend on the order of the sums,
// and ties (to the lower page) are real ties.
#pragma once

#include "common.cuh"
#include "paged_common.cuh"

namespace mlxvs_b200 {

struct SelectParams {
  const void* q;
  int64_t tokens, q_token, q_head;
  int heads, group, dim, shift;
  const int8_t* codes;
  const float* scales;
  int64_t pages;
  const int32_t* table;
  int64_t rows, width;
  const int32_t *requests, *lengths;
  FastDiv page;
  int n, first, last;
  int32_t* out;  // [tokens, heads, n]
};

constexpr int SELECT_WARPS = 8;
constexpr int SELECT_WARP_PAGES = 512;  // selected by one warp
constexpr int SELECT_CODES = 2 * 256;  // bytes of a token's query codes, at most

// d += a b: 16 x 32 by 32 x 8 signed bytes, 32-bit sums.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The threads that select for one token: a warp, or the whole block.
template <int WARPS>
__device__ __forceinline__ void select_sync() {
  if (WARPS == 1) __syncwarp();
  else __syncthreads();
}

// The n pages of the best keys (0: no page, 1: a score that is NaN, ~0: a forced
// page) of held pages, ascending, by WARPS warps.  The range of the keys is cut into 256 bins, then
// the bin that holds the n-th key again, until its count is taken whole or it
// is a single key (whose first pages are taken): two rounds for most rows, four
// at most.
template <int WARPS>
__device__ __forceinline__ void select_pages(const uint32_t* keys, int held, int n, int32_t* out,
                                             uint32_t* bins, uint32_t (*shared)[4]) {
  constexpr int THREADS = 32 * WARPS;
  constexpr uint32_t FORCED = 0xFFFFFFFFu;
  const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
  const int tid = warp * 32 + lane;
  // ---- range and counts
  uint32_t lo = FORCED, hi = 0, forced = 0, valid = 0;
#pragma unroll 4
  for (int b = tid; b < held; b += THREADS) {
    const uint32_t key = keys[b];
    forced += key == FORCED;
    if (key != 0 && key != FORCED) lo = min(lo, key), hi = max(hi, key), ++valid;
  }
  lo = __reduce_min_sync(~0u, lo), hi = __reduce_max_sync(~0u, hi);
  forced = __reduce_add_sync(~0u, forced), valid = __reduce_add_sync(~0u, valid);
  if (WARPS > 1) {
    if (lane == 0)
      shared[warp][0] = lo, shared[warp][1] = hi, shared[warp][2] = forced, shared[warp][3] = valid;
    __syncthreads();
    lo = FORCED, hi = forced = valid = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      lo = min(lo, shared[w][0]), hi = max(hi, shared[w][1]);
      forced += shared[w][2], valid += shared[w][3];
    }
    __syncthreads();
  }
  // taken: keys above `limit`, and the first `equals` of those equal to it
  uint32_t limit = 0, equals = 0, need = (uint32_t)n - min((uint32_t)n, forced);
  if (need == 0) limit = FORCED, equals = n;
  while (valid > need && need > 0) {
    const int bits = 32 - __clz(hi - lo), shift = max(bits - 8, 0);
    for (int i = tid; i < 256; i += THREADS) bins[i] = 0;
    select_sync<WARPS>();
#pragma unroll 4
    for (int b = tid; b < held; b += THREADS) {
      const uint32_t key = keys[b];
      if (key >= lo && key <= hi) atomicAdd(&bins[(key - lo) >> shift], 1u);
    }
    select_sync<WARPS>();
    // lane l holds bins 255 - 8 l .. 248 - 8 l: down in keys (every warp alike)
    uint32_t count[8], mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine += count[i] = bins[255 - 8 * lane - i];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += y;
    }
    // the first lane whose count passes `need` (the bins hold more than that)
    const int owner = __ffs(__ballot_sync(~0u, upto >= need)) - 1;
    uint32_t above = upto - mine, bin = 0, in_bin = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bin = 255 - 8 * lane - i, in_bin = count[i];
      if (above + count[i] >= need) break;
      above += count[i];
    }
    bin = __shfl_sync(~0u, bin, owner), in_bin = __shfl_sync(~0u, in_bin, owner);
    need -= __shfl_sync(~0u, above, owner);
    lo += bin << shift;
    // the bin's end, which may lie past the largest 32-bit number (scores of over 1.7e38)
    const uint32_t width = (1u << shift) - 1;
    if (hi - lo > width) hi = lo + width;
    if (in_bin == need) {
      limit = lo - 1;  // lo > 0: keys of pages are
      break;
    }
    if (shift == 0) {
      limit = lo, equals = need;
      break;
    }
    valid = in_bin;
    select_sync<WARPS>();
  }
  // ---- out, in page order: each warp its share of the pages
  const int share = ((held + THREADS - 1) / THREADS) * 32;
  const int begin = warp * share, end = min(held, begin + share);
  uint32_t done = 0, before = 0;  // taken, and equal to the limit, so far
  if (WARPS > 1) {
    uint32_t above = 0, equal = 0;
    for (int b = begin + lane; b < end; b += 32) {
      const uint32_t key = keys[b];
      above += key > limit, equal += key == limit && key != 0;
    }
    above = __reduce_add_sync(~0u, above), equal = __reduce_add_sync(~0u, equal);
    if (lane == 0) shared[warp][0] = above, shared[warp][1] = equal;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) done += shared[w][0], before += shared[w][1];
      all += shared[w][0];
    }
    done += min(before, equals);
    uint32_t all_equal = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all_equal += shared[w][1];
    all += min(all_equal, equals);
    for (int i = (int)all + tid; i < n; i += THREADS) out[i] = -1;
  }
  for (int b0 = begin; b0 < end; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t key = b < end ? keys[b] : 0;
    const bool equal = key == limit && key != 0;
    const uint32_t eq = __ballot_sync(~0u, equal);
    const uint32_t place = before + __popc(eq & ((1u << lane) - 1));
    const bool take = key > limit || (equal && place < equals);
    const uint32_t tk = __ballot_sync(~0u, take);
    if (take) out[done + __popc(tk & ((1u << lane) - 1))] = b;
    done += __popc(tk), before += __popc(eq);
  }
  if (WARPS == 1)
    for (int i = (int)done + lane; i < n; i += 32) out[i] = -1;
}

// A cluster of blocks per TT tokens and key head.  The tensor cores score 16
// pages against up to 8 tokens at a time (page codes as the 16-row operand,
// read straight from global memory: the order of the channels is free, so a
// lane's 16 consecutive bytes serve four operand words).  The blocks of the
// cluster share the pages and put the keys into the first one's shared memory,
// where one warp per token, or the block for its only token, selects.
//
// Bound: the codes are read once per tile (once per token when TT is 1), the
// products are nearly free; what is left is the latency of table -> codes ->
// keys -> bins, and for prompts the instructions of the selection.  Both want
// many blocks per SM: fetching the codes a step ahead as well took 143
// registers and made prompts of 5,229 tokens slower (97 -> 144 us).  Now those
// take 56 us (8 to start, 18 for the query codes, 14 for the scores, 16 for the
// selection), 32 single tokens with up to 500 pages 11.5 us, and 7 with up to 3,900
// pages (27 MB of codes) 21.5 us, of which 9 for the scores and 8 for the selection.
//
// SEG: 64-byte segments of a page's codes (dim up to 32 SEG).
template <class T, int TT, int SEG>
__global__ void __launch_bounds__(SELECT_WARPS * 32, SEG == 8 ? 2 : 4) paged_select_kernel(const SelectParams p) {
  extern __shared__ uint32_t keys[];  // [TT][width] order bits of the scores, 0: no page
  __shared__ __align__(16) int8_t qc[TT][SELECT_CODES];  // q- then q+ codes
  __shared__ uint32_t hist[TT][256];
  __shared__ uint32_t counts[SELECT_WARPS][4];
  uint32_t rank, cluster;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster));
  const int64_t t0 = (int64_t)(blockIdx.x / cluster) * TT;
  const int h = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // ---- the tile's tokens, one per lane: row of the table and pages held
  int my_row = -1, my_held = 0;
  if (lane < TT && t0 + lane < p.tokens) {
    const int64_t t = t0 + lane;
    const int64_t row = p.requests ? p.requests[t] : t;
    if (row >= 0 && row < p.rows) {
      my_row = (int)row;
      my_held = min((int)p.page.div((uint32_t)max(p.lengths[t], 0) + p.page.d - 1), (int)p.width);
    }
  }
  const int bytes = 2 * p.dim;  // codes of a page
  const int stride = (int)cluster * SELECT_WARPS;

  // places of 16 pages' codes (rows lane / 4 and lane / 4 + 8 of the operand),
  // fetched one step ahead
  auto ids_of = [&](int row, int held, int g) {
    const int32_t* table = p.table + (int64_t)row * p.width;
    const int b = g * 16 + lane / 4;
    int2 id = make_int2(b < held ? table[b] : -1, b + 8 < held ? table[b + 8] : -1);
    if (id.x >= p.pages) id.x = -1;
    if (id.y >= p.pages) id.y = -1;
    return id;
  };
  // the tokens of one request together, in the order of their first ones
  uint32_t rest = __ballot_sync(~0u, my_held > 0);
  int row = -1, held = 0;
  auto next_request = [&] {
    row = __shfl_sync(~0u, my_row, __ffs(rest) - 1);
    rest &= ~__ballot_sync(~0u, my_row == row);
    held = __reduce_max_sync(~0u, my_row == row ? my_held : 0);
  };
  const int g0 = (int)rank * SELECT_WARPS + warp;
  int2 next_ids = make_int2(-1, -1);
  if (rest != 0) {
    next_request();
    next_ids = ids_of(row, held, g0);
  }
  if (TT == 1 && warp > 0 && row >= 0)
    // the warps that make no query codes fetch their first pages' codes to L2
    for (int i = 128 * (lane & 1); i < bytes; i += 256) {
      const int64_t at = (int64_t)((lane & 2) ? next_ids.y : next_ids.x) * p.heads + h;
      if (at >= 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.codes + at * bytes + i));
    }

  // ---- query codes, one warp per token: LANES lanes of eight channels, the
  // other lanes of the warp take other heads
  if (warp < TT) {
    for (int i = lane; i < SELECT_CODES / 4; i += 32)
      reinterpret_cast<uint32_t*>(qc[warp])[i] = 0;
    __syncwarp();
    if (__shfl_sync(~0u, my_held, warp) > 0) {
      const int64_t t = t0 + warp;
      const int lanes = p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32;
      const int c = (lane & (lanes - 1)) * 8, step = 32 / lanes;
      const bool mine = c < p.dim;
      const T* q = static_cast<const T*>(p.q) + t * p.q_token + (int64_t)h * p.group * p.q_head + c;
      // the first heads' values stay in registers between the two passes
      constexpr int HELD = 4;
      uint4 first[HELD];
#pragma unroll
      for (int u = 0; u < HELD; ++u) {
        const int g = lane / lanes + u * step;
        first[u] = mine && g < p.group ? *reinterpret_cast<const uint4*>(q + g * p.q_head)
                                       : make_uint4(0, 0, 0, 0);
      }
      float top = 0.0f;
      auto measure = [&](const uint4& x) {
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(to_float(e[i])));
      };
#pragma unroll
      for (int u = 0; u < HELD; ++u) measure(first[u]);
      if (mine)
        for (int g = lane / lanes + HELD * step; g < p.group; g += step)
          measure(*reinterpret_cast<const uint4*>(q + g * p.q_head));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      const float by = exp2_int(code_exponent(top));
      // sums of the rounded values and of their magnitudes: whole numbers of
      // at most 128 * 127, exact as floats
      float sum[8], size[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = size[i] = 0.0f;
      auto add = [&](const uint4& x) {
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = to_float(e[i]) * by;
          // 1.5 * 2^23 added and taken off: rounded to nearest even
          const float r = fmaxf(-127.0f, fminf(127.0f, y)) + 12582912.0f - 12582912.0f;
          const float z = y == y ? r : 0.0f;
          sum[i] += z, size[i] += fabsf(z);
        }
      };
#pragma unroll
      for (int u = 0; u < HELD; ++u) add(first[u]);
      if (mine)
        for (int g = lane / lanes + HELD * step; g < p.group; g += step)
          add(*reinterpret_cast<const uint4*>(q + g * p.q_head));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        for (int o = lanes; o < 32; o <<= 1) {
          sum[i] += __shfl_xor_sync(~0u, sum[i], o);
          size[i] += __shfl_xor_sync(~0u, size[i], o);
        }
      if (mine && lane < lanes) {
        uint32_t down[2] = {0, 0}, up[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int u = (int)(size[i] + sum[i]) >> 1, d = (int)(size[i] - sum[i]) >> 1;
          down[i / 4] |= ((uint32_t)(-(d >> p.shift)) & 255u) << (8 * (i & 3));
          up[i / 4] |= (uint32_t)(u >> p.shift) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2*>(&qc[warp][c]) = make_uint2(down[0], down[1]);
        *reinterpret_cast<uint2*>(&qc[warp][p.dim + c]) = make_uint2(up[0], up[1]);
      }
    }
  }
  __syncthreads();

  // ---- scores
  const uint32_t my_keys = (uint32_t)__cvta_generic_to_shared(keys);
  uint32_t first_keys;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first_keys) : "r"(my_keys));
  if (cluster > 1)  // every block of the cluster has started before any writes there
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
  uint4 b[SEG];  // the column's query codes: token lane / 4
#pragma unroll
  for (int i = 0; i < SEG; ++i)
    b[i] = lane / 4 < TT
               ? *reinterpret_cast<const uint4*>(
                     &qc[TT == 1 ? 0 : lane / 4][64 * i + 16 * (lane & 3)])
               : make_uint4(0, 0, 0, 0);
  // this lane's two tokens of a result
  const int w0 = 2 * (lane & 3);
  const int row_w[2] = {__shfl_sync(~0u, my_row, w0), __shfl_sync(~0u, my_row, w0 + 1)};
  const int held_w[2] = {__shfl_sync(~0u, my_held, w0), __shfl_sync(~0u, my_held, w0 + 1)};
  while (row >= 0) {
    const int groups = (held + 15) / 16;
    for (int g = g0; g < groups; g += stride) {
      const int b0 = g * 16 + lane / 4, b1 = b0 + 8;
      const int2 id = next_ids;
      next_ids = ids_of(row, held, g + stride);
      const int64_t at0 = (int64_t)id.x * p.heads + h, at1 = (int64_t)id.y * p.heads + h;
      const int8_t* c0 = p.codes + at0 * bytes + 16 * (lane & 3);
      const int8_t* c1 = p.codes + at1 * bytes + 16 * (lane & 3);
      const float scale0 = id.x >= 0 ? p.scales[at0] : 0.0f;
      const float scale1 = id.y >= 0 ? p.scales[at1] : 0.0f;
      int dot[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < SEG; ++i) {
        const bool in = 64 * i + 16 * (lane & 3) < bytes;
        const uint4 x = in && id.x >= 0 ? *reinterpret_cast<const uint4*>(c0 + 64 * i)
                                        : make_uint4(0, 0, 0, 0);
        const uint4 y = in && id.y >= 0 ? *reinterpret_cast<const uint4*>(c1 + 64 * i)
                                        : make_uint4(0, 0, 0, 0);
        mma_s8(dot, x.x, y.x, x.y, y.y, b[i].x, b[i].y);
        mma_s8(dot, x.z, y.z, x.w, y.w, b[i].z, b[i].w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (TT == 1 && (i & 1)) continue;
        const int w = w0 + (i & 1);  // token of the result
        const int page = i < 2 ? b0 : b1;
        if (w >= TT || row_w[i & 1] != row || page >= held_w[i & 1]) continue;
        uint32_t key = 0;
        if ((i < 2 ? id.x : id.y) >= 0) {
          // + 0.0f: a zero score has one form.  A NaN score (a scale that is not a
          // number, or an infinite one times zero) comes after all others: by its
          // bits it would be a forced page, of which there may be no more than n.
          const float score = (float)dot[i] * (i < 2 ? scale0 : scale1) + 0.0f;
          key = page < p.first || page >= held_w[i & 1] - p.last ? 0xFFFFFFFFu
                : score == score                                 ? order_bits(score)
                                                                 : 1u;
        }
        const uint32_t at = (uint32_t)(w * p.width + page);
        if (cluster > 1)
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(first_keys + 4 * at), "r"(key)
                       : "memory");
        else
          keys[at] = key;
      }
    }
    if (rest == 0) break;
    next_request();
    next_ids = ids_of(row, held, g0);
  }
  if (cluster > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
  else
    __syncthreads();
  if (rank != 0) return;
  if (TT == 1) {
    // few pages: one warp is quicker than a block's barriers (32 tokens with up
    // to 500 pages 12.2 -> 11.3 us; up to 2048 pages it makes no difference)
    const int mine = __shfl_sync(~0u, my_held, 0);
    int32_t* out = p.out + (t0 * p.heads + h) * p.n;
    if (mine > SELECT_WARP_PAGES)
      select_pages<SELECT_WARPS>(keys, mine, p.n, out, hist[0], counts);
    else if (warp == 0)
      select_pages<1>(keys, mine, p.n, out, hist[0], nullptr);
  } else if (warp < TT && t0 + warp < p.tokens) {
    select_pages<1>(keys + (int64_t)warp * p.width, __shfl_sync(~0u, my_held, warp), p.n,
                    p.out + ((t0 + warp) * p.heads + h) * p.n, hist[warp], nullptr);
  }
}

}  // namespace mlxvs_b200
