// Page selection: the n pages of its request that each new token and key
// head attends to.
//
// The score of a page is an upper bound of q . key over its rows, summed over
// the query heads of the key head, in 8 bits: with the page's bounds lo, hi
// and the parts q+ = max(q, 0), q- = min(q, 0),
//     q . key <= q+ . hi + q- . lo   for every key of the page.
// The query heads share one power of two that puts their largest magnitude in
// [64, 128); each is rounded to whole numbers of at most 127, the parts are
// summed over the heads and shifted right by ceil(log2 G), which leaves codes
// of at most 127.  The dot products are whole numbers below 2^24
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

// A cluster of blocks per TT tokens and key head.  The tensor cores score 16
// pages against up to 8 tokens at a time (page codes as the 16-row operand,
// read straight from global memory: the order of the channels is free, so a
// lane's 16 consecutive bytes serve four operand words).  The blocks of the
// cluster share the pages and put the keys into the first one's shared memory,
// where one warp per token selects: a radix selection of the n-th key in
// 8-bit digits, then one pass in page order.
//
// Bound: the codes are read once per tile (once per token when TT is 1), the
// products are nearly free; what is left is the latency of table -> codes ->
// keys -> four digits.
template <class T, int TT>
__global__ void __launch_bounds__(SELECT_WARPS * 32) paged_select_kernel(const SelectParams p) {
  extern __shared__ uint32_t keys[];  // [TT][width] order bits of the scores, 0: no page
  __shared__ __align__(16) int8_t qc[TT][SELECT_CODES];  // q- then q+ codes
  __shared__ uint32_t hist[TT][256];
  __shared__ int s_row[TT], s_held[TT];
  uint32_t rank, cluster;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster));
  const int64_t t0 = (int64_t)(blockIdx.x / cluster) * TT;
  const int h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // ---- query codes, one warp per token
  if (warp < TT) {
    const int64_t t = t0 + warp;
    int64_t row = t < p.tokens ? (p.requests ? p.requests[t] : t) : -1;
    int held = 0;
    if (row >= 0 && row < p.rows)
      held = min((int)p.page.div((uint32_t)max(p.lengths[t], 0) + p.page.d - 1), (int)p.width);
    else
      row = -1;
    if (lane == 0) s_row[warp] = (int)row, s_held[warp] = held;
    for (int i = lane; i < SELECT_CODES / 4; i += 32)
      reinterpret_cast<uint32_t*>(qc[warp])[i] = 0;
    __syncwarp();
    if (held > 0) {
      const T* q = static_cast<const T*>(p.q) + t * p.q_token + (int64_t)h * p.group * p.q_head;
      const bool mine = lane * 8 < p.dim;  // eight channels a lane
      float top = 0.0f;
      if (mine)
        for (int g = 0; g < p.group; ++g) {
          const uint4 x = *reinterpret_cast<const uint4*>(q + g * p.q_head + lane * 8);
          const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(to_float(e[i])));
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      const float by = exp2_int(code_exponent(top));
      if (mine) {
        int up[8] = {}, down[8] = {};
        for (int g = 0; g < p.group; ++g) {
          const uint4 x = *reinterpret_cast<const uint4*>(q + g * p.q_head + lane * 8);
          const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float y = to_float(e[i]) * by;
            const int c = y == y ? __float2int_rn(fmaxf(-127.0f, fminf(127.0f, y))) : 0;
            up[i] += max(c, 0), down[i] += max(-c, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          qc[warp][lane * 8 + i] = (int8_t)(-(down[i] >> p.shift));
          qc[warp][p.dim + lane * 8 + i] = (int8_t)(up[i] >> p.shift);
        }
      }
    }
  }
  __syncthreads();

  // ---- scores
  const int bytes = 2 * p.dim;  // codes of a page
  const int segments = (bytes + 63) / 64;
  const uint32_t my_keys = (uint32_t)__cvta_generic_to_shared(keys);
  uint32_t first_keys;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first_keys) : "r"(my_keys));
  if (cluster > 1)  // every block of the cluster has started before any writes there
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
  uint4 b[SELECT_CODES / 64];  // the column's query codes: token lane / 4
#pragma unroll
  for (int i = 0; i < SELECT_CODES / 64; ++i)
    b[i] = lane / 4 < TT ? *reinterpret_cast<const uint4*>(
                               &qc[TT == 1 ? 0 : lane / 4][64 * i + 16 * (lane & 3)])
                         : make_uint4(0, 0, 0, 0);
  for (int u = 0; u < TT; ++u) {
    // the tokens of one request together, at the first of them
    const int row = s_row[u];
    int held = s_held[u];
    if (TT > 1) {
      bool again = row < 0;
      for (int w = 0; w < u; ++w) again |= s_row[w] == row;
      if (again) continue;
      for (int w = u + 1; w < TT; ++w)
        if (s_row[w] == row) held = max(held, s_held[w]);
    } else if (row < 0) {
      continue;
    }
    const int32_t* table = p.table + (int64_t)row * p.width;
    const int groups = (held + 15) / 16;
    for (int g = rank * SELECT_WARPS + warp; g < groups; g += cluster * SELECT_WARPS) {
      const int b0 = g * 16 + lane / 4, b1 = b0 + 8;
      int32_t page0 = b0 < held ? table[b0] : -1, page1 = b1 < held ? table[b1] : -1;
      if (page0 >= p.pages) page0 = -1;
      if (page1 >= p.pages) page1 = -1;
      const int8_t* c0 = p.codes + ((int64_t)page0 * p.heads + h) * bytes + 16 * (lane & 3);
      const int8_t* c1 = p.codes + ((int64_t)page1 * p.heads + h) * bytes + 16 * (lane & 3);
      const float scale0 = page0 >= 0 ? p.scales[(int64_t)page0 * p.heads + h] : 0.0f;
      const float scale1 = page1 >= 0 ? p.scales[(int64_t)page1 * p.heads + h] : 0.0f;
      int dot[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < SELECT_CODES / 64; ++i) {
        if (i >= segments) break;
        const bool in = 64 * i + 16 * (lane & 3) < bytes;
        const uint4 x = in && page0 >= 0 ? *reinterpret_cast<const uint4*>(c0 + 64 * i)
                                         : make_uint4(0, 0, 0, 0);
        const uint4 y = in && page1 >= 0 ? *reinterpret_cast<const uint4*>(c1 + 64 * i)
                                         : make_uint4(0, 0, 0, 0);
        mma_s8(dot, x.x, y.x, x.y, y.y, b[i].x, b[i].y);
        mma_s8(dot, x.z, y.z, x.w, y.w, b[i].z, b[i].w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int w = 2 * (lane & 3) + (i & 1);  // token of the result
        const int page = i < 2 ? b0 : b1;
        if (w >= TT || s_row[w] != row || page >= s_held[w]) continue;
        uint32_t key = 0;
        if ((i < 2 ? page0 : page1) >= 0)
          // + 0.0f: a zero score has one form
          key = page < p.first || page >= s_held[w] - p.last
                    ? 0xFFFFFFFFu
                    : order_bits((float)dot[i] * (i < 2 ? scale0 : scale1) + 0.0f);
        const uint32_t at = 4 * (uint32_t)(w * p.width + page);
        if (cluster > 1)
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(first_keys + at), "r"(key)
                       : "memory");
        else
          keys[w * p.width + page] = key;
      }
    }
  }
  if (cluster > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
  else
    __syncthreads();
  if (rank != 0 || warp >= TT || t0 + warp >= p.tokens) return;

  // ---- selection, one warp per token
  const uint32_t* row_keys = keys + (int64_t)warp * p.width;
  const int held = s_held[warp];
  int32_t* out = p.out + ((t0 + warp) * p.heads + h) * p.n;
  uint32_t* bins = hist[warp];
  uint32_t prefix = 0, left = p.n;
  const bool all = held <= p.n;
  if (!all)
    for (int shift = 24; shift >= 0; shift -= 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) bins[lane + 32 * i] = 0;
      __syncwarp();
      for (int b = lane; b < held; b += 32) {
        const uint32_t key = row_keys[b];
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&bins[(key >> shift) & 255u], 1u);
      }
      __syncwarp();
      // lane l holds bins 255 - 8 l .. 248 - 8 l, so lanes go down in keys
      uint32_t count[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += count[i] = bins[255 - 8 * lane - i];
      uint32_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += y;
      }
      // the lane where the count passes `left`; the keys counted are at least n
      const uint32_t reach = __ballot_sync(~0u, upto >= left);
      const int owner = reach ? __ffs(reach) - 1 : 31;
      uint32_t above = upto - mine, digit = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        digit = 255 - 8 * lane - i;
        if (above + count[i] >= left || i == 7) break;
        above += count[i];
      }
      digit = __shfl_sync(~0u, digit, owner);
      above = __shfl_sync(~0u, above, owner);
      prefix |= digit << shift;
      left -= above;
      __syncwarp();
    }
  // pages above the threshold and its first `left` equals, in page order
  uint32_t done = 0, equals = 0;
  for (int b0 = 0; b0 < held; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t key = b < held ? row_keys[b] : 0;
    const bool equal = !all && key == prefix && key != 0;
    const uint32_t eq = __ballot_sync(~0u, equal);
    const uint32_t rank_eq = equals + __popc(eq & ((1u << lane) - 1));
    const bool take = key != 0 && (all || key > prefix || (equal && rank_eq < left));
    const uint32_t tk = __ballot_sync(~0u, take);
    if (take) out[done + __popc(tk & ((1u << lane) - 1))] = b;
    done += __popc(tk), equals += __popc(eq);
  }
  for (int i = (int)done + lane; i < p.n; i += 32) out[i] = -1;
}

}  // namespace mlxvs_b200
