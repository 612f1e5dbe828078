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

constexpr int SELECT_THREADS = 256;

// One block per token and key head; scores in shared memory, then a radix
// selection of the n best by (score, lower page) in 8-bit digits.
template <class T>
__global__ void __launch_bounds__(SELECT_THREADS) paged_select_kernel(const SelectParams p) {
  extern __shared__ uint32_t keys[];  // order bits of the scores, 0: no page
  __shared__ __align__(16) int8_t qc[512];  // q- then q+ codes
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_left;
  __shared__ float sh_top[SELECT_THREADS / 32];
  __shared__ uint32_t warp_count[2][SELECT_THREADS / 32];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* out = p.out + (t * p.heads + h) * p.n;
  const int64_t row = p.requests ? p.requests[t] : t;
  int length = p.lengths[t];
  if (row < 0 || row >= p.rows) length = 0;
  const int held = min((int)p.page.div((uint32_t)max(length, 0) + p.page.d - 1), (int)p.width);
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + (int64_t)h * p.group * p.q_head;
  float top = 0.0f;
  for (int i = tid; i < p.group * p.dim; i += SELECT_THREADS)
    top = fmaxf(top, fabsf(to_float(q[(i / p.dim) * p.q_head + i % p.dim])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if (lane == 0) sh_top[warp] = top;
  __syncthreads();
  for (int w = 0; w < SELECT_THREADS / 32; ++w) top = fmaxf(top, sh_top[w]);
  const float by = exp2_int(code_exponent(top));
  if (tid < p.dim) {
    int up = 0, down = 0;
    for (int g = 0; g < p.group; ++g) {
      const float x = to_float(q[g * p.q_head + tid]) * by;
      const int c = x == x ? (int)rintf(fmaxf(-127.0f, fminf(127.0f, x))) : 0;
      if (c > 0) up += c;
      else down -= c;
    }
    qc[tid] = (int8_t)(-(down >> p.shift));
    qc[p.dim + tid] = (int8_t)(up >> p.shift);
  }
  __syncthreads();
  const int32_t* table = p.table + row * p.width;
  const int words = p.dim / 2;  // 2 * dim codes, four to a word
  const int* qw = reinterpret_cast<const int*>(qc);
  for (int b = tid; b < held; b += SELECT_THREADS) {
    const int32_t page = table[b];
    uint32_t key = 0;
    if (page >= 0 && page < p.pages) {
      if (b < p.first || b >= held - p.last) {
        key = 0xFFFFFFFFu;
      } else {
        const int* c = reinterpret_cast<const int*>(p.codes + ((int64_t)page * p.heads + h) * 2 * p.dim);
        int dot = 0;
        for (int i = 0; i < words; ++i) dot = __dp4a(c[i], qw[i], dot);
        // + 0.0f: a zero score has one form
        key = order_bits((float)dot * p.scales[(int64_t)page * p.heads + h] + 0.0f);
      }
    }
    keys[b] = key;
  }
  __syncthreads();
  // threshold: the n-th largest key and how many of its equals are taken
  uint32_t prefix = 0, left = p.n;
  bool all = held <= p.n;
  if (!all) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      hist[tid] = 0;
      __syncthreads();
      for (int b = tid; b < held; b += SELECT_THREADS) {
        const uint32_t key = keys[b];
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0;
        int digit = 255;
        for (; digit > 0; --digit) {
          if (above + hist[digit] >= left) break;
          above += hist[digit];
        }
        sh_prefix = prefix | ((uint32_t)digit << shift);
        sh_left = left - above;
      }
      __syncthreads();
      prefix = sh_prefix, left = sh_left;
      __syncthreads();
    }
  }
  // pages above the threshold, and its first `left` equals, in page order
  uint32_t done = 0, equals = 0;
  for (int b0 = 0; b0 < held; b0 += SELECT_THREADS) {
    const int b = b0 + tid;
    const uint32_t key = b < held ? keys[b] : 0;
    const bool equal = !all && key == prefix && key != 0;
    const uint32_t eq = __ballot_sync(~0u, equal);
    if (lane == 0) warp_count[0][warp] = __popc(eq);
    __syncthreads();
    uint32_t rank = equals, total = 0;
    for (int w = 0; w < SELECT_THREADS / 32; ++w) {
      if (w < warp) rank += warp_count[0][w];
      total += warp_count[0][w];
    }
    rank += __popc(eq & ((1u << lane) - 1));
    const bool take = key != 0 && (all || key > prefix || (equal && rank < left));
    const uint32_t tk = __ballot_sync(~0u, take);
    if (lane == 0) warp_count[1][warp] = __popc(tk);
    __syncthreads();
    uint32_t at = done, taken = 0;
    for (int w = 0; w < SELECT_THREADS / 32; ++w) {
      if (w < warp) at += warp_count[1][w];
      taken += warp_count[1][w];
    }
    at += __popc(tk & ((1u << lane) - 1));
    if (take) out[at] = b;
    done += taken, equals += total;
    __syncthreads();
  }
  for (int i = (int)done + tid; i < p.n; i += SELECT_THREADS) out[i] = -1;
}

}  // namespace mlxvs_b200
