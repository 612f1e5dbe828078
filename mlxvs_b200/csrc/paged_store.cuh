// Writes of new key and value rows to their slots, and the 8-bit bounds of
// the pages that got one.
//
// A page's bounds are, per key head and channel, the least and the largest
// key among its rows, rounded outward to multiples of one power of two that
// puts the page's largest magnitude in [64, 128): codes lo, hi in [-127, 127]
// and scale 2^-e with lo * scale <= key <= hi * scale (but for the last half
// step below 128, which saturates at 127).  Minima, maxima, products by powers of two,
// floor and ceil are exact, so the codes are a function of the page's rows
// alone: storing a page in one step or row by row gives the same bits.
#pragma once

#include "paged_common.cuh"

namespace mlxvs_b200 {

struct StoreParams {
  const void *k, *v;
  int64_t tokens;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
  const int64_t* slots;
  void *keys, *values;
  int64_t key_page, key_row, key_head, value_page, value_row, value_head;
  int64_t pages;
  FastDiv page;
  int heads, dim;
  float k_inverse, v_inverse;  // reciprocals of the cache's scales
  int8_t* codes;   // [pages, heads, 2, dim], null: no bounds
  float* scales;   // [pages, heads]
};

// One block per token.  The block of the last new row of a page reads the
// page's rows back (the earlier new ones from the input, since other blocks
// write them) and makes its bounds, one warp per key head.
template <class T, class C>
__global__ void __launch_bounds__(256) paged_store_kernel(const StoreParams p) {
  const int64_t t = blockIdx.x;
  const int64_t slot = p.slots[t];
  const int64_t P = p.page.d;
  if (slot < 0 || slot >= p.pages * P) return;
  const int64_t page = slot / P, row = slot % P;
  const T* k = static_cast<const T*>(p.k);
  const T* v = static_cast<const T*>(p.v);
  C* keys = static_cast<C*>(p.keys);
  C* values = static_cast<C*>(p.values);
  for (int i = threadIdx.x; i < p.heads * p.dim; i += blockDim.x) {
    const int h = i / p.dim, d = i % p.dim;
    keys[page * p.key_page + row * p.key_row + h * p.key_head + d] =
        from_float<C>(to_float(k[t * p.k_token + h * p.k_head + d]) * p.k_inverse);
    values[page * p.value_page + row * p.value_row + h * p.value_head + d] =
        from_float<C>(to_float(v[t * p.v_token + h * p.v_head + d]) * p.v_inverse);
  }
  if (p.codes == nullptr) return;
  if (t + 1 < p.tokens && p.slots[t + 1] == slot + 1 && row + 1 < P) return;
  int64_t fresh = 1;  // new rows of this page: the tokens t - fresh + 1 .. t
  while (fresh <= row && fresh <= t && p.slots[t - fresh] == slot - fresh) ++fresh;
  const int lane = threadIdx.x & 31;
  for (int h = threadIdx.x >> 5; h < p.heads; h += blockDim.x >> 5) {
    float lo[8], hi[8], top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      lo[j] = INFINITY, hi[j] = -INFINITY;
      if (d >= p.dim) continue;
      for (int64_t r = 0; r <= row; ++r) {
        const int64_t back = row - r;
        float x;
        if (back < fresh)
          x = to_float(from_float<C>(to_float(k[(t - back) * p.k_token + h * p.k_head + d]) *
                                     p.k_inverse));
        else
          x = to_float(keys[page * p.key_page + r * p.key_row + h * p.key_head + d]);
        lo[j] = fminf(lo[j], x), hi[j] = fmaxf(hi[j], x);
      }
      if (lo[j] > hi[j]) lo[j] = hi[j] = 0.0f;  // nothing but NaN
      top = fmaxf(top, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const int e = code_exponent(top);
    const float by = exp2_int(e);
    int8_t* codes = p.codes + ((page * p.heads + h) * 2) * p.dim;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      if (d >= p.dim) continue;
      codes[d] = (int8_t)fmaxf(fminf(floorf(lo[j] * by), 127.0f), -127.0f);
      codes[p.dim + d] = (int8_t)fminf(fmaxf(ceilf(hi[j] * by), -127.0f), 127.0f);
    }
    if (lane == 0) p.scales[page * p.heads + h] = exp2_int(-e);
  }
}

}  // namespace mlxvs_b200
