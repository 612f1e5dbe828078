// Writes of new key and value rows to their slots, and the 8-bit bounds of
// the pages that got one.
//
// A page's bounds are, per key head and channel, the least and the largest
// key among its rows, rounded outward to multiples of one power of two that
// puts the page's largest magnitude in [64, 128): codes lo, hi in [-127, 127]
// and scale 2^-e with lo * scale <= key <= hi * scale, but for magnitudes of more
// than 127 steps, which saturate: short by up to the step below 128, or without
// limit where e has ended at -100.  Minima, maxima, products by powers of two,
// floor and ceil are exact, so the codes are a function of the page's rows
// alone: storing a page in one step or row by row gives the same bits.
#pragma once

#include <type_traits>

#include "paged_attention.cuh"
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

constexpr int STORE_WARPS = 8;

template <class T>
struct alignas(sizeof(T) * 8) Eight {
  T x[8];
};

// Eight values times `by`, rounded to C.
template <class T, class C>
__device__ __forceinline__ Eight<C> rounded(const Eight<T>& x, float by) {
  Eight<C> y;
  if (std::is_same<T, C>::value && by == 1.0f) return *reinterpret_cast<const Eight<C>*>(&x);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<T>(w[i]);
    if (sizeof(C) == 1) {
      reinterpret_cast<__nv_fp8x2_storage_t*>(&y)[i] = __nv_cvt_float2_to_fp8x2(
          make_float2(v.x * by, v.y * by), __NV_SATFINITE, __NV_E4M3);
    } else {
      reinterpret_cast<uint32_t*>(&y)[i] = pack2<T>(v.x * by, v.y * by);
    }
  }
  return y;
}

// Running minima and maxima of eight channels in pairs of 16-bit values.  NaN is
// passed over; scaling by a positive number and rounding keep the order, so
// the bounds of what is stored are the stored bounds of the input.
template <class T>
struct Range;
template <>
struct Range<__half> {
  __half2 lo[4], hi[4];
  __device__ __forceinline__ Range() {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      lo[i] = __float2half2_rn(INFINITY), hi[i] = __float2half2_rn(-INFINITY);
  }
  __device__ __forceinline__ void take(int i, uint32_t w) {
    const __half2 x = *reinterpret_cast<const __half2*>(&w);
    lo[i] = __hmin2(lo[i], x), hi[i] = __hmax2(hi[i], x);
  }
};
template <>
struct Range<__nv_bfloat16> {
  __nv_bfloat162 lo[4], hi[4];
  __device__ __forceinline__ Range() {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      lo[i] = __float2bfloat162_rn(INFINITY), hi[i] = __float2bfloat162_rn(-INFINITY);
  }
  __device__ __forceinline__ void take(int i, uint32_t w) {
    const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w);
    lo[i] = __hmin2(lo[i], x), hi[i] = __hmax2(hi[i], x);
  }
};

// One warp per key head and chunk of up to 16 tokens, LANES lanes per row (8
// channels each, so 16-byte loads), ROWS rows side by side.  First it copies
// the chunk's rows; then, for each page whose last new row lies in the chunk,
// it reads the page's rows (the new ones from the input, which other warps may
// still be writing to the cache, the older ones from the cache) and makes its
// bounds.  The second reading of new rows hits L2.
//
// A page's new rows are tokens in a row, one row on for each token; a skipped
// token among them leaves its row as it was.  So row r of a page is new if token
// te - re + r has its slot (te: the page's last token, re: its row), and a token
// is its page's last unless the next token that is not skipped has its slot as
// many rows on as it comes tokens later.
//
// Bound: the copies by HBM; single tokens by the latency of slot -> rows of
// the page -> codes.  13,881 tokens of 8 heads of 128 into e4m3 take 24.1 us (86
// MB, 3.6 TB/s), 16.6 without bounds, into bf16 28.9 (114 MB, 4.0 TB/s); 128
// single tokens 6.5 us.
template <class T, class C, int LANES>
__global__ void __launch_bounds__(STORE_WARPS * 32)
    paged_store_kernel(const StoreParams p, const int chunk) {
  constexpr int ROWS = 32 / LANES;
  const int lane = threadIdx.x & 31, sub = lane / LANES, d = (lane % LANES) * 8;
  const int h = blockIdx.y * STORE_WARPS + (threadIdx.x >> 5);
  if (h >= p.heads) return;
  const bool mine = d < p.dim;
  const int64_t P = p.page.d;
  const int64_t t0 = (int64_t)blockIdx.x * chunk;
  const int count = (int)min((int64_t)chunk, p.tokens - t0);
  const T* k = static_cast<const T*>(p.k) + h * p.k_head + d;
  const T* v = static_cast<const T*>(p.v) + h * p.v_head + d;
  C* keys = static_cast<C*>(p.keys) + h * p.key_head + d;
  C* values = static_cast<C*>(p.values) + h * p.value_head + d;

  // one token per lane: its page and row, and whether it is its page's last
  const int64_t end = p.pages * P;  // of the slots
  int64_t slot = -1, page = -1;
  int row = 0;
  bool last = false, unsure = false;  // unsure: the next token is a skipped one
  if (lane < count) {
    slot = p.slots[t0 + lane];
    if (slot >= 0 && slot < end) {
      page = slot / P, row = (int)(slot - page * P);
      last = true;
      if (row + 1 < P && t0 + lane + 1 < p.tokens) {
        const int64_t next = p.slots[t0 + lane + 1];
        last = next != slot + 1;
        unsure = next < 0 || next >= end;
      }
    }
  }
  constexpr int UNROLL = 4;
  for (int i0 = 0; i0 < count; i0 += ROWS * UNROLL) {
    Eight<T> kx[UNROLL], vx[UNROLL];
    int64_t pg[UNROLL];
    int r[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = i0 + u * ROWS + sub;
      pg[u] = __shfl_sync(~0u, page, i & 31), r[u] = __shfl_sync(~0u, row, i & 31);
      if (i >= count || !mine) pg[u] = -1;
      if (pg[u] >= 0) {
        kx[u] = *reinterpret_cast<const Eight<T>*>(k + (t0 + i) * p.k_token);
        vx[u] = *reinterpret_cast<const Eight<T>*>(v + (t0 + i) * p.v_token);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (pg[u] >= 0) {
        *reinterpret_cast<Eight<C>*>(keys + pg[u] * p.key_page + r[u] * p.key_row) =
            rounded<T, C>(kx[u], p.k_inverse);
        *reinterpret_cast<Eight<C>*>(values + pg[u] * p.value_page + r[u] * p.value_row) =
            rounded<T, C>(vx[u], p.v_inverse);
      }
  }
  if (p.codes == nullptr) return;

  for (uint32_t some = __ballot_sync(~0u, unsure); some != 0; some &= some - 1) {
    const int i = __ffs(some) - 1;
    const int64_t t = t0 + i, s = __shfl_sync(~0u, slot, i);
    const int reach = (int)min(P - 1 - __shfl_sync(~0u, row, i), p.tokens - 1 - t);
    bool more = false;
    for (int j0 = 2; j0 <= reach; j0 += 32) {
      const int j = j0 + lane;
      const int64_t later = j <= reach ? p.slots[t + j] : -1;
      const uint32_t there = __ballot_sync(~0u, later >= 0 && later < end);
      if (there != 0) {
        more = __shfl_sync(~0u, later == s + j, __ffs(there) - 1);
        break;
      }
    }
    if (lane == i) last = !more;
  }
  for (uint32_t ends = __ballot_sync(~0u, last); ends != 0; ends &= ends - 1) {
    const int e = __ffs(ends) - 1;
    const int64_t te = t0 + e;
    const int64_t pg = __shfl_sync(~0u, page, e), se = __shfl_sync(~0u, slot, e);
    const int re = __shfl_sync(~0u, row, e);
    // new rows without a gap, from the last one back: begin to re
    int begin = re;
    bool gap = false;  // a skipped token lies before them
    while (begin > 0) {
      const int back = re - begin + 1 + lane;  // this lane's row is re - back
      const bool inside = back <= re && back <= te;
      const int64_t s = inside ? p.slots[te - back] : 0;
      const uint32_t all = __ballot_sync(~0u, inside && s == se - back);
      const uint32_t skips = __ballot_sync(~0u, inside && (s < 0 || s >= end));
      const int run = all == ~0u ? 32 : __ffs(~all) - 1;
      begin -= run;
      if (run < 32) {
        gap = skips >> run & 1;
        break;
      }
    }
    // old rows as they are stored (e4m3 as the float16 it is exactly), new ones
    // as they came
    using Old = typename std::conditional<sizeof(C) == 1, __half, T>::type;
    Range<Old> old_range;
    Range<T> new_range;
    if (mine) {
      const C* old = keys + pg * p.key_page;
      const T* fresh = k + (te - re) * p.k_token;  // of the page's row 0, were it new
      auto take_old = [&](int r) {
        const Eight<C> x = *reinterpret_cast<const Eight<C>*>(old + r * p.key_row);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          old_range.take(i, sizeof(C) == 1
                                ? widen_e4m3(reinterpret_cast<const uint16_t*>(&x)[i])
                                : reinterpret_cast<const uint32_t*>(&x)[i]);
      };
      auto take_new = [&](int r) {
        const Eight<T> x = *reinterpret_cast<const Eight<T>*>(fresh + r * p.k_token);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          new_range.take(i, reinterpret_cast<const uint32_t*>(&x)[i]);
      };
      if (!gap) {
#pragma unroll 8
        for (int r = sub; r < begin; r += ROWS) take_old(r);
      } else {
        for (int r = sub; r < begin; r += ROWS) {
          const int64_t t = te - re + r;
          if (t >= 0 && p.slots[t] == se - re + r) take_new(r);
          else take_old(r);
        }
      }
#pragma unroll 8
      for (int r = begin + sub; r <= re; r += ROWS) take_new(r);
    }
    float lo[8], hi[8];
    {
      const Eight<C> new_lo =
          rounded<T, C>(*reinterpret_cast<const Eight<T>*>(new_range.lo), p.k_inverse);
      const Eight<C> new_hi =
          rounded<T, C>(*reinterpret_cast<const Eight<T>*>(new_range.hi), p.k_inverse);
      const Old* old_lo = reinterpret_cast<const Old*>(old_range.lo);
      const Old* old_hi = reinterpret_cast<const Old*>(old_range.hi);
      const T* raw_lo = reinterpret_cast<const T*>(new_range.lo);
      const T* raw_hi = reinterpret_cast<const T*>(new_range.hi);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = to_float(old_lo[i]), hi[i] = to_float(old_hi[i]);
        if (to_float(raw_lo[i]) <= to_float(raw_hi[i])) {  // some new row is not NaN
          lo[i] = fminf(lo[i], to_float(new_lo.x[i]));
          hi[i] = fmaxf(hi[i], to_float(new_hi.x[i]));
        }
      }
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) {
        lo[i] = fminf(lo[i], __shfl_xor_sync(~0u, lo[i], o));
        hi[i] = fmaxf(hi[i], __shfl_xor_sync(~0u, hi[i], o));
      }
      if (lo[i] > hi[i]) lo[i] = hi[i] = 0.0f;  // nothing but NaN
      top = fmaxf(top, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const int x = code_exponent(top);
    const float by = exp2_int(x);
    if (mine && sub == 0) {
      Eight<int8_t> a, b;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a.x[i] = (int8_t)fmaxf(fminf(floorf(lo[i] * by), 127.0f), -127.0f);
        b.x[i] = (int8_t)fminf(fmaxf(ceilf(hi[i] * by), -127.0f), 127.0f);
      }
      int8_t* codes = p.codes + ((pg * p.heads + h) * 2) * p.dim + d;
      *reinterpret_cast<Eight<int8_t>*>(codes) = a;
      *reinterpret_cast<Eight<int8_t>*>(codes + p.dim) = b;
    }
    if (lane == 0) p.scales[pg * p.heads + h] = exp2_int(-x);
  }
}

}  // namespace mlxvs_b200
