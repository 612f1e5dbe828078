// Attention of new tokens over a paged key-value cache.
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// over the keys of a token: the first `length` of its request, or those of
// them that lie in the pages selected for it.
#pragma once

#include "paged_common.cuh"

namespace mlxvs_b200 {

struct AttentionParams {
  const void* q;
  int64_t tokens, q_token, q_head;
  int heads, group, dim;
  const void *keys, *values;
  int64_t key_page, key_row, key_head, value_page, value_row, value_head;
  int64_t pages;
  FastDiv page;
  const int32_t* table;
  int64_t rows, width;
  const int32_t *requests, *lengths;
  const int32_t* selected;  // [tokens, heads, n] or null
  int n;
  float scale, v_scale;  // scale: of the scores, with the keys' scale
  void* out;             // [tokens, heads * group, dim]
  float* lse;            // [tokens, heads * group] or null
};

constexpr int ATTENTION_WARPS = 8;

// One block per token and query head, a key per warp at a time.
template <class T, class C>
__global__ void __launch_bounds__(ATTENTION_WARPS * 32)
    paged_attention_kernel(const AttentionParams p) {
  __shared__ float part[ATTENTION_WARPS][256];
  __shared__ float part_m[ATTENTION_WARPS], part_l[ATTENTION_WARPS];
  const int64_t t = blockIdx.x;
  const int hq = blockIdx.y, h = hq / p.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = p.requests ? p.requests[t] : t;
  int length = p.lengths[t];
  if (row < 0 || row >= p.rows) length = 0;
  const int P = (int)p.page.d;
  length = (int)min((int64_t)max(length, 0), p.width * P);
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + hq * p.q_head;
  float qr[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int d = lane + 32 * j;
    qr[j] = d < p.dim ? to_float(q[d]) * p.scale : 0.0f;
    o[j] = 0.0f;
  }
  const int32_t* selected = p.selected ? p.selected + (t * p.heads + h) * p.n : nullptr;
  const int64_t count = selected ? (int64_t)p.n * P : length;
  for (int64_t i = warp; i < count; i += ATTENTION_WARPS) {
    const int in_list = (int)(i / P), in = (int)(i % P);
    const int b = selected ? selected[in_list] : in_list;
    if (b < 0 || (int64_t)b * P + in >= length) continue;
    const int64_t page = p.table[row * p.width + b];
    if (page < 0 || page >= p.pages) continue;
    const C* key = static_cast<const C*>(p.keys) + page * p.key_page + in * p.key_row + h * p.key_head;
    const C* value =
        static_cast<const C*>(p.values) + page * p.value_page + in * p.value_row + h * p.value_head;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      if (d < p.dim) s += qr[j] * to_float(key[d]);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.0f : expf(m - top);
    const float e = s == -INFINITY ? 0.0f : expf(s - top);
    l = l * keep + e;
    m = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      if (d < p.dim) o[j] = o[j] * keep + e * to_float(value[d]);
    }
  }
  if (lane == 0) part_m[warp] = m, part_l[warp] = l;
#pragma unroll
  for (int j = 0; j < 8; ++j) part[warp][lane + 32 * j] = o[j];
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < ATTENTION_WARPS; ++w) top = fmaxf(top, part_m[w]);
  float weight[ATTENTION_WARPS];
  for (int w = 0; w < ATTENTION_WARPS; ++w) {
    weight[w] = part_m[w] == -INFINITY ? 0.0f : expf(part_m[w] - top);
    sum += weight[w] * part_l[w];
  }
  T* out = static_cast<T*>(p.out) + (t * p.heads * p.group + hq) * p.dim;
  for (int d = threadIdx.x; d < p.dim; d += blockDim.x) {
    float x = 0.0f;
    for (int w = 0; w < ATTENTION_WARPS; ++w) x += weight[w] * part[w][d];
    out[d] = from_float<T>(sum != 0.0f ? x / sum * p.v_scale : 0.0f);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[t * p.heads * p.group + hq] = sum != 0.0f ? top + logf(sum) : -INFINITY;
}

}  // namespace mlxvs_b200
