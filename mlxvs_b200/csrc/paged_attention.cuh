// Attention of new tokens over a paged key-value cache.
//
//   s_j = scale * q . k_j,  o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m)
//
// (scores in units of log 2) over the keys of a token: the first `length` of
// its request, or those of them that lie in the pages selected for it.
//
// Bound: every byte of a token's keys and values is read once for all query
// heads of a key head, 2 G multiply-adds per element of two bytes (one with an
// 8-bit cache), so HBM bounds it.  The work is cut along the keys: the tiles
// of all (token, key head) rows form one sequence, each block takes an equal
// range of it, and rows that a range's end cuts leave partial sums (maximum,
// sum, weighted values) that a second kernel joins in the order of the keys.
//
// Measured, with the joining kernel: 64 requests of 0 to 5,000 keys (bf16, 8 key
// heads of 4) 67 us, 5.7 TB/s; 200 requests of up to 16,000 keys (f16, 4 key heads
// of 16) 405 us, 6.5 TB/s, the rate of a copy, and up to 455 where the power limit
// lowers the clock; 3 requests of up to 200,001 keys in e4m3 (8 key heads of 8) 171
// us, 5.4 TB/s, where the warps' conversions and the short ring show.
//
// Several tokens of a request are rows of their own, each of which reads the keys
// again: 2,048 tokens that see up to 12,000 keys (bf16, 4 key heads of 8) take 3.7
// ms, 17 times their operations' floor (e4m3 3.1 ms); 64 requests of 4 tokens and
// 8,000 keys 603 us against 161 for the bytes (e4m3 324 against 81).
#pragma once

#include <type_traits>

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
  float scale, v_scale;  // scale: of the scores, with the keys' scale and log2(e)
  void* out;             // [tokens, heads * group, dim]
  float* lse;            // [tokens, heads * group] or null
  float* part;           // [blocks][2][8 NT heads][DP + 2]: sums, maximum, sum
  int4* cut;             // [blocks]: the row that the block's start cuts
  int whole;             // a row for each block, none cut
};

// ------------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// 16 bytes to shared memory, past L1.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src)
               : "memory");
}
// Zeros where !valid (src is not read then).
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// d += a b: 16 x 16 by 16 x 8, float32 sums.
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two floats rounded to 16 bits (lo in the low half), and what rounding left.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 x = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
}

// Two values cut to a magnitude that no sum of products with the weights'
// remainders carries to infinity (float16: 65,504, its largest; bfloat16: 2^110,
// whose remainders are at most 1/2).  A remainder may be 0 or negative, and
// times an infinite value it would make a NaN of the infinity that the weight's
// first term gives.  (A float16 weight below 2^-32 of the largest is zero and
// still makes one, as a float32 weight that underflows does.)  Prompts of 5,229
// tokens 738 -> 754 us, 200 requests of up to 16,000 keys 463 -> 471 us (calls).
template <class T>
__device__ __forceinline__ uint32_t finite2(uint32_t x);
template <>
__device__ __forceinline__ uint32_t finite2<__half>(uint32_t x) {
  uint32_t r;  // the smaller magnitude, with the signs' product
  asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x7BFF7BFFu));
  return r;
}
template <>
__device__ __forceinline__ uint32_t finite2<__nv_bfloat16>(uint32_t x) {
  uint32_t r;
  asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x76807680u));
  return r;
}

// Two e4m3 (the low 16 bits of x) as two float16: exact.
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n"
      : "=r"(r)
      : "r"(x));
  return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ softmax
// Weights are 2^(s - m) with a reference m that follows the running maximum: it
// is LIFT below the maximum when it is raised, and raised when a score passes it
// by LIFT + 8.  So weights stay below 2^(LIFT + 8) and the largest one of a row is
// at least 2^LIFT.  In float16 LIFT is 7: weights up to 2^15 of 65,504, and the
// smallest steps, 2^-24, are 2^-31 of the largest weight, so that what many small
// weights behind a large one lose stays below the output's rounding up to 2^20
// keys.  bfloat16 has the exponents of float32.
template <class M>
struct Lift {
  static constexpr float value = std::is_same<M, __half>::value ? 7.0f : 0.0f;
};
// Rounded so that the weights' bounds hold for scores of any size.
template <class M>
__device__ __forceinline__ float reference(float maximum) {
  return __fadd_ru(maximum, -Lift<M>::value);
}
template <class M>
__device__ __forceinline__ float raised_past(float m) {
  return __fadd_rd(m, Lift<M>::value + 8.0f);
}

// sum += x with what the addition loses kept in `lost` (Kahan, 1965): a thread's
// sum of weights has one term per key, too many for plain float32 sums behind a
// large one.
__device__ __forceinline__ void add_kept(float& sum, float& lost, float x) {
  const float y = x - lost, t = sum + y;
  lost = (t - sum) - y;
  sum = t;
}

// ------------------------------------------------------------------ shapes
// T: type of the queries, C: of the cache, DP: the head dimension padded to
// 64, 128 or 256, NT: query heads in eights (8 or 16 at a time).
template <class T, class C, int DP, int NT>
struct AttentionShape {
  static constexpr bool EIGHT = sizeof(C) == 1;
  static constexpr int PITCH = DP * (int)sizeof(C);  // bytes of a row in shared memory
  static constexpr int KT = PITCH <= 128 ? 32 : 16;  // keys of a warp's step
  static constexpr int STEP = 2 * KT * PITCH;        // bytes of a warp's step
  // Warps, blocks per SM as registers allow, and the ring that shared memory
  // leaves each: three blocks with rings of two steps against two with three took
  // 166 for 175 us on long 8-bit caches, and 20 for 23 us on short lists of pages
  // (the products' latency counts there), the same on others.  Rows of 512 bytes:
  // two blocks of three warps against one of four 149 for 197 us (8 requests up
  // to 112,749 keys, 2 key heads of 16, bf16; the kernel alone).  There the sums'
  // compensation costs 8 us in registers.
  static constexpr int WARPS = STEP > 8192 ? 3 : 4;
  static constexpr int BLOCKS = STEP <= 8192 && NT == 1 && DP <= 128 ? 3 : 2;
  static constexpr int STAGES =
      STEP > 8192 ? 2 : (BLOCKS == 3 ? 2 : 3) * (8192 / STEP);
  static constexpr int KEYS = WARPS * KT;  // keys of a tile
  static constexpr int HEADS = 8 * NT;
  static constexpr int RING = WARPS * STAGES * STEP;
  static constexpr int SMEM = RING + HEADS * DP * 4;
  static constexpr int PART = HEADS * (DP + 2);  // floats of a partial result
};

// A row's end (joining the warps, writing, fetching queries) takes as long as
// about this many tiles, so it counts as such in the cut of the work: without
// it the blocks that got many short rows were the last to end by far.
constexpr int ROW_COST = 2;

// The row (token, key head, chunk of query heads) of a place in the sequence.
struct AttentionRow {
  int64_t t;       // token
  int h, chunk;    // key head, chunk of query heads
  int64_t start;   // the place of the row's first tile, behind its cost
  int tiles;
};

// ------------------------------------------------------------------ kernel
// A block works through its range of tiles.  In a tile each warp has KT keys
// of its own and a ring of STAGES of them in shared memory, filled by
// asynchronous copies and synchronised by the warp alone (16-byte copies rather
// than tiled ones: rows may lie in pages of any size).  Scores and sums
// are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the 16-row side
// of the tensor cores' tile holds keys or channels, never padding, and the
// 8-column side the query heads.  The weights' reference is raised only when a
// score passes the maximum it was taken from by 8, so the sums are rescaled a few
// times a row instead of every step.
//
// The weights are two 16-bit terms (value and remainder), since one would add a
// rounding up to as large as the output's own, and more where values cancel; the
// products that costs hide behind the loads (e4m3 cache of 200,001 keys: 172 us
// with two terms, 171 with one).  An 8-bit cache's values are exact in float16,
// to which the queries are scaled by a power of two per head.
template <class T, class C, int DP, int NT, bool SPARSE>
__global__ void __launch_bounds__(AttentionShape<T, C, DP, NT>::WARPS * 32,
                                  AttentionShape<T, C, DP, NT>::BLOCKS)
    paged_attention_kernel(const AttentionParams p) {
  using S = AttentionShape<T, C, DP, NT>;
  using M = typename std::conditional<S::EIGHT, __half, T>::type;  // tensor core type
  constexpr int KT = S::KT, MT = KT / 16, THREADS = S::WARPS * 32;
  extern __shared__ __align__(1024) uint8_t ring[];
  float* sum_o = reinterpret_cast<float*>(ring + S::RING);  // [HEADS][DP]
  __shared__ float sh_m[S::WARPS][S::HEADS], sh_l[S::WARPS][S::HEADS];
  __shared__ int64_t sh_scan[S::WARPS + 1];
  __shared__ int64_t sh_found[2];  // the token that holds the first tile, its start
  __shared__ uint32_t sh_valid[S::WARPS][S::STAGES];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = (int)p.page.d;
  const int chunks = (p.group + S::HEADS - 1) / S::HEADS;
  const int per_token = p.heads * chunks;  // rows of a token

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  auto length_of = [&](int64_t t) -> int {
    const int64_t r = p.requests ? p.requests[t] : t;
    if (r < 0 || r >= p.rows) return 0;
    return (int)min((int64_t)max(p.lengths[t], 0), min(p.width * P, (int64_t)INT32_MAX));
  };
  auto tiles_of = [&](int64_t t) -> int {
    if (SPARSE) return (int)(((int64_t)p.n * P + S::KEYS - 1) / S::KEYS);
    return max(1, (length_of(t) + S::KEYS - 1) / S::KEYS);
  };

  // ---- this block's range of places, and the row it begins in
  int64_t total;
  int64_t x, x1, per;
  AttentionRow row;
  if (p.whole) {
    row.t = blockIdx.x / per_token;
    row.h = (int)(blockIdx.x % per_token) / chunks, row.chunk = (int)(blockIdx.x % per_token) % chunks;
    row.tiles = tiles_of(row.t);
    row.start = x = 0, x1 = per = row.tiles;
  } else if (SPARSE) {
    row.tiles = tiles_of(0);
    const int places = row.tiles + ROW_COST;
    total = p.tokens * per_token * places;
    per = max((int64_t)1, (total + gridDim.x - 1) / gridDim.x);
    x = blockIdx.x * per, x1 = min(x + per, total);
    const int64_t index = x / places;
    row.t = index / per_token;
    row.start = index * places + ROW_COST;
    row.h = (int)(index % per_token) / chunks, row.chunk = (int)(index % per_token) % chunks;
  } else {
    const int64_t each = (p.tokens + THREADS - 1) / THREADS;
    const int64_t ta = min(tid * each, p.tokens), tb = min(ta + each, p.tokens);
    int64_t mine = 0;
    for (int64_t t = ta; t < tb; ++t) mine += tiles_of(t) + ROW_COST;
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) sh_scan[warp] = sum;
    __syncthreads();
    total = 0;
    int64_t before = sum - mine;
#pragma unroll
    for (int w = 0; w < S::WARPS; ++w) {
      if (w < warp) before += sh_scan[w];
      total += sh_scan[w];
    }
    total *= per_token;
    per = max((int64_t)1, (total + gridDim.x - 1) / gridDim.x);
    x = blockIdx.x * per, x1 = min(x + per, total);
    int64_t at = before * per_token;
    if (x >= at && x < at + mine * per_token)
      for (int64_t t = ta; t < tb; ++t) {
        const int64_t next = at + (int64_t)(tiles_of(t) + ROW_COST) * per_token;
        if (x < next) {
          sh_found[0] = t, sh_found[1] = at;
          break;
        }
        at = next;
      }
    __syncthreads();
    if (x < x1) {
      row.t = sh_found[0];
      row.tiles = tiles_of(row.t);
      const int places = row.tiles + ROW_COST;
      const int index = (int)((x - sh_found[1]) / places);
      row.start = sh_found[1] + (int64_t)index * places + ROW_COST;
      row.h = index / chunks, row.chunk = index % chunks;
    }
  }
  // the block's first tile, and how many places are left from there: a range
  // that ends within a row's cost leaves the row to the next block
  const bool cut = x < x1 && x > row.start;
  if (tid == 0 && !p.whole) {
    // a row that this block's start cuts, listed by the first block that cuts it
    const bool first = cut && row.start >= x - per;
    const int64_t last = first ? (row.start + row.tiles - 1) / per : 0;
    p.cut[blockIdx.x] =
        first ? make_int4((int)row.t, row.h, row.chunk, (int)last) : make_int4(-1, 0, 0, 0);
  }
  x = max(x, row.start);
  if (x >= x1) return;

  const uint32_t my_ring = smem_address(ring) + warp * S::STAGES * S::STEP;
  // columns past dim are never copied: zero for good
  if (p.dim < DP) {
    for (int i = tid; i < S::RING / 16; i += THREADS)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }

  // swizzle: the 16-byte chunk of a row moves so that 8 rows of one chunk
  // column lie in different banks
  constexpr int CH = S::PITCH / 16;  // chunks of a row
  auto chunk_at = [](int r, int c) -> uint32_t {
    const int s = CH >= 8 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & (CH - 1)));
    return r * S::PITCH + s * 16;
  };

  // ---- the loading side runs STAGES - 1 tiles ahead of the products, across
  // the ends of rows: while one row's results are written, the next one's
  // first tiles are on their way
  struct {
    int64_t t;
    int h, chunk, tile, tiles, length;
    const int32_t* table;
  } ahead;
  auto enter = [&](int64_t t) {  // the loading side's token
    const int64_t request = p.requests ? p.requests[t] : t;
    ahead.t = t;
    ahead.length = length_of(t);
    ahead.table = p.table + request * p.width;
    if (!SPARSE) ahead.tiles = max(1, (ahead.length + S::KEYS - 1) / S::KEYS);
  };
  ahead.h = row.h, ahead.chunk = row.chunk, ahead.tile = (int)(x - row.start);
  ahead.tiles = row.tiles;
  enter(row.t);
  // where this lane's key of the next tile lies: its page (-1: none) and the
  // offsets of its row in it, with the key head's
  int page;
  int64_t key_at, value_at;
  bool located;  // there is a next tile
  int64_t ahead_x = x;
  auto locate = [&] {
    page = -1;
    located = ahead_x < x1;
    if (!located) return;
    const int64_t j = (int64_t)ahead.tile * S::KEYS + warp * KT + lane;
    if (lane < KT && j < (SPARSE ? (int64_t)p.n * P : (int64_t)ahead.length)) {
      const int pos = (int)p.page.div((uint32_t)j), in = (int)j - pos * P;
      int b = pos;
      if (SPARSE) {
        b = p.selected[(ahead.t * p.heads + ahead.h) * p.n + pos];
        if (b >= p.width || (int64_t)b * P + in >= ahead.length) b = -1;
      }
      if (b >= 0) page = ahead.table[b];
      key_at = in * p.key_row + ahead.h * p.key_head;
      value_at = in * p.value_row + ahead.h * p.value_head;
    }
    ++ahead_x;
    if (++ahead.tile == ahead.tiles) {
      ahead.tile = 0;
      ahead_x += ROW_COST;
      if (++ahead.chunk == chunks) {
        ahead.chunk = 0;
        if (++ahead.h == p.heads) {
          ahead.h = 0;
          if (ahead.t + 1 < p.tokens) enter(ahead.t + 1);
        }
      }
    }
  };
  auto load = [&](int stage) {
    if (page >= p.pages) page = -1;
    const uint32_t valid = __ballot_sync(~0u, page >= 0);
    if (lane == 0) sh_valid[warp][stage] = valid;
    // offsets in bytes from the first key and value
    const int64_t koff = (page * p.key_page + key_at) * (int64_t)sizeof(C);
    const int64_t voff = (page * p.value_page + value_at) * (int64_t)sizeof(C);
    constexpr int LANES = CH < 8 ? CH : 8;  // lanes of a row
    constexpr int ROWS = 32 / LANES;
    const int c0 = lane % LANES, r0 = lane / LANES;
    const uint8_t* keys = static_cast<const uint8_t*>(p.keys) + c0 * 16;
    const uint8_t* values = static_cast<const uint8_t*>(p.values) + c0 * 16;
    const uint32_t at = my_ring + stage * S::STEP;
    const int bytes = p.dim * (int)sizeof(C) - c0 * 16;  // of a row, from this lane's chunk
    if (valid == (KT == 32 ? ~0u : (1u << KT) - 1)) {
#pragma unroll
      for (int g = 0; g < KT / ROWS; ++g) {
        const int r = g * ROWS + r0;
        const uint8_t* k = keys + __shfl_sync(~0u, koff, r);
        const uint8_t* v = values + __shfl_sync(~0u, voff, r);
#pragma unroll
        for (int cc = 0; cc < CH; cc += LANES)
          if (cc * 16 < bytes) {
            const uint32_t to = at + chunk_at(r, cc + c0);
            copy16(to, k + cc * 16);
            copy16(to + KT * S::PITCH, v + cc * 16);
          }
      }
    } else {
      // rows that are not there become zeros
#pragma unroll
      for (int g = 0; g < KT / ROWS; ++g) {
        const int r = g * ROWS + r0;
        const bool there = valid >> r & 1;
        const int64_t ko = __shfl_sync(~0u, koff, r), vo = __shfl_sync(~0u, voff, r);
#pragma unroll
        for (int cc = 0; cc < CH; cc += LANES)
          if (cc * 16 < bytes) {
            const uint32_t to = at + chunk_at(r, cc + c0);
            copy16_or_zero(to, there ? keys + ko + cc * 16 : keys, there);
            copy16_or_zero(to + KT * S::PITCH, there ? values + vo + cc * 16 : values, there);
          }
      }
    }
  };
  locate();
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s) {
    if (located) load(s);
    copy_commit();
    locate();
  }

  // ---- queries: B operands, head n = lane / 4 of each eight
  uint32_t qf[DP / 16][NT][2];
  float factor[NT][2];  // of the scores of heads 2 (lane % 4) + {0, 1}
  auto fetch_queries = [&] {
    const int head0 = row.h * p.group + row.chunk * S::HEADS;
    const int heads = min(S::HEADS, p.group - row.chunk * S::HEADS);
    const T* q = static_cast<const T*>(p.q) + row.t * p.q_token + (int64_t)head0 * p.q_head;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + lane / 4;
      const T* qn = q + (int64_t)min(n, heads - 1) * p.q_head;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        const int d0 = s * 16 + (S::EIGHT ? 4 : 2) * (lane % 4), d1 = d0 + (S::EIGHT ? 2 : 8);
        const bool live = n < heads;
        qf[s][nt][0] = live && d0 < p.dim ? *reinterpret_cast<const uint32_t*>(qn + d0) : 0u;
        qf[s][nt][1] = live && d1 < p.dim ? *reinterpret_cast<const uint32_t*>(qn + d1) : 0u;
      }
    }
  };
  auto scale_queries = [&] {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      factor[nt][0] = factor[nt][1] = p.scale;
      if (S::EIGHT) {
        // the largest magnitude to [64, 128): exact in float16 down to 2^-21 of it
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 v = unpack2<T>(qf[s][nt][i]);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        const int e = query_exponent(top);
        const float by = exp2_int(e), back = exp2_int(-e) * p.scale;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 v = unpack2<T>(qf[s][nt][i]);
            qf[s][nt][i] = pack2<M>(v.x * by, v.y * by);
          }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          factor[nt][i] = __shfl_sync(~0u, back, (2 * (lane % 4) + i) * 4);
      }
    }
  };
  fetch_queries();

  int stage = 0;
  while (x < x1) {
    // ------------------------------------------------ one row's piece
    const int tile0 = (int)(x - row.start);
    const int tile1 = (int)min((int64_t)row.tiles, x1 - row.start);
    scale_queries();
    float o[DP / 16][NT][4], m[NT][2], l[NT][2], lost[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = lost[nt][0] = lost[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    }

    for (int tile = tile0; tile < tile1; ++tile) {
      copy_wait<S::STAGES - 2>();
      __syncwarp();
      {
        int to = stage + S::STAGES - 1;
        if (to >= S::STAGES) to -= S::STAGES;
        if (located) load(to);
        copy_commit();
        locate();
      }
      const uint32_t valid = sh_valid[warp][stage];
      const uint32_t kat = my_ring + stage * S::STEP, vat = kat + KT * S::PITCH;
      if (++stage == S::STAGES) stage = 0;
      if (valid == 0) continue;

      // ---- S^T = K Q^T
      float st[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          st[mt][nt][0] = st[mt][nt][1] = st[mt][nt][2] = st[mt][nt][3] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16 + (lane & 15);
        if (S::EIGHT) {
#pragma unroll
          for (int s = 0; s < DP / 16; s += 2) {
            uint32_t a[4];  // keys 0-7, 8-15 of chunk s, then of chunk s + 1
            load_matrices(a, kat + chunk_at(r, s + (lane >> 4)));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t w[4] = {widen_e4m3(a[2 * u]), widen_e4m3(a[2 * u + 1]),
                                     widen_e4m3(a[2 * u] >> 16), widen_e4m3(a[2 * u + 1] >> 16)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<M>(st[mt][nt], w, qf[s + u][nt][0], qf[s + u][nt][1]);
            }
          }
        } else {
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) {
            uint32_t a[4];
            load_matrices(a, kat + chunk_at(r, 2 * s + (lane >> 4)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<M>(st[mt][nt], a, qf[s][nt][0], qf[s][nt][1]);
          }
        }
      }
      // ---- scores, masked; a raised reference where one passes it by far
      bool raise = false;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float& s = st[mt][nt][i];
            s *= factor[nt][i & 1];
            if (!((valid >> (mt * 16 + (i >> 1) * 8 + lane / 4)) & 1)) s = -INFINITY;
            raise |= s > raised_past<M>(m[nt][i & 1]);
          }
      if (__any_sync(~0u, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              top = fmaxf(top, fmaxf(st[mt][nt][i], st[mt][nt][i + 2]));
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, w));
            const float to = fmaxf(m[nt][i], reference<M>(top));
            const float keep = m[nt][i] == -INFINITY ? 0.0f : exp2_approx(m[nt][i] - to);
            m[nt][i] = to;
            l[nt][i] *= keep, lost[nt][i] *= keep;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) o[k][nt][i] *= keep, o[k][nt][i + 2] *= keep;
          }
      }
      // ---- weights, and O^T += V^T P^T
      float more[NT][2];  // the tile's weights
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) more[nt][0] = more[nt][1] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t b[NT][2], rest[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0];
          const float m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float w0 = exp2_approx(st[mt][nt][2 * u] - m0);
            const float w1 = exp2_approx(st[mt][nt][2 * u + 1] - m1);
            more[nt][0] += w0, more[nt][1] += w1;
            const uint32_t both = pack2<M>(w0, w1);
            b[nt][u] = transpose8x8(both);
            const float2 r = unpack2<M>(both);
            rest[nt][u] = transpose8x8(pack2<M>(w0 - r.x, w1 - r.y));
          }
        }
        if (S::EIGHT) {
          const int r = mt * 16 + (lane & 15);
#pragma unroll
          for (int s = 0; s < DP / 16; s += 2) {
            uint32_t a[4];  // keys 0-7, 8-15 of chunk s, then of chunk s + 1
            load_matrices_t(a, vat + chunk_at(r, s + (lane >> 4)));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // bytes (key, channel): 00 01 10 11 -> 00 10 01 11: rows 0-7 of the
              // tile are the even channels of the chunk, rows 8-15 the odd ones
              const uint32_t e0 = __byte_perm(a[2 * u], 0, 0x3120);
              const uint32_t e1 = __byte_perm(a[2 * u + 1], 0, 0x3120);
              const uint32_t w[4] = {widen_e4m3(e0), widen_e4m3(e0 >> 16), widen_e4m3(e1),
                                     widen_e4m3(e1 >> 16)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<M>(o[s + u][nt], w, b[nt][0], b[nt][1]);
                mma16816<M>(o[s + u][nt], w, rest[nt][0], rest[nt][1]);
              }
            }
          }
        } else {
          const int r = mt * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) {
            uint32_t a[4];
            load_matrices_t(a, vat + chunk_at(r, 2 * s + ((lane >> 3) & 1)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<M>(o[s][nt], a, b[nt][0], b[nt][1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = finite2<M>(a[i]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<M>(o[s][nt], a, rest[nt][0], rest[nt][1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) add_kept(l[nt][i], lost[nt][i], more[nt][i]);
    }
    // ---- on to the next row, whose queries are fetched meanwhile
    const AttentionRow ended = row;
    row.start += row.tiles + ROW_COST;
    x = row.start;
    if (x < x1) {
      if (++row.chunk == chunks) {
        row.chunk = 0;
        if (++row.h == p.heads) row.h = 0, row.t += 1, row.tiles = tiles_of(row.t);
      }
      fetch_queries();
    }

    // ---- join the warps in their order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], w);
        if (lane < 4) {
          sh_m[warp][nt * 8 + 2 * lane + i] = m[nt][i];
          sh_l[warp][nt * 8 + 2 * lane + i] = l[nt][i];
        }
      }
    __syncthreads();
    float weight[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < S::WARPS; ++w)
          top = fmaxf(top, sh_m[w][nt * 8 + 2 * (lane % 4) + i]);
        weight[nt][i] = m[nt][i] == -INFINITY ? 0.0f : exp2_approx(m[nt][i] - top);
      }
#pragma unroll
    for (int w = 0; w < S::WARPS; ++w) {
      if (w == warp) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d = k * 16 + (S::EIGHT ? 2 * (lane / 4) + (i >> 1)
                                               : lane / 4 + 8 * (i >> 1));
              float& to = sum_o[(nt * 8 + 2 * (lane % 4) + (i & 1)) * DP + d];
              const float y = o[k][nt][i] * weight[nt][i & 1];
              to = w == 0 ? y : to + y;
            }
      }
      __syncthreads();
    }
    // ---- write the row, or its part
    const bool whole = tile0 == 0 && tile1 == ended.tiles;
    const int head0 = ended.h * p.group + ended.chunk * S::HEADS;  // first query head
    const int heads = min(S::HEADS, p.group - ended.chunk * S::HEADS);
    float* part = p.part + ((int64_t)blockIdx.x * 2 + (tile0 == 0)) * S::PART;
    for (int n = warp; n < heads; n += S::WARPS) {
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < S::WARPS; ++w) top = fmaxf(top, sh_m[w][n]);
#pragma unroll
      for (int w = 0; w < S::WARPS; ++w)
        sum += sh_m[w][n] == -INFINITY ? sh_l[w][n] : sh_l[w][n] * exp2_approx(sh_m[w][n] - top);
      if (whole) {
        const int64_t hq = ended.t * p.heads * p.group + head0 + n;
        T* out = static_cast<T*>(p.out) + hq * p.dim;
        const float by = sum != 0.0f ? p.v_scale / sum : 0.0f;
        for (int d = 2 * lane; d < p.dim; d += 64) {
          const float2 y = *reinterpret_cast<const float2*>(sum_o + n * DP + d);
          *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(y.x * by, y.y * by);
        }
        if (p.lse && lane == 0)
          p.lse[hq] = sum != 0.0f ? (top + log2f(sum)) * 0.693147180559945f : -INFINITY;
      } else {
        for (int d = lane; d < DP; d += 32) part[n * (DP + 2) + d] = sum_o[n * DP + d];
        if (lane == 0) part[n * (DP + 2) + DP] = top, part[n * (DP + 2) + DP + 1] = sum;
      }
    }
    __syncthreads();
  }
  copy_wait<0>();
}

// Joins the parts of a cut row, one block per cut and query head: parts in the
// order of the keys, so the sums do not depend on which block ended first.
template <class T, int DP, int NT>
__global__ void __launch_bounds__(DP) paged_attention_join_kernel(const AttentionParams p) {
  constexpr int HEADS = 8 * NT, PART = HEADS * (DP + 2);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = p.cut[blockIdx.x];
  if (cut.x < 0) return;
  const int n = blockIdx.y;
  if (cut.z * HEADS + n >= p.group) return;
  // the block before holds the row's beginning, the others follow in slot 0
  const int parts = cut.w - (int)blockIdx.x + 2;
  auto part = [&](int i) {
    return p.part + ((int64_t)(blockIdx.x - 1 + i) * 2 + (i == 0)) * PART + n * (DP + 2);
  };
  const int d = threadIdx.x;
  float top = -INFINITY;
  for (int i = 0; i < parts; ++i) top = fmaxf(top, part(i)[DP]);
  float sum = 0.0f, y = 0.0f;
  for (int i = 0; i < parts; ++i) {
    const float* from = part(i);
    const float w = from[DP] == -INFINITY ? (from[DP + 1] != 0.0f ? 1.0f : 0.0f)
                                          : exp2_approx(from[DP] - top);
    sum += w * from[DP + 1];
    y += w * from[d];
  }
  const int64_t hq = ((int64_t)cut.x * p.heads + cut.y) * p.group + cut.z * HEADS + n;
  if (d < p.dim)
    static_cast<T*>(p.out)[hq * p.dim + d] =
        from_float<T>(sum != 0.0f ? y * (p.v_scale / sum) : 0.0f);
  if (p.lse && d == 0)
    p.lse[hq] = sum != 0.0f ? (top + log2f(sum)) * 0.693147180559945f : -INFINITY;
}

}  // namespace mlxvs_b200
