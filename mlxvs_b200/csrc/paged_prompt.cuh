// Attention of prompts over selected pages: many neighbouring tokens of a
// request, each with its own list of pages.
//
// Neighbouring tokens select the same pages often (their queries are alike)
// and, out of a limited number of pages, by chance.  So a block takes a tile
// of tokens and one key head, marks in shared memory which of its tokens
// selected which page, and walks the pages that any of them selected once:
// each page is loaded once for the tile instead of once per token, and each
// warp multiplies it only by the queries of those of its own tokens that
// selected it.  As in paged_attention.cuh the products are transposed
// (S^T = K Q^T, O^T = V^T P^T): a token's query heads are the 8 columns, so no
// work is spent on tokens that did not select the page.
//
// Bound: 5,229 tokens with 16 of up to 230 pages of 64 each (bf16, 4 key heads of
// 8, 89 GFLOP) take 693 us, 128 TFLOP/s, and 799 over an e4m3 cache.  Parts switched
// off in turn when they took 672 (without the care for infinite values and small
// weights): the loads
// alone take 298 us (the tiles still read 2.5 GB from L2) and hide behind the
// products, which alone take 635; of those the waits for the slowest warp of a
// stage cost 76, the scores 224, the weights 69, the values 171 and the lists and
// ends 95.  A token reads each of its pages from shared memory by itself (32 KB
// for 8 query heads), so shared memory, not the tensor cores (257 us at the warp
// instructions' full rate), is what the products run into.  128-row tensor core
// tiles would multiply every token by every page of the tile: with pages chosen
// alike they would win, with pages chosen by chance they do eight times the
// work.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "paged_attention.cuh"

namespace mlxvs_b200 {

template <class T, class C, int DP>
struct PromptShape {
  static constexpr bool EIGHT = sizeof(C) == 1;
  static constexpr int WARPS = 11;                 // and one that loads: 3 per SM partition
  static constexpr int NT = DP == 256 ? 1 : 2;     // column groups (8 heads) of a warp
  static constexpr int COLUMNS = WARPS * NT;       // of a block
  static constexpr int SLOTS = 64;                 // keys of a stage
  static constexpr int BOX = DP * (int)sizeof(C) < 128 ? DP * (int)sizeof(C) : 128;
  static constexpr int BOXES = DP * (int)sizeof(C) / BOX;  // 128-byte columns of a row
  static constexpr int STAGE = 2 * SLOTS * DP * (int)sizeof(C);
  static constexpr int Q_BYTES = COLUMNS * 8 * DP * 2;
  static constexpr int WINDOW = 1024;              // pages marked at a time
  // what shared memory leaves (227 KB, 4 KB of static arrays and alignment)
  static constexpr int ROOM = 232448 - 4096 - Q_BYTES - WINDOW * 12;
  static constexpr int STAGES = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
  static constexpr int SMEM = 1024 + STAGES * STAGE + Q_BYTES + WINDOW * 12;
};

struct PromptParams {
  AttentionParams a;
  int tile;         // tokens of a block
  int per_token;    // column groups of a token (1, or 2 for more than 8 heads)
  int slots;        // key slots of a page piece in a stage: 16, 32, 48 or 64
  int pieces;       // pieces of a page: more than one when it has over 64 rows
  uint32_t* error;
  uint64_t limit_ns;
};

// Tiled load of a 4-D tensor (channel, head, row, page); the channel's
// coordinate starts a 128-byte (or 64-byte) box, so the copy is 16-byte aligned.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// 16 MT keys of a stage from slot `first` on, for the column groups in WHICH (a
// bit each); limit: how many of the keys each sees.
//
// The bodies are kept short on purpose: the warps are at different pages at
// any time, and a body unrolled over a whole page made them wait for
// instructions more than for anything else (2.2 ms in all instead of 0.67).  Two independent tiles (of keys,
// or of column groups) are in flight in each, to cover the latency of the chain
// products -> weights -> products.
template <class T, class C, int DP, int NT, int WHICH, int MT>
__device__ __forceinline__ void prompt_keys(float (&o)[DP / 16][NT][4], float (&m)[NT][2],
                                            float (&l)[NT][2], float (&lost)[NT][2], uint32_t keys, uint32_t values,
                                            uint32_t queries, int first, const int (&limit)[NT],
                                            const float (*factor)[8]) {
  using S = PromptShape<T, C, DP>;
  using M = typename std::conditional<S::EIGHT, __half, T>::type;
  const int lane = threadIdx.x & 31;
  auto chunk_at = [](int r, int c) -> uint32_t {
    constexpr int PER = S::BOX / 16;
    const int inside = PER == 8 ? ((c & 7) ^ (r & 7)) : ((c & 3) ^ ((r >> 1) & 3));
    return (c / PER) * (S::SLOTS * S::BOX) + r * S::BOX + inside * 16;
  };
  // ---- S^T = K Q^T
  float st[MT][NT][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      st[mt][nt][0] = st[mt][nt][1] = st[mt][nt][2] = st[mt][nt][3] = 0.0f;
  // A loop over an 8-bit cache's steps, for which the widening makes the bodies
  // twice as long: 5,229 tokens and their selection 1,064 us unrolled, 856 rolled
  // (a 16-bit cache's 748 and 815).
#pragma unroll(S::EIGHT ? 1 : DP / 32)
  for (int s = 0; s < DP / 16; s += 2) {
    uint32_t q[NT][4];  // operands of steps s and s + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      if (WHICH >> nt & 1)
        load_matrices(q[nt], queries + (uint32_t)(nt * 8 + (lane & 7)) * (DP * 2) +
                                 (((2 * s + (lane >> 3)) ^ (lane & 7)) << 4));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = first + mt * 16 + (lane & 15);
      if (S::EIGHT) {
        uint32_t a[4];
        load_matrices(a, keys + chunk_at(r, s + (lane >> 4)));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t w[4] = {widen_e4m3(a[2 * u]), widen_e4m3(a[2 * u + 1]),
                                 widen_e4m3(a[2 * u] >> 16), widen_e4m3(a[2 * u + 1] >> 16)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (WHICH >> nt & 1)
              mma16816<M>(st[mt][nt], w, q[nt][2 * u], q[nt][2 * u + 1]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a[4];
          load_matrices(a, keys + chunk_at(r, 2 * (s + u) + (lane >> 4)));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (WHICH >> nt & 1)
              mma16816<M>(st[mt][nt], a, q[nt][2 * u], q[nt][2 * u + 1]);
        }
      }
    }
  }
  // ---- scores, masked; the reference is raised where one passes it by far
  bool raise = false, partial = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (WHICH >> nt & 1) {
      const float2 f = *reinterpret_cast<const float2*>(&factor[nt][2 * (lane & 3)]);
      partial |= limit[nt] < 16 * MT;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& x = st[mt][nt][i];
          x *= i & 1 ? f.y : f.x;
          if (mt * 16 + (i >> 1) * 8 + lane / 4 >= limit[nt]) x = -INFINITY;
          raise |= x > raised_past<M>(m[nt][i & 1]);
        }
    }
  if (__any_sync(~0u, raise)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      if (WHICH >> nt & 1)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) top = fmaxf(top, fmaxf(st[mt][nt][i], st[mt][nt][i + 2]));
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
  // ---- weights
  uint32_t b[MT][NT][2], rest[MT][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (WHICH >> nt & 1) {
      const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0];
      const float m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
      float more[2] = {0.0f, 0.0f};
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float w0 = exp2_approx(st[mt][nt][2 * u] - m0);
          const float w1 = exp2_approx(st[mt][nt][2 * u + 1] - m1);
          more[0] += w0, more[1] += w1;
          const uint32_t both = pack2<M>(w0, w1);
          b[mt][nt][u] = transpose8x8(both);
          const float2 r = unpack2<M>(both);
          rest[mt][nt][u] = transpose8x8(pack2<M>(w0 - r.x, w1 - r.y));
        }
      add_kept(l[nt][0], lost[nt][0], more[0]);
      add_kept(l[nt][1], lost[nt][1], more[1]);
    }
  // ---- O^T += V^T P^T
  auto products = [&](auto masked) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      // Values of keys that a token does not see count as zero, whatever they
      // hold (a weight of zero times NaN or infinity would not): masks of the
      // operand's two keys in each half.
      uint32_t see[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = mt * 16 + 8 * u + 2 * (lane & 3);
          see[nt][u] =
              (key < limit[nt] ? 0xFFFFu : 0u) | (key + 1 < limit[nt] ? 0xFFFF0000u : 0u);
        }
      auto multiply = [&](uint32_t (&w)[4], int s) {
        auto product = [&](const uint32_t (&weights)[NT][2]) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (WHICH >> nt & 1) {
              uint32_t x[4] = {w[0], w[1], w[2], w[3]};
              if (decltype(masked)::value)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] &= see[nt][i / 2];
              mma16816<M>(o[s][nt], x, weights[nt][0], weights[nt][1]);
            }
        };
        product(b[mt]);
        if (!S::EIGHT)  // an 8-bit cache has no infinities
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = finite2<M>(w[i]);
        product(rest[mt]);
      };
      if (S::EIGHT) {
        const int r = first + mt * 16 + (lane & 15);
#pragma unroll
        for (int s = 0; s < DP / 16; s += 2) {
          uint32_t a[4];
          load_matrices_t(a, values + chunk_at(r, s + (lane >> 4)));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t e0 = __byte_perm(a[2 * u], 0, 0x3120);
            const uint32_t e1 = __byte_perm(a[2 * u + 1], 0, 0x3120);
            uint32_t w[4] = {widen_e4m3(e0), widen_e4m3(e0 >> 16), widen_e4m3(e1),
                             widen_e4m3(e1 >> 16)};
            multiply(w, s + u);
          }
        }
      } else {
        const int r = first + mt * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          uint32_t a[4];
          load_matrices_t(a, values + chunk_at(r, 2 * s + ((lane >> 3) & 1)));
          multiply(a, s);
        }
      }
    }
  };
  if (partial) products(std::true_type{});
  else products(std::false_type{});
}

template <class T, class C, int DP>
__global__ void __launch_bounds__((PromptShape<T, C, DP>::WARPS + 1) * 32, 1)
    paged_prompt_kernel(const PromptParams pp, const __grid_constant__ CUtensorMap key_map,
                        const __grid_constant__ CUtensorMap value_map) {
  using S = PromptShape<T, C, DP>;
  using M = typename std::conditional<S::EIGHT, __half, T>::type;
  constexpr int THREADS = (S::WARPS + 1) * 32, NT = S::NT;
  const AttentionParams& p = pp.a;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + ((1024 - (smem_address(raw) & 1023)) & 1023);
  uint8_t* q_mem = ring + S::STAGES * S::STAGE;  // [COLUMNS][8 heads][DP] of M
  uint32_t* marks = reinterpret_cast<uint32_t*>(q_mem + S::Q_BYTES);  // [WINDOW] column bits
  uint2* list = reinterpret_cast<uint2*>(marks + S::WINDOW);          // [WINDOW] page, columns
  __shared__ uint64_t full[S::STAGES], empty[S::STAGES];
  __shared__ float sh_factor[S::COLUMNS][8];
  __shared__ int s_row[S::COLUMNS], s_length[S::COLUMNS];  // per column group
  __shared__ int s_count[THREADS / 32];
  __shared__ int abort_flag;  // a wait gave up
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = (int)p.page.d;
  const int chunks = (p.group + 15) / 16;
  const int h = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
  const int64_t t0 = (int64_t)blockIdx.x * pp.tile;
  const int head_first = chunk * 16;                       // of the key head's query heads
  const int head_count = min(16, p.group - head_first);
  // column group c: token t0 + c / per_token, its heads head_first + 8 (c % per_token) ..
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], S::WARPS);
    }
    fence_barrier_init();
    tma_prefetch_desc(&key_map);
    tma_prefetch_desc(&value_map);
  }
  for (int c = tid; c < S::COLUMNS; c += THREADS) {
    const int64_t t = t0 + c / pp.per_token;
    int64_t row = -1;
    int length = 0;
    if (c / pp.per_token < pp.tile && t < p.tokens) {
      row = p.requests ? p.requests[t] : t;
      if (row < 0 || row >= p.rows) row = -1;
      else length = (int)min((int64_t)max(p.lengths[t], 0), min(p.width * P, (int64_t)INT32_MAX));
    }
    s_row[c] = (int)row, s_length[c] = length;
  }
  // ---- queries into shared memory: [column group][head][chunk of 16 bytes],
  // the chunks swizzled by the head
  constexpr int QC = DP / 8;  // 16-byte chunks of a head's query
  auto q_at = [](int column, int head, int c) -> uint32_t {
    return (uint32_t)(column * 8 + head) * (DP * 2) + ((c ^ head) << 4);
  };
  if (warp < S::WARPS)
    for (int i = warp * 8; i < S::COLUMNS * 8; i += S::WARPS * 8)
      for (int head = 0; head < 8; ++head) {
        const int column = i / 8;
        const int64_t t = t0 + column / pp.per_token;
        const int local = head_first + (column % pp.per_token) * 8 + head;
        const bool live = column / pp.per_token < pp.tile && t < p.tokens &&
                          local < head_first + head_count;
        const T* q = static_cast<const T*>(p.q) + t * p.q_token +
                     (int64_t)(h * p.group + local) * p.q_head;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (live && lane < QC && lane * 8 < p.dim)
          x = *reinterpret_cast<const uint4*>(q + lane * 8);
        if (S::EIGHT) {
          uint32_t* w = reinterpret_cast<uint32_t*>(&x);
          float top = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 v = unpack2<T>(w[j]);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
          const int e = query_exponent(top);
          const float by = exp2_int(e);
          if (lane == 0) sh_factor[column][head] = exp2_int(-e) * p.scale;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 v = unpack2<T>(w[j]);
            w[j] = pack2<M>(v.x * by, v.y * by);
          }
          // the order in which an 8-bit key's fragments hold the channels:
          // pairs 0 2 4 6 1 3 5 7 of each 16, two lanes to 16 channels
          uint4 other;
          other.x = __shfl_xor_sync(~0u, x.x, 1), other.y = __shfl_xor_sync(~0u, x.y, 1);
          other.z = __shfl_xor_sync(~0u, x.z, 1), other.w = __shfl_xor_sync(~0u, x.w, 1);
          x = lane & 1 ? make_uint4(other.y, other.w, x.y, x.w)
                       : make_uint4(x.x, x.z, other.x, other.z);
        } else if (lane == 0) {
          sh_factor[column][head] = p.scale;
        }
        if (lane < QC) *reinterpret_cast<uint4*>(q_mem + q_at(column, head, lane)) = x;
      }
  __syncthreads();

  const uint32_t ring_at = smem_address(ring), q_base = smem_address(q_mem);
  const int entries = S::SLOTS / pp.slots;  // page pieces of a stage
  uint32_t stage = 0, phase = 0;            // of the next stage, by both sides
  float o[DP / 16][NT][4], m[NT][2], l[NT][2], lost[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = lost[nt][0] = lost[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
  }
  bool alive = true;

  uint32_t issued = 0;  // stages that the loading lane has filled

  const int my_row = lane < S::COLUMNS ? s_row[lane] : -1;
  const int my_length = lane < S::COLUMNS ? s_length[lane] : 0;
  for (uint32_t rest = __ballot_sync(~0u, my_row >= 0); rest != 0;) {
    // the tokens of one request together
    const int row = __shfl_sync(~0u, my_row, __ffs(rest) - 1);
    const uint32_t same = __ballot_sync(~0u, my_row == row);
    rest &= ~same;
    const int longest = __reduce_max_sync(~0u, my_row == row ? my_length : 0);
    const int held = (int)p.page.div((uint32_t)longest + P - 1);
    const int32_t* table = p.table + (int64_t)row * p.width;
    for (int w0 = 0; w0 < held; w0 += S::WINDOW) {
      // ---- the window's pages that some token selected, ascending
      const int span = min(S::WINDOW, held - w0);
      for (int i = tid; i < span; i += THREADS) marks[i] = 0;
      __syncthreads();
      for (int i = tid; i < pp.tile * p.n; i += THREADS) {
        const int token = i / p.n, c = token * pp.per_token;
        if (s_row[c] != row) continue;
        const int b = p.selected[((t0 + token) * p.heads + h) * p.n + i % p.n];
        if (b >= w0 && b < w0 + span && (int64_t)b * P < s_length[c])
          atomicOr(&marks[b - w0], (pp.per_token == 2 ? 3u : 1u) << c);
      }
      __syncthreads();
      int listed = 0;
      for (int i0 = 0; i0 < span; i0 += THREADS) {
        const int i = i0 + tid;
        const uint32_t mark = i < span ? marks[i] : 0;
        int32_t page = mark ? table[w0 + i] : -1;
        const bool take = page >= 0 && page < p.pages;
        const uint32_t votes = __ballot_sync(~0u, take);
        if (lane == 0) s_count[warp] = __popc(votes);
        __syncthreads();
        int at = listed;
        for (int w = 0; w < THREADS / 32; ++w) {
          if (w < warp) at += s_count[w];
          listed += s_count[w];
        }
        if (take) {
          list[at + __popc(votes & ((1u << lane) - 1))] = make_uint2(w0 + i, mark);
          marks[i] = page;
        }
        __syncthreads();
      }
      const int units = listed * pp.pieces;
      const int stages = (units + entries - 1) / entries;

      if (warp == S::WARPS) {
        // ---- the loading warp: one lane issues the tiled copies of a stage
        if (lane == 0)
          for (int i = 0; i < stages && alive; ++i) {
            if (!mbar_wait(&empty[stage], phase ^ 1, &abort_flag, pp.limit_ns)) {
              alive = false;
              break;
            }
            const int from = i * entries, to = min(from + entries, units);
            const int rows = min(P, pp.slots);
            mbar_arrive_expect_tx(&full[stage],
                                  (uint32_t)(to - from) * 2 * S::BOXES * rows * S::BOX);
            for (int e = from; e < to; ++e) {
              const int b = list[e / pp.pieces].x, piece = e % pp.pieces;
              const int page = marks[b - w0];
              uint8_t* dst = ring + stage * S::STAGE + (e - from) * pp.slots * S::BOX;
#pragma unroll
              for (int x = 0; x < S::BOXES; ++x) {
                const int column = x * (S::BOX / (int)sizeof(C));
                tma_load_4d(dst + x * S::SLOTS * S::BOX, &key_map, &full[stage], column, h,
                            piece * S::SLOTS, page);
                tma_load_4d(dst + S::STAGE / 2 + x * S::SLOTS * S::BOX, &value_map,
                            &full[stage], column, h, piece * S::SLOTS, page);
              }
            }
            ++issued;
            if (++stage == S::STAGES) stage = 0, phase ^= 1;
          }
        __syncwarp();
      } else {
        for (int i = 0; i < stages; ++i) {
          if (alive) alive = mbar_wait(&full[stage], phase, &abort_flag, pp.limit_ns);
          alive = __all_sync(~0u, alive);
          if (!alive) break;
          const uint32_t kat = ring_at + stage * S::STAGE, vat = kat + S::STAGE / 2;
          const int from = i * entries, to = min(from + entries, units);
          for (int e = from; e < to; ++e) {
            const uint2 entry = list[e / pp.pieces];
            const uint32_t mine = (entry.y >> (warp * NT)) & ((1u << NT) - 1);
            if (mine == 0) continue;
            const int piece = e % pp.pieces;
            const int key0 = (int)entry.x * P + piece * S::SLOTS;
            const int rows = min(P - piece * S::SLOTS, pp.slots);
            int limit[NT], most = 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              limit[nt] = mine >> nt & 1 ? min(s_length[warp * NT + nt] - key0, rows) : 0;
              most = max(most, limit[nt]);
            }
            const int slot = (e - from) * pp.slots;
            const uint32_t queries = q_base + (uint32_t)warp * NT * 8 * DP * 2;
            const float(*factor)[8] = &sh_factor[warp * NT];
            int k = 0;
            auto step = [&](auto which, auto tiles) {
              constexpr int MT = decltype(tiles)::value;
              prompt_keys<T, C, DP, NT, decltype(which)::value, MT>(
                  o, m, l, lost, kat, vat, queries, slot + k, limit, factor);
              k += 16 * MT;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) limit[nt] -= 16 * MT;
            };
            using One = std::integral_constant<int, 1>;
            using Two = std::integral_constant<int, 2>;
            using Both = std::integral_constant<int, (1 << NT) - 1>;
            if (mine == 1) {
#pragma unroll 1
              while (k + 32 <= pp.slots && k < most) step(One{}, Two{});
              if (k < most) step(One{}, One{});
            } else if (NT == 2 && mine == 2) {
#pragma unroll 1
              while (k + 32 <= pp.slots && k < most)
                step(std::integral_constant<int, NT == 2 ? 2 : 1>{}, Two{});
              if (k < most) step(std::integral_constant<int, NT == 2 ? 2 : 1>{}, One{});
            } else if (NT == 2) {
#pragma unroll 1
              while (k + 32 <= pp.slots && k < most) step(Both{}, Two{});
              if (k < most) step(Both{}, One{});
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[stage]);
          if (++stage == S::STAGES) stage = 0, phase ^= 1;
        }
      }
      // before the next window's marks; a role that gave up says so to all
      if (!alive) abort_flag = 1;
      __syncthreads();
      if (abort_flag) break;
    }
    if (abort_flag) break;
  }
  if (abort_flag) {
    // the copies in flight land (or are given up too) before the block ends
    if (warp == S::WARPS && lane == 0) {
      int never = 0;
      atomicOr(pp.error, ERR_WAIT_PRODUCER);
      for (uint32_t i = issued - min(issued, (uint32_t)S::STAGES); i < issued; ++i)
        mbar_wait(&full[i % S::STAGES], (i / S::STAGES) & 1, &never, pp.limit_ns);
    }
    __syncthreads();
    return;
  }
  if (warp == S::WARPS) return;

  // ---- results: through the column group's own query memory, then in rows
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int column = warp * NT + nt;
    const int64_t t = t0 + column / pp.per_token;
    if (column / pp.per_token >= pp.tile || t >= p.tokens) continue;
    const int local = (column % pp.per_token) * 8;
    const int live = min(8, head_count - local);
    float by[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], w);
      by[i] = l[nt][i] != 0.0f ? p.v_scale / l[nt][i] : 0.0f;
      const int head = 2 * (lane & 3) + i;
      if (p.lse && lane < 4 && head < live)
        p.lse[t * p.heads * p.group + h * p.group + head_first + local + head] =
            l[nt][i] != 0.0f ? (m[nt][i] + log2f(l[nt][i])) * 0.693147180559945f : -INFINITY;
    }
    T* mem = reinterpret_cast<T*>(q_mem) + column * 8 * DP;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = k * 16 + (S::EIGHT ? 2 * (lane / 4) + (i >> 1) : lane / 4 + 8 * (i >> 1));
        const int head = 2 * (lane & 3) + (i & 1);
        mem[head * DP + ((((d >> 3) ^ head) << 3) | (d & 7))] =
            from_float<T>(o[k][nt][i] * by[i & 1]);
      }
    __syncwarp();
    T* out = static_cast<T*>(p.out) +
             (t * p.heads * p.group + h * p.group + head_first + local) * p.dim;
    for (int i = lane; i < live * QC; i += 32) {
      const int head = i / QC, c = i % QC;
      if (c * 8 < p.dim)
        *reinterpret_cast<uint4*>(out + head * p.dim + c * 8) =
            *reinterpret_cast<const uint4*>(mem + head * DP + ((c ^ head) << 3));
    }
  }
}

}  // namespace mlxvs_b200
