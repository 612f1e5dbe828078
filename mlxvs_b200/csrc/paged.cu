// Host side of the paged key-value cache: argument checks and launches.
#include "paged.h"

#include <cmath>
#include <cstring>
#include <type_traits>

#include "host.h"
#include "paged_attention.cuh"
#include "paged_prompt.cuh"
#include "paged_select.cuh"
#include "paged_store.cuh"
#include "paged_tables.cuh"

namespace mlxvs_b200 {

namespace {

constexpr int MAX_DIM = 256;
constexpr int MAX_PAGE = 1024;
constexpr int MAX_SELECTED = 256;

// Argument checks: the message is only put together when one fails (a call's
// checks would otherwise take longer than its launch).
#define REQUIRE(ok, msg)                                          \
  do {                                                            \
    if (!(ok)) throw std::invalid_argument(std::string(op) + (msg)); \
  } while (0)

int type_size(int type) { return type == MLXVS_FLOAT8_E4M3 ? 1 : 2; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Calls f(T{}, C{}) with the element types of queries and cache.
template <class F>
void dispatch_types(int type, int cache_type, F&& f) {
  if (type == MLXVS_FLOAT16 && cache_type == MLXVS_FLOAT16)
    f(__half{}, __half{});
  else if (type == MLXVS_FLOAT16)
    f(__half{}, __nv_fp8_e4m3{});
  else if (cache_type == MLXVS_BFLOAT16)
    f(__nv_bfloat16{}, __nv_bfloat16{});
  else
    f(__nv_bfloat16{}, __nv_fp8_e4m3{});
}

void check_types(const char* op, int type, int cache_type) {
  REQUIRE(type == MLXVS_FLOAT16 || type == MLXVS_BFLOAT16,
          "queries, keys and values must be float16 or bfloat16.");
  REQUIRE(cache_type == type || cache_type == MLXVS_FLOAT8_E4M3,
          "the cache must have their type or be float8_e4m3.");
}

// Shape, strides and alignment of the cache's tensors.
void check_cache(const char* op, const mlxvs_paged_cache& c, bool rows) {
  REQUIRE(c.pages >= 0 && c.pages < (1LL << 31), "the number of pages must be in [0, 2^31).");
  REQUIRE(c.page_size >= 1 && c.page_size <= MAX_PAGE, "page_size must be in [1, 1024].");
  REQUIRE(c.heads >= 1 && c.heads <= 4096, "the key heads must be in [1, 4096].");
  const int unit = 16 / type_size(c.type);
  const int d_unit = rows ? unit : 8;
  REQUIRE(c.dim >= d_unit && c.dim <= MAX_DIM && c.dim % d_unit == 0,
          "the head dimension must be a multiple of " + std::to_string(d_unit) +
                                " and at most 256.");
  if (!rows) return;
  REQUIRE(c.pages == 0 || (c.keys != nullptr && c.values != nullptr),
          "keys and values must not be NULL.");
  REQUIRE(aligned16(c.keys) && aligned16(c.values), "keys and values must be 16-byte aligned.");
  // a dimension of one element may have any stride
  const int64_t strides[6][2] = {
      {c.pages, c.key_page_stride},   {c.page_size, c.key_row_stride},
      {c.heads, c.key_head_stride},   {c.pages, c.value_page_stride},
      {c.page_size, c.value_row_stride}, {c.heads, c.value_head_stride}};
  for (const auto& s : strides)
    REQUIRE(s[0] <= 1 || (s[1] >= 0 && s[1] % unit == 0),
            "the cache's strides must be multiples of 16 bytes and not negative.");
  REQUIRE(std::isfinite(c.key_scale) && c.key_scale > 0 && std::isfinite(c.value_scale) &&
              c.value_scale > 0, "k_scale and v_scale must be positive and finite.");
  REQUIRE(std::isfinite(1.0f / c.key_scale) && std::isfinite(1.0f / c.value_scale),
          "k_scale and v_scale must have finite reciprocals.");
}

void check_codes(const char* op, const mlxvs_paged_cache& c) {
  REQUIRE(c.codes != nullptr && c.scales != nullptr, "codes and scales must not be NULL.");
  REQUIRE(aligned16(c.codes), "codes must be 16-byte aligned.");
}

void check_queries(const char* op, const mlxvs_paged_cache& c,
                   const mlxvs_paged_queries& q) {
  check_types(op, q.type, c.type);
  REQUIRE(q.tokens >= 0 && q.tokens < (1LL << 31), "the tokens must be in [0, 2^31).");
  REQUIRE(q.heads >= 1 && q.heads % c.heads == 0 && q.heads / c.heads <= 128,
          "the query heads must be 1 to 128 times the key heads.");
  REQUIRE(q.rows >= 0 && q.rows < (1LL << 31) && q.width >= 0 && q.width < (1LL << 31),
          "the table must be int32 [requests, width].");
  REQUIRE(q.tokens == 0 || (q.q != nullptr && q.lengths != nullptr),
          "q and lengths must not be NULL.");
  REQUIRE(q.table != nullptr || q.rows * q.width == 0, "table must not be NULL.");
  REQUIRE(q.requests != nullptr || q.tokens <= q.rows,
          "without requests every token needs a row of the table.");
  REQUIRE(aligned16(q.q) &&
              (q.tokens <= 1 || (q.token_stride >= 0 && q.token_stride % 8 == 0)) &&
              (q.heads <= 1 || (q.head_stride >= 0 && q.head_stride % 8 == 0)),
          "q must be 16-byte aligned, with strides of multiples of 16 bytes.");
}

// What the kernels' static arrays may take of a block's shared memory.
constexpr int STATIC_SMEM = 16384;

// More than 48 KB of shared memory, static arrays among it, has to be asked for.
// The limit belongs to the kernel, not to the call, and other threads launch it
// too: `most` is one number for all of a kernel's calls.
template <class K>
void allow_smem(K* kernel, size_t bytes, size_t most) {
  if (bytes > 32 * 1024)
    CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
}

// The attention kernel on every SM and, when it may have cut rows, the kernel
// that joins them, launched so that it is ready when the first one ends.
template <class T, class C, int DP, int NT>
void launch_attention(AttentionParams p, DeviceInfo& dev, Scratch& scratch, cudaStream_t s) {
  using S = AttentionShape<T, C, DP, NT>;
  auto* kernel = p.selected ? paged_attention_kernel<T, C, DP, NT, true>
                            : paged_attention_kernel<T, C, DP, NT, false>;
  allow_smem(kernel, S::SMEM, S::SMEM);
  // Rows of few tiles are not cut: a block each, and no second kernel.  Longest
  // possible rows of 8 tiles: two requests of up to 300 keys 8.1 -> 6.0 us in a
  // graph (and one launch less on the host), 415 tokens with 9 pages of 24 and
  // their selection 31.3 -> 30.0 us.
  const int64_t keys = (p.selected ? (int64_t)p.n : p.width) * p.page.d;
  const int64_t all = p.tokens * p.heads * ((p.group + S::HEADS - 1) / S::HEADS);
  if (keys <= 8 * S::KEYS && all < (1LL << 31)) {
    p.whole = 1;
    ProfScope prof("paged_attention", s);
    kernel<<<(unsigned)all, S::WARPS * 32, S::SMEM, s>>>(p);
    CK(cudaGetLastError());
    return;
  }
  const int blocks = dev.sms * S::BLOCKS;
  p.cut = scratch.alloc<int4>(blocks + ((size_t)blocks * 2 * S::PART + 3) / 4);
  p.part = reinterpret_cast<float*>(p.cut + blocks);
  {
    ProfScope prof("paged_attention", s);
    kernel<<<blocks, S::WARPS * 32, S::SMEM, s>>>(p);
    CK(cudaGetLastError());
  }
  ProfScope prof("paged_attention_join", s);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks, std::min(p.group, S::HEADS));
  config.blockDim = dim3(DP);
  config.stream = s;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  CK(cudaLaunchKernelEx(&config, paged_attention_join_kernel<T, DP, NT>, p));
}

// Keys or values as a 4-D tensor (channel, head, row, page) whose boxes are
// up to 128 bytes of channels and 64 rows of one head and page.
template <class C>
CUtensorMap cache_map(const void* base, const AttentionParams& p, int64_t head_stride,
                      int64_t row_stride, int64_t page_stride, int box_bytes) {
  CUtensorMap m;
  std::memset(&m, 0, sizeof(m));
  const cuuint64_t size = sizeof(C);
  const cuuint64_t dims[4] = {(cuuint64_t)p.dim, (cuuint64_t)p.heads, p.page.d,
                              (cuuint64_t)p.pages};
  // a dimension of one element may have any stride: one that the map accepts
  const cuuint64_t strides[3] = {dims[1] > 1 ? head_stride * size : 16,
                                 dims[2] > 1 ? row_stride * size : 16,
                                 dims[3] > 1 ? page_stride * size : 16};
  const cuuint32_t box[4] = {(cuuint32_t)(box_bytes / size), 1, std::min(p.page.d, 64u), 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = encode_fn()(
      &m, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
      const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
      box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    throw std::runtime_error("[mlxvs_b200] cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return m;
}

// Whether selected pages are walked by tiles of tokens: prompts with enough
// tiles for the SMs, and a cache that a tensor map can describe.  Pages of under
// 16 rows would leave most of a stage empty.  A tile walks its requests one after
// another, so it needs many tokens of each; the host knows the tokens and the
// table's rows, idle ones among them, so what it asks for is 32 tokens a row.
// Attention of 16 pages of 64 a token, by tiles and by rows of their own pages:
// 400 tokens (8 key heads of 4, bf16) of 200 requests 564 and 247 us, of 50
// requests 255 and 244, of 25 189 and 197, of one 142 and 172; 1,000 tokens (4 key
// heads of 8) of 125 requests 328 and 305, of 31 211 and 221, of 10 195 and 221;
// 5,229 tokens of 3 requests 768 and 1110.
template <class T, class C, int DP>
bool prompt_tiles(const AttentionParams& p, const DeviceInfo& dev) {
  using S = PromptShape<T, C, DP>;
  if (p.selected == nullptr || p.tokens < 32 * p.rows || p.page.d < 16 || p.pages == 0) return false;
  const int64_t limit = (1LL << 40) / (int64_t)sizeof(C);
  for (int64_t s : {p.key_page, p.value_page})
    if (p.pages > 1 && (s == 0 || s >= limit)) return false;
  for (int64_t s : {p.key_row, p.value_row})
    if (s == 0 || s >= limit) return false;
  for (int64_t s : {p.key_head, p.value_head})
    if (p.heads > 1 && (s == 0 || s >= limit)) return false;
  const int64_t tile = S::COLUMNS / (p.group > 8 ? 2 : 1);
  return (p.tokens + tile - 1) / tile * p.heads * ((p.group + 15) / 16) >= dev.sms;
}

template <class T, class C, int DP>
void launch_prompt(const AttentionParams& p, DeviceInfo& dev, cudaStream_t s) {
  using S = PromptShape<T, C, DP>;
  PromptParams pp;
  pp.a = p;
  pp.per_token = p.group > 8 ? 2 : 1;
  pp.tile = S::COLUMNS / pp.per_token;
  pp.slots = std::min((int)(p.page.d + 15) / 16 * 16, S::SLOTS);
  pp.pieces = (int)(p.page.d + S::SLOTS - 1) / S::SLOTS;
  pp.error = dev.err;
  pp.limit_ns = WAIT_LIMIT_NS;
  const CUtensorMap keys =
      cache_map<C>(p.keys, p, p.key_head, p.key_row, p.key_page, S::BOX);
  const CUtensorMap values =
      cache_map<C>(p.values, p, p.value_head, p.value_row, p.value_page, S::BOX);
  auto* kernel = paged_prompt_kernel<T, C, DP>;
  allow_smem(kernel, S::SMEM, S::SMEM);
  const dim3 grid((unsigned)((p.tokens + pp.tile - 1) / pp.tile),
                  p.heads * ((p.group + 15) / 16));
  ProfScope prof("paged_prompt", s);
  kernel<<<grid, (S::WARPS + 1) * 32, S::SMEM, s>>>(pp, keys, values);
  CK(cudaGetLastError());
}

}  // namespace

void paged_tables(const int32_t* past, const int32_t* fresh, int64_t requests, int page_size,
                  const int32_t* free_pages, int64_t num_free, int32_t* table, int64_t width,
                  int64_t num_tokens, int32_t* starts, int32_t* token_requests,
                  int32_t* lengths, int64_t* slots, int32_t* used, cudaStream_t s) {
  const char* op = "[mlxvs::paged_tables] ";
  REQUIRE(requests >= 0 && requests < (1LL << 31), "the requests must be in [0, 2^31).");
  REQUIRE(page_size >= 1 && page_size <= MAX_PAGE, "page_size must be in [1, 1024].");
  REQUIRE(num_tokens >= 0 && num_tokens < (1LL << 31) - TABLES_TOKENS,
          "num_tokens must be in [0, 2^31).");
  REQUIRE(num_free >= 0 && width >= 0 && width < (1LL << 31),
          "the table must be int32 [requests, width].");
  REQUIRE(requests == 0 || (past != nullptr && fresh != nullptr),
          "past and fresh must not be NULL.");
  REQUIRE(requests * width == 0 || table != nullptr, "table must not be NULL.");
  REQUIRE(num_free == 0 || free_pages != nullptr, "free_pages must not be NULL.");
  REQUIRE(starts != nullptr && used != nullptr &&
              (num_tokens == 0 ||
               (token_requests != nullptr && lengths != nullptr && slots != nullptr)), "outputs must not be NULL.");
  device_info();
  const TablesParams p{past,  fresh,      requests, FastDiv((uint32_t)page_size), free_pages,
                       num_free, table,  width,    num_tokens, starts, token_requests,
                       lengths, slots, used};
  const unsigned blocks =
      (unsigned)std::max<int64_t>(1, (num_tokens + TABLES_TOKENS - 1) / TABLES_TOKENS);
  ProfScope prof("paged_tables", s);
  // one pass over up to 256 requests, or 1024 (a request a thread is quicker)
  if (requests <= TABLES_THREADS)
    paged_tables_kernel<1><<<blocks, TABLES_THREADS, 0, s>>>(p);
  else
    paged_tables_kernel<4><<<blocks, TABLES_THREADS, 0, s>>>(p);
  CK(cudaGetLastError());
}

void paged_store(const mlxvs_paged_cache& c, const void* k, const void* v, int type,
                 int64_t tokens, int64_t k_token, int64_t k_head, int64_t v_token,
                 int64_t v_head, const int64_t* slots, cudaStream_t s) {
  const char* op = "[mlxvs::paged_store] ";
  check_types(op, type, c.type);
  check_cache(op, c, true);
  REQUIRE(tokens >= 0 && tokens < (1LL << 31), "the tokens must be in [0, 2^31).");
  REQUIRE(tokens == 0 || (k != nullptr && v != nullptr && slots != nullptr),
          "k, v and slots must not be NULL.");
  REQUIRE(aligned16(k) && aligned16(v), "k and v must be 16-byte aligned.");
  for (int64_t x : {k_token, v_token})
    REQUIRE(tokens <= 1 || (x >= 0 && x % 8 == 0),
            "the strides of k and v must be multiples of 16 bytes.");
  for (int64_t x : {k_head, v_head})
    REQUIRE(c.heads <= 1 || (x >= 0 && x % 8 == 0),
            "the strides of k and v must be multiples of 16 bytes.");
  // rows that share memory would be written by several blocks at a time
  REQUIRE((c.pages <= 1 || (c.key_page_stride > 0 && c.value_page_stride > 0)) &&
              (c.page_size <= 1 || (c.key_row_stride > 0 && c.value_row_stride > 0)) &&
              (c.heads <= 1 || (c.key_head_stride > 0 && c.value_head_stride > 0)),
          "the cache's rows must lie apart: strides of 0 can only be read.");
  if (c.codes != nullptr || c.scales != nullptr) check_codes(op, c);
  DeviceInfo& dev = device_info();
  if (tokens == 0 || c.pages == 0) return;
  StoreParams p{k, v, tokens, k_token, k_head, v_token, v_head, slots, c.keys, c.values,
                c.key_page_stride, c.key_row_stride, c.key_head_stride,
                c.value_page_stride, c.value_row_stride, c.value_head_stride,
                c.pages, FastDiv((uint32_t)c.page_size), c.heads, c.dim,
                1.0f / c.key_scale, 1.0f / c.value_scale, c.codes, c.scales};
  // Chunks of one token while that fills the GPU (single tokens end a page's
  // rows each, so a chunk of them would go one after another), 16 at most (of 4,
  // 8, 16 and 32: 28.9, 24.0, 23.7 and 27.4 us for 13,881 tokens).
  const int64_t chunk =
      std::max<int64_t>(1, std::min<int64_t>(16, tokens * c.heads / (dev.sms * 16)));
  const dim3 grid((unsigned)((tokens + chunk - 1) / chunk),
                  (c.heads + STORE_WARPS - 1) / STORE_WARPS);
  ProfScope prof("paged_store", s);
  dispatch_types(type, c.type, [&](auto t, auto ct) {
    auto lanes = [&](auto n) {
      paged_store_kernel<decltype(t), decltype(ct), decltype(n)::value>
          <<<grid, STORE_WARPS * 32, 0, s>>>(p, (int)chunk);
    };
    if (c.dim <= 64) lanes(std::integral_constant<int, 8>{});
    else if (c.dim <= 128) lanes(std::integral_constant<int, 16>{});
    else lanes(std::integral_constant<int, 32>{});
  });
  CK(cudaGetLastError());
}

void paged_select(const mlxvs_paged_cache& c, const mlxvs_paged_queries& q, int n, int first,
                  int last, int32_t* pages, cudaStream_t s) {
  const char* op = "[mlxvs::paged_select] ";
  check_cache(op, c, false);
  check_codes(op, c);
  check_queries(op, c, q);
  REQUIRE(n >= 1 && n <= MAX_SELECTED, "n must be in [1, 256].");
  REQUIRE(first >= 0 && last >= 0 && first <= n && last <= n - first,
          "first and last must be at least 0 and together at most n.");
  REQUIRE(q.tokens == 0 || pages != nullptr, "pages must not be NULL.");
  DeviceInfo& dev = device_info();
  // keys of one token and the static arrays must fit a block's shared memory
  const int64_t room = (dev.max_smem - STATIC_SMEM) / 4;
  REQUIRE(q.width <= room,
          "the table must have at most " + std::to_string(room) + " pages a request.");
  if (q.tokens == 0) return;
  int shift = 0;
  while ((1 << shift) < q.heads / c.heads) ++shift;
  const SelectParams p{q.q, q.tokens, q.token_stride, q.head_stride, c.heads,
                       q.heads / c.heads, c.dim, shift, c.codes, c.scales, c.pages, q.table,
                       q.rows, q.width, q.requests, q.lengths, FastDiv((uint32_t)c.page_size),
                       n, first, last, pages};
  // Prompts (more tokens than requests) share the pages' codes between 8 tokens
  // of a tile; single tokens have pages of their own.  By tiles and by tokens: 400
  // tokens (8 key heads of 4, up to 63 pages) of 200 requests 15 and 31 us, of one
  // 10 and 30; 5,229 tokens of 3 requests 58 and 229.  Clusters share the pages
  // of few tiles among more SMs: 7 requests of up to 250,000 keys took 91 us
  // without clusters and 33 with up to 8 blocks, 256 rows of up to 500 pages 23
  // us without and 31 with 4.
  const bool tiles = q.tokens > q.rows && 8 * q.width <= room;
  const int64_t units = (q.tokens + (tiles ? 7 : 0)) / (tiles ? 8 : 1);
  int cluster = 1;
  while (cluster < 8 && units * c.heads * cluster < 2 * dev.sms && cluster * 128 < q.width)
    cluster *= 2;
  ProfScope prof("paged_select", s);
  dispatch_types(q.type, q.type, [&](auto t, auto) {
    using T = decltype(t);
    auto* kernel = p.dim <= 64    ? tiles ? paged_select_kernel<T, 8, 2>
                                          : paged_select_kernel<T, 1, 2>
                   : p.dim <= 128 ? tiles ? paged_select_kernel<T, 8, 4>
                                          : paged_select_kernel<T, 1, 4>
                   : tiles        ? paged_select_kernel<T, 8, 8>
                                  : paged_select_kernel<T, 1, 8>;
    const size_t smem = (size_t)(tiles ? 8 : 1) * q.width * 4;
    allow_smem(kernel, smem, dev.max_smem - STATIC_SMEM);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(units * cluster), c.heads);
    config.blockDim = dim3(SELECT_WARPS * 32);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    CK(cudaLaunchKernelEx(&config, kernel, p));
  });
}

void paged_attention(const mlxvs_paged_cache& c, const mlxvs_paged_queries& q,
                     const int32_t* pages, int n, float scale, void* out, float* lse,
                     cudaStream_t s) {
  const char* op = "[mlxvs::paged_attention] ";
  check_cache(op, c, true);
  check_queries(op, c, q);
  REQUIRE(pages == nullptr || (n >= 1 && n <= (1 << 20)),
          "pages must be int32 [tokens, key heads, n], n at most 2^20.");
  REQUIRE(std::isfinite(scale), "scale must be finite.");
  REQUIRE(q.tokens == 0 || out != nullptr, "out must not be NULL.");
  REQUIRE(aligned16(out), "out must be 16-byte aligned.");
  DeviceInfo& dev = device_info();
  if (q.tokens == 0) return;
  const float log2e = 1.44269504088896f;
  AttentionParams p{q.q, q.tokens, q.token_stride, q.head_stride, c.heads, q.heads / c.heads,
                    c.dim, c.keys, c.values, c.key_page_stride, c.key_row_stride,
                    c.key_head_stride, c.value_page_stride, c.value_row_stride,
                    c.value_head_stride, c.pages, FastDiv((uint32_t)c.page_size), q.table,
                    q.rows, q.width, q.requests, q.lengths, pages, n, scale * c.key_scale * log2e,
                    c.value_scale, out, lse, nullptr, nullptr, 0};
  Scratch scratch(s);
  dispatch_types(q.type, c.type, [&](auto t, auto ct) {
    auto shaped = [&](auto dp, auto nt) {
      launch_attention<decltype(t), decltype(ct), decltype(dp)::value, decltype(nt)::value>(
          p, dev, scratch, s);
    };
    auto wide = [&](auto dp) {
      if (prompt_tiles<decltype(t), decltype(ct), decltype(dp)::value>(p, dev))
        launch_prompt<decltype(t), decltype(ct), decltype(dp)::value>(p, dev, s);
      else if (p.group <= 8) shaped(dp, std::integral_constant<int, 1>{});
      else shaped(dp, std::integral_constant<int, 2>{});
    };
    if (p.dim <= 64) wide(std::integral_constant<int, 64>{});
    else if (p.dim <= 128) wide(std::integral_constant<int, 128>{});
    else wide(std::integral_constant<int, 256>{});
  });
}

}  // namespace mlxvs_b200
