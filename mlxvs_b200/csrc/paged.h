// Internal C++ API of the paged key-value cache (device pointers, stream
// ordered): page tables and slot maps of a step, cache writes with the pages'
// 8-bit bounds, page selection and attention.  No counterpart in the
// reference.  Errors: std::invalid_argument for bad arguments,
// std::runtime_error for CUDA failures.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "mlxvs_c.h"

namespace mlxvs_b200 {

void paged_tables(const int32_t* past, const int32_t* fresh, int64_t requests, int page_size,
                  const int32_t* free_pages, int64_t num_free, int32_t* table, int64_t width,
                  int64_t num_tokens, int32_t* starts, int32_t* token_requests,
                  int32_t* lengths, int64_t* slots, int32_t* used, cudaStream_t s);

void paged_store(const mlxvs_paged_cache& cache, const void* k, const void* v, int type,
                 int64_t tokens, int64_t k_token_stride, int64_t k_head_stride,
                 int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots,
                 cudaStream_t s);

void paged_select(const mlxvs_paged_cache& cache, const mlxvs_paged_queries& queries, int n,
                  int first, int last, int32_t* pages, cudaStream_t s);

void paged_attention(const mlxvs_paged_cache& cache, const mlxvs_paged_queries& queries,
                     const int32_t* pages, int n, float scale, void* out, float* lse,
                     cudaStream_t s);

}  // namespace mlxvs_b200
