// Arguments of the paged-cache kernels (paged_append.cu, paged_rows.cu,
// paged_decode.cu, paged_prompt.cu)
// and the device helpers that they share: where a row stands, which keys it
// sees, where a key lives.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "m5b_internal.h"

namespace m5b {

// The batch and its cache (m5b_paged_batch with narrow integers; the ABI
// layer has checked that they fit).  Strides in elements.
struct PagedBatch {
  int tokens, batch, q_heads, kv_heads, group, head_dim;
  const int32_t* query_start;
  const int32_t* seq_lens;
  void* k_cache;
  void* v_cache;
  int num_pages, page_size;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int32_t* page_table;
  int max_pages;
  int64_t table_stride;
  int capacity;  // min(max_pages * page_size, INT_MAX): positions that pages can hold
};

struct PagedAppendArgs {
  PagedBatch b;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  const void* cos;
  const void* sin;
  int table_dtype, table_rows, rope_half, interleaved;
  void* q_out;
  int units;  // whole 16-channel units in 16-byte accesses
  int sms;
};

struct PagedAttnArgs {
  PagedBatch b;
  const void* q;
  int64_t q_token, q_head;
  void* out;
  int64_t o_token, o_head;
  float* lse;
  int max_query_len;
  float scale, softcap;
  const float* slopes;
  int window;  // INT_MAX: none
  const int32_t* prefix_lens;
  int* tickets;          // [kPagedTickets], zero between launches (decode kernel)
  void* workspace;       // the tiled kernels' PagedPartials
  unsigned int* status;  // device status word (bounded-wait errors)
};

// Tensor maps of the caches, {channel, slot, head, page}, boxes of 64
// channels x box_rows slots, 128-byte swizzle.
constexpr int kPagedBlock = 64;  // keys of a block of the tiled kernels
struct PagedMaps {
  CUtensorMap k, v;
  int box_rows;
  // The prompt kernel's rows, {channel, head, token}, boxes of 64 channels x a
  // group of heads x as many tokens as make 128 rows; where the group divides 128.
  CUtensorMap q;
  int has_q;
};

cudaError_t launch_paged_append(const PagedAppendArgs& a, int x_dtype, int cache_dtype,
                                cudaStream_t stream);
cudaError_t launch_paged_attention_rows(const PagedAttnArgs& a, int dtype, cudaStream_t stream);
// The tiled kernels: 16-bit types, 64 or 128 channels, pages of 2^k >= 8
// slots, everything on the 16-byte grid.
constexpr int kPagedTickets = 1024;  // CTAs of a decode launch, at most
constexpr int kDecodeRows = 16;  // rows per kv head and sequence that the decode kernel is for
cudaError_t launch_paged_decode(const PagedAttnArgs& a, const PagedMaps& m, int dtype, int sms,
                                cudaStream_t stream);
int64_t paged_decode_workspace(int head_dim, int sms);
cudaError_t launch_paged_prompt(const PagedAttnArgs& a, const PagedMaps& m, int dtype, int sms,
                                cudaStream_t stream);
int64_t paged_prompt_workspace(int head_dim, int sms);

// Rows of sequence b, clipped to the batch's rows whatever query_start holds.
__device__ __forceinline__ int2 paged_rows(const PagedBatch& b, int seq) {
  const int lo = max(0, min(b.query_start[seq], b.tokens));
  const int hi = max(lo, min(b.query_start[seq + 1], b.tokens));
  return make_int2(lo, hi);
}

// The sequence that row t belongs to, or -1: the last b with query_start[b] <= t.
__device__ __forceinline__ int paged_find(const PagedBatch& b, int t) {
  int lo = 0, hi = b.batch + 1;  // first index in [lo, hi) whose start is > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (b.query_start[mid] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  return (lo == 0 || lo > b.batch) ? -1 : lo - 1;
}

// Length of sequence b, its new rows included.
__device__ __forceinline__ int paged_len(const PagedBatch& b, int seq) {
  return max(0, b.seq_lens[seq]);
}

// The page of position p (0 <= p < capacity) of sequence seq, or -1.
__device__ __forceinline__ int paged_page(const PagedBatch& b, int seq, int p) {
  const int page = b.page_table[seq * b.table_stride + p / b.page_size];
  return (page >= 0 && page < b.num_pages) ? page : -1;
}

}  // namespace m5b
