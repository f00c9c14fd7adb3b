// C-ABI entry points of the paged key/value cache (declared in
// include/m5b200.h): contract checks, kernel choice, launches.  Nothing here
// allocates or synchronizes, and nothing throws.
#include <cfloat>
#include <cmath>
#include <cstdio>

#include "m5b200.h"
#include "paged.cuh"

using namespace m5b;

namespace {

int einval(const char* msg) { return set_last_error(M5B_EINVAL, msg); }
int eunsupported(const char* msg) { return set_last_error(M5B_EUNSUPPORTED, msg); }

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return set_last_error(M5B_OK, "");
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return set_last_error(M5B_ECUDA, msg);
}

bool float_dtype(int64_t dt) { return dt == M5B_F32 || dt == M5B_F16 || dt == M5B_BF16; }
bool fits_int(int64_t v) { return v >= 0 && v <= INT_MAX; }

int take_batch(const m5b_paged_batch& s, PagedBatch& d) {
  if (s.tokens < 0 || s.batch < 1 || s.q_heads < 1 || s.kv_heads < 1 || s.head_dim < 1)
    return einval("tokens, batch, heads and head_dim must be positive");
  if (s.q_heads % s.kv_heads) return einval("q_heads must be a multiple of kv_heads");
  if (s.num_pages < 1 || s.page_size < 1 || s.max_pages < 0 || s.table_stride < 0)
    return einval("the cache needs pages and a page table");
  if (!float_dtype(s.cache_dtype)) return einval("cache dtype must be float16, bfloat16 or float32");
  if (!fits_int(s.tokens) || !fits_int(s.batch) || !fits_int(s.num_pages) ||
      !fits_int(s.page_size) || !fits_int(s.max_pages) || s.q_heads > 65535 || s.head_dim > 65535)
    return eunsupported("batch or cache dimensions exceed the index range");
  // (the kernels round rows up to whole tiles, and count a token's channels)
  if (s.tokens * s.q_heads > INT_MAX - 4096 || (s.q_heads + 2 * s.kv_heads) * s.head_dim > INT_MAX)
    return eunsupported("tokens x heads or heads x head_dim exceed the index range");
  if (!s.query_start || !s.seq_lens || !s.k_cache || !s.v_cache || (!s.page_table && s.max_pages > 0))
    return einval("query_start, seq_lens, the caches and the page table are required");
  d = PagedBatch{};
  d.tokens = static_cast<int>(s.tokens);
  d.batch = static_cast<int>(s.batch);
  d.q_heads = static_cast<int>(s.q_heads);
  d.kv_heads = static_cast<int>(s.kv_heads);
  d.group = d.q_heads / d.kv_heads;
  d.head_dim = static_cast<int>(s.head_dim);
  d.query_start = s.query_start;
  d.seq_lens = s.seq_lens;
  d.k_cache = s.k_cache;
  d.v_cache = s.v_cache;
  d.num_pages = static_cast<int>(s.num_pages);
  d.page_size = static_cast<int>(s.page_size);
  d.k_page = s.k_page_stride;
  d.k_head = s.k_head_stride;
  d.k_slot = s.k_slot_stride;
  d.v_page = s.v_page_stride;
  d.v_head = s.v_head_stride;
  d.v_slot = s.v_slot_stride;
  d.page_table = s.page_table;
  d.max_pages = static_cast<int>(s.max_pages);
  d.table_stride = s.table_stride;
  const int64_t capacity = s.max_pages * s.page_size;
  d.capacity = capacity > INT_MAX ? INT_MAX : static_cast<int>(capacity);
  return M5B_OK;
}

constexpr int64_t kTicketBytes = M5B_PAGED_COUNTER_BYTES;  // first in the workspace
static_assert(kTicketBytes == kPagedTickets * sizeof(int), "a counter for each ticket");

bool pow2(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }
bool grid16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Whether the tiled kernels can take the call: 16-bit elements, 64 or 128
// channels, pages of 2^k >= 8 slots (a box of the swizzled copy is whole
// 8-row groups) and all rows on the 16-byte grid.
bool tiled(const PagedAttnArgs& a, int64_t dtype) {
  const PagedBatch& b = a.b;
  if (dtype == M5B_F32 || (b.head_dim != 64 && b.head_dim != 128)) return false;
  if (!pow2(b.page_size) || b.page_size < 8) return false;
  const int64_t strides[] = {b.k_page, b.k_head, b.k_slot, b.v_page, b.v_head, b.v_slot,
                             a.q_token, a.q_head, a.o_token, a.o_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return false;
  return grid16(b.k_cache) && grid16(b.v_cache) && grid16(a.q) && grid16(a.out);
}

// Whether appending can go by 16-channel units: heads and their rotated part
// are whole units, and all rows (8 table entries too) are on the 16-byte grid.
// 9914 rows of 32 + 8 + 8 heads of 128 take 47 us so, 127 by channel pairs.
bool whole_units(const PagedAppendArgs& a) {
  const PagedBatch& b = a.b;
  if (b.head_dim % 16 || b.head_dim > 1024 || a.rope_half % 8) return false;
  const int64_t strides[] = {b.k_page, b.k_head, b.k_slot, b.v_page, b.v_head, b.v_slot,
                             a.k_token, a.k_head, a.v_token, a.v_head, a.q_token, a.q_head};
  for (int64_t s : strides)
    if (s % 8) return false;
  return grid16(b.k_cache) && grid16(b.v_cache) && grid16(a.q) && grid16(a.k) && grid16(a.v) &&
         grid16(a.q_out) && (!a.rope_half || (grid16(a.cos) && grid16(a.sin)));
}

// Boxes of up to kPagedBlock slots x 64 channels of one head of one page.
bool cache_map(CUtensorMap* map, const void* ptr, const PagedBatch& b, bool f16, int64_t page,
               int64_t head, int64_t slot, int box_rows) {
  const uint64_t dims[4] = {uint64_t(b.head_dim), uint64_t(b.page_size), uint64_t(b.kv_heads),
                            uint64_t(b.num_pages)};
  const uint64_t strides[3] = {uint64_t(slot) * 2, uint64_t(head) * 2, uint64_t(page) * 2};
  const uint32_t box[4] = {64, uint32_t(box_rows), 1, 1};
  return make_swizzled_map16(map, f16, 4, ptr, dims, strides, box);
}

void row_map(PagedMaps& m, const PagedAttnArgs& a, int64_t dtype) {
  const PagedBatch& b = a.b;
  m.has_q = 0;
  if (128 % b.group || a.q_head == 0 || a.q_token == 0) return;
  const uint64_t dims[3] = {uint64_t(b.head_dim), uint64_t(b.q_heads), uint64_t(b.tokens)};
  const uint64_t strides[2] = {uint64_t(a.q_head) * 2, uint64_t(a.q_token) * 2};
  const uint32_t box[3] = {64, uint32_t(b.group), uint32_t(128 / b.group)};
  m.has_q = make_swizzled_map16(&m.q, dtype == M5B_F16, 3, a.q, dims, strides, box) ? 1 : 0;
}

bool cache_maps(PagedMaps& m, const PagedAttnArgs& a, int64_t dtype) {
  const PagedBatch& b = a.b;
  m.box_rows = b.page_size < kPagedBlock ? b.page_size : kPagedBlock;
  return cache_map(&m.k, b.k_cache, b, dtype == M5B_F16, b.k_page, b.k_head, b.k_slot, m.box_rows) &&
         cache_map(&m.v, b.v_cache, b, dtype == M5B_F16, b.v_page, b.v_head, b.v_slot, m.box_rows);
}

}  // namespace

extern "C" {

int m5b_paged_append(const m5b_paged_append_args* s, void* stream) {
  if (!s) return einval("arguments are NULL");
  PagedAppendArgs a{};
  int rc = take_batch(s->b, a.b);
  if (rc) return rc;
  if (!float_dtype(s->x_dtype)) return einval("input dtype must be float16, bfloat16 or float32");
  if (s->rope_half < 0 || 2 * s->rope_half > s->b.head_dim)
    return einval("the rotated channels must fit the head");
  if (s->rope_half > 0) {
    if (!s->cos || !s->sin || s->table_rows < 1) return einval("cos and sin tables are required");
    if (!float_dtype(s->table_dtype)) return einval("cos and sin must have floating dtype");
    if (!fits_int(s->table_rows)) return eunsupported("cos and sin tables exceed the index range");
  }
  if (s->b.tokens == 0) return set_last_error(M5B_OK, "");
  if (!s->k || !s->v) return einval("k and v are required");
  if (s->q && !s->q_out) return einval("q_out is required with q");
  a.q = s->q;
  a.k = s->k;
  a.v = s->v;
  a.q_token = s->q_token_stride;
  a.q_head = s->q_head_stride;
  a.k_token = s->k_token_stride;
  a.k_head = s->k_head_stride;
  a.v_token = s->v_token_stride;
  a.v_head = s->v_head_stride;
  a.cos = s->cos;
  a.sin = s->sin;
  a.table_dtype = static_cast<int>(s->table_dtype);
  a.table_rows = static_cast<int>(s->table_rows);
  a.rope_half = static_cast<int>(s->rope_half);
  a.interleaved = s->interleaved ? 1 : 0;
  a.q_out = s->q_out;
  a.units = whole_units(a) ? 1 : 0;
  if ((rc = current_device_state(nullptr, &a.sms))) return rc;
  return launched(launch_paged_append(a, static_cast<int>(s->x_dtype),
                                      static_cast<int>(s->b.cache_dtype),
                                      static_cast<cudaStream_t>(stream)),
                  "paged append launch");
}

int64_t m5b_paged_attention_workspace_bytes(int64_t head_dim) {
  int sms = 0;
  if ((head_dim != 64 && head_dim != 128) || current_device_state(nullptr, &sms)) return 0;
  const int64_t few = paged_decode_workspace(static_cast<int>(head_dim), sms);
  const int64_t many = paged_prompt_workspace(static_cast<int>(head_dim), sms);
  return kTicketBytes + (few > many ? few : many);
}

int m5b_paged_attention(const m5b_paged_attention_args* s, void* stream) {
  if (!s) return einval("arguments are NULL");
  PagedAttnArgs a{};
  int rc = take_batch(s->b, a.b);
  if (rc) return rc;
  if (s->b.head_dim > 256) return eunsupported("head_dim above 256 is unsupported");
  // (as fp32, in which the kernels scale, times log2 e too: -inf * 0 would make
  // hidden scores NaN)
  const float scale = static_cast<float>(s->scale);
  if (!(scale > 0.0f) || !std::isfinite(scale * 1.4426950408889634f))
    return einval("scale must be a positive finite real scalar");
  if (!(s->softcap >= 0.0) || !std::isfinite(static_cast<float>(s->softcap)) ||
      (s->softcap > 0.0 && s->softcap < FLT_MIN))
    return einval("softcap must be a positive finite real scalar");
  if (s->window < 0) return einval("window must be positive");
  if (s->max_query_len < 0) return einval("max_query_len must not be negative");
  if (s->b.tokens == 0) return set_last_error(M5B_OK, "");
  if (!s->q || !s->out) return einval("q and out are required");
  a.q = s->q;
  a.q_token = s->q_token_stride;
  a.q_head = s->q_head_stride;
  a.out = s->out;
  a.o_token = s->out_token_stride;
  a.o_head = s->out_head_stride;
  a.lse = s->lse;
  a.max_query_len = s->max_query_len > INT_MAX ? INT_MAX : static_cast<int>(s->max_query_len);
  a.scale = scale;
  a.softcap = static_cast<float>(s->softcap);
  a.slopes = s->slopes;
  a.window = s->window == 0 || s->window > INT_MAX ? INT_MAX : static_cast<int>(s->window);
  a.prefix_lens = s->prefix_lens;
  const int dtype = static_cast<int>(s->b.cache_dtype);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tiled(a, dtype)) {
    int sms = 0;
    rc = current_device_state(&a.status, &sms);
    if (rc) return rc;
    a.tickets = static_cast<int*>(s->workspace);
    a.workspace = static_cast<uint8_t*>(s->workspace) + kTicketBytes;
    if (!s->workspace || !grid16(s->workspace) || 2 * sms > kPagedTickets ||
        s->workspace_bytes < m5b_paged_attention_workspace_bytes(a.b.head_dim))
      return einval("workspace of m5b_paged_attention_workspace_bytes(head_dim) bytes required");
    // Up to 16 rows a kv head the decode kernel, beyond that the prompt kernel,
    // for 4 (16) rows: 158 (165) against 179 us for 4 sequences of 60000 keys,
    // 54 (55) against 58 for 16 of 4000, 9.4 (12.9) against 13.7 for one of 517;
    // for 24 rows, two tiles of 16: 305 against 184 and 69 against 59.
    const bool few = int64_t(a.max_query_len) * a.b.group <= kDecodeRows;
    PagedMaps m{};
    if (!few) row_map(m, a, dtype);
    if (cache_maps(m, a, dtype))
      return launched(few ? launch_paged_decode(a, m, dtype, sms, st)
                          : launch_paged_prompt(a, m, dtype, sms, st),
                      "paged attention launch");
  }
  return launched(launch_paged_attention_rows(a, dtype, st),
                  "paged attention launch");
}

}  // extern "C"
