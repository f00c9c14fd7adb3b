// Appending keys and values to a paged cache, positions rotated on the way
// (m5b_paged_append).
//
// One CTA per new row; a thread takes channel pairs of the row's query, key
// and value heads in turn.  A rotated pair is
//   (a c - b s, b c + a s)
// with one rounding per product and sum in FP32, then one to the cache's type.
#include "paged.cuh"

namespace m5b {
namespace {

constexpr int kThreads = 256;

template <typename TX, typename TC>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppendArgs a) {
  const PagedBatch& b = a.b;
  const int t = blockIdx.x;
  const int d = b.head_dim;
  __shared__ int s_pos, s_page;
  if (threadIdx.x == 0) {
    const int seq = paged_find(b, t);
    int pos = -1, page = -1;
    if (seq >= 0) {
      const int2 rows = paged_rows(b, seq);
      pos = paged_len(b, seq) - (rows.y - t);
      if (pos >= 0 && pos < b.capacity) page = paged_page(b, seq, pos);
      if (a.rope_half > 0 && pos >= a.table_rows) pos = page = -1;
    }
    s_pos = pos;
    s_page = page;
  }
  __syncthreads();
  const int pos = s_pos, page = s_page;
  const int64_t slot = pos >= 0 ? pos % b.page_size : 0;
  const int pairs = (d + 1) / 2, r = a.rope_half;
  const int heads = (a.q ? b.q_heads : 0) + 2 * b.kv_heads;
  for (int u = threadIdx.x; u < heads * pairs; u += kThreads) {
    int h = u / pairs;
    const int p = u % pairs;
    const TX* src;
    TC* dst;
    bool turn = r > 0, store;
    const int nq = a.q ? b.q_heads : 0;
    if (h < nq) {
      src = static_cast<const TX*>(a.q) + int64_t(t) * a.q_token + h * a.q_head;
      dst = static_cast<TC*>(a.q_out) + (int64_t(t) * b.q_heads + h) * d;
      store = true;
    } else if (h < nq + b.kv_heads) {
      h -= nq;
      src = static_cast<const TX*>(a.k) + int64_t(t) * a.k_token + h * a.k_head;
      dst = static_cast<TC*>(b.k_cache) + page * b.k_page + h * b.k_head + slot * b.k_slot;
      store = page >= 0;
    } else {
      h -= nq + b.kv_heads;
      src = static_cast<const TX*>(a.v) + int64_t(t) * a.v_token + h * a.v_head;
      dst = static_cast<TC*>(b.v_cache) + page * b.v_page + h * b.v_head + slot * b.v_slot;
      store = page >= 0;
      turn = false;
    }
    if (!store) continue;
    int i0 = 2 * p, i1 = 2 * p + 1;
    if (turn && !a.interleaved && p < r) i0 = p, i1 = p + r;
    if (pos < 0) {  // only queries get here
      dst[i0] = from_f32<TC>(0.0f);
      if (i1 < d) dst[i1] = from_f32<TC>(0.0f);
      continue;
    }
    float x = to_f32(src[i0]), y = i1 < d ? to_f32(src[i1]) : 0.0f;
    if (turn && p < r) {
      const float c = load_param(a.cos, a.table_dtype, int64_t(pos) * r + p);
      const float s = load_param(a.sin, a.table_dtype, int64_t(pos) * r + p);
      const float x0 = x;
      x = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
      y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x0, s));
    }
    dst[i0] = from_f32<TC>(x);
    if (i1 < d) dst[i1] = from_f32<TC>(y);
  }
}

template <typename TX, typename TC>
cudaError_t launch(const PagedAppendArgs& a, cudaStream_t stream) {
  paged_append_kernel<TX, TC><<<a.b.tokens, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename TX>
cudaError_t by_cache(const PagedAppendArgs& a, int cache_dtype, cudaStream_t stream) {
  switch (cache_dtype) {
    case DT_F32: return launch<TX, float>(a, stream);
    case DT_F16: return launch<TX, __half>(a, stream);
    default: return launch<TX, __nv_bfloat16>(a, stream);
  }
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& a, int x_dtype, int cache_dtype,
                                cudaStream_t stream) {
  switch (x_dtype) {
    case DT_F32: return by_cache<float>(a, cache_dtype, stream);
    case DT_F16: return by_cache<__half>(a, cache_dtype, stream);
    default: return by_cache<__nv_bfloat16>(a, cache_dtype, stream);
  }
}

}  // namespace m5b
