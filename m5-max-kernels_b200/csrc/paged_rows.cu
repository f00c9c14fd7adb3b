// Attention over a paged cache, one CTA per (row, query head): any head
// dimension up to 256, any page size, any strides, FP32 / FP16 / BF16
// (m5b_paged_attention).
//
// The row's keys come in chunks of 32, dealt to the CTA's warps in turn.  In
// a chunk a lane takes one key: x = scale q.k (capped, biased, masked); then
// the warp keeps the running maximum m and sum l of its row,
//   m' = max(m, max x),  l' = l e^(m - m') + sum e^(x - m'),
//   o' = o e^(m - m') + sum e^(x - m') v,
// with the lanes across the channels for the last sum.  The warps' (m, l, o)
// are joined the same way at the end.  All sums are FP32.  Hidden keys and
// values are never used, whatever they hold.
#include "paged.cuh"

namespace m5b {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxDim = 256;
constexpr int kPerLane = kMaxDim / 32;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_rows_kernel(const PagedAttnArgs a) {
  const PagedBatch& b = a.b;
  const int t = blockIdx.x / b.q_heads, h = blockIdx.x % b.q_heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int d = b.head_dim, kvh = h / b.group;
  __shared__ float s_q[kMaxDim];
  __shared__ float s_o[kWarps][kMaxDim];
  __shared__ float s_m[kWarps], s_l[kWarps];

  const int seq = paged_find(b, t);
  int len = 0, pos = -1, prefix = 0;
  if (seq >= 0) {
    const int2 rows = paged_rows(b, seq);
    len = paged_len(b, seq);
    pos = len - (rows.y - t);
    len = min(len, b.capacity);
    if (a.prefix_lens) prefix = max(0, min(a.prefix_lens[seq], len));
  }
  const T* q = static_cast<const T*>(a.q) + int64_t(t) * a.q_token + h * a.q_head;
  for (int i = threadIdx.x; i < d; i += kWarps * 32) s_q[i] = to_f32(q[i]);
  __syncthreads();

  const float slope = a.slopes ? a.slopes[h] : 0.0f;
  float m = -INFINITY, l = 0.0f, o[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) o[i] = 0.0f;
  // chunks [0, pre) hold the prefix, [from, end) the row's own window
  const int pre = prefix / 32 + (prefix % 32 != 0);
  const int last = min(pos, len - 1);
  const int first = (pos >= a.window) ? pos - a.window + 1 : 0;
  const int from = max(pre, first / 32), end = last >= 0 ? last / 32 + 1 : 0;
  const int chunks = pre + max(0, end - from);
  for (int i = warp; i < chunks; i += kWarps) {
    const int j0 = (i < pre ? i : from + i - pre) * 32, j = j0 + lane;
    const bool seen = j < len && (j < prefix || (j <= pos && pos - j < a.window));
    const int page = seen ? paged_page(b, seq, j) : -1;
    float x = -INFINITY;
    const T* v = nullptr;
    if (seen) {
      float dot = 0.0f;
      if (page >= 0) {
        const int slot = j % b.page_size;
        const T* k = static_cast<const T*>(b.k_cache) + page * b.k_page + kvh * b.k_head +
                     slot * b.k_slot;
        v = static_cast<const T*>(b.v_cache) + page * b.v_page + kvh * b.v_head + slot * b.v_slot;
        for (int c = 0; c < d; ++c) dot = fmaf(s_q[c], to_f32(k[c]), dot);
      }
      x = dot * a.scale;
      if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
      x -= slope * fabsf(static_cast<float>(pos - j));
    }
    float top = x;
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, s));
    if (__all_sync(~0u, x == -INFINITY)) continue;  // (a NaN score goes on into the sums)
    const float m2 = fmaxf(m, top), keep = expf(m - m2), p = expf(x - m2);
    m = m2;
    l = l * keep + p;  // of this lane's keys; summed over the lanes at the end
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) o[c] *= keep;
    const uint32_t any = __ballot_sync(~0u, page >= 0);
    for (int k = 0; k < 32; ++k) {
      if (!((any >> k) & 1u)) continue;
      const float pk = __shfl_sync(~0u, p, k);
      const T* vk = reinterpret_cast<const T*>(
          __shfl_sync(~0u, reinterpret_cast<unsigned long long>(v), k));
#pragma unroll
      for (int c = 0; c < kPerLane; ++c)
        if (c * 32 + lane < d) o[c] = fmaf(pk, to_f32(vk[c * 32 + lane]), o[c]);
    }
  }
#pragma unroll
  for (int s = 16; s; s >>= 1) l += __shfl_xor_sync(~0u, l, s);
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) s_o[warp][c * 32 + lane] = o[c];
  __syncthreads();

  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
  float share[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    share[w] = s_l[w] == 0.0f ? 0.0f : expf(s_m[w] - top);
    sum += s_l[w] * share[w];
  }
  T* out = static_cast<T*>(a.out) + int64_t(t) * a.o_token + h * a.o_head;
  for (int i = threadIdx.x; i < d; i += kWarps * 32) {
    float y = 0.0f;
    for (int w = 0; w < kWarps; ++w) y += s_o[w][i] * share[w];
    out[i] = from_f32<T>(sum == 0.0f ? 0.0f : y / sum);
  }
  if (a.lse && threadIdx.x == 0)
    a.lse[int64_t(t) * b.q_heads + h] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

template <typename T>
cudaError_t launch(const PagedAttnArgs& a, cudaStream_t stream) {
  paged_rows_kernel<T><<<a.b.tokens * a.b.q_heads, kWarps * 32, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_attention_rows(const PagedAttnArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case DT_F32: return launch<float>(a, stream);
    case DT_F16: return launch<__half>(a, stream);
    default: return launch<__nv_bfloat16>(a, stream);
  }
}

}  // namespace m5b
