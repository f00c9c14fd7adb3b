// Appending keys and values to a paged cache, positions rotated on the way
// (m5b_paged_append).
//
// A rotated pair of channels is
//   (fma(a, c, -(b s)), fma(b, c, a s))
// in FP32, rounded once more to the cache's type.
// Two kernels with the same arithmetic: whole 16-channel units in 16-byte
// accesses, up to eight rows a CTA and the heads over several if need be, and a
// channel pair at a time, one CTA per row, for everything else (head dimensions
// and rotated widths that units do not divide, operands off the 16-byte grid).
#include "paged.cuh"

namespace m5b {
namespace {

constexpr int kThreads = 256;
constexpr int kUnitThreads = 384;  // most threads of a CTA of the unit kernel, three on an SM
constexpr int kUnitRows = 8;       // most rows
constexpr int kUnitTables = 2048;  // cos and sin of a CTA's rows, at most

// The row's position and page, by one warp: a 32-way search in query_start,
// so that two rounds of loads find one of up to 1024 sequences.
struct Place {
  int pos, page, slot;  // -1: none
};
__device__ __forceinline__ Place place_of(const PagedAppendArgs& a, int t) {
  const PagedBatch& b = a.b;
  const int lane = threadIdx.x % 32;
  int lo = 0, n = b.batch + 1;  // the first start > t is among [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const bool past = i >= lo + n || b.query_start[i] > t;
    const uint32_t m = __ballot_sync(~0u, past);
    const int k = m ? __ffs(m) - 1 : 32;  // starts at lo + 0 .. (k - 1) step are <= t
    if (k == 0) break;
    const int from = lo + (k - 1) * step + 1;
    n = min(lo + n, lo + k * step) - from;
    lo = from;
  }
  Place p{-1, -1, 0};
  if (lo == 0 || lo > b.batch) return p;
  const int seq = lo - 1;
  const int2 rows = paged_rows(b, seq);
  p.pos = paged_len(b, seq) - (rows.y - t);
  if (p.pos < 0 || (a.rope_half > 0 && p.pos >= a.table_rows))
    p.pos = -1;
  else if (p.pos < b.capacity)
    p.page = paged_page(b, seq, p.pos), p.slot = p.pos % b.page_size;
  return p;
}

// Eight elements as they were read, and as fp32.
template <typename T> struct Raw8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) {  // (read once)
    w = __ldcs(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const T* h = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(h[i]);
  }
};
template <> struct Raw8<float> {
  float4 u, v;
  __device__ __forceinline__ void load(const float* p) {
    u = *reinterpret_cast<const float4*>(p);
    v = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  }
};
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const void* base, int64_t i) {
  Raw8<T> r;
  r.load(static_cast<const T*>(base) + i);
  r.get(x);
}
__device__ __forceinline__ void load8(float (&x)[8], const void* base, int dtype, int64_t i) {
  if (dtype == DT_F32)
    load8<float>(x, base, i);
  else if (dtype == DT_BF16)
    load8<__nv_bfloat16>(x, base, i);
  else
    load8<__half>(x, base, i);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  __align__(16) T h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(x[i]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// A thread owns 16 channels of one head in all rows of its CTA, as two vectors
// of 8: those that rotate together (j and j + R, or the 16 neighbours), or two
// neighbours that are copied.  Bound by DRAM, every element read and written
// once, as long as enough loads are on their way: the places of the CTA's rows
// (a chain of four loads each) are looked up at once, a warp each, then their
// table entries, which all heads share; and a row's elements are loaded while
// the row before it is turned and stored.  9914 rows of 32 + 8 + 8 heads of 128
// channels: 47 us, 5.3 TB/s (a row a CTA 64 us, without the shared tables 63).
template <typename TX, typename TC, bool INTERLEAVED>
__global__ void __launch_bounds__(kUnitThreads, 3)
    paged_append_units(const PagedAppendArgs a, int rows_per_cta) {
  __shared__ Place place[kUnitRows];
  __shared__ __align__(16) float tables[kUnitTables];
  grid_dependency_wait();
  grid_dependents_launch();
  const PagedBatch& b = a.b;
  const int d = b.head_dim, n = d / 16, r8 = a.rope_half / 8;
  const int unit = blockIdx.y * blockDim.x + threadIdx.x, u = unit % n;
  const int t0 = blockIdx.x * rows_per_cta, count = min(rows_per_cta, b.tokens - t0);
  int h = unit / n;
  const int nq = a.q ? b.q_heads : 0;
  const bool mine = h < nq + 2 * b.kv_heads, query = h < nq, value = h >= nq + b.kv_heads;
  const bool turns = u < r8 && !value;
  int c0 = 16 * u, c1 = 16 * u + 8;  // first channels of the two vectors
  if (!INTERLEAVED && r8 > 0 && !value) {
    c0 = turns ? 8 * u : 16 * r8 + 16 * (u - r8);
    c1 = turns ? 8 * (u + r8) : c0 + 8;
  }
  const TX* src;
  int64_t src_step;
  TC* dst;
  int64_t page_step, slot_step;
  if (query) {
    src = static_cast<const TX*>(a.q) + h * a.q_head;
    src_step = a.q_token;
    dst = static_cast<TC*>(a.q_out) + h * d;
    page_step = int64_t(b.q_heads) * d;  // (of rows)
    slot_step = 0;
  } else if (!value) {
    h -= nq;
    src = static_cast<const TX*>(a.k) + h * a.k_head;
    src_step = a.k_token;
    dst = static_cast<TC*>(b.k_cache) + h * b.k_head;
    page_step = b.k_page;
    slot_step = b.k_slot;
  } else {
    h -= nq + b.kv_heads;
    src = static_cast<const TX*>(a.v) + h * a.v_head;
    src_step = a.v_token;
    dst = static_cast<TC*>(b.v_cache) + h * b.v_head;
    page_step = b.v_page;
    slot_step = b.v_slot;
  }
  src += t0 * src_step;
  Raw8<TX> raw[2], ahead[2];
  if (mine) {
    raw[0].load(src + c0);
    raw[1].load(src + c1);
  }
  for (int i = threadIdx.x / 32; i < count; i += blockDim.x / 32) {
    const Place p = place_of(a, t0 + i);
    if (threadIdx.x % 32 == 0) place[i] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * 2 * r8; i += blockDim.x) {  // [row][cos, sin][8 r8]
    const int row = i / (2 * r8), j = i % (2 * r8), pos = place[row].pos;
    float x[8];
    if (pos >= 0) {
      load8(x, j < r8 ? a.cos : a.sin, a.table_dtype, int64_t(pos) * a.rope_half + 8 * (j % r8));
      store8(tables + 8 * i, x);
    }
  }
  __syncthreads();
  if (!mine) return;
  for (int i = 0; i < count; ++i) {
    const Place at = place[i];
    if (i + 1 < count) {
      src += src_step;
      ahead[0].load(src + c0);
      ahead[1].load(src + c1);
    }
    float x[2][8];
    raw[0].get(x[0]);
    raw[1].get(x[1]);
    if (turns && at.pos >= 0) {
      float c[8], s[8];
      load8<float>(c, tables, 16 * r8 * i + 8 * u);
      load8<float>(s, tables, 16 * r8 * i + 8 * (r8 + u));
      if (INTERLEAVED) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float& p = x[k / 4][2 * (k % 4)];
          float& q = x[k / 4][2 * (k % 4) + 1];
          const float p0 = p;
          p = __fmaf_rn(p, c[k], -__fmul_rn(q, s[k]));
          q = __fmaf_rn(q, c[k], __fmul_rn(p0, s[k]));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; k += 2) {  // (packed: the same operations on two pairs)
          const float2 p = make_float2(x[0][k], x[0][k + 1]), q = make_float2(x[1][k], x[1][k + 1]);
          const float2 c2 = make_float2(c[k], c[k + 1]), s2 = make_float2(s[k], s[k + 1]);
          const float2 lo = __ffma2_rn(p, c2, __fmul2_rn(q, make_float2(-s2.x, -s2.y)));
          const float2 hi = __ffma2_rn(q, c2, __fmul2_rn(p, s2));
          x[0][k] = lo.x, x[0][k + 1] = lo.y, x[1][k] = hi.x, x[1][k + 1] = hi.y;
        }
      }
    }
    if (query && at.pos < 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[0][k] = x[1][k] = 0.0f;
    }
    if (query || at.page >= 0) {
      TC* to = dst + (query ? t0 + i : at.page) * page_step + at.slot * slot_step;
      store8(to + c0, x[0]);
      store8(to + c1, x[1]);
    }
    raw[0] = ahead[0];
    raw[1] = ahead[1];
  }
}

template <typename TX, typename TC>
__global__ void __launch_bounds__(kThreads) paged_append_pairs(const PagedAppendArgs a) {
  const PagedBatch& b = a.b;
  const int t = blockIdx.x;
  const int d = b.head_dim;
  const Place at = place_of(a, t);
  const int pos = at.pos, page = at.page;
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
      x = __fmaf_rn(x, c, -__fmul_rn(y, s));
      y = __fmaf_rn(y, c, __fmul_rn(x0, s));
    }
    dst[i0] = from_f32<TC>(x);
    if (i1 < d) dst[i1] = from_f32<TC>(y);
  }
}

template <typename TX, typename TC>
cudaError_t launch(const PagedAppendArgs& a, cudaStream_t stream) {
  if (!a.units) {
    paged_append_pairs<TX, TC><<<a.b.tokens, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
  }
  // the heads' units over as many CTAs as their threads need; so many rows a
  // CTA that full waves of three CTAs an SM share the rows evenly
  const int units = ((a.q ? a.b.q_heads : 0) + 2 * a.b.kv_heads) * (a.b.head_dim / 16);
  const int across = (units + kUnitThreads - 1) / kUnitThreads;
  int most = a.rope_half > 0 ? kUnitTables / (2 * a.rope_half) : kUnitRows;
  most = most < kUnitRows ? most : kUnitRows;
  const int64_t work = int64_t(a.b.tokens) * across, slots = 3 * a.sms;
  const int64_t waves = (work + slots * most - 1) / (slots * most);
  const int rows = static_cast<int>((work + slots * waves - 1) / (slots * waves));
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.b.tokens + rows - 1) / rows), static_cast<unsigned>(across));
  cfg.blockDim = dim3(static_cast<unsigned>(((units + across - 1) / across + 31) / 32 * 32));
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return a.interleaved ? cudaLaunchKernelEx(&cfg, paged_append_units<TX, TC, true>, a, rows)
                       : cudaLaunchKernelEx(&cfg, paged_append_units<TX, TC, false>, a, rows);
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
