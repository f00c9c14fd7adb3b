// Appending keys and values to a paged cache, positions rotated on the way
// (m5b_paged_append).
//
// A rotated pair of channels is
//   (a c - b s, b c + a s)
// with one rounding per product and sum in FP32, then one to the cache's type.
// One CTA per new row.  Two kernels with the same arithmetic: whole 16-channel
// units in 16-byte accesses, and a channel pair at a time for everything else
// (head dimensions and rotated widths that units do not divide, operands off
// the 16-byte grid).
#include "paged.cuh"

namespace m5b {
namespace {

constexpr int kThreads = 256;
constexpr int kUnitThreads = 512;  // most threads of a row's CTA
constexpr int kTurns = 2;          // units a thread has on their way at a time

// The row's position and page, by one warp: a 32-way search in query_start,
// so that two rounds of loads find one of up to 1024 sequences.
struct Place {
  int pos, page;  // -1: none
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
  Place p{-1, -1};
  if (lo == 0 || lo > b.batch) return p;
  const int seq = lo - 1;
  const int2 rows = paged_rows(b, seq);
  p.pos = paged_len(b, seq) - (rows.y - t);
  if (p.pos < 0 || (a.rope_half > 0 && p.pos >= a.table_rows))
    p.pos = -1;
  else if (p.pos < b.capacity)
    p.page = paged_page(b, seq, p.pos);
  return p;
}

// Eight elements as they were read, and as fp32.
template <typename T> struct Raw8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
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

// 16 channels a thread and turn, as two vectors of 8: those that rotate
// together (j and j + R, or the 16 neighbours), or two neighbours that are
// copied.  The turns of a thread fall on the same channels of other heads, so
// the tables are read once, and the launch has threads for two turns, whose
// loads are on their way while the row's place is looked up.  Bound by DRAM:
// every element is read and written once.
template <typename TX, typename TC>
__global__ void __launch_bounds__(kUnitThreads) paged_append_units(const PagedAppendArgs a) {
  grid_dependency_wait();
  grid_dependents_launch();
  const PagedBatch& b = a.b;
  const int t = blockIdx.x, d = b.head_dim, n = d / 16, r8 = a.rope_half / 8;
  const int u = threadIdx.x % n, h0 = threadIdx.x / n, step = blockDim.x / n;
  const int nq = a.q ? b.q_heads : 0, heads = nq + 2 * b.kv_heads;
  const bool turns = u < r8;
  // first channels of the two vectors, in rotated heads and in values
  int c0 = 16 * u, c1 = 16 * u + 8;
  if (!a.interleaved && r8 > 0) {
    c0 = turns ? 8 * u : 16 * r8 + 16 * (u - r8);
    c1 = turns ? 8 * (u + r8) : c0 + 8;
  }
  Raw8<TX> raw[kTurns][2];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      int h = base + i * step;
      if (h >= heads) continue;
      const TX* src;
      int v0 = c0, v1 = c1;
      if (h < nq) {
        src = static_cast<const TX*>(a.q) + int64_t(t) * a.q_token + h * a.q_head;
      } else if ((h -= nq) < b.kv_heads) {
        src = static_cast<const TX*>(a.k) + int64_t(t) * a.k_token + h * a.k_head;
      } else {
        src = static_cast<const TX*>(a.v) + int64_t(t) * a.v_token + (h - b.kv_heads) * a.v_head;
        v0 = 16 * u, v1 = 16 * u + 8;
      }
      raw[i][0].load(src + v0);
      raw[i][1].load(src + v1);
    }
  };
  fetch(h0);
  const Place at = place_of(a, t);
  const int64_t slot = at.pos >= 0 ? at.pos % b.page_size : 0;
  float c[8], s[8];
  if (turns && at.pos >= 0) {
    load8(c, a.cos, a.table_dtype, int64_t(at.pos) * a.rope_half + 8 * u);
    load8(s, a.sin, a.table_dtype, int64_t(at.pos) * a.rope_half + 8 * u);
  }
  for (int base = h0; base < heads; base += kTurns * step) {
    if (base != h0) fetch(base);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      int h = base + i * step;
      if (h >= heads) continue;
      TC* dst;
      int v0 = c0, v1 = c1;
      bool rotate = turns;
      float x[2][8];
      raw[i][0].get(x[0]);
      raw[i][1].get(x[1]);
      if (h < nq) {
        dst = static_cast<TC*>(a.q_out) + (int64_t(t) * b.q_heads + h) * d;
        if (at.pos < 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[0][k] = x[1][k] = 0.0f;
          rotate = false;
        }
      } else {
        if (at.page < 0) continue;
        if ((h -= nq) < b.kv_heads) {
          dst = static_cast<TC*>(b.k_cache) + at.page * b.k_page + h * b.k_head + slot * b.k_slot;
        } else {
          dst = static_cast<TC*>(b.v_cache) + at.page * b.v_page + (h - b.kv_heads) * b.v_head +
                slot * b.v_slot;
          rotate = false;
          v0 = 16 * u, v1 = 16 * u + 8;
        }
      }
      if (rotate) {
        if (a.interleaved) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float& p = x[k / 4][2 * (k % 4)];
            float& q = x[k / 4][2 * (k % 4) + 1];
            const float p0 = p;
            p = __fsub_rn(__fmul_rn(p, c[k]), __fmul_rn(q, s[k]));
            q = __fadd_rn(__fmul_rn(q, c[k]), __fmul_rn(p0, s[k]));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float p0 = x[0][k], q0 = x[1][k];
            x[0][k] = __fsub_rn(__fmul_rn(p0, c[k]), __fmul_rn(q0, s[k]));
            x[1][k] = __fadd_rn(__fmul_rn(q0, c[k]), __fmul_rn(p0, s[k]));
          }
        }
      }
      store8(dst + v0, x[0]);
      store8(dst + v1, x[1]);
    }
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
      x = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
      y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x0, s));
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
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.b.tokens));
  const int n = a.b.head_dim / 16, heads = (a.q ? a.b.q_heads : 0) + 2 * a.b.kv_heads;
  const int round = n > 32 ? n : 32, want = (heads * n + kTurns - 1) / kTurns;
  const int threads = (want + round - 1) / round * round;
  cfg.blockDim = dim3(static_cast<unsigned>(threads < kUnitThreads ? threads : kUnitThreads));
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_append_units<TX, TC>, a);
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
