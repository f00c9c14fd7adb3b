// E4M3 quantization with a scale for each block of 128 channels: of one row
// (activations), or of 128 rows (weights).
//
//   v = x, or silu(gate) x = (gate / (1 + exp(-gate))) x, in fp32
//   scale = max|v| / 448 over the block, 1 where that is 0
//   code  = E4M3(RN32(v / scale)), nearest even, saturating
//
// One pass: a block of one row lives in 16 lanes, 8 channels each (one 16-byte
// load of a 16-bit type), its peak goes through four shuffles; a block of 128
// rows lives in the registers of one CTA.  Bound by memory: size + 1 bytes a
// value and 4 a block.
//
// The peak is taken on the values' bit patterns without the sign, which order
// like the values and put NaN above infinity, so that a block with either gets
// a scale that is not finite, and its products are not either.
#include "grouped.cuh"

namespace m5b {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct Raw8 {  // eight values as they are in memory
  uint32_t w[2 * sizeof(T)];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    r.w[4 * i] = v.x;
    r.w[4 * i + 1] = v.y;
    r.w[4 * i + 2] = v.z;
    r.w[4 * i + 3] = v.w;
  }
  return r;
}
// The first `count` of eight values, zeros behind them.
template <typename T>
__device__ __forceinline__ Raw8<T> load8_upto(const T* p, int count) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) r.w[i] = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= count) break;
    if constexpr (sizeof(T) == 4)
      r.w[i] = __float_as_uint(p[i]);
    else
      r.w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if constexpr (sizeof(T) == 4) {
      f = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    } else if constexpr (DTypeOf<T>::value == DT_BF16) {
      f = bf16x2_f2(r.w[i]);
    } else {
      f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
    }
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint32_t peak8(const float* v) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

__device__ __forceinline__ float silu(float g) {
  return __fdiv_rn(g, __fadd_rn(1.0f, expf(-g)));
}

__device__ __forceinline__ float block_scale(uint32_t peak) {
  const float s = __fdiv_rn(__uint_as_float(peak), 448.0f);
  return s == 0.0f ? 1.0f : s;
}

// Codes of eight values.  Where neither the scale nor its reciprocal leaves the
// normal range, quot_pair_div is the correctly rounded quotient wherever that
// is not far below the smallest code's half (2^-10); elsewhere divides.
__device__ __forceinline__ uint2 codes8(const float* v, float scale) {
  uint32_t w[4];
  if (scale >= kI8DivMinScale && scale <= 0x1p100f) {
    const I8Div d = i8_div(__frcp_rn(scale), scale);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __nv_cvt_float2_to_fp8x2(quot_pair_div(make_float2(v[2 * i], v[2 * i + 1]), d),
                                      __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  }
  return make_uint2(e4m3_word_exact(v[0], v[1], v[2], v[3], scale),
                    e4m3_word_exact(v[4], v[5], v[6], v[7], scale));
}

__device__ __forceinline__ void store8(uint8_t* q, uint2 codes, bool vec, int count) {
  if (vec) {
    *reinterpret_cast<uint2*>(q) = codes;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) q[i] = static_cast<uint8_t>((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)));
}

template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load_any(const T* p, int count) {
  if constexpr (VEC) {  // (k is a multiple of 8: all eight or none)
    if (count > 0) return load8(p);
    return Raw8<T>{};
  } else {
    return load8_upto(p, count);
  }
}

// Blocks of one row.  Half-warp h of the grid takes blocks h, h + halves, ...,
// UNROLL of them at a time, whose loads are all on their way before the first is
// used.
template <typename T, bool GATE, bool VEC, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    block_quant_rows_kernel(const BlockQuantArgs a, unsigned blocks_per_row, unsigned total) {
  const int sub = threadIdx.x & 15;
  const unsigned halves = gridDim.x * (kThreads / 16);
  const unsigned first = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4);
  const T* x = static_cast<const T*>(a.x);
  const T* gate = static_cast<const T*>(a.gate);
  // (whole warps leave the loop together: the shuffles below name all lanes)
  for (unsigned b0 = first - (first & 1u); b0 < total; b0 += halves * UNROLL) {
    Raw8<T> rx[UNROLL], rg[UNROLL];
    int64_t at[UNROLL];
    int count[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const unsigned b = b0 + (first & 1u) + u * halves;
      const unsigned row = b / blocks_per_row;
      const unsigned col = (b - row * blocks_per_row) * 128u + sub * 8u;
      int64_t left = b < total ? a.k - col : 0;
      at[u] = int64_t(row) * a.k + col;
      count[u] = static_cast<int>(left < 0 ? 0 : left > 8 ? 8 : left);
      int64_t src = row;
      bool have = true;
      if (a.index && b < total) {
        src = a.index[row];
        have = src >= 0 && src < a.x_rows;  // else a row of zeros
      }
      rx[u] = load_any<T, VEC>(x + src * a.x_row + col, have ? count[u] : 0);
      if constexpr (GATE)
        rg[u] = load_any<T, VEC>(gate + src * a.gate_row + col, have ? count[u] : 0);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const unsigned b = b0 + (first & 1u) + u * halves;
      float v[8];
      unpack8(rx[u], v);
      if constexpr (GATE) {
        float s[8];
        unpack8(rg[u], s);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(silu(s[i]), v[i]);
      }
      uint32_t peak = peak8(v);
#pragma unroll
      for (int d = 8; d; d >>= 1) peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, d));
      const float scale = block_scale(peak);
      if (b < total && sub == 0) a.scales[b] = scale;
      if (count[u] > 0) store8(a.q + at[u], codes8(v, scale), VEC, count[u]);
    }
  }
}

// Blocks of 128 rows, one a CTA: thread t has channels 8 (t % 16) .. + 7 of rows
// t / 16 + 16 i.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    block_quant_square_kernel(const BlockQuantArgs a, unsigned blocks_per_row,
                              unsigned row_blocks) {
  __shared__ uint32_t s_peak[kThreads / 32];
  const unsigned b = blockIdx.x;
  const unsigned rb = b / blocks_per_row;  // batch * row_blocks + row block
  const unsigned batch = rb / row_blocks;
  const int64_t row0 = int64_t(rb - batch * row_blocks) * 128 + (threadIdx.x >> 4);
  const int64_t col = int64_t(b - rb * blocks_per_row) * 128 + (threadIdx.x & 15) * 8;
  const int64_t left = a.k - col;
  const int count = static_cast<int>(left < 0 ? 0 : left > 8 ? 8 : left);
  const T* x = static_cast<const T*>(a.x) + batch * a.x_batch + col;
  Raw8<T> r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    r[i] = load_any<T, VEC>(x + row * a.x_row, row < a.rows ? count : 0);
  }
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v[8];
    unpack8(r[i], v);
    peak = max(peak, peak8(v));
  }
  peak = __reduce_max_sync(0xffffffffu, peak);
  if ((threadIdx.x & 31) == 0) s_peak[threadIdx.x >> 5] = peak;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) peak = max(peak, s_peak[i]);
  const float scale = block_scale(peak);
  if (threadIdx.x == 0) a.scales[b] = scale;
  uint8_t* q = a.q + int64_t(batch) * a.rows * a.k + col;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    if (row >= a.rows || count == 0) continue;
    float v[8];
    unpack8(r[i], v);
    store8(q + row * a.k, codes8(v, scale), VEC, count);
  }
}

template <typename T, bool VEC>
cudaError_t launch(const BlockQuantArgs& a, bool square, cudaStream_t stream) {
  const unsigned per_row = static_cast<unsigned>((a.k + 127) / 128);
  if (square) {
    const unsigned row_blocks = static_cast<unsigned>((a.rows + 127) / 128);
    block_quant_square_kernel<T, VEC><<<static_cast<unsigned>(a.batch) * row_blocks * per_row,
                                        kThreads, 0, stream>>>(a, per_row, row_blocks);
    return cudaGetLastError();
  }
  const unsigned total = static_cast<unsigned>(a.rows) * per_row;
  constexpr int UNROLL = sizeof(T) == 4 ? 2 : 4;
  const unsigned per_cta = kThreads / 16 * UNROLL;
  unsigned grid = (total + per_cta - 1) / per_cta;
  const unsigned most = static_cast<unsigned>(a.sms) * 8;
  if (grid > most) grid = most;
  if (a.gate)
    block_quant_rows_kernel<T, true, VEC, 2><<<grid, kThreads, 0, stream>>>(a, per_row, total);
  else
    block_quant_rows_kernel<T, false, VEC, UNROLL><<<grid, kThreads, 0, stream>>>(a, per_row, total);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_quantize(const BlockQuantArgs& a, int dtype, bool square,
                                  cudaStream_t stream) {
  switch (dtype) {
    case DT_BF16:
      return a.vec ? launch<__nv_bfloat16, true>(a, square, stream)
                   : launch<__nv_bfloat16, false>(a, square, stream);
    case DT_F16:
      return a.vec ? launch<__half, true>(a, square, stream)
                   : launch<__half, false>(a, square, stream);
    case DT_F32:
      return a.vec ? launch<float, true>(a, square, stream)
                   : launch<float, false>(a, square, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace m5b
