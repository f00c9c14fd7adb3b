// E4M3 quantization with a scale for each block of 128 channels: of one row
// (activations), or of 128 rows (weights).
//
//   v = x, or silu(gate) x = gate / (1 + exp(-gate)) x, in fp32
//   scale = max|v| / 448 over the block, 1 where that is 0
//   code  = E4M3(RN32(v / scale)), nearest even, saturating; -0 gives code 0 where
//           quotients go by multiplications (x - q s is +0), 0x80 where they are divided
//
// One pass: a block of one row lives in eight lanes, 16 channels each (32 bytes
// of a 16-bit type, one 16-byte store of codes), its peak goes through three
// shuffles; a block of 128 rows lives in the registers of one CTA.  Bound by
// memory: size + 1 bytes a value and 4 a block.
//
// The peak is taken on the values' bit patterns without the sign, which order
// like the values and put NaN above infinity, so that a block with either gets
// a scale that is not finite, and its products are not either.
#include "grouped.cuh"

namespace m5b {

namespace {

constexpr int kThreads = 256;
constexpr int kLane = 16;                // channels a thread
constexpr int kLanes = 128 / kLane;      // threads of a block's row
constexpr int kRows = kThreads / kLanes;  // rows of blocks that a CTA has at a time

template <typename T>
struct Raw {  // kLane values as they are in memory
  uint32_t w[kLane * sizeof(T) / 4];
};

template <typename T>
__device__ __forceinline__ Raw<T> load(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[i];
    r.w[4 * i] = v.x;
    r.w[4 * i + 1] = v.y;
    r.w[4 * i + 2] = v.z;
    r.w[4 * i + 3] = v.w;
  }
  return r;
}
// The first `count` values, zeros behind them.
template <typename T>
__device__ __forceinline__ Raw<T> load_upto(const T* p, int count) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r) / 4); ++i) r.w[i] = 0u;
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    if (i >= count) break;
    if constexpr (sizeof(T) == 4)
      r.w[i] = __float_as_uint(p[i]);
    else
      r.w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i])
                     << (16 * (i & 1));
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_any(const T* p, int count) {
  if constexpr (VEC) {  // (k is a multiple of kLane: all values or none)
    if (count > 0) return load(p);
    return Raw<T>{};
  } else {
    return load_upto(p, count);
  }
}

template <typename T>
__device__ __forceinline__ float2 pair(const Raw<T>& r, int i) {  // values 2 i, 2 i + 1
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
  else if constexpr (DTypeOf<T>::value == DT_BF16)
    return bf16x2_f2(r.w[i]);
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
}

// m = the larger magnitude of m and v, NaN if either is, under a sign of no meaning
// (magnitude() takes it off).
__device__ __forceinline__ void larger(float& m, float v) {
  asm("max.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(m) : "f"(v));
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The largest magnitude, as the bits of an fp32 number.
template <typename T>
__device__ __forceinline__ uint32_t peak_of(const Raw<T>& r) {
  if constexpr (sizeof(T) == 4) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kLane; ++i) larger(m, __uint_as_float(r.w[i]));
    return magnitude(m);
  } else {
    uint32_t m = 0u;
    // (the larger magnitude of each half, NaN if either is, under a sign of no meaning)
#pragma unroll
    for (int i = 0; i < kLane / 2; ++i) {
      if constexpr (DTypeOf<T>::value == DT_BF16)
        asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(r.w[i]));
      else
        asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(r.w[i]));
    }
    m &= 0x7FFF7FFFu;
    const uint32_t top = max(m >> 16, m & 0xFFFFu);
    if constexpr (DTypeOf<T>::value == DT_BF16) return top << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top))));
  }
}

// 1 / d of a packed pair of normal numbers whose reciprocals are normal: a Newton
// step after the approximation, right but for the rarest ulp.
__device__ __forceinline__ float2 reciprocal(float2 d, float2 nd) {
  float2 y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(d.y));
  return __ffma2_rn(__ffma2_rn(nd, y, make_float2(1.0f, 1.0f)), y, y);
}

// silu(g) x for |g| <= kSiluFast: exp(-g) = 2^t, t = -g log2 e in two parts (the
// constant in two, the product's rounding error from one multiply-add), of which
// the second, below 2^-17, is multiplied on: 2^(hi + lo) = 2^hi (1 + lo ln 2).
// The quotient is Markstein's, as in i8_pair_div.  Elsewhere exp may be infinite:
// silu() divides.
constexpr float kSiluFast = 80.0f;
__device__ __forceinline__ float2 silu_fast(float2 g, float2 x) {
  const float2 one = make_float2(1.0f, 1.0f);
  const float2 l_hi = make_float2(-0x1.715476p+0f, -0x1.715476p+0f);    // -log2 e
  const float2 l_lo = make_float2(-0x1.4ae0c0p-26f, -0x1.4ae0c0p-26f);  // what that lacks
  const float2 ln2 = make_float2(0x1.62e430p-1f, 0x1.62e430p-1f);
  const float2 hi = __fmul2_rn(g, l_hi);
  const float2 lo =
      __ffma2_rn(g, l_lo, __ffma2_rn(g, l_hi, make_float2(-hi.x, -hi.y)));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(hi.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(hi.y));
  e = __ffma2_rn(e, __fmul2_rn(lo, ln2), e);
  const float2 d = __fadd2_rn(one, e);
  const float2 nd = make_float2(-d.x, -d.y);
  const float2 y = reciprocal(d, nd);
  const float2 q = __fmul2_rn(g, y);
  return __fmul2_rn(__ffma2_rn(__ffma2_rn(nd, q, g), y, q), x);
}
__device__ __forceinline__ float silu(float g) {
  return __fdiv_rn(g, __fadd_rn(1.0f, expf(-g)));
}

// A block's scale, and whether quotients by it may go by multiplications: where
// peak / 448, its reciprocal and the residuals below stay normal.
struct Scale {
  float s;
  bool fast;
};
__device__ __forceinline__ Scale block_scale(uint32_t peak) {
  const float p = __uint_as_float(peak);
  Scale r;
  r.fast = p >= 0x1p-80f && p <= 0x1p100f;
  if (r.fast) {  // RN(p / 448): Markstein's step with RN(1 / 448)
    const float q = __fmul_rn(p, 1.0f / 448.0f);
    r.s = __fmaf_rn(__fmaf_rn(-448.0f, q, p), 1.0f / 448.0f, q);
  } else {
    r.s = __fdiv_rn(p, 448.0f);
    if (r.s == 0.0f) r.s = 1.0f;
  }
  return r;
}

// Stores the codes of kLane values, of which the first `count` exist.  The
// quotient RN(v / s) decides at ties, wherever it is not far below half the
// smallest code (2^-10): quot_pair_div.
template <bool VEC, class Pair>
__device__ __forceinline__ void store_codes(uint8_t* q, int count, Scale scale, Pair pair_at) {
  uint32_t w[kLane / 4];
  if (scale.fast) {
    I8Div d;
    d.ns = make_float2(-scale.s, -scale.s);
    d.y = reciprocal(make_float2(scale.s, scale.s), d.ns);
#pragma unroll
    for (int i = 0; i < kLane / 4; ++i)
      w[i] = __nv_cvt_float2_to_fp8x2(quot_pair_div(pair_at(2 * i), d), __NV_SATFINITE,
                                      __NV_E4M3) |
             static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(quot_pair_div(pair_at(2 * i + 1), d),
                                                            __NV_SATFINITE, __NV_E4M3))
                 << 16;
  } else {
#pragma unroll
    for (int i = 0; i < kLane / 4; ++i) {
      const float2 a = pair_at(2 * i), b = pair_at(2 * i + 1);
      w[i] = e4m3_word_exact(a.x, a.y, b.x, b.y, scale.s);
    }
  }
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (i < count) q[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
  }
}

// Blocks of one row.  A group of eight lanes takes blocks b, b + stride, ...,
// UNROLL of them at a time, whose loads are all on their way before the first is
// used.
template <typename T, bool GATE, bool VEC, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    block_quant_rows_kernel(const BlockQuantArgs a, unsigned blocks_per_row, unsigned total) {
  const int sub = threadIdx.x % kLanes;
  const unsigned stride = gridDim.x * kRows;
  const unsigned row_step = stride / blocks_per_row;
  const unsigned col_step = stride - row_step * blocks_per_row;
  const T* x = static_cast<const T*>(a.x);
  const T* gate = static_cast<const T*>(a.gate);
  const int k = static_cast<int>(a.k), x_rows = static_cast<int>(a.x_rows);
  unsigned b = blockIdx.x * kRows + threadIdx.x / kLanes;
  unsigned row = b / blocks_per_row, block = b - row * blocks_per_row;
  grid_dependency_wait();
  grid_dependents_launch();  // (a product that follows sets itself up meanwhile)
  // (whole warps leave the loop together: the shuffles below name all lanes)
  while (b - threadIdx.x % 32 / kLanes < total) {
    Raw<T> rx[UNROLL], rg[UNROLL];
    int64_t at[UNROLL];
    int count[UNROLL];
    unsigned which[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int col = static_cast<int>(block * 128) + sub * kLane;
      const int left = b < total ? k - col : 0;
      which[u] = b;
      at[u] = int64_t(row) * k + col;
      count[u] = left < 0 ? 0 : left > kLane ? kLane : left;
      int src = static_cast<int>(row);
      int here = count[u];
      if (a.index && here > 0) {
        src = a.index[row];
        if (src < 0 || src >= x_rows) here = 0;  // a row of zeros
      }
      rx[u] = load_any<T, VEC>(x + src * a.x_row + col, here);
      if constexpr (GATE) rg[u] = load_any<T, VEC>(gate + src * a.gate_row + col, here);
      b += stride;
      row += row_step;
      block += col_step;
      if (block >= blocks_per_row) {
        block -= blocks_per_row;
        ++row;
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float2 v[kLane / 2];
      uint32_t peak = 0u;
      if constexpr (GATE) {
        if (peak_of(rg[u]) <= __float_as_uint(kSiluFast)) {
#pragma unroll
          for (int i = 0; i < kLane / 2; ++i) v[i] = silu_fast(pair(rg[u], i), pair(rx[u], i));
        } else {
#pragma unroll
          for (int i = 0; i < kLane / 2; ++i) {
            const float2 g = pair(rg[u], i), f = pair(rx[u], i);
            v[i] = make_float2(__fmul_rn(silu(g.x), f.x), __fmul_rn(silu(g.y), f.y));
          }
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < kLane / 2; ++i) {
          larger(m, v[i].x);
          larger(m, v[i].y);
        }
        peak = magnitude(m);
      } else {
        peak = peak_of(rx[u]);
      }
#pragma unroll
      for (int d = kLanes / 2; d; d >>= 1)
        peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, d));
      const Scale scale = block_scale(peak);
      if (which[u] < total && sub == 0) a.scales[which[u]] = scale.s;
      if (count[u] > 0)
        store_codes<VEC>(a.q + at[u], count[u], scale, [&](int i) {
          if constexpr (GATE)
            return v[i];
          else
            return pair(rx[u], i);
        });
    }
  }
}

// Blocks of 128 rows, one a CTA: thread t has channels 16 (t % 8) .. + 15 of rows
// t / 8 + 32 i.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    block_quant_square_kernel(const BlockQuantArgs a, unsigned blocks_per_row,
                              unsigned row_blocks) {
  constexpr int N = 128 / kRows;
  __shared__ uint32_t s_peak[kThreads / 32];
  const unsigned b = blockIdx.x;
  const unsigned rb = b / blocks_per_row;  // batch * row_blocks + row block
  const unsigned batch = rb / row_blocks;
  const int64_t row0 = int64_t(rb - batch * row_blocks) * 128 + threadIdx.x / kLanes;
  const int64_t col = int64_t(b - rb * blocks_per_row) * 128 + threadIdx.x % kLanes * kLane;
  const int64_t left = a.k - col;
  const int count = static_cast<int>(left < 0 ? 0 : left > kLane ? kLane : left);
  const T* x = static_cast<const T*>(a.x) + batch * a.x_batch + col;
  grid_dependency_wait();
  grid_dependents_launch();
  Raw<T> r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t row = row0 + kRows * i;
    r[i] = load_any<T, VEC>(x + row * a.x_row, row < a.rows ? count : 0);
  }
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) peak = max(peak, peak_of(r[i]));
  peak = __reduce_max_sync(0xffffffffu, peak);
  if (threadIdx.x % 32 == 0) s_peak[threadIdx.x / 32] = peak;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) peak = max(peak, s_peak[i]);
  const Scale scale = block_scale(peak);
  if (threadIdx.x == 0) a.scales[b] = scale.s;
  uint8_t* q = a.q + int64_t(batch) * a.rows * a.k + col;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t row = row0 + kRows * i;
    if (row < a.rows && count > 0)
      store_codes<VEC>(q + row * a.k, count, scale, [&](int j) { return pair(r[i], j); });
  }
}

// With programmatic launch (grid_dependency_wait): the start overlaps the end of
// the kernel before.
template <class... Params, class... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), unsigned grid, cudaStream_t stream,
                              Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, bool VEC>
cudaError_t launch(const BlockQuantArgs& a, bool square, cudaStream_t stream) {
  const unsigned per_row = static_cast<unsigned>((a.k + 127) / 128);
  if (square) {
    const unsigned row_blocks = static_cast<unsigned>((a.rows + 127) / 128);
    return launch_overlapped(block_quant_square_kernel<T, VEC>,
                             static_cast<unsigned>(a.batch) * row_blocks * per_row, stream, a,
                             per_row, row_blocks);
  }
  const unsigned total = static_cast<unsigned>(a.rows) * per_row;
  constexpr int UNROLL = sizeof(T) == 4 ? 1 : 2;
  unsigned grid = (total + kRows - 1) / kRows;
  // As many CTAs as are resident (48 registers a thread): 8 an SM take 21.7 us for
  // 10662 rows of 4096 to experts, 5 take 19.7, 64 take 31 (10.7 instructions an
  // element; 4096 x 16384 33 us, 6.1 TB/s).  Gated, where the arithmetic of one hides
  // the loads of another, 20: 51.6 us for 9914 x 5376 against 54.7 with 5 (50.3 since;
  // 23.5 instructions an element).
  const unsigned most = static_cast<unsigned>(a.sms) * (a.gate ? 20 : 5);
  if (grid > most) grid = most;
  return a.gate ? launch_overlapped(block_quant_rows_kernel<T, true, VEC, 1>, grid, stream, a,
                                    per_row, total)
                : launch_overlapped(block_quant_rows_kernel<T, false, VEC, UNROLL>, grid, stream, a,
                                    per_row, total);
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
