// Attention of few rows over a paged cache (m5b_paged_attention when a
// sequence has at most kDecodeRows rows per kv head: decoding, drafts).
//
// Every key and value is used by at most 16 rows, 16 flop a byte: the bound is
// DRAM, and the kernel is a stream of the cache through shared
// memory.  A producer warp fills a ring with key blocks (64 keys, K and V) by
// TMA, one box per page; each consumer warp takes 16 of the block's keys for
// 16 packed rows (mma.sync m16n8k16, whose 16-row tile fits a group of heads;
// tcgen05's 128 rows would be padding) with its own running maximum and sum,
//   t = x log2 e,  p = 2^(t - m),  l += sum p,  o += p V,
// fp32 but for p, which is rounded to the cache's type for the product (its
// relative error enters the output once, at the size of the output's own
// rounding).  m is near the row's maximum (kGrow).  At a tile's end the warps'
// parts are added through shared memory.  paged_sched.cuh deals the blocks out
// evenly whatever the lengths are; the parts of a split tile are joined by
// whichever CTA finishes its part last (a ticket per tile tells), always in the
// same order.
//
// 64 sequences of up to 8191 keys, 32 + 8 heads of 128: 182 us, 5.7 TB/s; all
// of 8000 and more 6.5 TB/s, the rate of a copy.  What short calls pay is the
// start (lengths, table, first block) and the joins, 10 us together.
#include <cfloat>

#include "paged_sched.cuh"

namespace m5b {
namespace {

constexpr int kBlock = kPagedBlock;  // keys per ring stage

template <int D> struct Cfg {
  static constexpr int ROWS = kDecodeRows;
  static constexpr int WARPS = 4;  // consumers, a slice of 16 keys each
  static constexpr int THREADS = (WARPS + 1) * 32;
  static constexpr int PER_SM = 2;
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = kBlock * 128;           // 64 channels of a block
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;    // K or V of a block
  static constexpr int STAGES = D == 64 ? 6 : 3;
  static constexpr int JOIN_BYTES = 2 * 16 * D * 4;
  static constexpr int SMEM = STAGES * 2 * TILE_BYTES + JOIN_BYTES + 1024;  // + Small
  struct Small {
    uint64_t full[STAGES], empty[STAGES];
    PagedWalkScratch<THREADS> scratch;
    float2 join_ml[2][16];
    int last;
    volatile int abort_flag;
  };
  static_assert(sizeof(Small) <= 1024, "shared memory layout");
};

template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <int N> __device__ __forceinline__ void consumers_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}

// A warp's scores q.k scaled and capped; r = scale / softcap.  Scores up to the
// cap go by tanh_ratio, those beyond by tanh(y) = 1 - 2 / (e^2y + 1), which would
// leave small ones off by 1e-7 of the cap, however large that is.
__device__ __forceinline__ void cap_scores(float (&s)[2][4], float scale, float softcap, float r) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(s[i / 4][i % 4]));
  const bool within = __all_sync(~0u, top * r <= 1.0f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float &x0 = s[i / 4][i % 4], &x1 = s[i / 4][i % 4 + 1];
    const float2 x = make_float2(x0, x1), y = __fmul2_rn(x, make_float2(r, r));
    const float2 in = __fmul2_rn(__fmul2_rn(x, make_float2(scale, scale)),
                                 tanh_ratio(__fmul2_rn(y, y)));
    x0 = in.x;
    x1 = in.y;
    if (!within) {
      if (!(fabsf(y.x) <= 1.0f))
        x0 = softcap * (1.0f - __fdividef(2.0f, ex2(y.x * (2.0f * kLog2e)) + 1.0f));
      if (!(fabsf(y.y) <= 1.0f))
        x1 = softcap * (1.0f - __fdividef(2.0f, ex2(y.y * (2.0f * kLog2e)) + 1.0f));
    }
  }
}

template <typename T, int D, bool MOD>
__global__ void __launch_bounds__(Cfg<D>::THREADS, Cfg<D>::PER_SM)
    paged_decode_kernel(const PagedAttnArgs a, const __grid_constant__ PagedMaps maps) {
  using C = Cfg<D>;
  constexpr int ROWS = C::ROWS, STAGES = C::STAGES;
  // (no static shared memory: the ring starts on the swizzle's 1024-byte grid)
  extern __shared__ __align__(1024) uint8_t ring[];
  float2* join = reinterpret_cast<float2*>(ring + STAGES * 2 * C::TILE_BYTES);
  typename C::Small& small = *reinterpret_cast<typename C::Small*>(
      ring + STAGES * 2 * C::TILE_BYTES + C::JOIN_BYTES);
  uint64_t *full = small.full, *empty = small.empty;
  auto& join_ml = small.join_ml;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], C::WARPS);
    }
    small.abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  grid_dependency_wait();
  grid_dependents_launch();
  PagedWalk<ROWS, kBlock> walk =
      paged_walk<ROWS, kBlock, C::THREADS>(a, small.scratch);  // (syncs)
  PagedPiece p;
  int stage = 0, phase = 0;

  if (warp == C::WARPS) {  // ---- producer
    const int boxes = kBlock / maps.box_rows * C::HALVES;
    const int row = lane / C::HALVES * maps.box_rows, half = lane % C::HALVES;
    int issued = 0;
    bool ok = true;
    while (ok && walk.next(a, p)) {
      const int window = paged_window<ROWS>(a, p.s, p.rt);
      for (int i = p.begin; i < p.end; ++i) {
        const int key = p.r.at(i) * kBlock + row;
        int page = a.b.num_pages, slot = 0;  // out of range: zeros
        if (lane < boxes && key < p.s.keys && (key < p.s.prefix || key > window - maps.box_rows)) {
          const int at = paged_page(a.b, p.seq, key);
          if (at >= 0) page = at;
          slot = key % a.b.page_size;
        }
        ok = mbar_wait_bounded(&empty[stage], phase ^ 1, &small.abort_flag, a.status,
                               DEV_TIMEOUT_PRODUCER);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        uint8_t* dst = ring + stage * 2 * C::TILE_BYTES + half * C::HALF_BYTES + row * 128;
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::TILE_BYTES);
        __syncwarp();
        if (lane < boxes) {
          tma_load_4d(dst, &maps.k, &full[stage], half * 64, slot, p.head, page);
          tma_load_4d(dst + C::TILE_BYTES, &maps.v, &full[stage], half * 64, slot, p.head, page);
        }
        ++issued;
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
    }
    if (!ok) {  // let the copies in flight land before the CTA ends
      for (int i = 0; i < STAGES && i < issued; ++i) {
        if (--stage < 0) stage = STAGES - 1, phase ^= 1;
        const unsigned long long start = globaltimer_ns();
        while (!mbar_try_wait(&full[stage], phase) && globaltimer_ns() - start < kWaitLimitNs) {
        }
      }
    }
    return;
  }

  // ---- consumers
  const int slice = warp;
  const int g = lane / 4, t4 = lane % 4;
  const int group = a.b.group;
  const PagedPartials<ROWS, D> parts(a.workspace, gridDim.x);
  // ldmatrix row addresses inside a block: lanes 0-7, 8-15, 16-23, 24-31 give
  // the rows of the four 8 x 8 matrices
  const int lrow = slice * 16 + (lane & 7);
  const int k_row = lrow + ((lane >> 4) & 1) * 8, k_chunk = (lane >> 3) & 1;  // keys 0-7 | 8-15 last
  const int v_row = lrow + ((lane >> 3) & 1) * 8, v_chunk = (lane >> 4) & 1;  // channels last
  const float cap_ratio = MOD && a.softcap > 0.0f ? fminf(a.scale / a.softcap, FLT_MAX) : 0.0f;
  bool ok = true;
  // (a warp whose wait gave up still walks along, for the barriers' sake)
  while (walk.next(a, p)) {
    const int first = p.rt * ROWS;
    const int rows = p.s.n * group;
    uint32_t q[D / 16][4];
    int pos[2];
    float slope[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int packed = first + g + i * 8;
      const bool in = packed < rows;
      const int tok = min(packed, rows - 1) / group, h = p.head * group + packed % group;
      pos[i] = p.s.pos0 + tok;
      if (MOD && a.slopes && in) slope[i] = a.slopes[h];
      const T* src = static_cast<const T*>(a.q) + int64_t(p.s.row0 + tok) * a.q_token + h * a.q_head + t4 * 2;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][i] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        q[k][i + 2] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
      }
    }
    const int pos_lo = p.s.pos0 + p.rt * ROWS / group;
    const int pos_hi = p.s.pos0 + min(p.rt * ROWS + ROWS - 1, rows - 1) / group;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

    for (int i = p.begin; i < p.end; ++i) {
      const int block0 = p.r.at(i) * kBlock;
      if (ok) ok = mbar_wait_bounded(&full[stage], phase, &small.abort_flag, a.status, DEV_TIMEOUT_MMA);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      const uint32_t kbase = smem_u32(ring + stage * 2 * C::TILE_BYTES);
      const uint32_t vbase = kbase + C::TILE_BYTES;
      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];
        const int chunk = (k * 2 + k_chunk) & 7;
        ldsm4(b, kbase + (k / 4) * C::HALF_BYTES + k_row * 128 + ((chunk ^ (k_row & 7)) << 4));
        mma16816<T>(s[0], q[k], b[0], b[1]);
        mma16816<T>(s[1], q[k], b[2], b[3]);
      }
      const int key0 = block0 + slice * 16 + t4 * 2;
      if (MOD && a.softcap > 0.0f) {
        cap_scores(s, a.scale, a.softcap, cap_ratio);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e / 4][e % 4] *= a.scale;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (MOD) s[n][e] -= slope[e / 2] * fabsf(static_cast<float>(pos[e / 2] - key0 - n * 8 - (e & 1)));
          s[n][e] *= kLog2e;
        }
      // (differences: positions reach the last 32-bit one)
      const bool open = p.s.keys - block0 >= kBlock &&
                        (p.s.prefix - block0 >= kBlock ||
                         (pos_lo - block0 >= kBlock - 1 && pos_hi - block0 < a.window));
      if (!open) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + n * 8 + (e & 1), at = pos[e / 2];
            if (key >= p.s.keys ||
                (key >= p.s.prefix && (key > at || at - key >= a.window)))
              s[n][e] = -INFINITY;
          }
        // slots behind the sequence's end may hold NaN, which a zero
        // probability would not stop: blank them
        const int live = p.s.keys - block0 - slice * 16;
        if (live < 16) {
          for (int r = max(live, 0); r < 16; ++r)
            for (int c = lane; c < C::HALVES * 8; c += 32)
              *reinterpret_cast<uint4*>(ring + stage * 2 * C::TILE_BYTES + C::TILE_BYTES +
                                        (c / 8) * C::HALF_BYTES + (slice * 16 + r) * 128 +
                                        (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          __syncwarp();
        }
      }
      float top[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 2));
      }
      constexpr float below = kBelow<T>, lag = kGrow + below;
      if (__any_sync(~0u, top[0] > m[0] + lag || top[1] > m[1] + lag)) {
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float m2 = fmaxf(m[r], top[r] - below);
          f[r] = m[r] == -INFINITY ? 0.0f : ex2(m[r] - m2);
          m[r] = m2;
          l[r] *= f[r];
        }
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          o[c][0] *= f[0];
          o[c][1] *= f[0];
          o[c][2] *= f[1];
          o[c][3] *= f[1];
        }
      }
      const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = ex2(s[n][e] - base[e / 2]);
          l[e / 2] += s[n][e];
        }
      const uint32_t pa[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]),
                              pack2<T>(s[1][0], s[1][1]), pack2<T>(s[1][2], s[1][3])};
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t b[4];
        const int chunk = (c * 2 + v_chunk) & 7;
        ldsm4_t(b, vbase + (c / 4) * C::HALF_BYTES + v_row * 128 + ((chunk ^ (v_row & 7)) << 4));
        mma16816<T>(o[2 * c], pa, b[0], b[1]);
        mma16816<T>(o[2 * c + 1], pa, b[2], b[3]);
      }
      // The stage's next copy comes by the async proxy, which the arrival alone
      // does not hold behind ldmatrix (and the zeros above): without the fence a
      // copy out of L2 could overtake the last ones and change V under them.
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      if (++stage == STAGES) stage = 0, phase ^= 1;
    }

    // join the four key slices: 2, 3 into 0, 1, then 1 into 0
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(~0u, l[r], 1);
      l[r] += __shfl_xor_sync(~0u, l[r], 2);
    }
    consumers_sync<C::WARPS * 32>();  // the last join's readers are done
#pragma unroll
    for (int step = 2; step >= 1; --step) {
      const int buf = step == 2 ? slice & 1 : 1;
      float2* at = join + buf * (16 * D / 2);
      const bool give = step == 2 ? slice >= 2 : slice == 1;
      const bool take = step == 2 ? slice < 2 : slice == 0;
      if (give) {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          at[(2 * c) * 32 + lane] = make_float2(o[c][0], o[c][1]);
          at[(2 * c + 1) * 32 + lane] = make_float2(o[c][2], o[c][3]);
        }
        if (t4 == 0) {
          join_ml[buf][g] = make_float2(m[0], l[0]);
          join_ml[buf][g + 8] = make_float2(m[1], l[1]);
        }
      }
      consumers_sync<C::WARPS * 32>();
      if (take) {
        float f0[2], f1[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 ml = join_ml[buf][g + r * 8];
          const float m2 = fmaxf(m[r], ml.x);
          f0[r] = m[r] == -INFINITY ? 0.0f : ex2(m[r] - m2);
          f1[r] = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m2);
          m[r] = m2;
          l[r] = l[r] * f0[r] + ml.y * f1[r];
        }
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const float2 x = at[(2 * c) * 32 + lane], y = at[(2 * c + 1) * 32 + lane];
          o[c][0] = o[c][0] * f0[0] + x.x * f1[0];
          o[c][1] = o[c][1] * f0[0] + x.y * f1[0];
          o[c][2] = o[c][2] * f0[1] + y.x * f1[1];
          o[c][3] = o[c][3] * f0[1] + y.y * f1[1];
        }
      }
    }
    const bool whole = p.whole();
    if (slice == 0) {
      const int64_t slot = 2 * int64_t(blockIdx.x) + (p.begin == 0 ? 1 : 0);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int packed = first + g + r * 8;
        if (packed >= rows) continue;
        if (whole) {
          const int64_t tok = p.s.row0 + packed / group;
          const int h = p.head * group + packed % group;
          const bool none = l[r] == 0.0f;  // (NaN is something)
          const float inv = none ? 0.0f : 1.0f / l[r];
          T* out = static_cast<T*>(a.out) + tok * a.o_token + h * a.o_head + t4 * 2;
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint32_t*>(out + c * 8) =
                pack2<T>(o[c][2 * r] * inv, o[c][2 * r + 1] * inv);
          if (a.lse && t4 == 0)
            a.lse[tok * a.b.q_heads + h] = none ? -INFINITY : (m[r] + log2f(l[r])) * kLn2;
        } else {
          const int64_t at = slot * ROWS + g + r * 8;
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<float2*>(parts.o + at * D + c * 8 + t4 * 2) =
                make_float2(o[c][2 * r], o[c][2 * r + 1]);
          if (t4 == 0) parts.ml[at] = make_float2(m[r], l[r]);
        }
      }
    }
    if (!whole) {  // the last CTA to get here joins the tile's parts
      __threadfence();
      consumers_sync<C::WARPS * 32>();
      const int from = static_cast<int>(paged_div(p.tile_at, walk.share));
      const int to = static_cast<int>(paged_div(p.tile_at + p.r.blocks - 1, walk.share));
      if (threadIdx.x == 0) small.last = atomicAdd(&a.tickets[from], 1) == to - from;
      consumers_sync<C::WARPS * 32>();
      if (small.last) {
        __threadfence();
        // (four rows a warp at once would hold more loads in flight yet, but
        // cost a step of few rows more in code than it gains the others)
        const int n = min(ROWS, rows - first);
        int r = warp;
#pragma unroll 1
        for (; r + C::WARPS < n; r += 2 * C::WARPS)
          paged_join_rows<T, ROWS, D, 2, C::WARPS>(a, parts, from, to - from + 1, r, p.s.row0, p.head, first);
        if (r < n)
          paged_join_rows<T, ROWS, D, 1, C::WARPS>(a, parts, from, to - from + 1, r, p.s.row0, p.head, first);
        if (threadIdx.x == 0) a.tickets[from] = 0;
      }
    }
  }
  paged_zero_outside<T, D>(a, int64_t(blockIdx.x) * (C::WARPS * 32) + threadIdx.x,
                           int64_t(gridDim.x) * (C::WARPS * 32));
}

template <typename T, int D, bool MOD>
cudaError_t launch(const PagedAttnArgs& a, const PagedMaps& m, int sms, cudaStream_t stream) {
  using C = Cfg<D>;
  auto kern = paged_decode_kernel<T, D, MOD>;
  static std::atomic<long long> shape[kMaxLaunchDevices];
  int dev = 0, n = 0, per_sm = 0;
  cudaError_t e = launch_shape(reinterpret_cast<const void*>(kern), C::THREADS, C::SMEM, shape,
                               &dev, &n, &per_sm);
  if (e != cudaSuccess) return e;
  const int ctas = sms * C::PER_SM;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, m);
}

template <typename T, int D>
cudaError_t by_scores(const PagedAttnArgs& a, const PagedMaps& m, int sms, cudaStream_t stream) {
  return a.softcap > 0.0f || a.slopes ? launch<T, D, true>(a, m, sms, stream)
                                      : launch<T, D, false>(a, m, sms, stream);
}

}  // namespace

int64_t paged_decode_workspace(int head_dim, int sms) {
  return head_dim == 64 ? PagedPartials<kDecodeRows, 64>::bytes(2 * sms)
                        : PagedPartials<kDecodeRows, 128>::bytes(2 * sms);
}

cudaError_t launch_paged_decode(const PagedAttnArgs& a, const PagedMaps& m, int dtype, int sms,
                                cudaStream_t stream) {
  if (dtype == DT_F16)
    return a.b.head_dim == 64 ? by_scores<__half, 64>(a, m, sms, stream)
                              : by_scores<__half, 128>(a, m, sms, stream);
  return a.b.head_dim == 64 ? by_scores<__nv_bfloat16, 64>(a, m, sms, stream)
                            : by_scores<__nv_bfloat16, 128>(a, m, sms, stream);
}

}  // namespace m5b
