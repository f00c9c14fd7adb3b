// Attention of many rows over a paged cache (m5b_paged_attention for prompts
// and chunks of them): tcgen05 matrix products with the softmax between them.
//
// One CTA per SM works on a tile of 256 packed rows of a kv head, as two
// halves of 128 rows (an MMA's height).  Per step of 64 keys and half:
//   S = Q K^T          A, B from shared memory, 128 x 64 fp32 in TMEM
//   t = S scale log2 e, p = 2^(t - m), l += sum p   one thread a row
//   O += P V           P (the cache's type) from TMEM over S, V from shared memory
// Roles: two warpgroups, one per half, each thread owning a row of S and O;
// one thread issuing the MMAs in the order  PV0(s) QK0(s+2) PV1(s) QK1(s+2);
// one warp filling a ring with K and V blocks by TMA, one box per page.  O
// takes 2 x 128 columns of TMEM, S 2 x 2 x 64: with two buffers a half, the
// scores of step s + 1 are there when the softmax of step s ends, and neither
// the softmax nor the tensor cores wait for a chain through the other.  (One
// S buffer of 128 keys a half fits as well, but chains softmax -> PV -> QK ->
// softmax: 1.64 ms against TIME for two prompts of 8192, 32 heads.)  P
// overwrites its S.  m only follows the maximum when that has grown by more
// than 2^8; then O is rescaled in place.  The rows of the next tile are loaded
// during this one, into a second buffer.
//
// Bound by shared memory's bandwidth in the products: an MMA of 128 x 64 x 16
// reads 6 KB where its 32 cycles have 4, so that a step takes 8 * 48 + 4 * 64
// cycles a half at D = 128, 80 % of the tensor cores' rate; the exponentials,
// 128 * 64 / 16 = 512 cycles a half, fit beside them.
#include "paged_sched.cuh"

namespace m5b {
namespace {

constexpr int kBlock = kPagedBlock;  // keys per step
constexpr int kRows = 256;     // packed rows per tile, two halves
constexpr float kGrow = 8.0f;  // log2 of the growth that m may lag behind
constexpr int kThreads = 384;  // warps 0-3, 4-7: halves; 8: MMA; 9: TMA
constexpr int kMmaWarp = 8, kTmaWarp = 9;

template <int D> struct Cfg {
  static constexpr int HALVES = D / 64;              // 64-channel halves of a row
  static constexpr int Q_HALF = 128 * 128;           // 128 rows x 64 channels
  static constexpr int Q_BYTES = HALVES * Q_HALF;    // the rows of one half tile
  static constexpr int HALF_BYTES = kBlock * 128;    // 64 keys x 64 channels
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
  static constexpr int STAGES = D == 64 ? 16 : 6;
  static constexpr int SMEM = 4 * Q_BYTES + STAGES * TILE_BYTES + 1024;
  struct Small {
    uint64_t full[STAGES], empty[STAGES];
    uint64_t q_full[2][2], s_full[2][2], p_full[2][2];  // [half][buffer]
    uint64_t pv_done[2], o_full[2], drain;  // after every PV, after a piece's last
    long long scratch[kThreads / 32 + 4];
    uint32_t tmem;
    volatile int abort_flag;
  };
  static_assert(sizeof(Small) <= 1024, "shared memory layout");
};
// TMEM columns: S [half][buffer] of 64, O [half] of 128
constexpr uint32_t kColS = 0, kColO = 256;

template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// MN-major B operand (V: keys down, channels along 128-byte rows, 128-byte
// swizzle): 64-channel halves HALF_BYTES apart, 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t addr, uint32_t half_bytes) {
  uint64_t d = static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((half_bytes >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
// D (TMEM) (+)= A (TMEM) B (shared memory)
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
               "l"(__cvta_generic_to_global(src)), "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
// x of one score: capped and biased, in log2 units.
__device__ __forceinline__ float modify(float x, float softcap, float slope, int pos, int key) {
  if (softcap > 0.0f)  // tanh(y) = 1 - 2 / (e^2y + 1)
    x = softcap * (1.0f - __fdividef(2.0f, ex2(x * (2.0f * kLog2e / softcap)) + 1.0f));
  return (x - slope * fabsf(static_cast<float>(pos - key))) * kLog2e;
}

// One step of the MMA thread's stream: first or last of its piece, second half
// in use.
struct Step {
  bool valid, first, last, two;
};

template <typename T, int D, bool MOD>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prompt_kernel(const PagedAttnArgs a, const __grid_constant__ PagedMaps maps) {
  using C = Cfg<D>;
  constexpr int STAGES = C::STAGES;
  // (no static shared memory: the tiles start on the swizzle's 1024-byte grid)
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const q_smem = smem;  // [buffer][half]
  uint8_t* const ring = smem + 4 * C::Q_BYTES;
  typename C::Small& sm =
      *reinterpret_cast<typename C::Small*>(ring + STAGES * C::TILE_BYTES);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int h = 0; h < 2; ++h) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.q_full[h][i], 4);
        mbar_init(&sm.s_full[h][i], 1);
        mbar_init(&sm.p_full[h][i], 4);
      }
      mbar_init(&sm.pv_done[h], 1);
      mbar_init(&sm.o_full[h], 1);
    }
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  grid_dependency_wait();
  grid_dependents_launch();
  PagedWalk<kRows, kBlock> walk = paged_walk<kRows, kBlock, kThreads>(a, sm.scratch);  // (syncs)
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const int group = a.b.group;

  if (warp == kTmaWarp) {  // ---- K and V blocks, in the order K0 K1 V0 K2 V1 ...
    const int boxes = kBlock / maps.box_rows * C::HALVES;
    const int row = lane / C::HALVES * maps.box_rows, half = lane % C::HALVES;
    int stage = 0, phase = 0, issued = 0;
    bool ok = true;
    auto load = [&](const CUtensorMap* map, int head, int page, int slot) {
      ok = mbar_wait_bounded(&sm.empty[stage], phase ^ 1, &sm.abort_flag, a.status,
                             DEV_TIMEOUT_PRODUCER);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], C::TILE_BYTES);
      __syncwarp();
      if (lane < boxes)
        tma_load_4d(ring + stage * C::TILE_BYTES + half * C::HALF_BYTES + row * 128, map,
                    &sm.full[stage], half * 64, slot, head, page);
      ++issued;
      if (++stage == STAGES) stage = 0, phase ^= 1;
    };
    PagedPiece p;
    int head = -1, page = 0, slot = 0;  // of the step before
    while (ok && walk.next(a, p)) {
      for (int i = p.begin; ok && i < p.end; ++i) {
        const int key = p.r.at(i) * kBlock + row;
        int page2 = a.b.num_pages, slot2 = 0;  // out of range: zeros
        if (lane < boxes && key < p.s.keys) {
          const int at = paged_page(a.b, p.seq, key);
          if (at >= 0) page2 = at;
          slot2 = key % a.b.page_size;
        }
        load(&maps.k, p.head, page2, slot2);
        if (ok && head >= 0) load(&maps.v, head, page, slot);
        head = p.head, page = page2, slot = slot2;
      }
    }
    if (ok && head >= 0) load(&maps.v, head, page, slot);
    if (!ok) {  // let the copies in flight land before the CTA ends
      for (int i = 0; i < STAGES && i < issued; ++i) {
        if (--stage < 0) stage = STAGES - 1, phase ^= 1;
        const unsigned long long start = globaltimer_ns();
        while (!mbar_try_wait(&sm.full[stage], phase) && globaltimer_ns() - start < kWaitLimitNs) {
        }
      }
    }
  } else if (warp == kMmaWarp) {  // ---- matrix products, all by one thread
    if (elect_one()) {
      constexpr int kind = DTypeOf<T>::value == DT_BF16 ? KIND_BF16 : KIND_F16;
      constexpr uint32_t idesc_s = make_idesc(kind, 128, kBlock);
      constexpr uint32_t idesc_o = make_idesc(kind, 128, D) | (1u << 16);  // B is MN-major
      const uint64_t q_desc = smem_desc_k128(smem_u32(q_smem));
      const uint64_t k_desc = smem_desc_k128(smem_u32(ring));
      const uint64_t v_desc = smem_desc_mn128(smem_u32(ring), C::HALF_BYTES);
      int stage = 0, phase = 0;
      int qt[2] = {0, 0}, si[2] = {0, 0}, pi[2] = {0, 0};  // pieces, QK and PV steps of the halves
      bool ok = true;
      auto wait = [&](uint64_t* bar, int parity) {
        if (ok) ok = mbar_wait_bounded(bar, parity, &sm.abort_flag, a.status, DEV_TIMEOUT_MMA);
        return ok;
      };
      PagedPiece p{};
      int at = 0;
      bool open = false;
      auto advance = [&]() {
        Step s{};
        if (!open || at == p.end) {
          open = walk.next(a, p);
          if (!open) return s;
          at = p.begin;
        }
        s.valid = true;
        s.first = at == p.begin;
        s.two = p.s.n * group - p.rt * kRows > 128;
        s.last = ++at == p.end;
        return s;
      };
      auto take = [&](int& st) {  // the next stage of the ring, filled
        st = stage;
        wait(&sm.full[stage], phase);
        if (++stage == STAGES) stage = 0, phase ^= 1;
        tc_fence_after();
      };
      auto qk = [&](int h, int st, const Step& s) {  // S_h = Q_h K^T
        if (s.first) {
          wait(&sm.q_full[h][qt[h] & 1], (qt[h] >> 1) & 1);
          ++qt[h];
          tc_fence_after();
        }
        if (!ok) return;
        const int buf = si[h]++ & 1;
        const uint64_t qd = q_desc + ((((qt[h] - 1) & 1) * 2 + h) * C::Q_BYTES >> 4);
        const uint64_t kd = k_desc + (st * C::TILE_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma<KIND_F16>(tmem + kColS + h * 128 + buf * 64,
                           qd + (((k / 4) * C::Q_HALF + (k % 4) * 32) >> 4),
                           kd + (((k / 4) * C::HALF_BYTES + (k % 4) * 32) >> 4), idesc_s, k > 0);
        tc_commit(&sm.s_full[h][buf]);
      };
      auto pv = [&](int h, int st, const Step& s) {  // O_h (+)= P_h V
        const int buf = pi[h] & 1;
        wait(&sm.p_full[h][buf], (pi[h] >> 1) & 1);
        ++pi[h];
        tc_fence_after();
        if (!ok) return;
        const uint64_t vd = v_desc + (st * C::TILE_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < kBlock / 16; ++k)
          tc_mma_ts(tmem + kColO + h * 128, tmem + kColS + h * 128 + buf * 64 + k * 8,
                    vd + (k * 2048 >> 4), idesc_o, !s.first || k > 0);
        tc_commit(&sm.pv_done[h]);
        if (s.last) tc_commit(&sm.o_full[h]);
      };

      Step cur = advance(), nx1 = advance();
      int ks = 0, vs = 0;
      for (int i = 0; i < 2; ++i) {
        const Step& s = i ? nx1 : cur;
        if (!ok || !s.valid) break;
        take(ks);
        qk(0, ks, s);
        if (s.two) qk(1, ks, s);
        tc_commit(&sm.empty[ks]);
      }
      while (ok && cur.valid) {
        const Step nx2 = advance();
        take(vs);
        pv(0, vs, cur);
        if (nx2.valid) {
          take(ks);
          qk(0, ks, nx2);
        }
        if (cur.two) pv(1, vs, cur);
        tc_commit(&sm.empty[vs]);
        if (nx2.valid) {
          if (nx2.two) qk(1, ks, nx2);
          tc_commit(&sm.empty[ks]);
        }
        cur = nx1;
        nx1 = nx2;
      }
      // every MMA has retired before TMEM is freed
      tc_commit(&sm.drain);
      const unsigned long long start = globaltimer_ns();
      while (!mbar_try_wait(&sm.drain, 0)) {
        if (globaltimer_ns() - start > kWaitLimitNs) {
          atomicOr(a.status, DEV_TIMEOUT_DRAIN);
          break;
        }
      }
    }
    __syncwarp();
  } else if (warp < kMmaWarp) {  // ---- softmax: thread `row` of half h
    const int h = warp / 4;
    const int row = threadIdx.x % 128;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    const uint32_t t_s = lanes + kColS + h * 128, t_o = lanes + kColO + h * 128;
    const PagedPartials<kRows, D> parts(a.workspace, gridDim.x);
    const float c = a.scale * kLog2e;
    int step = 0, piece = 0;  // of this half
    bool ok = true, any = false;
    auto wait = [&](uint64_t* bar, int parity) {
      ok = mbar_wait_bounded(bar, parity, &sm.abort_flag, a.status, DEV_TIMEOUT_EPILOGUE);
      ok = __all_sync(~0u, ok);
      tc_fence_after();
      return ok;
    };
    // Row `row` of a piece into the buffer of the half's piece number n.
    auto fetch = [&](const PagedPiece& p, int n) {
      const int packed = p.rt * kRows + h * 128 + row, rows = p.s.n * group;
      const bool in = packed < rows;
      const int tok = (in ? packed : rows - 1) / group, qh = p.head * group + packed % group;
      const T* src = static_cast<const T*>(a.q) + int64_t(p.s.row0 + tok) * a.q_token + qh * a.q_head;
      const uint32_t dst = smem_u32(q_smem + ((n & 1) * 2 + h) * C::Q_BYTES) + row * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        cp_async16(dst + (i / 8) * C::Q_HALF + (((i % 8) ^ (row & 7)) << 4), src + i * 8, in);
    };
    auto fetched = [&](int n) {
      cp_async_wait_all();
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[h][n & 1]);
    };
    // The next piece with rows for this half (the first half has some in all).
    auto next = [&](PagedPiece& p) {
      while (walk.next(a, p))
        if (h == 0 || p.s.n * group - p.rt * kRows > 128) return true;
      return false;
    };
    PagedPiece p, pn;
    bool have = next(p);
    if (have) {
      fetch(p, 0);
      fetched(0);
    }
    while (have && ok) {
      any = true;
      const int rows = p.s.n * group, packed = p.rt * kRows + h * 128 + row;
      const int tok = min(packed, rows - 1) / group;
      const int pos = p.s.pos0 + tok;
      const float slope = MOD && a.slopes && packed < rows
                              ? a.slopes[p.head * group + packed % group] : 0.0f;
      const int pos_lo = p.s.pos0 + (p.rt * kRows + h * 128) / group;
      const int pos_hi = p.s.pos0 + min(p.rt * kRows + h * 128 + 127, rows - 1) / group;
      float m = -INFINITY, l = 0.0f;
      bool more = false;
      for (int i = p.begin; i < p.end; ++i, ++step) {
        const int block0 = p.r.at(i) * kBlock, buf = step & 1;
        if (!wait(&sm.s_full[h][buf], (step >> 1) & 1)) break;
        if (i == p.begin) {  // the products with the last piece's rows are done
          more = next(pn);
          if (more) fetch(pn, piece + 1);
        }
        uint32_t s[2][32];
        tmem_ld32(t_s + buf * 64, s[0]);
        tmem_ld32(t_s + buf * 64 + 32, s[1]);
        tmem_wait_ld();
        if (MOD) {
#pragma unroll
          for (int e = 0; e < kBlock; ++e)
            s[e / 32][e % 32] = __float_as_uint(modify(__uint_as_float(s[e / 32][e % 32]) * a.scale,
                                                       a.softcap, slope, pos, block0 + e));
        }
        const bool open = block0 + kBlock <= p.s.keys &&
                          (block0 + kBlock <= p.s.prefix ||
                           (block0 + kBlock - 1 <= pos_lo && pos_hi - block0 < a.window));
        if (!open) {
          const int hi = min(pos, p.s.keys - 1) - block0;
          const int lo = (pos >= a.window ? pos - a.window + 1 : 0) - block0;
          const int pre = p.s.prefix - block0;
#pragma unroll
          for (int e = 0; e < kBlock; ++e)
            if (!(e < pre || (e <= hi && e >= lo))) s[e / 32][e % 32] = 0xff800000u;
          if (h == 0 && block0 + kBlock > p.s.keys) {
            // slots behind the sequence's end may hold NaN, which a zero
            // probability would not stop: blank them before PV is issued.  (V
            // of step s is the ring's load 2 s + 2, but for the last step.)
            const int at = 2 * step + (i + 1 == p.end && !more ? 1 : 2);
            if (!wait(&sm.full[at % STAGES], (at / STAGES) & 1)) break;
            const int dead = row / 2;  // two threads a key
            if (block0 + dead >= p.s.keys)
              for (int k = row % 2; k < C::HALVES * 8; k += 2)
                *reinterpret_cast<uint4*>(ring + (at % STAGES) * C::TILE_BYTES +
                                          (k / 8) * C::HALF_BYTES + dead * 128 + (k % 8) * 16) =
                    make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_shared();
          }
        }
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = __uint_as_float(s[q / 2][(q % 2) * 16]);
#pragma unroll
          for (int e = 1; e < 16; ++e)
            top[q] = fmaxf(top[q], __uint_as_float(s[q / 2][(q % 2) * 16 + e]));
        }
        float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (!MOD) high *= c;
        const bool grow = high > m + kGrow;
        if (__any_sync(~0u, grow)) {
          const float m2 = grow ? high : m;
          const float f = m == -INFINITY ? 0.0f : ex2(m - m2);
          m = m2;
          l *= f;
          if (i > p.begin) {
            // O holds the steps before this one, once they are done.  (S of
            // this step says so of all but the last, so that the parity is
            // not two phases off.)
            if (!wait(&sm.pv_done[h], (step - 1) & 1)) break;
            uint32_t o[32];
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              tmem_ld32(t_o + q * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(t_o + q * 32, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float2 sum[2] = {};
        const float2 c2 = make_float2(c, c), b2 = make_float2(-base, -base);
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float2 x = make_float2(__uint_as_float(s[e / 16][(2 * e) % 32]),
                                 __uint_as_float(s[e / 16][(2 * e) % 32 + 1]));
          x = MOD ? __fadd2_rn(x, b2) : __ffma2_rn(x, c2, b2);
          x.x = ex2(x.x);
          x.y = ex2(x.y);
          sum[e & 1] = __fadd2_rn(sum[e & 1], x);
          pk[e] = pack2<T>(x.x, x.y);
        }
        tmem_st32(t_s + buf * 64, pk);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[h][buf]);
        if (i == p.begin && more) fetched(piece + 1);
      }
      if (!ok) break;

      if (!wait(&sm.o_full[h], piece & 1)) break;
      const bool whole = p.whole(), in = packed < rows;
      const float inv = whole ? (l > 0.0f ? 1.0f / l : 0.0f) : 1.0f;
      const int qh = p.head * group + packed % group;
      const int64_t t = p.s.row0 + tok;
      T* out = static_cast<T*>(a.out) + t * a.o_token + qh * a.o_head;
      const int64_t part = (2 * int64_t(blockIdx.x) + (p.begin == 0 ? 1 : 0)) * kRows + h * 128 + row;
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        uint32_t o[32];
        tmem_ld32(t_o + q * 32, o);
        tmem_wait_ld();
        if (!in) continue;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = pack2<T>(__uint_as_float(o[e + 2 * k]) * inv, __uint_as_float(o[e + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(out + q * 32 + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(parts.o + part * D + q * 32 + e) =
                make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      if (in && whole && a.lse)
        a.lse[t * a.b.q_heads + qh] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
      if (in && !whole) parts.ml[part] = make_float2(m, l);
      tc_fence_before();
      if (!more) break;
      p = pn;
      ++piece;
    }
    if (h == 0 && row == 0)  // (p is the CTA's last piece)
      paged_write_split(&parts.split[blockIdx.x], any ? &p : nullptr, walk.share, kRows, group);
    paged_zero_outside<T, D>(a, int64_t(blockIdx.x) * 256 + threadIdx.x, int64_t(gridDim.x) * 256);
  }
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <typename T, int D, bool MOD>
cudaError_t launch(const PagedAttnArgs& a, const PagedMaps& m, int sms, cudaStream_t stream) {
  using C = Cfg<D>;
  auto kern = paged_prompt_kernel<T, D, MOD>;
  static std::atomic<long long> shape[kMaxLaunchDevices];
  int dev = 0, n = 0, per_sm = 0;
  cudaError_t e = launch_shape(reinterpret_cast<const void*>(kern), kThreads, C::SMEM, shape, &dev,
                               &n, &per_sm);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, a, m);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(sms), 16);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, kRows, D>, a, sms);
}

template <typename T, int D>
cudaError_t by_scores(const PagedAttnArgs& a, const PagedMaps& m, int sms, cudaStream_t stream) {
  return a.softcap > 0.0f || a.slopes ? launch<T, D, true>(a, m, sms, stream)
                                      : launch<T, D, false>(a, m, sms, stream);
}

}  // namespace

int64_t paged_prompt_workspace(int head_dim, int sms) {
  return head_dim == 64 ? PagedPartials<kRows, 64>::bytes(sms) : PagedPartials<kRows, 128>::bytes(sms);
}

cudaError_t launch_paged_prompt(const PagedAttnArgs& a, const PagedMaps& m, int dtype, int sms,
                                cudaStream_t stream) {
  if (dtype == DT_F16)
    return a.b.head_dim == 64 ? by_scores<__half, 64>(a, m, sms, stream)
                              : by_scores<__half, 128>(a, m, sms, stream);
  return a.b.head_dim == 64 ? by_scores<__nv_bfloat16, 64>(a, m, sms, stream)
                            : by_scores<__nv_bfloat16, 128>(a, m, sms, stream);
}

}  // namespace m5b
