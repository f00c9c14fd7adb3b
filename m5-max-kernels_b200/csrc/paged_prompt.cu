// Attention of many rows over a paged cache (m5b_paged_attention for prompts
// and chunks of them): tcgen05 matrix products with the softmax between them.
//
// One CTA per SM works on a tile of 256 packed rows of a kv head, as two
// halves of 128 rows (an MMA's height).  Per block of 128 keys and half:
//   S = Q K^T          A, B from shared memory, 128 x 128 fp32 in TMEM
//   t = S scale log2 e, p = 2^(t - m), l += sum p   one thread a row
//   O += P V           P (the cache's type) from TMEM over S, V from shared memory
// Roles: two warpgroups, one per half, each thread owning a row of S and O;
// one warp issuing the MMAs in the order  PV0(j) QK0(j+1) PV1(j) QK1(j+1),  so
// that one half's softmax runs under the other half's products; one warp
// filling a ring with K and V blocks by TMA, one box per page.  S, P and O of
// both halves take the 512 columns of TMEM: P overwrites S, and since MMAs
// retire in order, S of block j + 1 being there also says that P of block j
// is used up and O is up to date.  m only follows the maximum when that has
// grown by more than 2^8; then O is rescaled in place.  Rows are loaded for
// the next tile while the last block's softmax runs.
//
// The products take 4 * 128 * 128 * D flop a half and block, 1024 cycles at
// D = 128; the exponentials 128 * 128 / 16 = 1024 cycles of the SM's special
// function units: the kernel is bound by both alike.
#include "paged_sched.cuh"

namespace m5b {
namespace {

constexpr int kBlock = 128;    // keys per block
constexpr int kRows = 256;     // packed rows per tile, two halves
constexpr float kGrow = 8.0f;  // log2 of the growth that m may lag behind
constexpr int kThreads = 384;  // warps 0-3, 4-7: halves; 8: MMA; 9: TMA
constexpr int kMmaWarp = 8, kTmaWarp = 9;

template <int D> struct Cfg {
  static constexpr int HALVES = D / 64;               // 64-channel halves of a row
  static constexpr int HALF_BYTES = 128 * 128;        // 128 rows x 64 channels
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
  static constexpr int STAGES = D == 64 ? 8 : 5;
  static constexpr int SMEM = (2 + STAGES) * TILE_BYTES + 1024;
  struct Small {
    uint64_t full[STAGES], empty[STAGES];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], drain;
    long long scratch[kThreads / 32 + 4];
    uint32_t tmem;
    volatile int abort_flag;
  };
  static_assert(sizeof(Small) <= 1024, "shared memory layout");
};
// TMEM columns
constexpr uint32_t kColS = 0, kColO = 256;  // S0 S1 O0 O1, 128 columns each

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
template <int N> __device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// x of one score: capped and biased, in log2 units.
__device__ __forceinline__ float modify(float x, float softcap, float slope, int pos, int key) {
  if (softcap > 0.0f)  // tanh(y) = 1 - 2 / (e^2y + 1)
    x = softcap * (1.0f - __fdividef(2.0f, ex2(x * (2.0f * kLog2e / softcap)) + 1.0f));
  return (x - slope * fabsf(static_cast<float>(pos - key))) * kLog2e;
}

// One block of the MMA warp's stream.
struct Step {
  bool valid, first, last, two;  // first / last block of its piece; second half in use
  int live;                      // keys of the block that exist
};

template <typename T, int D, bool MOD>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prompt_kernel(const PagedAttnArgs a, const __grid_constant__ PagedMaps maps) {
  using C = Cfg<D>;
  constexpr int STAGES = C::STAGES;
  // (no static shared memory: the tiles start on the swizzle's 1024-byte grid)
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const q_smem = smem;  // two halves of rows
  uint8_t* const ring = smem + 2 * C::TILE_BYTES;
  typename C::Small& sm =
      *reinterpret_cast<typename C::Small*>(smem + (2 + STAGES) * C::TILE_BYTES);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&sm.q_full[h], 4);
      mbar_init(&sm.s_full[h], 1);
      mbar_init(&sm.p_full[h], 4);
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

  if (warp >= 8) {
    regs_dec<72>();
    if (warp == kTmaWarp) {  // ---- K and V blocks
      const int boxes = kBlock / maps.box_rows * C::HALVES;
      const int row = lane / C::HALVES * maps.box_rows, half = lane % C::HALVES;
      int stage = 0, phase = 0, issued = 0;
      bool ok = true;
      PagedPiece p;
      while (ok && walk.next(a, p)) {
        for (int i = p.begin; ok && i < p.end; ++i) {
          const int key = p.r.at(i) * kBlock + row;
          int page = a.b.num_pages, slot = 0;  // out of range: zeros
          if (lane < boxes && key < p.s.keys) {
            const int at = paged_page(a.b, p.seq, key);
            if (at >= 0) page = at;
            slot = key % a.b.page_size;
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = mbar_wait_bounded(&sm.empty[stage], phase ^ 1, &sm.abort_flag, a.status,
                                   DEV_TIMEOUT_PRODUCER);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], C::TILE_BYTES);
            __syncwarp();
            if (lane < boxes)
              tma_load_4d(ring + stage * C::TILE_BYTES + half * C::HALF_BYTES + row * 128,
                          kv ? &maps.v : &maps.k, &sm.full[stage], half * 64, slot, p.head, page);
            ++issued;
            if (++stage == STAGES) stage = 0, phase ^= 1;
          }
        }
      }
      if (!ok) {  // let the copies in flight land before the CTA ends
        for (int i = 0; i < STAGES && i < issued; ++i) {
          if (--stage < 0) stage = STAGES - 1, phase ^= 1;
          const unsigned long long start = globaltimer_ns();
          while (!mbar_try_wait(&sm.full[stage], phase) && globaltimer_ns() - start < kWaitLimitNs) {
          }
        }
      }
    } else if (warp == kMmaWarp) {  // ---- matrix products
      constexpr int kind = DTypeOf<T>::value == DT_BF16 ? KIND_BF16 : KIND_F16;
      constexpr uint32_t idesc_s = make_idesc(kind, 128, kBlock);
      constexpr uint32_t idesc_o = make_idesc(kind, 128, D) | (1u << 16);  // B is MN-major
      int stage = 0, phase = 0;
      int ph_q[2] = {0, 0}, ph_p[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, int parity) {
        if (ok) ok = mbar_wait_bounded(bar, parity, &sm.abort_flag, a.status, DEV_TIMEOUT_MMA);
        ok = __all_sync(~0u, ok);
        tc_fence_after();
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
        s.live = p.s.keys - p.r.at(at) * kBlock;
        s.last = ++at == p.end;
        return s;
      };
      auto qk = [&](int h, int st) {  // S_h = Q_h K^T
        if (lane == 0) {
          const uint32_t qa = smem_u32(q_smem + h * C::TILE_BYTES);
          const uint32_t ka = smem_u32(ring + st * C::TILE_BYTES);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k / 4) * C::HALF_BYTES + (k % 4) * 32;
            tc_mma<KIND_F16>(tmem + kColS + h * 128, smem_desc_k128(qa + off),
                             smem_desc_k128(ka + off), idesc_s, k > 0);
          }
          tc_commit(&sm.s_full[h]);
        }
        __syncwarp();
      };
      auto pv = [&](int h, int st, const Step& s) {  // O_h (+)= P_h V
        if (lane == 0) {
          const uint32_t va = smem_u32(ring + st * C::TILE_BYTES);
#pragma unroll
          for (int k = 0; k < kBlock / 16; ++k)
            tc_mma_ts(tmem + kColO + h * 128, tmem + kColS + h * 128 + k * 8,
                      smem_desc_mn128(va + k * 2048, C::HALF_BYTES), idesc_o, !s.first || k > 0);
          if (s.last) tc_commit(&sm.o_full[h]);
        }
        __syncwarp();
      };
      auto release = [&](int st) {
        if (lane == 0) tc_commit(&sm.empty[st]);
        __syncwarp();
      };
      auto take = [&](int& st) {  // the next stage of the ring, filled
        st = stage;
        const bool r = wait(&sm.full[stage], phase);
        if (++stage == STAGES) stage = 0, phase ^= 1;
        return r;
      };

      Step cur = advance();
      int ks = 0, vs = 0;
      if (cur.valid && wait(&sm.q_full[0], 0) && take(ks)) {
        ph_q[0] ^= 1;
        qk(0, ks);
        if (cur.two) {
          if (wait(&sm.q_full[1], 0)) qk(1, ks);
          ph_q[1] ^= 1;
        }
        if (ok) release(ks);
      }
      while (ok && cur.valid) {
        const Step nxt = advance();
        if (!take(vs)) break;
        if (cur.live < kBlock) {
          // slots behind the sequence's end may hold NaN, which a zero
          // probability would not stop: blank them
          uint8_t* v = ring + vs * C::TILE_BYTES;
          for (int r = max(cur.live, 0); r < kBlock; ++r)
            if (lane < C::HALVES * 8)
              *reinterpret_cast<uint4*>(v + (lane / 8) * C::HALF_BYTES + r * 128 + (lane % 8) * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_shared();
          __syncwarp();
        }
        if (!wait(&sm.p_full[0], ph_p[0])) break;
        ph_p[0] ^= 1;
        pv(0, vs, cur);
        if (nxt.valid) {
          if (nxt.first) {
            if (!wait(&sm.q_full[0], ph_q[0])) break;
            ph_q[0] ^= 1;
          }
          if (!take(ks)) break;
          qk(0, ks);
        }
        if (cur.two) {
          if (!wait(&sm.p_full[1], ph_p[1])) break;
          ph_p[1] ^= 1;
          pv(1, vs, cur);
        }
        release(vs);
        if (nxt.valid) {
          if (nxt.two) {
            if (nxt.first) {
              if (!wait(&sm.q_full[1], ph_q[1])) break;
              ph_q[1] ^= 1;
            }
            qk(1, ks);
          }
          release(ks);
        }
        cur = nxt;
      }
      // every MMA has retired before TMEM is freed
      if (lane == 0) {
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
    }
  } else {  // ---- softmax: thread `row` of half h
    regs_inc<216>();
    const int h = warp / 4;
    const int row = threadIdx.x % 128;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    const uint32_t t_s = lanes + kColS + h * 128, t_o = lanes + kColO + h * 128;
    const PagedPartials<kRows, D> parts(a.workspace, gridDim.x);
    const float c = a.scale * kLog2e;
    int ph_s = 0, ph_o = 0;
    bool ok = true, any = false;

    // The piece's own row: its token and head, and its copy into shared memory.
    auto fetch = [&](const PagedPiece& p) {
      const int packed = p.rt * kRows + h * 128 + row, rows = p.s.n * group;
      const bool in = packed < rows;
      const int tok = (in ? packed : rows - 1) / group, qh = p.head * group + packed % group;
      const T* src = static_cast<const T*>(a.q) + int64_t(p.s.row0 + tok) * a.q_token + qh * a.q_head;
      const uint32_t dst = smem_u32(q_smem + h * C::TILE_BYTES) + row * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        cp_async16(dst + (i / 8) * C::HALF_BYTES + (((i % 8) ^ (row & 7)) << 4), src + i * 8, in);
    };
    auto fetched = [&]() {
      cp_async_wait_all();
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[h]);
    };
    // The next piece with rows for this half (the first half has some in all).
    PagedPiece seen;  // last piece of the walk
    auto next = [&](PagedPiece& p) {
      while (walk.next(a, p)) {
        any = true;
        seen = p;
        if (h == 0 || p.s.n * group - p.rt * kRows > 128) return true;
      }
      return false;
    };
    PagedPiece p, pn;
    bool have = next(p);
    if (have) {
      fetch(p);
      fetched();
    }
    while (have && ok) {
      const int rows = p.s.n * group, packed = p.rt * kRows + h * 128 + row;
      const int tok = min(packed, rows - 1) / group;
      const int pos = p.s.pos0 + tok;
      const float slope = MOD && a.slopes && packed < rows
                              ? a.slopes[p.head * group + packed % group] : 0.0f;
      const int pos_lo = p.s.pos0 + (p.rt * kRows + h * 128) / group;
      const int pos_hi = p.s.pos0 + min(p.rt * kRows + h * 128 + 127, rows - 1) / group;
      float m = -INFINITY, l = 0.0f;
      bool more = false;
      for (int i = p.begin; i < p.end; ++i) {
        const int block0 = p.r.at(i) * kBlock;
        ok = mbar_wait_bounded(&sm.s_full[h], ph_s, &sm.abort_flag, a.status, DEV_TIMEOUT_EPILOGUE);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        ph_s ^= 1;
        tc_fence_after();
        if (i + 1 == p.end) {  // Q K^T of this tile is done: bring the next tile's rows
          more = next(pn);
          if (more) fetch(pn);
        }
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(t_s + q * 32, s[q]);
        tmem_wait_ld();
        if (MOD) {
#pragma unroll
          for (int e = 0; e < 128; ++e)
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
          for (int e = 0; e < 128; ++e)
            if (!(e < pre || (e <= hi && e >= lo))) s[e / 32][e % 32] = 0xff800000u;
        }
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = __uint_as_float(s[q][0]);
#pragma unroll
          for (int e = 1; e < 32; ++e) top[q] = fmaxf(top[q], __uint_as_float(s[q][e]));
        }
        float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (!MOD) high *= c;
        const bool grow = high > m + kGrow;
        if (__any_sync(~0u, grow)) {
          const float m2 = grow ? high : m;
          const float f = m == -INFINITY ? 0.0f : ex2(m - m2);
          m = m2;
          l *= f;
          if (i > p.begin) {  // O holds the blocks before this one
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
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int at = q * 64 + 2 * e;
            float2 x = make_float2(__uint_as_float(s[at / 32][at % 32]),
                                   __uint_as_float(s[at / 32][at % 32 + 1]));
            x = MOD ? __fadd2_rn(x, b2) : __ffma2_rn(x, c2, b2);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum[e & 1] = __fadd2_rn(sum[e & 1], x);
            pk[e] = pack2<T>(x.x, x.y);
          }
          tmem_st32(t_s + q * 32, pk);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[h]);
      }
      if (!ok) break;
      if (more) fetched();

      ok = mbar_wait_bounded(&sm.o_full[h], ph_o, &sm.abort_flag, a.status, DEV_TIMEOUT_EPILOGUE);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      ph_o ^= 1;
      tc_fence_after();
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
      p = pn;
      have = more;
    }
    if (h == 0 && row == 0)
      paged_write_split(&parts.split[blockIdx.x], any ? &seen : nullptr, walk.share, kRows, group);
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
