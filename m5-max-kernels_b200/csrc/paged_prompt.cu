// Attention of many rows over a paged cache (m5b_paged_attention for prompts
// and chunks of them): tcgen05 matrix products with the softmax between them.
//
// One CTA per SM works on a tile of 256 packed rows of a kv head, as two
// halves of 128 rows (an MMA's height).  Per step of 64 keys and half:
//   S = Q K^T          A, B from shared memory, 128 x 64 fp32 in TMEM
//   t = S scale log2 e, p = 2^(t - m), l += sum p   one thread a row
//   O += P V           P (the cache's type) from TMEM over S, V from shared memory
// Roles: two warpgroups, one per half, each thread owning a row of S and O; one
// thread per half issuing its MMAs, PV(s) QK(s+2) PV(s+1) ... (a wait on an
// mbarrier costs an issuing thread some 55 cycles even when there is nothing
// to wait for, and the tensor cores' queue holds but four to six MMAs: by one
// thread for both halves a step took 2090 cycles); one warp filling a ring
// with K and V blocks by TMA, one box per page; one warp finding the CTA's
// pieces of tiles and loading their rows, one piece ahead.  O
// takes 2 x 128 columns of TMEM, S 2 x 2 x 64: with two buffers a half, the
// scores of step s + 1 are there when the softmax of step s ends, and neither
// the softmax nor the tensor cores wait for a chain through the other.  (One
// S buffer of 128 keys a half fits as well, but chains softmax -> PV -> QK ->
// softmax: 1.64 ms against TIME for two prompts of 8192, 32 heads.)  P
// overwrites its S.  m only follows the row's maximum when that has grown by
// more than 2^8, which the softmax finds out after the fact: it takes the
// exponentials with the old m, looks at the largest, and in the rare case
// takes them again after rescaling O in place.
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
constexpr float kGrow = 8.0f;           // log2 of the growth that m may lag behind
constexpr int kFmaPairs = 3;             // of 8 pairs of exponentials, those by ex2_fma
constexpr int kThreads = 384;  // warps 0-3, 4-7: halves; 8, 9: their MMAs; 10: K, V; 11: rows
constexpr int kMmaWarp = 8, kTmaWarp = 10, kRowWarp = 11;

// What the CTA's other warps need to know of a piece.
struct Piece {
  int begin, end;       // steps; end == 0: there is no piece any more
  int pre, from;        // PagedBlocks
  int keys, prefix, pos0;
  int rows, first;      // packed rows of the sequence's kv head, first of the tile
  int row0, head, whole, slot;
};

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
    uint64_t q_full[2], q_empty[2];          // [buffer] of rows and pieces
    uint64_t s_full[2][2], p_full[2][2];     // [half][buffer]
    uint64_t pv_done[2], o_full[2], drain[2];  // after every PV, after a piece's last
    uint64_t landed;                            // a V block to be blanked
    long long scratch[kThreads / 32 + 4];
    Piece piece[2];
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
// 2^x of a pair on the FMA pipes, for x < 100: x = n + f with n the nearest
// integer (adding 1.5 * 2^23 leaves it in the low bits), 2^f by a polynomial,
// n added to its exponent.  The coefficients are the minimax fit of the
// relative error on [-1/2, 1/2] (Remez exchange): 7.5e-5 with four, for bf16
// probabilities (their rounding: up to 3.9e-3), 2.6e-6 with five, for fp16
// (4.9e-4).  Below -126 the result stays near 2^-126, not zero: a row that saw
// no key is known by its m.
template <typename T> __device__ __forceinline__ float2 ex2_fma(float2 x) {
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const float2 big = make_float2(12582912.0f, 12582912.0f);
  const float2 neg = make_float2(-12582912.0f, -12582912.0f), one = make_float2(-1.0f, -1.0f);
  const float2 r = __fadd2_rn(x, big);
  const float2 f = __ffma2_rn(__fadd2_rn(r, neg), one, x);
  float2 p;
  if (DTypeOf<T>::value == DT_BF16) {
    p = __ffma2_rn(make_float2(0x1.c3f76p-5f, 0x1.c3f76p-5f), f, make_float2(0x1.f0de1ap-3f, 0x1.f0de1ap-3f));
    p = __ffma2_rn(p, f, make_float2(0x1.62f31ap-1f, 0x1.62f31ap-1f));
    p = __ffma2_rn(p, f, make_float2(0x1.fff692p-1f, 0x1.fff692p-1f));
  } else {
    p = __ffma2_rn(make_float2(0x1.3997d6p-7f, 0x1.3997d6p-7f), f, make_float2(0x1.ca144p-5f, 0x1.ca144p-5f));
    p = __ffma2_rn(p, f, make_float2(0x1.ec06dap-3f, 0x1.ec06dap-3f));
    p = __ffma2_rn(p, f, make_float2(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
    p = __ffma2_rn(p, f, make_float2(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  }
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(r.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(r.y) << 23)));
}

// x of one score: capped and biased, in log2 units.
__device__ __forceinline__ float modify(float x, float softcap, float slope, int pos, int key) {
  if (softcap > 0.0f)  // tanh(y) = 1 - 2 / (e^2y + 1)
    x = softcap * (1.0f - __fdividef(2.0f, ex2(x * (2.0f * kLog2e / softcap)) + 1.0f));
  return (x - slope * fabsf(static_cast<float>(pos - key))) * kLog2e;
}

// One step of an MMA thread's stream: first or last of its piece, one that its
// half takes part in, with the rows in buffer buf.
struct Step {
  bool valid, first, last, mine;
  int buf;
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
      mbar_init(&sm.empty[i], 2);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&sm.q_full[h], 1);
      mbar_init(&sm.q_empty[h], 10);  // the softmax warps and the MMA threads
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.s_full[h][i], 1);
        mbar_init(&sm.p_full[h][i], 4);
      }
      mbar_init(&sm.pv_done[h], 1);
      mbar_init(&sm.o_full[h], 1);
      mbar_init(&sm.drain[h], 1);
    }
    mbar_init(&sm.landed, 1);
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
    int blank = -1, blank_from = 0, ph_landed = 0;  // a stage whose last keys are to be blanked
    bool ok = true;
    auto load = [&](const CUtensorMap* map, int head, int page, int slot, int live) {
      if (ok)
        ok = mbar_wait_bounded(&sm.empty[stage], phase ^ 1, &sm.abort_flag, a.status,
                               DEV_TIMEOUT_PRODUCER);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      uint64_t* bar = live < kBlock ? &sm.landed : &sm.full[stage];
      if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE_BYTES);
      __syncwarp();
      if (lane < boxes)
        tma_load_4d(ring + stage * C::TILE_BYTES + half * C::HALF_BYTES + row * 128, map, bar,
                    half * 64, slot, head, page);
      if (live < kBlock) blank = stage, blank_from = max(live, 0);
      ++issued;
      if (++stage == STAGES) stage = 0, phase ^= 1;
    };
    // Slots behind the sequence's end may hold NaN, which a zero probability
    // would not stop: V blocks that reach there land here first and are
    // blanked, while the K block after them is on its way.
    auto finish = [&]() {
      if (blank < 0) return;
      if (ok)
        ok = mbar_wait_bounded(&sm.landed, ph_landed, &sm.abort_flag, a.status,
                               DEV_TIMEOUT_PRODUCER);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      ph_landed ^= 1;
      uint8_t* v = ring + blank * C::TILE_BYTES;
      for (int i = blank_from * C::HALVES * 8 + lane; i < kBlock * C::HALVES * 8; i += 32)
        *reinterpret_cast<uint4*>(v + (i / 8 % C::HALVES) * C::HALF_BYTES + i / (C::HALVES * 8) * 128 +
                                  i % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.full[blank]);
      blank = -1;
    };
    PagedPiece p;
    int head = -1, page = 0, slot = 0, live = 0;  // of the step before
    while (ok && walk.next(a, p)) {
      for (int i = p.begin; ok && i < p.end; ++i) {
        const int block0 = p.r.at(i) * kBlock, key = block0 + row;
        int page2 = a.b.num_pages, slot2 = 0;  // out of range: zeros
        if (lane < boxes && key < p.s.keys) {
          const int at = paged_page(a.b, p.seq, key);
          if (at >= 0) page2 = at;
          slot2 = key % a.b.page_size;
        }
        load(&maps.k, p.head, page2, slot2, kBlock);
        finish();
        if (head >= 0) load(&maps.v, head, page, slot, live);
        head = p.head, page = page2, slot = slot2, live = p.s.keys - block0;
      }
    }
    finish();
    if (head >= 0) load(&maps.v, head, page, slot, live);
    finish();
    if (!ok) {  // let the copies in flight land before the CTA ends
      for (int i = 0; i < STAGES && i < issued; ++i) {
        if (--stage < 0) stage = STAGES - 1, phase ^= 1;
        const unsigned long long start = globaltimer_ns();
        while (!(stage == blank ? mbar_try_wait(&sm.landed, ph_landed)
                                : mbar_try_wait(&sm.full[stage], phase)) &&
               globaltimer_ns() - start < kWaitLimitNs) {
        }
      }
    }
  } else if (warp == kRowWarp) {  // ---- pieces and their rows
    constexpr int CH = D / 8;  // 16-byte chunks of a row
    const int chunk = lane % CH;
    bool ok = true, any = false;
    PagedPiece p;
    for (int n = 0; ok; ++n) {
      const int buf = n & 1;
      const bool more = walk.next(a, p);
      any |= more;
      ok = mbar_wait_bounded(&sm.q_empty[buf], (n >> 1 & 1) ^ 1, &sm.abort_flag, a.status,
                             DEV_TIMEOUT_PRODUCER);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      const int rows = p.s.n * group, first = p.rt * kRows;
      if (more) {
        const int here = min(rows - first, kRows), all = here > 128 ? kRows : 128;
        int r = lane / CH, tok = (first + r) / group, g = (first + r) % group;
        for (; r < all; r += 32 / CH) {
          const bool in = r < here;
          const T* src = static_cast<const T*>(a.q) + int64_t(p.s.row0 + (in ? tok : 0)) * a.q_token +
                         (p.head * group + g) * a.q_head + chunk * 8;
          cp_async16(smem_u32(q_smem + buf * 2 * C::Q_BYTES + (r / 128) * C::Q_BYTES +
                              (chunk / 8) * C::Q_HALF + (r % 128) * 128 +
                              (((chunk % 8) ^ (r & 7)) << 4)), src, in);
          for (g += 32 / CH; g >= group; g -= group) ++tok;
        }
      }
      if (lane == 0) {
        Piece d{};
        if (more) {
          d.begin = p.begin;
          d.end = p.end;
          d.pre = p.r.pre;
          d.from = p.r.from;
          d.keys = p.s.keys;
          d.prefix = p.s.prefix;
          d.pos0 = p.s.pos0;
          d.rows = rows;
          d.first = first;
          d.row0 = p.s.row0;
          d.head = p.head;
          d.whole = p.whole();
          d.slot = 2 * blockIdx.x + (p.begin == 0 ? 1 : 0);
        }
        sm.piece[buf] = d;
      }
      cp_async_wait_all();
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[buf]);
      if (!more) break;
    }
    if (lane == 0)  // (p is the last piece)
      paged_write_split(&PagedPartials<kRows, D>(a.workspace, gridDim.x).split[blockIdx.x],
                        any ? &p : nullptr, walk.share, kRows, group);
  } else if (warp >= kMmaWarp) {  // ---- matrix products of half h, by one thread
    const int h = warp - kMmaWarp;
    if (elect_one()) {
      constexpr int kind = DTypeOf<T>::value == DT_BF16 ? KIND_BF16 : KIND_F16;
      constexpr uint32_t idesc_s = make_idesc(kind, 128, kBlock);
      constexpr uint32_t idesc_o = make_idesc(kind, 128, D) | (1u << 16);  // B is MN-major
      const uint64_t q_desc = smem_desc_k128(smem_u32(q_smem + h * C::Q_BYTES));
      const uint64_t k_desc = smem_desc_k128(smem_u32(ring));
      const uint64_t v_desc = smem_desc_mn128(smem_u32(ring), C::HALF_BYTES);
      const uint32_t t_s = tmem + kColS + h * 128, t_o = tmem + kColO + h * 128;
      int stage = 0, phase = 0;
      int piece = -1, si = 0, pi = 0;  // QK and PV steps of this half
      int left = 0;  // steps of the piece
      bool ok = true, mine = false, ended = false;
      auto wait = [&](uint64_t* bar, int parity) {
        if (ok) ok = mbar_wait_bounded(bar, parity, &sm.abort_flag, a.status, DEV_TIMEOUT_MMA);
        tc_fence_after();
      };
      auto advance = [&]() {
        Step s{};
        if (ended) return s;
        if (left == 0) {
          ++piece;
          wait(&sm.q_full[piece & 1], piece >> 1 & 1);
          if (ok) {
            const Piece& d = sm.piece[piece & 1];
            left = d.end - d.begin;
            mine = h == 0 || d.rows - d.first > 128;
            mbar_arrive(&sm.q_empty[piece & 1]);
          }
          ended = !ok || left == 0;
          if (ended) return s;
          s.first = true;
        }
        s.valid = true;
        s.mine = mine;
        s.buf = piece & 1;
        s.last = --left == 0;
        return s;
      };
      // The next stage of the ring, once it is filled, for a step of this half
      // or of the other alone.
      auto use = [&](bool mine, auto&& products) {
        const int st = stage;
        wait(&sm.full[st], phase);
        if (++stage == STAGES) stage = 0, phase ^= 1;
        if (mine && ok) {
          products(st * C::TILE_BYTES >> 4);
          tc_commit(&sm.empty[st]);
        } else {
          mbar_arrive(&sm.empty[st]);
        }
      };
      auto qk = [&](const Step& s) {  // S = Q K^T
        use(s.mine, [&](int off) {
          const int buf = si++ & 1;
          const uint64_t qd = q_desc + (s.buf * 2 * C::Q_BYTES >> 4), kd = k_desc + off;
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            tc_mma<KIND_F16>(t_s + buf * 64, qd + (((k / 4) * C::Q_HALF + (k % 4) * 32) >> 4),
                             kd + (((k / 4) * C::HALF_BYTES + (k % 4) * 32) >> 4), idesc_s, k > 0);
          tc_commit(&sm.s_full[h][buf]);
        });
      };
      auto pv = [&](const Step& s) {  // O (+)= P V
        use(s.mine, [&](int off) {
          const int buf = pi & 1;
          wait(&sm.p_full[h][buf], (pi >> 1) & 1);
          ++pi;
          const uint64_t vd = v_desc + off;
#pragma unroll
          for (int k = 0; k < kBlock / 16; ++k)
            tc_mma_ts(t_o, t_s + buf * 64 + k * 8, vd + (k * 2048 >> 4), idesc_o, !s.first || k > 0);
          tc_commit(&sm.pv_done[h]);
          if (s.last) tc_commit(&sm.o_full[h]);
        });
      };
      Step cur = advance();
      if (cur.valid) qk(cur);
      Step nx1 = advance();
      if (nx1.valid) qk(nx1);
      while (ok && cur.valid) {
        pv(cur);
        // (a piece's rows may have to wait for the softmax of the piece two
        // before, which needs this PV)
        const Step nx2 = advance();
        if (nx2.valid) qk(nx2);
        cur = nx1;
        nx1 = nx2;
      }
      // every MMA has retired before TMEM is freed
      tc_commit(&sm.drain[h]);
      const unsigned long long start = globaltimer_ns();
      while (!mbar_try_wait(&sm.drain[h], 0)) {
        if (globaltimer_ns() - start > kWaitLimitNs) {
          atomicOr(a.status, DEV_TIMEOUT_DRAIN);
          break;
        }
      }
    }
    __syncwarp();
  } else {  // ---- softmax: thread `row` of half h
    const int h = warp / 4;
    const int row = threadIdx.x % 128;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    const uint32_t t_s = lanes + kColS + h * 128, t_o = lanes + kColO + h * 128;
    const float c = MOD ? 1.0f : a.scale * kLog2e;
    int step = 0, outs = 0;  // steps and pieces of this half
    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) {
      if (!__all_sync(~0u, mbar_try_wait(bar, parity))) {
        ok = mbar_wait_bounded(bar, parity, &sm.abort_flag, a.status, DEV_TIMEOUT_EPILOGUE);
        ok = __all_sync(~0u, ok);
      }
      tc_fence_after();
      return ok;
    };
    for (int piece = 0;; ++piece) {
      const int qb = piece & 1;
      if (!wait(&sm.q_full[qb], piece >> 1 & 1)) break;
      const Piece& d = sm.piece[qb];
      const int end = d.end, packed = d.first + h * 128 + row;
      if (end == 0) break;
      if (d.rows - d.first <= h * 128) {  // no rows for this half
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_empty[qb]);
        continue;
      }
      const int tok = min(packed, d.rows - 1) / group, head = d.head * group + packed % group;
      const int pos = d.pos0 + tok;
      const float slope = MOD && a.slopes && packed < d.rows ? a.slopes[head] : 0.0f;
      const int pre = d.pre, from = d.from, prefix = d.prefix;
      // this row sees keys [0, prefix) and [row_lo, row_hi]; all rows see [all_lo, all_hi]
      const int row_lo = pos >= a.window ? pos - a.window + 1 : 0, row_hi = min(pos, d.keys - 1);
      const int pos_lo = d.pos0 + (d.first + h * 128) / group;
      const int pos_hi = d.pos0 + min(d.first + h * 128 + 127, d.rows - 1) / group;
      const int all_lo = pos_hi >= a.window ? pos_hi - a.window + 1 : 0, all_hi = min(pos_lo, d.keys - 1);
      const int begin = d.begin;
      float m = -INFINITY, l = 0.0f;
      for (int i = begin; i < end; ++i, ++step) {
        const int block0 = (i < pre ? i : from + i - pre) * kBlock, buf = step & 1;
        if (!wait(&sm.s_full[h][buf], (step >> 1) & 1)) break;
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
        if (!(block0 + kBlock <= prefix || (block0 >= all_lo && block0 + kBlock - 1 <= all_hi))) {
          const int hi = row_hi - block0, lo = row_lo - block0, pr = prefix - block0;
#pragma unroll
          for (int e = 0; e < kBlock; ++e)
            if (!(e < pr || (e <= hi && e >= lo))) s[e / 32][e % 32] = 0xff800000u;
        }
        uint32_t pk[32];
        float2 sum[2];
        float over;  // the largest t - m
        auto exponentials = [&]() {
          const float base = m == -INFINITY ? 0.0f : -m;
          const float2 c2 = make_float2(c, c), b2 = make_float2(base, base);
          float top[2] = {-INFINITY, -INFINITY};
          sum[0] = sum[1] = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {  // (16 at a time, to have them in flight)
            float2 x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int at = 2 * (e + k);
              x[k] = __ffma2_rn(make_float2(__uint_as_float(s[at / 32][at % 32]),
                                            __uint_as_float(s[at / 32][at % 32 + 1])), c2, b2);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) top[k & 1] = fmaxf(top[k & 1], fmaxf(x[k].x, x[k].y));
#pragma unroll
            for (int k = 0; k < 8; ++k)
              x[k] = k % 8 < kFmaPairs ? ex2_fma<T>(x[k]) : make_float2(ex2(x[k].x), ex2(x[k].y));
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              sum[k & 1] = __fadd2_rn(sum[k & 1], x[k]);
              pk[e + k] = pack2<T>(x[k].x, x[k].y);
            }
          }
          over = fmaxf(top[0], top[1]);
        };
        auto maximum = [&]() {
          float top[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            top[q] = __uint_as_float(s[q / 2][(q % 2) * 16]);
#pragma unroll
            for (int e = 1; e < 16; ++e)
              top[q] = fmaxf(top[q], __uint_as_float(s[q / 2][(q % 2) * 16 + e]));
          }
          return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
        };
        if (i == begin) m = maximum();
        exponentials();
        // (a row without any key so far has no m yet)
        if (__any_sync(~0u, over > (m == -INFINITY ? -INFINITY : kGrow))) {
          // O holds the steps before this one, once they are done.  (S of this
          // step says so of all but the last, so that the parity is not two
          // phases off.)
          if (!wait(&sm.pv_done[h], (step - 1) & 1)) break;
          const float m2 = fmaxf(m, maximum()), f = m == -INFINITY ? 0.0f : ex2(m - m2);
          m = m2;
          l *= f;
          uint32_t o[32];
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            tmem_ld32(t_o + q * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(t_o + q * 32, o);
          }
          exponentials();
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st32(t_s + buf * 64, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[h][buf]);
      }
      if (!ok) break;

      if (!wait(&sm.o_full[h], outs++ & 1)) break;
      const bool in = packed < d.rows;
      const int64_t t = d.row0 + tok;
      if (d.whole) {
        // by way of the rows' buffer, which is done with: a thread has a row,
        // a row's stores shall be whole lines
        const float inv = m > -INFINITY ? 1.0f / l : 0.0f;
        uint8_t* const stage = q_smem + (qb * 2 + h) * C::Q_BYTES;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          tmem_ld32(t_o + q * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = pack2<T>(__uint_as_float(o[e * 8 + 2 * k]) * inv,
                              __uint_as_float(o[e * 8 + 2 * k + 1]) * inv);
            const int chunk = q * 4 + e;
            *reinterpret_cast<uint4*>(stage + (chunk / 8) * C::Q_HALF + row * 128 +
                                      (((chunk % 8) ^ (row & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (in && a.lse) a.lse[t * a.b.q_heads + head] = (m + log2f(l)) * kLn2;
        __syncwarp();
        constexpr int CH = D / 8;
        const long long at = in ? t * a.o_token + head * a.o_head : -1;
#pragma unroll 4
        for (int i = 0; i < CH; ++i) {
          const int r = i * (32 / CH) + lane / CH, chunk = lane % CH, from_row = (warp % 4) * 32 + r;
          const long long to = __shfl_sync(~0u, at, r);
          const uint4 w = *reinterpret_cast<const uint4*>(
              stage + (chunk / 8) * C::Q_HALF + from_row * 128 + (((chunk % 8) ^ (from_row & 7)) << 4));
          if (to >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to + chunk * 8) = w;
        }
      } else {
        const PagedPartials<kRows, D> parts(a.workspace, gridDim.x);
        float* o_part = parts.o + int64_t(d.slot) * kRows * D + (h * 128 + row) * 4;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          tmem_ld32(t_o + q * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (in)
              *reinterpret_cast<uint4*>(o_part + (q * 8 + e / 4) * (kRows * 4)) =
                  make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
        if (in) parts.ml[int64_t(d.slot) * kRows + h * 128 + row] = make_float2(m, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_empty[qb]);
    }
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
  cfg.gridDim = dim3(static_cast<unsigned>(sms), D / 16);
  cfg.blockDim = dim3(kRows);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_join_columns_kernel<T, kRows, D>, a, sms);
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
