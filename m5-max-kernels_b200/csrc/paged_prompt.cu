// Attention of many rows over a paged cache (m5b_paged_attention for prompts
// and chunks of them): tcgen05 matrix products with the softmax between them.
//
// One CTA per SM works on a tile of 256 packed rows of a kv head, as two
// halves of 128 rows (an MMA's height).  Per step of 64 keys and half:
//   S = Q K^T          A, B from shared memory, 128 x 64 fp32 in TMEM
//   t = S scale log2 e, p = 2^(t - m), l += sum p   one thread a row
//   O += P V           P (the cache's type) from TMEM, V from shared memory
// Roles: two warpgroups, one per half, each thread owning a row of S and O; one
// thread issuing QK of both halves in turn and one issuing PV (a wait on an
// mbarrier costs an issuing thread some 55 cycles even when there is nothing
// to wait for, and the tensor cores' queue holds but four to six MMAs: a step
// took 2090 cycles when one thread issued all; a thread for each product of
// each half lets the halves fall into step, so that all wait at once: 1850);
// one warp filling a ring with K and V blocks by TMA, one box per page; one
// warp finding the CTA's pieces of tiles and loading their rows, one piece
// ahead.
//
// TMEM's 512 columns hold O (2 x 128), S (2 x 64) and P (2 x 2 x 32): QK of
// the next step starts when the softmax has read S, and PV of this one when P
// is there.  (Measured and not kept, with a thread per half issuing both of its
// products: two S buffers with P over them, whose reuse chains softmax, PV and
// QK, 1830 cycles; one S buffer of 128 keys, which needs fewer bytes of shared
// memory a flop but chains them all the more, 4250 for 128 keys.)  m is near the
// row's maximum (kGrow); where it changes, O is rescaled in place.  (Taking the
// exponentials with the old m first, and again in the rare case: 2200 cycles.)
// P is rounded to the cache's type for the product, once, at the size of the
// output's own rounding; sums, m and O are fp32.
//
// What bounds it: an MMA of 128 x 64 x 16 reads 6 KB of shared memory where its
// 32 cycles have room for 4, so the products take 8 * 48 + 4 * 64 cycles a half
// and step at D = 128, 1290 for both halves with the softmax beside them (a
// test of the two alone), 1460 here without the exponentials (TMA writes, the
// issuing threads' waits) and 1770 with them: two prompts of 8192 tokens, 32 +
// 8 heads, 1.17 ms, 940 TFLOP/s.
#include "paged_sched.cuh"

namespace m5b {
namespace {

constexpr int kBlock = kPagedBlock;  // keys per step
constexpr int kRows = 256;           // packed rows per tile, two halves
// Of 8 pairs of exponentials, those by ex2_fma: a prompt of 4096 tokens, 32 + 8
// heads, takes 179 us (188 with none), two of 8192, which the power limit slows,
// 1170 (1175 with none, 1172 with 2, 1226 with 4).  None where the scores are
// modified, whose arithmetic keeps the FMA pipes busy (162 us, 187 with 3, in the
// distance bias of 56 heads).
constexpr int kFmaPairs = 3;
constexpr int kThreads = 384;  // warps 0-3, 4-7: halves; 8: QK; 9: PV; 10: K, V; 11: rows
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
    uint64_t s_full[2], s_free[2];           // [half]
    uint64_t p_full[2][2];                   // [half][buffer]
    uint64_t pv_done[2][2];                  // [half][buffer]
    uint64_t o_full[2], drain[2];            // after a piece's last PV; [MMA thread]
    uint64_t landed;                         // a V block to be blanked
    PagedWalkScratch<kThreads> scratch;
    Piece piece[2];
    uint32_t tmem;
    volatile int abort_flag;
  };
  static_assert(STAGES % 2 == 0 && sizeof(Small) <= 1024, "shared memory layout");
};
// TMEM columns: S [half] of 64, P [half][buffer] of 32, O [half] of 128
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256;

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
template <int N> __device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
// 2^x of a pair on the FMA pipes, for x < 100: x = n + f with n the nearest
// integer (adding 1.5 * 2^23 leaves it in the low bits), 2^f by a polynomial
// 1 + f (c1 + ...), n added to its exponent.  The coefficients are the minimax
// fit of the relative error on [-1/2, 1/2] (Remez exchange), 2.9e-6 in fp32.
// The sum of these is an output, lse, so bf16 takes as many terms as fp16:
// with one less (1e-4, below its rounding of P all the same) two prompts of
// 8192 tokens took 1150 us instead of 1168; with one more (1.6e-7) 1183.
// From -127 down the result is zero, as hidden keys' has to be: the polynomial
// is 1 there, whose exponent bits n = -127 takes to none (down to -126 it leaves
// a number below 2^-126).
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  x.x = fmaxf(x.x, -127.0f);
  x.y = fmaxf(x.y, -127.0f);
  const float2 big = make_float2(12582912.0f, 12582912.0f), one = make_float2(1.0f, 1.0f);
  const float2 r = __fadd2_rn(x, big);
  const float2 f = __ffma2_rn(__fadd2_rn(r, make_float2(-12582912.0f, -12582912.0f)),
                              make_float2(-1.0f, -1.0f), x);
  float2 p = make_float2(0x1.3a02ccp-7f, 0x1.3a02ccp-7f);
  p = __ffma2_rn(p, f, make_float2(0x1.c9fc46p-5f, 0x1.c9fc46p-5f));
  p = __ffma2_rn(p, f, make_float2(0x1.ec0378p-3f, 0x1.ec0378p-3f));
  p = __ffma2_rn(p, f, make_float2(0x1.62e12cp-1f, 0x1.62e12cp-1f));
  p = __ffma2_rn(p, f, one);
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(r.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(r.y) << 23)));
}

// What is done to the scores: nothing, a bias, a cap (and, by a flag, a bias).
// Each has a kernel, for the sake of the instruction cache: one for both of the
// latter took 4 to 7 % longer.  So have caps above kFarCap.
enum Scores : int { kPlain = 0, kBiased = 1, kCapped = 2, kCappedFar = 3 };
constexpr float kFarCap = 64.0f;

// A row's 64 scores capped, biased and in log2 units; `ahead` is the row's
// position minus that of the first key.  Special functions would take as long
// as the exponentials do three times over, so scores within the cap, the usual
// case, go by tanh_ratio; a row with any beyond it takes
// tanh(y) = 1 - 2 / (e^2y + 1) for all of its 64, which leaves small scores off by
// up to 4e-7 of the cap.  (Each row for itself, though a warp of both kinds then
// takes both ways, 121 us instead of 107 for two prompts of 2048 tokens: some of
// its rows may be another sequence's, which shall not move a bit.)  With caps above
// kFarCap only the scores beyond take it, one by one (two prompts of 2048 tokens
// with scores beyond a cap of 100: 142 us instead of 107; none beyond: 89 both ways).
template <int SCORES>
__device__ __forceinline__ void modify(uint32_t (&s)[2][32], float scale, float softcap,
                                       bool biased, float slope, int ahead) {
  const float k = scale * kLog2e;
  if (SCORES >= kCapped) {
    // ((x r^2) x, not x^2 r^2: x^2 may be beyond the range; r^2 is not)
    const float r = fminf(scale / softcap, 0x1p63f);
    float top[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 64; e += 2)
      top[e / 2 & 1] = fmaxf(top[e / 2 & 1], fmaxf(fabsf(__uint_as_float(s[e / 32][e % 32])),
                                                   fabsf(__uint_as_float(s[e / 32][e % 32 + 1]))));
    if (fmaxf(top[0], top[1]) * r <= 1.0f) {
      const float2 r2 = make_float2(r * r, r * r), k2 = make_float2(k, k);
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const float2 x = make_float2(__uint_as_float(s[e / 32][e % 32]),
                                     __uint_as_float(s[e / 32][e % 32 + 1]));
        const float2 y = __fmul2_rn(__fmul2_rn(x, k2), tanh_ratio(__fmul2_rn(__fmul2_rn(x, r2), x)));
        s[e / 32][e % 32] = __float_as_uint(y.x);
        s[e / 32][e % 32 + 1] = __float_as_uint(y.y);
      }
    } else {
      const float cap = softcap * kLog2e, two = 2.0f * r * kLog2e;
#pragma unroll
      for (int e = 0; e < 64; ++e) {
        const float x = __uint_as_float(s[e / 32][e % 32]);
        float y = cap * (1.0f - __fdividef(2.0f, ex2(x * two) + 1.0f));
        if (SCORES == kCappedFar) {
          const float z = x * (r * r) * x;
          if (z <= 1.0f) y = x * k * tanh_ratio(make_float2(z, z)).x;
        }
        s[e / 32][e % 32] = __float_as_uint(y);
      }
    }
  } else {
    const float2 k2 = make_float2(k, k);
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
      const float2 y = __fmul2_rn(make_float2(__uint_as_float(s[e / 32][e % 32]),
                                              __uint_as_float(s[e / 32][e % 32 + 1])), k2);
      s[e / 32][e % 32] = __float_as_uint(y.x);
      s[e / 32][e % 32 + 1] = __float_as_uint(y.y);
    }
  }
  if (SCORES >= kCapped && !biased) return;
  const float down = -slope * kLog2e, first = static_cast<float>(ahead);
  if (__all_sync(~0u, ahead >= 63)) {  // no key is ahead of its row: the distance is linear
    const float2 d2 = make_float2(down, down), f2 = make_float2(first, first);
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
      const float2 y = __ffma2_rn(
          __fadd2_rn(f2, make_float2(-static_cast<float>(e), -static_cast<float>(e + 1))), d2,
          make_float2(__uint_as_float(s[e / 32][e % 32]), __uint_as_float(s[e / 32][e % 32 + 1])));
      s[e / 32][e % 32] = __float_as_uint(y.x);
      s[e / 32][e % 32 + 1] = __float_as_uint(y.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 64; ++e)
      s[e / 32][e % 32] = __float_as_uint(
          fmaf(down, fabsf(first - static_cast<float>(e)), __uint_as_float(s[e / 32][e % 32])));
  }
}

template <bool B> struct Flag {
  static constexpr bool value = B;
};

template <typename T, int D, int SCORES>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prompt_kernel(const PagedAttnArgs a, const __grid_constant__ PagedMaps maps) {
  using C = Cfg<D>;
  constexpr int STAGES = C::STAGES;
  constexpr bool MOD = SCORES != kPlain;
  constexpr int kBlankK = SCORES == kCapped;  // whether K blocks are blanked behind the end
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
      mbar_init(&sm.q_full[h], 1);
      mbar_init(&sm.q_empty[h], 10);  // the softmax warps and the MMA threads
      mbar_init(&sm.s_full[h], 1);
      mbar_init(&sm.s_free[h], 4);
      mbar_init(&sm.p_full[h][0], 4);
      mbar_init(&sm.p_full[h][1], 4);
      mbar_init(&sm.pv_done[h][0], 1);
      mbar_init(&sm.pv_done[h][1], 1);
      mbar_init(&sm.o_full[h], 1);
      mbar_init(&sm.drain[h], 1);
    }
    mbar_init(&sm.landed, 1 + kBlankK);
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

  // Registers: 256 threads of 208 and 128 of 88 make the 384 x 168 of the launch.
  if (warp >= kMmaWarp) {
    regs_dec<88>();
    if (warp == kTmaWarp) {  // ---- K and V blocks
      const int boxes = kBlock / maps.box_rows * C::HALVES;
      const int row = lane / C::HALVES * maps.box_rows, half = lane % C::HALVES;
      int stage = 0, phase = 0, issued = 0;
      // Slots behind the sequence's end may hold NaN, which a zero probability
      // would not stop: V blocks that reach there land here first and are
      // blanked, while the K block after them is on its way.  With caps that a
      // row takes in one form or the other their K blocks too, lest what an
      // unused slot holds choose.
      int blank = -1, blank_from = 0, ph_landed = 0;  // the V block's stage, its first unused key
      bool ok = true;
      auto load = [&](const CUtensorMap* map, int head, int page, int slot, bool last) {
        if (ok)
          ok = mbar_wait_relaxed(&sm.empty[stage], phase ^ 1, &sm.abort_flag, a.status,
                                 DEV_TIMEOUT_PRODUCER, 100);
        ok = __all_sync(~0u, ok);
        if (!ok) return;
        uint64_t* bar = last ? &sm.landed : &sm.full[stage];
        if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE_BYTES);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(ring + stage * C::TILE_BYTES + half * C::HALF_BYTES + row * 128, map, bar,
                      half * 64, slot, head, page);
        ++issued;
        if (++stage == STAGES) stage = 0, phase ^= 1;
      };
      auto finish = [&]() {
        if (blank < 0) return;
        if (ok)
          ok = mbar_wait_relaxed(&sm.landed, ph_landed, &sm.abort_flag, a.status,
                                 DEV_TIMEOUT_PRODUCER, 100);
        ok = __all_sync(~0u, ok);
        if (!ok) return;
        ph_landed ^= 1;
        uint8_t* at = ring + (blank - kBlankK) * C::TILE_BYTES;
        for (int b = 0; b <= kBlankK; ++b, at += C::TILE_BYTES)
          for (int i = blank_from * C::HALVES * 8 + lane; i < kBlock * C::HALVES * 8; i += 32)
            *reinterpret_cast<uint4*>(at + (i / 8 % C::HALVES) * C::HALF_BYTES + i / (C::HALVES * 8) * 128 +
                                      i % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_shared();
        __syncwarp();
        if (lane <= kBlankK) mbar_arrive(&sm.full[blank - lane]);
        blank = -1;
      };
      PagedPiece p;
      while (ok && walk.next(a, p)) {
        const int window = paged_window<kRows>(a, p.s, p.rt);
        for (int i = p.begin; ok && i < p.end; ++i) {
          const int block0 = p.r.at(i) * kBlock, key = block0 + row;
          int page = a.b.num_pages, slot = 0;  // out of range: zeros
          if (lane < boxes && key < p.s.keys &&
              (key < p.s.prefix || key > window - maps.box_rows)) {
            const int at = paged_page(a.b, p.seq, key);
            if (at >= 0) page = at;
            slot = key % a.b.page_size;
          }
          // (K blocks are in the even stages, V blocks in the odd ones after them)
          const bool last = p.s.keys - block0 < kBlock;
          if (kBlankK) finish();
          load(&maps.k, p.head, page, slot, kBlankK && last);
          if (!kBlankK) finish();
          if (last) blank = stage, blank_from = max(p.s.keys - block0, 0);
          load(&maps.v, p.head, page, slot, last);
        }
      }
      finish();
      if (!ok) {  // let the copies in flight land before the CTA ends
        for (int i = 0; i < STAGES && i < issued; ++i) {
          if (--stage < 0) stage = STAGES - 1, phase ^= 1;
          const bool late = blank >= 0 && stage <= blank && stage >= blank - kBlankK;
          const unsigned long long start = globaltimer_ns();
          while (!(late ? mbar_try_wait(&sm.landed, ph_landed)
                        : mbar_try_wait(&sm.full[stage], phase)) &&
                 globaltimer_ns() - start < kWaitLimitNs) {
          }
        }
      }
    } else if (warp == kRowWarp) {  // ---- pieces and their rows
      constexpr int CH = D / 8;  // 16-byte chunks of a row
      const int chunk = lane % CH;
      bool ok = true, any = false;
      int n = 0;
      PagedPiece p;
      for (;; ++n) {
        const int buf = n & 1;
        const bool more = walk.next(a, p);
        any |= more;
        ok = mbar_wait_relaxed(&sm.q_empty[buf], (n >> 1 & 1) ^ 1, &sm.abort_flag, a.status,
                               DEV_TIMEOUT_PRODUCER, 100);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        const int rows = p.s.n * group, first = p.rt * kRows;
        const bool by_tma = more && maps.has_q;
        if (more && !by_tma) {
          // a row after every 32 / CH; the pointer follows head and token
          constexpr int STEP = 32 / CH;
          const int here = min(rows - first, kRows), all = here > 128 ? kRows : 128;
          const int r0 = lane / CH;
          int g = (first + r0) % group;
          const T* src = static_cast<const T*>(a.q) +
                         int64_t(p.s.row0 + (first + r0) / group) * a.q_token +
                         (p.head * group + g) * a.q_head + chunk * 8;
          const int64_t next = (STEP / group) * a.q_token + (STEP % group) * a.q_head;
          const int64_t wrap = a.q_token - group * a.q_head;
          uint32_t dst = smem_u32(q_smem + buf * 2 * C::Q_BYTES + (chunk / 8) * C::Q_HALF);
#pragma unroll 4
          for (int r = r0; r < all; r += STEP) {
            cp_async16(dst + (r / 128) * C::Q_BYTES + (r % 128) * 128 + (((chunk % 8) ^ (r & 7)) << 4),
                       r < here ? src : static_cast<const T*>(a.q), r < here);
            src += next;
            g += STEP % group;
            if (g >= group) g -= group, src += wrap;
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
        if (by_tma) {
          // (rows behind the sequence's are another's: computed, not stored)
          __syncwarp();
          if (lane == 0) {
            const int halves = rows - first > 128 ? 2 : 1;
            mbar_arrive_expect_tx(&sm.q_full[buf], halves * C::Q_BYTES);
            for (int i = 0; i < halves * C::HALVES; ++i)
              tma_load_3d(q_smem + (buf * 2 + i / C::HALVES) * C::Q_BYTES + i % C::HALVES * C::Q_HALF,
                          &maps.q, &sm.q_full[buf], i % C::HALVES * 64, p.head * group,
                          p.s.row0 + (first + i / C::HALVES * 128) / group);
          }
        } else {
          cp_async_wait_all();
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.q_full[buf]);
        }
        if (!more) break;
      }
      // let the rows in flight land before the CTA ends
      for (int i = n - 1; !ok && maps.has_q && i >= 0 && i >= n - 2; --i) {
        const unsigned long long start = globaltimer_ns();
        while (!mbar_try_wait(&sm.q_full[i & 1], i >> 1 & 1) &&
               globaltimer_ns() - start < kWaitLimitNs) {
        }
      }
      if (lane == 0)  // (p is the last piece)
        paged_write_split(&PagedPartials<kRows, D>(a.workspace, gridDim.x).split[blockIdx.x],
                          any ? &p : nullptr, walk.share, kRows, group);
    } else {  // ---- QK or PV of both halves, by one thread
      const bool is_pv = warp != kMmaWarp;
      if (elect_one()) {
        constexpr int kind = DTypeOf<T>::value == DT_BF16 ? KIND_BF16 : KIND_F16;
        constexpr uint32_t idesc_s = make_idesc(kind, 128, kBlock);
        constexpr uint32_t idesc_o = make_idesc(kind, 128, D) | (1u << 16);  // B is MN-major
        const uint64_t q_desc = smem_desc_k128(smem_u32(q_smem));
        const uint64_t k_desc = smem_desc_k128(smem_u32(ring));
        const uint64_t v_desc = smem_desc_mn128(smem_u32(ring), C::HALF_BYTES);
        bool ok = true;
        auto wait = [&](uint64_t* bar, int parity) {
          if (ok) ok = mbar_wait_bounded(bar, parity, &sm.abort_flag, a.status, DEV_TIMEOUT_MMA);
          tc_fence_after();
        };
        // K blocks are in the ring's even stages, V blocks in the odd ones
        int stage = is_pv ? 1 : 0, phase = 0;
        int done[2] = {0, 0};  // steps of the halves
        for (int piece = 0; ok; ++piece) {
          wait(&sm.q_full[piece & 1], piece >> 1 & 1);
          if (!ok) break;
          const Piece& d = sm.piece[piece & 1];
          const int steps = d.end - d.begin, halves = d.rows - d.first > 128 ? 2 : 1;
          mbar_arrive(&sm.q_empty[piece & 1]);
          if (steps == 0) break;
          const uint64_t qd = q_desc + ((piece & 1) * 2 * C::Q_BYTES >> 4);
          for (int i = 0; ok && i < steps; ++i) {
            wait(&sm.full[stage], phase);
            const int at = stage * C::TILE_BYTES >> 4;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h >= halves) break;
              if (!is_pv) {  // S = Q K^T
                if (done[h] > 0) wait(&sm.s_free[h], (done[h] - 1) & 1);
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                  tc_mma<KIND_F16>(tmem + kColS + h * 64,
                                   qd + ((h * C::Q_BYTES + (k / 4) * C::Q_HALF + (k % 4) * 32) >> 4),
                                   k_desc + at + (((k / 4) * C::HALF_BYTES + (k % 4) * 32) >> 4),
                                   idesc_s, k > 0);
                tc_commit(&sm.s_full[h]);
              } else {  // O (+)= P V
                const int buf = done[h] & 1;
                wait(&sm.p_full[h][buf], (done[h] >> 1) & 1);
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < kBlock / 16; ++k)
                  tc_mma_ts(tmem + kColO + h * 128, tmem + kColP + h * 64 + buf * 32 + k * 8,
                            v_desc + at + (k * 2048 >> 4), idesc_o, i > 0 || k > 0);
                tc_commit(&sm.pv_done[h][buf]);
                if (i + 1 == steps) tc_commit(&sm.o_full[h]);
              }
              ++done[h];
            }
            if (ok) tc_commit(&sm.empty[stage]);
            stage += 2;
            if (stage >= STAGES) stage -= STAGES, phase ^= 1;
          }
        }
        // every MMA has retired before TMEM is freed
        uint64_t* drain = &sm.drain[warp - kMmaWarp];
        tc_commit(drain);
        const unsigned long long start = globaltimer_ns();
        while (!mbar_try_wait(drain, 0)) {
          if (globaltimer_ns() - start > kWaitLimitNs) {
            atomicOr(a.status, DEV_TIMEOUT_DRAIN);
            break;
          }
        }
      }
      __syncwarp();
    }
  } else {  // ---- softmax: thread `row` of half h
    regs_inc<208>();
    const int h = warp / 4;
    const int row = threadIdx.x % 128;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    const uint32_t t_s = lanes + kColS + h * 64, t_p = lanes + kColP + h * 64;
    const uint32_t t_o = lanes + kColO + h * 128;
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
      auto softmax = [&](auto masked, int i, int block0, bool open) {
        const int buf = step & 1;
        uint32_t s[2][32];
        tmem_ld32(t_s, s[0]);
        tmem_ld32(t_s + 32, s[1]);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_free[h]);
        if (MOD) modify<SCORES>(s, a.scale, a.softcap, a.slopes != nullptr, slope, pos - block0);
        if (decltype(masked)::value && !(MOD && open)) {
          const int hi = row_hi - block0, lo = row_lo - block0, pr = prefix - block0;
#pragma unroll
          for (int e = 0; e < kBlock; ++e)
            if (!(e < pr || (e <= hi && e >= lo))) s[e / 32][e % 32] = 0xff800000u;
        }
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t* x = &s[q / 2][(q % 2) * 16];
          top[q] = __uint_as_float(x[0]);
#pragma unroll
          for (int e = 1; e < 15; e += 2)
            top[q] = max_nan(top[q], max_nan(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
          top[q] = max_nan(top[q], __uint_as_float(x[15]));
        }
        // A row with a NaN or +inf among its scores gets m = NaN, which stays
        // and makes l and O NaN: ex2_fma would lose a single NaN score.
        const float high = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])) * c;
        const bool grow = !(high <= m + (kGrow + kBelow<T>)) && m == m;  // (m = -inf: any key)
        const bool any = __any_sync(~0u, grow);
        const float m2 = !grow ? m : high < INFINITY ? high - kBelow<T> : NAN;
        const float f = m == -INFINITY ? 0.0f : ex2(m - m2);
        m = m2;
        uint32_t pk[32];
        const float base = m == -INFINITY ? 0.0f : -m;
        const float2 c2 = make_float2(c, c), b2 = make_float2(base, base);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
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
          for (int k = 0; k < 8; ++k)
            x[k] = k % 8 < (MOD ? 0 : kFmaPairs) ? ex2_fma(x[k]) : make_float2(ex2(x[k].x), ex2(x[k].y));
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            sum[k & 1] = __fadd2_rn(sum[k & 1], x[k]);
            pk[e + k] = pack2<T>(x[k].x, x[k].y);
          }
        }
        l = l * f + (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        // (PV of two steps before has long been done with this buffer)
        if (step > 1 && !wait(&sm.pv_done[h][buf], ((step >> 1) - 1) & 1)) return;
        tmem_st32(t_p + buf * 32, pk);
        if (any && i > begin) {  // O holds the steps before this one, once they are done
          if (!wait(&sm.pv_done[h][buf ^ 1], ((step - 1) >> 1) & 1)) return;
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
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[h][buf]);
      };
      for (int i = begin; i < end; ++i, ++step) {
        const int block0 = (i < pre ? i : from + i - pre) * kBlock;
        if (!wait(&sm.s_full[h], step & 1)) break;
        // (two bodies, where they are short: scores that a branch may change
        // cost the other way too, but a body may outgrow the instruction cache)
        const bool open =
            prefix - block0 >= kBlock || (block0 >= all_lo && all_hi - block0 >= kBlock - 1);
        if (!MOD && open)
          softmax(Flag<false>(), i, block0, true);
        else
          softmax(Flag<true>(), i, block0, open);
        if (!ok) break;
      }
      if (!ok) break;

      if (!wait(&sm.o_full[h], outs++ & 1)) break;
      const bool in = packed < d.rows;
      const int64_t t = d.row0 + tok;
      if (d.whole) {
        // by way of the rows' buffer, which is done with: a thread has a row,
        // a row's stores shall be whole lines
        const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
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
      fence_proxy_async_shared();  // before the buffer's next rows come by TMA
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_empty[qb]);
    }
    paged_zero_outside<T, D>(a, int64_t(blockIdx.x) * 256 + threadIdx.x, int64_t(gridDim.x) * 256);
  }
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <typename T, int D, int SCORES>
cudaError_t launch(const PagedAttnArgs& a, const PagedMaps& m, int sms, cudaStream_t stream) {
  using C = Cfg<D>;
  auto kern = paged_prompt_kernel<T, D, SCORES>;
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
  if (a.softcap > kFarCap) return launch<T, D, kCappedFar>(a, m, sms, stream);
  if (a.softcap > 0.0f) return launch<T, D, kCapped>(a, m, sms, stream);
  return a.slopes ? launch<T, D, kBiased>(a, m, sms, stream) : launch<T, D, kPlain>(a, m, sms, stream);
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
