// Matrix products grouped by expert with ragged sizes, and E4M3 products with a
// scale for each block of 128 channels, on tcgen05 tensor cores.
//
//   out[t, n] = epilogue( sum_k a[t, k] * b[e, n, k] ),  e the group of row t
//
// The weights are the M operand of the MMAs and the rows of a group the N
// operand: a tile is 128 channels (256 for a CTA pair) by any multiple of 16
// (32) rows of one group, so that a group of few rows costs few columns, and a
// group of many is cut into equal tiles.  Rows of the next group or behind the
// last one that a tile's loads bring along are columns of their own, which are
// not stored.
//
// Block scales: a block of 128 channels of K (one 128-byte slice, four MMAs) is
// summed in TMEM by itself, and the epilogue warps add it, times the row's and
// the channel block's scale, to fp32 sums in registers:
//   sum[t, n] += (sa[t, g] * sb[n / 128, g]) * partial[t, n]
// while the MMAs of the next block fill another TMEM buffer.  Without block
// scales a tile's whole K range stays in TMEM.
//
// Roles: warps 0-7 epilogue, warp 8 TMA producer, warp 9 MMA issuer, 10 and 11
// none (registers move between whole warpgroups).  TMEM is
// read in 16 x 256-bit fragments: a thread holds pairs of neighbouring rows
// (columns of the accumulator) of four channels, so that one scale pair serves
// four packed multiply-adds, and stmatrix turns a fragment into rows of 32
// channels for 16-byte stores.
//
// K split over a cluster (single CTAs, one tile a cluster): each CTA sums its
// part of K; the sums of eight rows go to the CTA that owns them through
// distributed shared memory, which adds the parts in the order of the ranks.
#include "grouped.cuh"

namespace m5b {

namespace {

template <bool PAIR>
struct Cfg {
  static constexpr int TN = PAIR ? kPairTileRows : kSingleTileRows;
  static constexpr int TM = PAIR ? 256 : 128;              // channels of a tile
  static constexpr int W_BYTES = 128 * 128;                // this CTA's weights of a stage
  static constexpr int X_BYTES = (PAIR ? TN / 2 : TN) * 128;  // this CTA's rows of a stage
  static constexpr int STAGES = PAIR ? 6 : 7;
  static constexpr int BUFS = 512 / TN;                    // TMEM accumulators
  static constexpr int CHUNKS = TN / 64;                   // 32-row chunks of an epilogue warp
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 32 * (EPI_WARPS + 4);     // three warpgroups
  static constexpr int SCALE_SLOTS = 2;                    // of four blocks each
  static constexpr int SCALE_BYTES = SCALE_SLOTS * 4 * TN * 4;
  static constexpr int STORE_BYTES = EPI_WARPS * 2 * 512;
  static constexpr int EXCHANGE_BYTES = PAIR ? 0 : TN * 128 * 4;
  static constexpr int TABLE_BYTES = 2 * (kMaxGroups + 4) * 4;
  static constexpr int BAR_BYTES = (2 * STAGES + 2 * BUFS + SCALE_SLOTS + 2) * 8 + 16;
  static constexpr int SMEM_BYTES = 1024 + STAGES * (W_BYTES + X_BYTES) + EXCHANGE_BYTES +
                                    SCALE_BYTES + STORE_BYTES + TABLE_BYTES + BAR_BYTES;
  static_assert(SMEM_BYTES <= 232448, "shared memory per CTA exceeds 227 KB");
};

// Four 8-column groups of 16 TMEM lanes: thread t receives, for group i,
// r[4i], r[4i + 1]: lane t / 4, columns 8i + 2 (t % 4), + 1; r[4i + 2],
// r[4i + 3]: the same columns of lane t / 4 + 8.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Waits for this thread's TMEM loads; the 32 registers are named so that no use
// of them moves above the wait.
__device__ __forceinline__ void tmem_wait_frag(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b,
                                                  uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                   addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
// As tma_load_2d_pair, of a 3D box.
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map,
                                                 uint64_t* bar, int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar) & 0xFEFFFFFFu), "r"(x), "r"(y),
      "r"(z)
      : "memory");
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                              uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
// As mbar_wait_bounded, for data that other CTAs of the cluster stored.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity,
                                                  volatile int* abort, unsigned int* status,
                                                  unsigned int code) {
  const unsigned long long start = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((++spins & 255u) == 0u) {
      if (*abort) return false;
      if (globaltimer_ns() - start > kWaitLimitNs) {
        if (status) atomicOr(status, code);
        *abort = 1;
        return false;
      }
    }
  }
}

struct Tile {
  int group;
  int row0, rows;  // of the activations
  int cols;        // rows as columns of the MMAs: a multiple of 16 (CTA pairs: 32)
  int ch0;         // first channel
};

// Walks the tiles unit, unit + stride, ...; every role of a CTA (and both CTAs of
// a pair) sees the same ones.  first_row[e]: the first row of group e, clamped
// to the rows there are; first_tile[e]: the tiles of the groups before e.
template <bool PAIR>
struct Walk {
  const int* first_row;
  const int* first_tile;
  int groups, tile_rows, ch_tiles;
  int unit, stride, e;

  __device__ __forceinline__ bool next(Tile& t) {
    using C = Cfg<PAIR>;
    if (unit >= first_tile[groups]) return false;
    while (unit >= first_tile[e + 1]) ++e;
    const int rows = first_row[e + 1] - first_row[e];  // positive: the group has tiles
    const int row_tiles = (rows + tile_rows - 1) / tile_rows;
    // Bands of at most 16 row tiles, within which the channel tiles follow one
    // another: CTAs that run side by side share weights, and a band's rows stay in L2.
    const int u = unit - first_tile[e];
    const int band = u / (16 * ch_tiles);
    const int in_band = u - band * 16 * ch_tiles;
    const int left = row_tiles - 16 * band;
    const int wide = left < 16 ? left : 16;
    const int ch = in_band / wide;
    const int r = 16 * band + in_band - ch * wide;
    constexpr int STEP = PAIR ? 32 : 16;
    const int each = ((rows + row_tiles - 1) / row_tiles + STEP - 1) / STEP * STEP;
    t.group = e;
    t.row0 = first_row[e] + r * each;
    // (positive too: tile_rows is a multiple of STEP, so each <= tile_rows and
    // (row_tiles - 1) * each <= (row_tiles - 1) * tile_rows < rows)
    t.rows = rows - r * each < each ? rows - r * each : each;
    t.cols = (t.rows + STEP - 1) / STEP * STEP;
    t.ch0 = ch * C::TM;
    unit += stride;
    return true;
  }
};

template <int KIND>
__device__ __forceinline__ float2 frag_value(uint32_t a, uint32_t b) {
  if constexpr (KIND == KIND_I8)
    return make_float2(__int2float_rn(static_cast<int>(a)), __int2float_rn(static_cast<int>(b)));
  else
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
template <int KIND>
__device__ __forceinline__ uint32_t frag_add(uint32_t a, uint32_t b) {
  if constexpr (KIND == KIND_I8)
    return a + b;
  else
    return __float_as_uint(__fadd_rn(__uint_as_float(a), __uint_as_float(b)));
}

// Eight rows (row .. row + 7, of which the first `rows` exist) of this warp's 32
// channels from ch on.  v[0..3]: the pairs of rows 2 (lane % 4), + 1 of channels
// lane / 4, + 8, + 16, + 24.  stage: 512 bytes of the warp's.
__device__ __forceinline__ void store_rows8(const GroupedArgs& g, const float2 (&v)[4],
                                            uint8_t* stage, int64_t row, int rows, int ch,
                                            int lane) {
  if (g.out_dtype == DT_F32) {
    float* o = reinterpret_cast<float*>(g.out);
    const int r = 2 * (lane & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = ch + 8 * j + (lane >> 2);
      if (c >= g.n) continue;
      if (r < rows) o[(row + r) * g.out_row + c] = v[j].x;
      if (r + 1 < rows) o[(row + r + 1) * g.out_row + c] = v[j].y;
    }
    return;
  }
  uint32_t pk[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (g.out_dtype == DT_F16) {
      const __half2 h = __floats2half2_rn(v[j].x, v[j].y);
      pk[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      pk[j] = f2_bf16x2(v[j]);
    }
  }
  // row r's 64 bytes of channels, 16-byte pieces swizzled by r / 2: no bank conflicts
  const int r = lane & 7;
  stmatrix_x4_trans(smem_u32(stage) + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4), pk[0], pk[1],
                    pk[2], pk[3]);
  __syncwarp();
  uint16_t* o = reinterpret_cast<uint16_t*>(g.out);
  if (g.out_vec) {
    const int rr = lane >> 2, piece = lane & 3;
    const uint4 w =
        *reinterpret_cast<const uint4*>(stage + rr * 64 + ((piece ^ ((rr >> 1) & 3)) << 4));
    if (rr < rows && ch + 8 * piece < g.n)
      *reinterpret_cast<uint4*>(o + (row + rr) * g.out_row + ch + 8 * piece) = w;
  } else if (ch + lane < g.n) {
    for (int rr = 0; rr < rows && rr < 8; ++rr)
      o[(row + rr) * g.out_row + ch + lane] = *reinterpret_cast<const uint16_t*>(
          stage + rr * 64 + (((lane >> 3) ^ ((rr >> 1) & 3)) << 4) + (lane & 7) * 2);
  }
}

template <int KIND, bool BLOCKS, bool PAIR>
__global__ void __launch_bounds__(Cfg<PAIR>::THREADS, 1)
    grouped_gemm_kernel(const __grid_constant__ GroupedMaps maps, const GroupedArgs g) {
  using C = Cfg<PAIR>;
  constexpr int K_ELEMS = (KIND == KIND_BF16 || KIND == KIND_F16) ? 64 : 128;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_w = smem;
  uint8_t* s_x = s_w + C::STAGES * C::W_BYTES;
  uint8_t* s_exchange = s_x + C::STAGES * C::X_BYTES;
  float* s_scale = reinterpret_cast<float*>(s_exchange + C::EXCHANGE_BYTES);
  uint8_t* s_store = reinterpret_cast<uint8_t*>(s_scale) + C::SCALE_BYTES;
  int* s_row = reinterpret_cast<int*>(s_store + C::STORE_BYTES);  // [groups + 1]
  int* s_tile = s_row + kMaxGroups + 4;                           // [groups + 1]
  uint64_t* full = reinterpret_cast<uint64_t*>(s_tile + kMaxGroups + 4);
  uint64_t* empty = full + C::STAGES;
  uint64_t* acc_full = empty + C::STAGES;
  uint64_t* acc_empty = acc_full + C::BUFS;
  uint64_t* scale_full = acc_empty + C::BUFS;
  uint64_t* drain = scale_full + C::SCALE_SLOTS;
  uint64_t* parts = drain + 1;  // K split: the owned rows' sums of all ranks are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(parts + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int splits = PAIR ? 1 : g.k_splits;
  const uint32_t rank = (PAIR || splits > 1) ? cluster_rank() : 0;
  const bool leader = !PAIR || rank == 0;
  const int per = PAIR ? 2 : splits;  // CTAs of a unit

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < C::BUFS; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * C::EPI_WARPS);
    }
    for (int s = 0; s < C::SCALE_SLOTS; ++s) mbar_init(&scale_full[s], C::EPI_WARPS);
    mbar_init(drain, 1);
    mbar_init(parts, 32);  // eight groups of rows / splits owners, four warps, `splits` senders
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&maps.b);
    tma_prefetch_desc(PAIR ? &maps.a128 : &maps.a64);
    tma_prefetch_desc(&maps.a16);
  }
  if (warp == 9) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  // With programmatic launch all that stands above overlaps the previous kernel's end.
  grid_dependency_wait();
  // The groups' first rows, then the tiles before each group.
  const int ch_tiles = (g.n + C::TM - 1) / C::TM;
  for (int e = threadIdx.x; e <= g.groups; e += C::THREADS) {
    int r = g.group_start ? g.group_start[e] : (e == 0 ? 0 : g.rows);
    r = r < 0 ? 0 : r;
    s_row[e] = r < g.rows ? r : g.rows;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    int before = 0;
    for (int e0 = 0; e0 < g.groups; e0 += 32) {
      const int e = e0 + lane;
      int tiles = 0;
      if (e < g.groups) {
        const int rows = s_row[e + 1] - s_row[e];
        tiles = rows > 0 ? (rows + g.tile_rows - 1) / g.tile_rows * ch_tiles : 0;
      }
      int sum = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += v;
      }
      if (e < g.groups) s_tile[e] = before + sum - tiles;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) s_tile[g.groups] = before;
  }
  __syncthreads();
  if (PAIR || splits > 1) cluster_sync();  // every CTA's barriers exist before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  Walk<PAIR> walk{s_row, s_tile, g.groups, g.tile_rows, ch_tiles,
                  static_cast<int>(blockIdx.x) / per, static_cast<int>(gridDim.x) / per, 0};
  const int kb0 = PAIR ? 0 : static_cast<int>(int64_t(g.num_k_blocks) * rank / splits);
  const int kb1 = PAIR ? g.num_k_blocks
                       : static_cast<int>(int64_t(g.num_k_blocks) * (rank + 1) / splits);

  // The fp32 sums of a pair's tile are 128 registers a thread of the epilogue:
  // it takes over registers of the other warps.  (384 threads are launched with
  // 168 each; 2 * 216 + 64 <= 3 * 168.)
  constexpr bool MOVE_REGS = BLOCKS && PAIR;
  if (warp >= C::EPI_WARPS) {
    if constexpr (MOVE_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 8) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      Tile t;
      while (!*abort_flag && walk.next(t)) {
        const int x_rows = PAIR ? t.cols / 2 : t.cols;  // this CTA's
        const int x_row = t.row0 + (PAIR ? static_cast<int>(rank) * x_rows : 0);
        const int w_row = t.ch0 + (PAIR ? static_cast<int>(rank) * 128 : 0);
        const uint32_t bytes = C::W_BYTES + x_rows * 128;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag, g.status,
                                 DEV_TIMEOUT_PRODUCER))
            break;
          const int kx = kb * K_ELEMS;
          uint8_t* w = s_w + stage * C::W_BYTES;
          uint8_t* x = s_x + stage * C::X_BYTES;
          if constexpr (PAIR) {
            // The even CTA's barrier counts both CTAs' bytes.
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * bytes);
            tma_load_3d_pair(w, &maps.b, &full[stage], kx, w_row, t.group);
          } else {
            mbar_arrive_expect_tx(&full[stage], bytes);
            tma_load_3d(w, &maps.b, &full[stage], kx, w_row, t.group);
          }
          for (int r = 0; r < x_rows;) {
            const int left = x_rows - r;
            const int take = left >= 128 ? 128 : left >= 64 ? 64 : 16;
            const CUtensorMap* m = take == 128 ? &maps.a128 : take == 64 ? &maps.a64 : &maps.a16;
            if constexpr (PAIR)
              tma_load_2d_pair(x + r * 128, m, &full[stage], kx, x_row + r);
            else
              tma_load_2d(x + r * 128, m, &full[stage], kx, x_row + r);
            r += take;
          }
          ++issued;
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (*abort_flag && leader) {
        // Wait (bounded) for the copies already issued, so that none lands after
        // this CTA has gone.  (The even CTA's barriers count both CTAs' copies.)
        int s = stage, ph = phase;
        for (int i = 0; i < C::STAGES && i < issued; ++i) {
          s = (s == 0) ? C::STAGES - 1 : s - 1;
          if (s == C::STAGES - 1) ph ^= 1;
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(&full[s], ph)) {
            if (globaltimer_ns() - t0 > kWaitLimitNs) {
              atomicOr(g.status, DEV_TIMEOUT_DRAIN);
              break;
            }
          }
        }
      }
    }
    } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    if (leader && elect_one()) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      auto take_buffer = [&]() {
        ok = mbar_wait_bounded(&acc_empty[buf], buf_phase ^ 1u, abort_flag, g.status,
                               DEV_TIMEOUT_MMA);
        tc_fence_after();
        return ok;
      };
      auto give_buffer = [&]() {
        if constexpr (PAIR)
          tc_commit_pair(&acc_full[buf]);
        else
          tc_commit(&acc_full[buf]);
        if (++buf == C::BUFS) {
          buf = 0;
          buf_phase ^= 1u;
        }
      };
      Tile t;
      while (ok && walk.next(t)) {
        const uint32_t idesc = make_idesc(KIND, C::TM, t.cols);
        if (!BLOCKS && !take_buffer()) break;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (BLOCKS && !take_buffer()) break;
          ok = mbar_wait_bounded(&full[stage], phase, abort_flag, g.status, DEV_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(buf * C::TN);
          const uint32_t w = smem_u32(s_w + stage * C::W_BYTES);
          const uint32_t x = smem_u32(s_x + stage * C::X_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t accumulate = (k != 0 || (!BLOCKS && kb != kb0)) ? 1u : 0u;
            if constexpr (PAIR)
              tc_mma_pair<KIND>(d_tmem, smem_desc_k128(w + k * 32), smem_desc_k128(x + k * 32),
                                idesc, accumulate);
            else
              tc_mma<KIND>(d_tmem, smem_desc_k128(w + k * 32), smem_desc_k128(x + k * 32), idesc,
                           accumulate);
          }
          if constexpr (PAIR)
            tc_commit_pair(&empty[stage]);
          else
            tc_commit(&empty[stage]);
          if (BLOCKS) give_buffer();
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (!BLOCKS) give_buffer();
      }
      if (!ok) {
        // Aborted: let every MMA already issued retire before TMEM is freed.
        if constexpr (PAIR)
          tc_commit_pair(drain);
        else
          tc_commit(drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0)) {
          if (globaltimer_ns() - t0 > kWaitLimitNs) {
            atomicOr(g.status, DEV_TIMEOUT_DRAIN);
            break;
          }
        }
      }
    }
    }
  } else {
    if constexpr (MOVE_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // TMEM lanes 32 quarter ..: channels
    const int half = warp >> 2;    // chunks half, half + 2, ... of 32 rows
    const uint32_t tmem_warp = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t empty0 = PAIR ? map_to_rank(acc_empty, 0) : 0u;  // in the even CTA
    uint8_t* stage_out = s_store + warp * 1024;
    int out_buf = 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    auto wait_acc = [&]() {
      const bool ok = mbar_wait_bounded(&acc_full[buf], buf_phase, abort_flag, g.status,
                                        DEV_TIMEOUT_EPILOGUE);
      __syncwarp();
      tc_fence_after();
      return ok;
    };
    auto release_acc = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_cluster(empty0 + buf * 8);
        else
          mbar_arrive(&acc_empty[buf]);
      }
      if (++buf == C::BUFS) {
        buf = 0;
        buf_phase ^= 1u;
      }
    };
    auto load_chunk = [&](int c, uint32_t* r) {
      const uint32_t t = tmem_warp + static_cast<uint32_t>(buf * C::TN + (2 * c + half) * 32);
      tmem_ld_frag(t, r);
      tmem_ld_frag(t + (16u << 16), r + 16);
    };
    auto has_chunk = [&](const Tile& t, int c) { return (2 * c + half) * 32 < t.cols; };

    // Block scales: products sa * sb of four blocks ("a quad") for the tile's rows
    // go to a slot of shared memory together.  A warp writes its share of quad
    // q + 1 after it has finished quad q, for which it had waited until every
    // warp had written its share of q, having finished q - 1: two slots need no
    // second barrier.
    float sv[4];
    uint32_t quad = 0;  // written so far
    constexpr int PER_THREAD = C::TN * 4 / 256;  // values of a quad a thread brings
    auto fetch_quad = [&](const Tile& t, int kb) {
      const int64_t ch_block = t.ch0 / 128 + (PAIR ? static_cast<int>(rank) : 0);
      const float* sb = g.b_scales + t.group * g.bs_group + ch_block * g.bs_n;
      const bool ch_ok = ch_block * 128 < g.n;
#pragma unroll
      for (int j = 0; j < PER_THREAD; ++j) {
        const int i = static_cast<int>(threadIdx.x) + 256 * j;
        const int r = i % C::TN, k = kb + i / C::TN;
        sv[j] = 0.0f;
        if (r < t.rows && k < kb1 && ch_ok)
          sv[j] = __fmul_rn(__ldg(g.a_scales + (t.row0 + r) * g.as_row + k * g.as_k),
                            __ldg(sb + k * g.bs_k));
      }
    };
    auto put_quad = [&]() {
      float* s = s_scale + (quad % C::SCALE_SLOTS) * 4 * C::TN;
#pragma unroll
      for (int j = 0; j < PER_THREAD; ++j) s[threadIdx.x + 256 * j] = sv[j];
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_full[quad % C::SCALE_SLOTS]);
      ++quad;
    };

    Tile t, ahead;
    bool more = walk.next(t);
    if (BLOCKS && more) fetch_quad(t, kb0);
    bool ok = true;
    while (more && ok) {
      const bool more_ahead = walk.next(ahead);
      uint32_t acc[C::CHUNKS][32];
      if constexpr (BLOCKS) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0u;
        put_quad();
        uint32_t now = quad - 1;
        for (int kq = kb0; kq < kb1 && ok; kq += 4, ++now) {
          // (the quad after this one, of this tile or the next, is on its way meanwhile)
          if (kq + 4 < kb1) {
            fetch_quad(t, kq + 4);
          } else if (more_ahead) {
            fetch_quad(ahead, kb0);
          }
          ok = mbar_wait_bounded(&scale_full[now % C::SCALE_SLOTS],
                                 (now / C::SCALE_SLOTS) & 1u, abort_flag, g.status,
                                 DEV_TIMEOUT_EPILOGUE);
          __syncwarp();
          const float* sc = s_scale + (now % C::SCALE_SLOTS) * 4 * C::TN + half * 32 +
                            2 * (lane & 3);
          for (int kb = kq; kb < kq + 4 && kb < kb1 && ok; ++kb, sc += C::TN) {
            ok = wait_acc();
            if (!ok) break;
            uint32_t r[2][32];
            if (has_chunk(t, 0)) load_chunk(0, r[0]);
#pragma unroll
            for (int c = 0; c < C::CHUNKS; ++c) {
              if (!has_chunk(t, c)) break;
              tmem_wait_frag(r[c & 1]);
              if (c + 1 < C::CHUNKS && has_chunk(t, c + 1))
                load_chunk(c + 1, r[(c + 1) & 1]);
              else
                release_acc();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 s = *reinterpret_cast<const float2*>(sc + c * 64 + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int at = (j >> 1) * 16 + 4 * i + 2 * (j & 1);
                  const float2 v = __ffma2_rn(
                      make_float2(__uint_as_float(r[c & 1][at]),
                                  __uint_as_float(r[c & 1][at + 1])),
                      s,
                      make_float2(__uint_as_float(acc[c][at]), __uint_as_float(acc[c][at + 1])));
                  acc[c][at] = __float_as_uint(v.x);
                  acc[c][at + 1] = __float_as_uint(v.y);
                }
              }
            }
            if (!has_chunk(t, 0)) release_acc();  // no rows for this warp
          }
          if (ok && kq + 4 < kb1) put_quad();
        }
        if (!ok) break;
      } else {
        ok = wait_acc();
        if (!ok) break;
      }

      const int ch = t.ch0 + (PAIR ? static_cast<int>(rank) * 128 : 0) + quarter * 32;
      float sb[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      constexpr bool ROW_SCALES = !BLOCKS && (KIND == KIND_I8 || KIND == KIND_F8);
      if constexpr (ROW_SCALES) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = ch + 8 * j + (lane >> 2);
          if (n < g.n) sb[j] = __ldg(g.b_scales + t.group * g.bs_group + n * g.bs_n);
        }
      }
      // Rows 8 i .. 8 i + 7 of chunk c: registers r.
      auto finish = [&](const uint32_t* r, int c, int i) {
        const int first = (2 * c + half) * 32 + 8 * i;
        if (first >= t.rows) return;
        float2 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = (j >> 1) * 16 + 4 * i + 2 * (j & 1);
          v[j] = frag_value<KIND>(r[at], r[at + 1]);
        }
        if constexpr (ROW_SCALES) {
          const int r0 = first + 2 * (lane & 3);
          const float* sa = g.a_scales + int64_t(t.row0 + r0) * g.as_row;
          const float2 s = make_float2(r0 < t.rows ? __ldg(sa) : 0.0f,
                                       r0 + 1 < t.rows ? __ldg(sa + g.as_row) : 0.0f);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[j] = __fmul2_rn(__fmul2_rn(v[j], s), make_float2(sb[j], sb[j]));
        }
        store_rows8(g, v, stage_out + out_buf * 512, int64_t(t.row0) + first, t.rows - first, ch,
                    lane);
        out_buf ^= 1;
      };
      if (!PAIR && splits > 1) {
        if constexpr (!PAIR) {
          if constexpr (!BLOCKS) {
            if (has_chunk(t, 0)) {
              load_chunk(0, acc[0]);
              tmem_wait_frag(acc[0]);
            }
            release_acc();
          }
          // Rows 8 n .. 8 n + 7 of the tile belong to rank n % splits, as its
          // group n / splits; every rank's sums of them are [sender][quarter][part][lane].
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = half * 4 + i;
            const uint32_t owner = static_cast<uint32_t>(n % splits);
            if (8 * n < t.rows) {
              const uint32_t to =
                  map_to_rank(s_exchange, owner) +
                  ((((n / splits) * splits + rank) * 4 + quarter) * 2 * 32 + lane) * 16;
              st_cluster_v4(to, acc[0][4 * i], acc[0][4 * i + 1], acc[0][4 * i + 2],
                            acc[0][4 * i + 3]);
              st_cluster_v4(to + 512, acc[0][16 + 4 * i], acc[0][17 + 4 * i], acc[0][18 + 4 * i],
                            acc[0][19 + 4 * i]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_rank(parts, owner));
          }
          ok = mbar_wait_cluster(parts, 0, abort_flag, g.status, DEV_TIMEOUT_FIXUP);
          __syncwarp();
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = half * 4 + i;
            if (n % splits != static_cast<int>(rank) || 8 * n >= t.rows) continue;
            for (int s = 0; s < splits; ++s) {
              const uint4* from = reinterpret_cast<const uint4*>(s_exchange) +
                                  (((n / splits) * splits + s) * 4 + quarter) * 2 * 32 + lane;
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                const uint4 w = from[32 * p];
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  uint32_t& a = acc[0][16 * p + 4 * i + q];
                  a = s == 0 ? u[q] : frag_add<KIND>(a, u[q]);
                }
              }
            }
            finish(acc[0], 0, i);
          }
          more = false;  // one tile a cluster
        }
      } else {
        if constexpr (BLOCKS) {
#pragma unroll
          for (int c = 0; c < C::CHUNKS; ++c) {
            if (!has_chunk(t, c)) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) finish(acc[c], c, i);
          }
        } else {
          for (int c = 0; c < C::CHUNKS && has_chunk(t, c); ++c) {
            uint32_t r[32];
            load_chunk(c, r);
            tmem_wait_frag(r);
            if (!(c + 1 < C::CHUNKS && has_chunk(t, c + 1))) release_acc();
#pragma unroll
            for (int i = 0; i < 4; ++i) finish(r, c, i);
          }
          if (!has_chunk(t, 0)) release_acc();  // no rows for this warp
        }
        more = more_ahead;
      }
      t = ahead;
    }

    if (g.zero_rest && ok) {
      // Rows before the first group and behind the last.
      const int lo = s_row[0], hi = s_row[g.groups];
      const int64_t rest = int64_t(lo) + (g.rows - hi);
      const int64_t step = int64_t(gridDim.x) * 8;
      for (int64_t i = int64_t(blockIdx.x) * 8 + warp; i < rest; i += step) {
        const int64_t row = i < lo ? i : i - lo + hi;
        if (g.out_dtype == DT_F32) {
          float* o = reinterpret_cast<float*>(g.out) + row * g.out_row;
          for (int c = lane; c < g.n; c += 32) o[c] = 0.0f;
        } else {
          uint16_t* o = reinterpret_cast<uint16_t*>(g.out) + row * g.out_row;
          for (int c = lane; c < g.n; c += 32) o[c] = 0;
        }
      }
    }
  }

  // ------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (PAIR || splits > 1) cluster_sync();  // no CTA of the cluster touches this one any more
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, 512);
    else
      tmem_dealloc(tmem_base, 512);
  }
}

template <int KIND, bool BLOCKS, bool PAIR>
cudaError_t launch(const GroupedMaps& maps, const GroupedArgs& g, int grid, cudaStream_t stream) {
  using C = Cfg<PAIR>;
  auto kern = grouped_gemm_kernel<KIND, BLOCKS, PAIR>;
  static std::atomic<long long> shape[kMaxLaunchDevices];
  int dev = 0, sms = 0, per_sm = 0;
  cudaError_t e = launch_shape(reinterpret_cast<const void*>(kern), C::THREADS, C::SMEM_BYTES,
                               shape, &dev, &sms, &per_sm);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(C::THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n_attr = 0;
  const int cluster = PAIR ? 2 : g.k_splits;
  if (cluster > 1) {
    attr[n_attr].id = cudaLaunchAttributeClusterDimension;
    attr[n_attr].val.clusterDim.x = cluster;
    attr[n_attr].val.clusterDim.y = 1;
    attr[n_attr].val.clusterDim.z = 1;
    ++n_attr;
  }
  cfg.attrs = n_attr ? attr : nullptr;
  cfg.numAttrs = n_attr;
  e = cudaLaunchKernelEx(&cfg, kern, maps, g);
  if (e != cudaSuccess) return e;
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_grouped_gemm(const GroupedMaps& maps, const GroupedArgs& g, int kind,
                                bool blocks, bool pair, int grid, cudaStream_t stream) {
#define M5B_GROUPED(KIND_, BLOCKS_)                                             \
  return pair ? launch<KIND_, BLOCKS_, true>(maps, g, grid, stream)             \
              : launch<KIND_, BLOCKS_, false>(maps, g, grid, stream)
  switch (kind) {
    case KIND_I8: M5B_GROUPED(KIND_I8, false);
    case KIND_F8:
      if (blocks) M5B_GROUPED(KIND_F8, true);
      M5B_GROUPED(KIND_F8, false);
    case KIND_BF16: M5B_GROUPED(KIND_BF16, false);
    case KIND_F16: M5B_GROUPED(KIND_F16, false);
    default: return cudaErrorInvalidValue;
  }
#undef M5B_GROUPED
}

}  // namespace m5b
