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
// not stored.  (Block-scaled products on CTA pairs are the other way round, see
// ROWS_M: a scale for each column would cost the epilogue more than the MMAs take.)
//
// Block scales: a block of 128 channels of K (one 128-byte slice, four MMAs) is
// summed in TMEM by itself, and the epilogue warps add it, times the row's and
// the channel block's scale, to fp32 sums in registers:
//   sum[t, n] += (sa[t, g] * sb[n / 128, g]) * partial[t, n]
// while the MMAs of the next block fill another TMEM buffer.  Without block
// scales a tile's whole K range stays in TMEM.
//
// Roles: warps 0-7 epilogue, warp 8 TMA producer, warp 9 MMA issuer, warps 10 and
// 11 bring the block scales (products sa * sb, in shared memory).  TMEM is
// read by whole lanes: a thread holds one channel of 32 rows (ROWS_M: one row of
// 16 channels).  That goes at 840 bytes a clock and SM, where 16 x 256-bit
// fragments, which would need fewer scales a thread, came at 253, as long as
// the MMAs of a block take.
//
// K split over a cluster (single CTAs, one tile a cluster): each CTA sums its
// part of K; the sums of eight rows go to the CTA that owns them through
// distributed shared memory, which adds the parts in the order of the ranks.
#include <type_traits>

#include "grouped.cuh"

namespace m5b {

namespace {

template <int ADD, bool PAIR>
struct Cfg {
  static constexpr bool BLOCKS = ADD == GROUPED_ADD_SCALED;
  static constexpr bool PARTS = ADD == GROUPED_ADD_PARTS;  // blocks of an accumulator: four
  static constexpr bool ROWS_M = BLOCKS && PAIR;           // the rows are the M operand
  static constexpr int TN = PAIR ? 256 : kSingleTileRows;  // columns of an accumulator
  static constexpr int TM = PAIR ? 256 : 128;              // channels of a tile
  static constexpr int STEP = PAIR ? 32 : 16;              // columns come in these
  static constexpr int M_BYTES = 128 * 128;                // this CTA's M operand of a stage
  static constexpr int N_BYTES = (PAIR ? TN / 2 : TN) * 128;  // and its N operand
  static constexpr int FEW_ROWS = PAIR ? 64 : 16;          // a CTA's columns come in these, or all
  static constexpr int STAGES = PAIR ? 6 : 7;
  // Blocks of K that change hands between MMAs and epilogue together, each with an
  // accumulator of its own (few columns: a hand-over takes longer than a block).
  static constexpr int BATCH = BLOCKS && !PAIR ? 4 : 1;
  static constexpr int BUFS = 512 / (TN * BATCH);          // TMEM accumulators, or batches
  static constexpr int CHUNKS = TN / 64;                   // 32-column chunks of an epilogue warp
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 32 * (EPI_WARPS + 4);     // three warpgroups
  static constexpr int SCALE_SLOTS = ROWS_M ? 2 : 8;       // of four blocks of K each
  // Block scales' slots, or each epilogue warp's rows' scales.
  static constexpr int SCALE_BYTES =
      BLOCKS ? SCALE_SLOTS * 4 * TN * 4 : EPI_WARPS * CHUNKS * 32 * 4;
  static constexpr int STORE_WARP = ROWS_M ? 2048 : 1024;  // a warp's bytes to rearrange stores
  static constexpr int STORE_BYTES = EPI_WARPS * STORE_WARP;
  static constexpr int EXCHANGE_BYTES = PAIR ? 0 : TN * 128 * 4;
  static constexpr int TABLE_BYTES = 2 * (kMaxGroups + 4) * 4;
  static constexpr int BAR_BYTES = (2 * STAGES + 2 * BUFS + 2 * SCALE_SLOTS + 2) * 8 + 16 +
                                   SCALE_SLOTS * 16;
  static constexpr int SMEM_BYTES = 1024 + STAGES * (M_BYTES + N_BYTES) + EXCHANGE_BYTES +
                                    SCALE_BYTES + STORE_BYTES + TABLE_BYTES + BAR_BYTES;
  static_assert(SMEM_BYTES <= 232448, "shared memory per CTA exceeds 227 KB");
};

// Waits for this thread's TMEM load; its registers are named so that no use of
// them moves above the wait.
__device__ __forceinline__ void tmem_wait32(uint32_t* r) {
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
// The same in 16 columns.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
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
// Arrival on a barrier of another CTA that hands over TMEM only (the tcgen05 fence
// before it orders that): a release over the cluster would wait for every load
// that the thread has under way (1.9 us a block of 128 channels instead of 1.45
// where it had both).
__device__ __forceinline__ void mbar_arrive_tmem(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The two halves of a cluster barrier.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_cluster() {
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
// Arrival that a fence_cluster before it makes a release.
__device__ __forceinline__ void mbar_arrive_fenced(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
               : "memory");
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                              uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
// A wait's answer as the warp's: after a wait that gave up, lanes may have seen the barrier
// or the abort flag first, and the aligned instructions that follow need all of them or none.
__device__ __forceinline__ bool whole_warp(bool ok) { return __all_sync(0xffffffffu, ok); }

// mbar_wait_bounded of a whole warp, with few registers (the epilogue has none to
// spare): 32 bits of the clock, 4.3 s.  It votes on each look, which serves as the
// warp barrier that would follow: 4096 x 4096 x 16384 block-scaled 277 us, 290 with one.
__device__ __forceinline__ uint32_t globaltimer_lo() {
  uint32_t t;
  asm volatile("mov.u32 %0, %globaltimer_lo;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool mbar_wait_lean(uint32_t bar, uint32_t parity, uint32_t abort,
                                               unsigned int* status, unsigned int code) {
  uint32_t start = 0;
  bool first = true;
  while (true) {
    uint32_t ok, stop;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (whole_warp(ok)) return true;
    if (first) start = globaltimer_lo();
    first = false;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(stop) : "r"(abort) : "memory");
    if (!whole_warp(!stop)) return false;
    if (!whole_warp(globaltimer_lo() - start <= static_cast<uint32_t>(kWaitLimitNs))) {
      atomicOr(status, code);
      asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort), "r"(1) : "memory");
      return false;
    }
  }
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
template <class C>
struct Walk {
  const int* first_row;
  const int* first_tile;
  int groups, tile_rows, ch_tiles;
  int unit, stride, e;

  __device__ __forceinline__ bool next(Tile& t) {
    if (unit >= first_tile[groups]) return false;
    while (unit >= first_tile[e + 1]) ++e;
    const int rows = first_row[e + 1] - first_row[e];  // positive: the group has tiles
    const int u = unit - first_tile[e];
    int ch = u, r = 0, each = rows;  // one row tile
    if (rows > tile_rows) {
      const int row_tiles = (rows + tile_rows - 1) / tile_rows;
      // Bands of at most 16 row tiles, within which the channel tiles follow one
      // another: CTAs that run side by side share weights, and a band's rows stay in L2.
      const int band = u / (16 * ch_tiles);
      const int in_band = u - band * 16 * ch_tiles;
      const int left = row_tiles - 16 * band;
      const int wide = left < 16 ? left : 16;
      ch = in_band / wide;
      r = 16 * band + in_band - ch * wide;
      each = ((rows + row_tiles - 1) / row_tiles + C::STEP - 1) / C::STEP * C::STEP;
    }
    t.group = e;
    t.row0 = first_row[e] + r * each;
    // (positive too: tile_rows is a multiple of STEP, so each <= tile_rows and
    // (row_tiles - 1) * each <= (row_tiles - 1) * tile_rows < rows)
    t.rows = rows - r * each < each ? rows - r * each : each;
    t.cols = (t.rows + C::STEP - 1) / C::STEP * C::STEP;
    t.ch0 = ch * C::TM;
    unit += stride;
    return true;
  }
};

template <int KIND>
__device__ __forceinline__ float sum_value(uint32_t a) {
  if constexpr (KIND == KIND_I8)
    return __int2float_rn(static_cast<int>(a));
  else
    return __uint_as_float(a);
}
template <int KIND>
__device__ __forceinline__ uint32_t sum_add(uint32_t a, uint32_t b) {
  if constexpr (KIND == KIND_I8)
    return a + b;
  else
    return __float_as_uint(__fadd_rn(__uint_as_float(a), __uint_as_float(b)));
}

// Eight rows, of which the first `rows` exist, of this lane's channel.  at: the
// first row's 32 channels of the warp, of which `channels` exist; stage: 512 bytes
// of the warp's, in which 16-bit values become rows for 16-byte stores.
__device__ __forceinline__ void store_rows8(const GroupedArgs& g, const float2 (&v)[4],
                                            uint8_t* stage, uint8_t* at, int rows, int channels,
                                            int lane) {
  if (g.out_dtype == DT_F32) {
    float* o = reinterpret_cast<float*>(at) + lane;
    if (lane >= channels) return;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r < rows) *o = r & 1 ? v[r >> 1].y : v[r >> 1].x;
      o += g.out_row;
    }
    return;
  }
  uint16_t* mine = reinterpret_cast<uint16_t*>(stage) + lane;
#pragma unroll
  for (int r = 0; r < 8; r += 2) {
    uint32_t two;
    if (g.out_dtype == DT_F16) {
      const __half2 h = __float22half2_rn(v[r >> 1]);
      two = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      two = f2_bf16x2(v[r >> 1]);
    }
    mine[r * 32] = static_cast<uint16_t>(two);
    mine[r * 32 + 32] = static_cast<uint16_t>(two >> 16);
  }
  __syncwarp();
  uint16_t* o = reinterpret_cast<uint16_t*>(at);
  if (g.out_vec) {
    const int r = lane >> 2, piece = lane & 3;
    const uint4 w = *reinterpret_cast<const uint4*>(stage + lane * 16);
    if (r < rows && 8 * piece < channels)
      *reinterpret_cast<uint4*>(o + r * g.out_row + 8 * piece) = w;
  } else if (lane < channels) {
    for (int r = 0; r < rows && r < 8; ++r) o[r * g.out_row + lane] = mine[r * 32];
  }
}

// 64 bytes of channels, from ch on, of 32 rows (row .. row + 31, of which the first
// `rows` exist): 32 of a 16-bit type, 16 of fp32.  w: those of row row + lane.
// stage: 2 KB of the warp's, in which the rows' 16-byte pieces change hands, so
// that four lanes store a row's.
__device__ __forceinline__ void store_rows32(const GroupedArgs& g, const uint32_t (&w)[16],
                                             uint8_t* stage, int64_t row, int rows, int ch,
                                             int lane) {
  const int swizzle = (lane >> 1) & 3;  // of the pieces: no bank conflicts
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((j ^ swizzle) << 4)) =
        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  __syncwarp();
  const bool wide = g.out_dtype == DT_F32;
  uint8_t* o = static_cast<uint8_t*>(g.out);
  if (g.out_vec) {
    const int c = ch + (lane & 3) * (wide ? 4 : 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + 8 * i;
      const uint4 x = *reinterpret_cast<const uint4*>(
          stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
      if (r < rows && c < g.n)
        *reinterpret_cast<uint4*>(o + ((row + r) * g.out_row + c) * (wide ? 4 : 2)) = x;
    }
  } else {
    // (one row at a time: 32 values of two bytes, or 16 of four)
    const int at = lane * (wide ? 4 : 2);
    if (at < 64 && ch + lane < g.n) {
      for (int r = 0; r < rows && r < 32; ++r) {
        const uint8_t* from = stage + r * 64 + (((at >> 4) ^ ((r >> 1) & 3)) << 4) + (at & 15);
        const int64_t to = (row + r) * g.out_row + ch + lane;
        if (wide)
          reinterpret_cast<float*>(o)[to] = *reinterpret_cast<const float*>(from);
        else
          reinterpret_cast<uint16_t*>(o)[to] = *reinterpret_cast<const uint16_t*>(from);
      }
    }
  }
  __syncwarp();
}

template <int KIND, int ADD, bool PAIR>
__global__ void __launch_bounds__(Cfg<ADD, PAIR>::THREADS, 1)
    grouped_gemm_kernel(const __grid_constant__ GroupedMaps maps, const GroupedArgs g) {
  using C = Cfg<ADD, PAIR>;
  constexpr bool BLOCKS = C::BLOCKS, PARTS = C::PARTS;
  constexpr int K_ELEMS = (KIND == KIND_BF16 || KIND == KIND_F16) ? 64 : 128;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_m = smem;
  uint8_t* s_n = s_m + C::STAGES * C::M_BYTES;
  uint8_t* s_exchange = s_n + C::STAGES * C::N_BYTES;
  float* s_scale = reinterpret_cast<float*>(s_exchange + C::EXCHANGE_BYTES);
  uint8_t* s_store = reinterpret_cast<uint8_t*>(s_scale) + C::SCALE_BYTES;
  int* s_row = reinterpret_cast<int*>(s_store + C::STORE_BYTES);  // [groups + 1]
  int* s_tile = s_row + kMaxGroups + 4;                           // [groups + 1]
  uint64_t* full = reinterpret_cast<uint64_t*>(s_tile + kMaxGroups + 4);
  uint64_t* empty = full + C::STAGES;
  uint64_t* acc_full = empty + C::STAGES;
  uint64_t* acc_empty = acc_full + C::BUFS;
  uint64_t* scale_full = acc_empty + C::BUFS;
  uint64_t* scale_empty = scale_full + C::SCALE_SLOTS;
  uint64_t* drain = scale_empty + C::SCALE_SLOTS;
  uint64_t* parts = drain + 1;  // K split: the owned rows' sums of all ranks are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(parts + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // ROWS_M: the tile that a slot's scales begin, {first row, rows (0: no more), first channel}
  volatile int* slot_tile = reinterpret_cast<volatile int*>(tmem_slot + 2);

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
    for (int s = 0; s < C::SCALE_SLOTS; ++s) {
      mbar_init(&scale_full[s], 2);
      mbar_init(&scale_empty[s], C::EPI_WARPS);
    }
    mbar_init(drain, 1);
    mbar_init(parts, 32);  // eight groups of rows / splits owners, four warps, `splits` senders
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  // K split: the CTAs need one another's barriers only when they exchange their
  // sums, and nothing of one another after that: they arrive here and wait there.
  const bool exchange = !PAIR && splits > 1;
  __syncwarp();
  if (exchange) cluster_arrive();
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&maps.b);
    tma_prefetch_desc(PAIR ? &maps.a128 : &maps.a64);
    if (!C::ROWS_M) tma_prefetch_desc(PAIR ? &maps.a64 : &maps.a16);  // (else not encoded)
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
  // With programmatic launch all that stands before the first access to global
  // memory overlaps the previous kernel's end, and lets the next kernel start, which
  // waits in its turn: here where the bounds are read, else in every role, whose code
  // is cold too (2500 cycles from here to the first copy).
  auto inputs_ready = []() {
    grid_dependency_wait();
    grid_dependents_launch();
  };
  if (g.group_start) inputs_ready();
  // The groups' first rows, then the tiles before each group.
  const int ch_tiles = (g.n + C::TM - 1) / C::TM;
  if (!g.group_start) {
    if (threadIdx.x == 32) {
      s_row[0] = s_tile[0] = 0;
      s_row[1] = g.rows;
      s_tile[1] = (g.rows + g.tile_rows - 1) / g.tile_rows * ch_tiles;
    }
  } else {
    for (int e = threadIdx.x; e <= g.groups; e += C::THREADS) {
      int r = g.group_start[e];
      r = r < 0 ? 0 : r;
      s_row[e] = r < g.rows ? r : g.rows;
    }
    __syncthreads();
  }
  if (g.group_start && warp == 0) {
    // Bounds that do not ascend (which is the caller's to see to) are taken as the
    // largest before them: no two groups share a row, and there are no more tiles
    // than the host allows for.
    int most = 0;
    for (int e0 = 0; e0 <= g.groups; e0 += 32) {
      int r = e0 + lane <= g.groups ? s_row[e0 + lane] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, r, d);
        if (lane >= d) r = max(r, v);
      }
      r = max(r, most);
      if (e0 + lane <= g.groups) s_row[e0 + lane] = r;
      most = __shfl_sync(0xffffffffu, r, 31);
    }
    __syncwarp();
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
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // both CTAs' barriers exist before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  bool exchanged = false;  // this warp has sent its sums
  Walk<C> walk{s_row, s_tile, g.groups, g.tile_rows, ch_tiles,
                  static_cast<int>(blockIdx.x) / per, static_cast<int>(gridDim.x) / per, 0};
  const int kb0 = PAIR ? 0 : static_cast<int>(int64_t(g.num_k_blocks) * rank / splits);
  const int kb1 = PAIR ? g.num_k_blocks
                       : static_cast<int>(int64_t(g.num_k_blocks) * (rank + 1) / splits);

  // The fp32 sums of a pair's tile are 128 registers a thread of the epilogue:
  // it takes over registers of the other warps.  (384 threads are launched with
  // 168 each: 2 * 216 + 72 = 3 * 168.)
  constexpr bool MOVE_REGS = PAIR && ADD != GROUPED_ADD_NONE;
  if (warp >= C::EPI_WARPS) {
    if constexpr (MOVE_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ------------------------------------------------------------ producer
      if (elect_one()) {
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        Tile t;
        while (!*abort_flag && walk.next(t)) {
          // This CTA's part of the columns (of a pair's, half), and its 128 of M.
          const int n_rows = C::ROWS_M ? 128 : PAIR ? t.cols / 2 : t.cols;
          const int n_row =
              (C::ROWS_M ? t.ch0 : t.row0) + (PAIR ? static_cast<int>(rank) * n_rows : 0);
          const int m_row =
              (C::ROWS_M ? t.row0 : t.ch0) + (PAIR ? static_cast<int>(rank) * 128 : 0);
          // One box brings the columns' rows: of the next size, what lies behind the
          // tile's is not used.
          const bool few = n_rows <= C::FEW_ROWS;
          const CUtensorMap* columns = few ? (PAIR ? &maps.a64 : &maps.a16)
                                           : (PAIR ? &maps.a128 : &maps.a64);
          if (issued == 0 && !g.group_start) inputs_ready();
          const uint32_t bytes =
              C::M_BYTES + (C::ROWS_M ? 128 : few ? C::FEW_ROWS : C::N_BYTES / 128) * 128;
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, abort_flag, g.status,
                                   DEV_TIMEOUT_PRODUCER))
              break;
            const int kx = kb * K_ELEMS;
            uint8_t* m = s_m + stage * C::M_BYTES;
            uint8_t* n = s_n + stage * C::N_BYTES;
            if constexpr (PAIR) {
              // The even CTA's barrier counts both CTAs' bytes.
              if (leader) mbar_arrive_expect_tx(&full[stage], 2 * bytes);
            } else {
              mbar_arrive_expect_tx(&full[stage], bytes);
            }
            if constexpr (C::ROWS_M) {
              tma_load_2d_pair(m, &maps.a128, &full[stage], kx, m_row);
              tma_load_3d_pair(n, &maps.b, &full[stage], kx, n_row, t.group);
            } else {
              if constexpr (PAIR)
                tma_load_3d_pair(m, &maps.b, &full[stage], kx, m_row, t.group);
              else
                tma_load_3d(m, &maps.b, &full[stage], kx, m_row, t.group);
              if constexpr (PAIR)
                tma_load_2d_pair(n, columns, &full[stage], kx, n_row);
              else
                tma_load_2d(n, columns, &full[stage], kx, n_row);
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
        // (the limit of its waits must not count the previous kernel's time, for as long as
        // which the producer waits)
        if (!g.group_start) inputs_ready();
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
          const uint32_t idesc = make_idesc(KIND, PAIR ? 256 : 128, C::ROWS_M ? C::TN : t.cols);
          for (int kb = kb0; kb < kb1; ++kb) {
            const int in_batch = BLOCKS ? (kb - kb0) % C::BATCH : 0;
            // the accumulator's first and last block
            const bool first = BLOCKS ? in_batch == 0 : PARTS ? (kb - kb0) % 4 == 0 : kb == kb0;
            const bool last = (BLOCKS ? in_batch == C::BATCH - 1 : PARTS && (kb - kb0) % 4 == 3) ||
                              kb + 1 == kb1;
            // (all that the MMAs need is ready before the accumulator is)
            ok = mbar_wait_bounded(&full[stage], phase, abort_flag, g.status, DEV_TIMEOUT_MMA);
            if (!ok) break;
            const uint32_t d_tmem =
                tmem_base + static_cast<uint32_t>((buf * C::BATCH + in_batch) * C::TN);
            const uint64_t m = smem_desc_k128(smem_u32(s_m + stage * C::M_BYTES));
            const uint64_t n = smem_desc_k128(smem_u32(s_n + stage * C::N_BYTES));
            if (first && !take_buffer()) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 32 bytes of K further: 2 in the descriptors
              const uint32_t accumulate = (k != 0 || (!BLOCKS && !first)) ? 1u : 0u;
              if constexpr (PAIR)
                tc_mma_pair<KIND>(d_tmem, m + 2 * k, n + 2 * k, idesc, accumulate);
              else
                tc_mma<KIND>(d_tmem, m + 2 * k, n + 2 * k, idesc, accumulate);
            }
            if constexpr (PAIR)
              tc_commit_pair(&empty[stage]);
            else
              tc_commit(&empty[stage]);
            if (last) give_buffer();
            if (++stage == C::STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
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
    } else if constexpr (BLOCKS) {
      // ---------------------------------------------------------- block scales
      // Products sa * sb of four blocks of K ("a quad") a slot: of the tile's rows,
      // or (ROWS_M) of this CTA's 128 rows with each of the tile's channel blocks.
      if (!g.group_start) inputs_ready();
      const int me = static_cast<int>(threadIdx.x) - 320;
      uint32_t quad = 0;
      bool ok = true;
      Tile t;
      while (ok && walk.next(t)) {
        const float* sa = g.a_scales + t.row0 * g.as_row;
        const float* sb = g.b_scales + t.group * g.bs_group + t.ch0 / 128 * g.bs_n;
        // All loads of QUADS of them are under way before the first is used.
        // (Plain loads, here and below: the kernel before may have written the scales
        // after this one had started.)
        constexpr int ROWS = C::ROWS_M ? 2 : 1, COLS = ROWS, QUADS = C::ROWS_M ? 1 : 4;
        for (int k0 = kb0; k0 < kb1 && ok; k0 += 4 * QUADS) {
          float v[ROWS][4 * QUADS], w[COLS][4 * QUADS];
#pragma unroll
          for (int k = 0; k < 4 * QUADS; ++k) {
            const bool there = k0 + k < kb1;
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
              const int r = (C::ROWS_M ? static_cast<int>(rank) * 128 : 0) + me + 64 * i;
              v[i][k] = there && r < t.rows ? sa[r * g.as_row + (k0 + k) * g.as_k] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < COLS; ++j)
              w[j][k] = there && t.ch0 + j * 128 < g.n
                            ? sb[j * g.bs_n + (k0 + k) * g.bs_k]
                            : 0.0f;
          }
#pragma unroll
          for (int q = 0; q < QUADS; ++q) {
            if (k0 + 4 * q >= kb1) break;
            const uint32_t slot = quad % C::SCALE_SLOTS;
            ok = whole_warp(mbar_wait_bounded(&scale_empty[slot],
                                              ((quad / C::SCALE_SLOTS) & 1u) ^ 1u, abort_flag,
                                              g.status, DEV_TIMEOUT_PRODUCER));
            if (!ok) break;
            float* s = s_scale + slot * 4 * C::TN + me;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int j = 0; j < COLS; ++j)
                  s[k * C::TN + j * 128 + i * 64] = __fmul_rn(v[i][4 * q + k], w[j][4 * q + k]);
            if (C::ROWS_M && me == 0 && k0 == kb0) {
              slot_tile[slot * 4] = t.row0;
              slot_tile[slot * 4 + 1] = t.rows;
              slot_tile[slot * 4 + 2] = t.ch0;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&scale_full[slot]);
            ++quad;
          }
        }
      }
      if (C::ROWS_M && ok) {
        const uint32_t slot = quad % C::SCALE_SLOTS;
        ok = whole_warp(mbar_wait_bounded(&scale_empty[slot], ((quad / C::SCALE_SLOTS) & 1u) ^ 1u,
                                          abort_flag, g.status, DEV_TIMEOUT_PRODUCER));
        if (me == 0) slot_tile[slot * 4 + 1] = 0;
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&scale_full[slot]);
      }
    }
  } else {
    if constexpr (MOVE_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------ epilogue
    if (!g.group_start) inputs_ready();
    const int quarter = warp & 3;  // TMEM lanes 32 quarter ..: channels
    const int half = warp >> 2;    // of the 32-column chunks: every second, or (ROWS_M) half
    const uint32_t tmem_warp = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t empty0 = PAIR ? map_to_rank(acc_empty, 0) : 0u;  // in the even CTA
    uint8_t* stage_out = s_store + warp * C::STORE_WARP;
    float* row_scales = s_scale + warp * C::CHUNKS * 32;
    int out_buf = 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    auto wait_acc = [&]() {
      const bool ok = mbar_wait_lean(smem_u32(acc_full) + buf * 8, buf_phase,
                                     smem_u32(const_cast<int*>(abort_flag)), g.status,
                                     DEV_TIMEOUT_EPILOGUE);
      tc_fence_after();
      return ok;
    };
    auto release_acc = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_tmem(empty0 + buf * 8);
        else
          mbar_arrive(&acc_empty[buf]);
      }
      if (++buf == C::BUFS) {
        buf = 0;
        buf_phase ^= 1u;
      }
    };
    auto load_chunk = [&](int c, uint32_t (&r)[32]) {
      tmem_ld32(tmem_warp + static_cast<uint32_t>(buf * C::TN + (2 * c + half) * 32), r);
      tmem_wait32(r);
    };
    auto has_chunk = [&](const Tile& t, int c) { return (2 * c + half) * 32 < t.cols; };

    // sum += scale * r, of neighbouring columns.
    uint32_t acc[C::CHUNKS][32];
    auto add_columns = [&](auto& r, uint32_t* sum, auto scale) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(r) / 4); i += 2) {
        const float2 v = __ffma2_rn(
            make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), scale(i),
            make_float2(__uint_as_float(sum[i]), __uint_as_float(sum[i + 1])));
        sum[i] = __float_as_uint(v.x);
        sum[i + 1] = __float_as_uint(v.y);
      }
    };
    uint32_t quad = 0;
    Tile t;
    bool ok = true;
    auto wait_scales = [&]() {
      ok = mbar_wait_lean(smem_u32(scale_full) + quad % C::SCALE_SLOTS * 8,
                          (quad / C::SCALE_SLOTS) & 1u, smem_u32(const_cast<int*>(abort_flag)),
                          g.status, DEV_TIMEOUT_EPILOGUE);
      return ok;
    };
    while (ok) {
      if constexpr (C::ROWS_M) {
        // (the warps that bring the scales walk the tiles: there are no registers
        // for that here)
        if (!wait_scales()) break;
        volatile int* info = slot_tile + quad % C::SCALE_SLOTS * 4;
        t.row0 = info[0];
        t.rows = info[1];
        t.ch0 = info[2];
        if (t.rows == 0) break;
      } else {
        if (!walk.next(t)) break;
      }
      if constexpr (ADD != GROUPED_ADD_NONE) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0u;
      }
      if constexpr (PARTS) {
        for (int kb = kb0; kb < kb1; kb += 4) {
          ok = wait_acc();
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < C::CHUNKS; ++c) {
            if (!has_chunk(t, c)) break;
            uint32_t r[32];
            load_chunk(c, r);
            if (!(c + 1 < C::CHUNKS && has_chunk(t, c + 1))) release_acc();
            add_columns(r, acc[c], [](int) { return make_float2(1.0f, 1.0f); });
          }
          if (!has_chunk(t, 0)) release_acc();  // no rows for this warp
        }
      }
      if constexpr (C::ROWS_M) {
        // A thread has one row and this warp's 128 channels have one scale: one product.
        const float* sc = s_scale + half * 128 + quarter * 32 + lane;
#pragma unroll 1
        for (int kb = 0; kb < kb1; ++kb) {
          if ((kb & 3) == 0 && kb != 0 && !wait_scales()) break;
          const float one = sc[((quad % C::SCALE_SLOTS) * 4 + (kb & 3)) * C::TN];
          const float2 s = make_float2(one, one);
          ok = wait_acc();
          if (!ok) break;
          // 16 columns are added while the next 16 come.
          const uint32_t from = tmem_warp + static_cast<uint32_t>(buf * C::TN + half * 128);
          uint32_t r[2][16];
          tmem_ld16(from, r[0]);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            tmem_wait16(r[c & 1]);
            if (c < 7)
              tmem_ld16(from + 16 * (c + 1), r[(c + 1) & 1]);
            else
              release_acc();
            add_columns(r[c & 1], acc[c >> 1] + 16 * (c & 1), [&](int) { return s; });
          }
          if ((kb & 3) == 3 || kb + 1 == kb1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&scale_empty[quad % C::SCALE_SLOTS]);
            ++quad;
          }
        }
      } else if constexpr (BLOCKS) {
        for (int kq = kb0; kq < kb1 && ok; kq += 4, ++quad) {
          const uint32_t slot = quad % C::SCALE_SLOTS;
          ok = whole_warp(mbar_wait_bounded(&scale_full[slot], (quad / C::SCALE_SLOTS) & 1u,
                                            abort_flag, g.status, DEV_TIMEOUT_EPILOGUE));
          if (!ok) break;
          ok = wait_acc();
          if (!ok) break;
          if (has_chunk(t, 0)) {
            const float* sc = s_scale + slot * 4 * C::TN + half * 32;
            const uint32_t from =
                tmem_warp + static_cast<uint32_t>(buf * C::BATCH * C::TN + half * 32);
            // (two at a time: more need more registers than there are)
#pragma unroll
            for (int k0 = 0; k0 < 4; k0 += 2) {
              uint32_t r[2][32];
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (kq + k0 + k < kb1) tmem_ld32(from + (k0 + k) * C::TN, r[k]);
#pragma unroll
              for (int k = 0; k < 2; ++k) tmem_wait32(r[k]);
              if (k0 == 2) release_acc();
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (kq + k0 + k < kb1)
                  add_columns(r[k], acc[0], [&](int i) {
                    return *reinterpret_cast<const float2*>(sc + (k0 + k) * C::TN + i);
                  });
            }
          } else {
            release_acc();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&scale_empty[slot]);
        }
      }
      // Scales of rows and channels: this thread's channel, and a row of each chunk.
      const int ch = t.ch0 + (PAIR ? static_cast<int>(rank) * 128 : 0) + quarter * 32;
      constexpr bool ROW_SCALES = !BLOCKS && (KIND == KIND_I8 || KIND == KIND_F8);
      float sb = 1.0f;
      if constexpr (ROW_SCALES) {
        if (ch + lane < g.n) sb = g.b_scales[t.group * g.bs_group + (ch + lane) * g.bs_n];
        __syncwarp();  // (all lanes are done with the last tile's)
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) {
          const int r = (2 * c + half) * 32 + lane;
          row_scales[c * 32 + lane] =
              r < t.rows ? g.a_scales[(int64_t(t.row0) + r) * g.as_row] : 0.0f;
        }
        __syncwarp();
      }
      const int channels = g.n - ch;  // from this warp's first on
      uint8_t* out = static_cast<uint8_t*>(g.out) +
                     (t.row0 * g.out_row + ch) * (g.out_dtype == DT_F32 ? 4 : 2);
      const int64_t out_step = 8 * g.out_row * (g.out_dtype == DT_F32 ? 4 : 2);
      if constexpr (ADD == GROUPED_ADD_NONE) ok = wait_acc();
      if (!ok) break;

      if constexpr (C::ROWS_M) {
        const int row0 = static_cast<int>(rank) * 128 + quarter * 32;
        const int rows = t.rows - row0, ch0 = t.ch0 + half * 128;
        const int64_t first = int64_t(t.row0) + row0;
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) {
          uint32_t w[16];
          if (g.out_dtype == DT_F32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = acc[c][i];
            store_rows32(g, w, stage_out, first, rows, ch0 + 32 * c, lane);
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = acc[c][16 + i];
            store_rows32(g, w, stage_out, first, rows, ch0 + 32 * c + 16, lane);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 two = make_float2(__uint_as_float(acc[c][2 * i]),
                                             __uint_as_float(acc[c][2 * i + 1]));
              if (g.out_dtype == DT_F16) {
                const __half2 h = __float22half2_rn(two);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
              } else {
                w[i] = f2_bf16x2(two);
              }
            }
            store_rows32(g, w, stage_out, first, rows, ch0 + 32 * c, lane);
          }
        }
        continue;
      }
      // Rows 8 i .. 8 i + 7 of chunk c, whose sums r holds.
      auto finish = [&](const uint32_t (&r)[32], int c, int i) {
        const int eight = (2 * c + half) * 4 + i;
        if (8 * eight >= t.rows) return;
        float2 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = make_float2(sum_value<KIND>(r[8 * i + 2 * j]),
                             sum_value<KIND>(r[8 * i + 2 * j + 1]));
        if constexpr (ROW_SCALES) {
          const float4* sa = reinterpret_cast<const float4*>(row_scales + c * 32 + 8 * i);
          const float4 lo = sa[0], hi = sa[1];
          const float2 by = make_float2(sb, sb);
          v[0] = __fmul2_rn(__fmul2_rn(v[0], make_float2(lo.x, lo.y)), by);
          v[1] = __fmul2_rn(__fmul2_rn(v[1], make_float2(lo.z, lo.w)), by);
          v[2] = __fmul2_rn(__fmul2_rn(v[2], make_float2(hi.x, hi.y)), by);
          v[3] = __fmul2_rn(__fmul2_rn(v[3], make_float2(hi.z, hi.w)), by);
        }
        store_rows8(g, v, stage_out + out_buf * 512, out + eight * out_step, t.rows - 8 * eight,
                    channels, lane);
        out_buf ^= 1;
      };
      if (exchange) {
        if constexpr (!PAIR) {
          cluster_wait();  // (one tile a cluster: once)
          if constexpr (ADD == GROUPED_ADD_NONE) {
            if (has_chunk(t, 0)) load_chunk(0, acc[0]);
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
              st_cluster_v4(to, acc[0][8 * i], acc[0][8 * i + 1], acc[0][8 * i + 2],
                            acc[0][8 * i + 3]);
              st_cluster_v4(to + 512, acc[0][8 * i + 4], acc[0][8 * i + 5], acc[0][8 * i + 6],
                            acc[0][8 * i + 7]);
            }
          }
          // One fence for all: a release each would be four of them in a row.
          __syncwarp();
          fence_cluster();
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t owner = static_cast<uint32_t>((half * 4 + i) % splits);
            if (lane == 0) mbar_arrive_fenced(map_to_rank(parts, owner));
          }
          __syncwarp();
          cluster_arrive();
          exchanged = true;
          ok = whole_warp(
              mbar_wait_cluster(parts, 0, abort_flag, g.status, DEV_TIMEOUT_FIXUP));
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
                  uint32_t& a = acc[0][8 * i + 4 * p + q];
                  a = s == 0 ? u[q] : sum_add<KIND>(a, u[q]);
                }
              }
            }
            finish(acc[0], 0, i);
          }
        }
      } else {
        if constexpr (ADD != GROUPED_ADD_NONE) {
#pragma unroll
          for (int c = 0; c < C::CHUNKS; ++c) {
            if (!has_chunk(t, c)) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) finish(acc[c], c, i);
          }
        } else {
#pragma unroll
          for (int c = 0; c < C::CHUNKS; ++c) {
            if (!has_chunk(t, c)) break;
            uint32_t r[32];
            load_chunk(c, r);
            if (!(c + 1 < C::CHUNKS && has_chunk(t, c + 1))) release_acc();
#pragma unroll
            for (int i = 0; i < 4; ++i) finish(r, c, i);
          }
          if (!has_chunk(t, 0)) release_acc();  // no rows for this warp
        }
      }
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
  if constexpr (PAIR) cluster_sync();  // the peer no longer touches this CTA
  if (exchange) {  // no CTA of the cluster sends to this one any more
    __syncwarp();
    if (!exchanged) {
      cluster_wait();
      cluster_arrive();
    }
    cluster_wait();
  }
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, 512);
    else
      tmem_dealloc(tmem_base, 512);
  }
}

template <int KIND, int ADD, bool PAIR>
cudaError_t launch(const GroupedMaps& maps, const GroupedArgs& g, int grid, cudaStream_t stream) {
  using C = Cfg<ADD, PAIR>;
  auto kern = grouped_gemm_kernel<KIND, ADD, PAIR>;
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
  // (programmatic launch, see grid_dependency_wait)
  attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
  ++n_attr;
  cfg.attrs = attr;
  cfg.numAttrs = n_attr;
  return cudaLaunchKernelEx(&cfg, kern, maps, g);
}

template <int KIND, int ADD>
int split_clusters(int splits) {
  using C = Cfg<ADD, false>;
  auto kern = grouped_gemm_kernel<KIND, ADD, false>;
  static std::atomic<int> known[kMaxLaunchDevices][4];  // + 1; of 1, 2, 4, 8
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxLaunchDevices) return 0;
  std::atomic<int>& slot = known[dev][splits == 8 ? 3 : splits == 4 ? 2 : splits == 2 ? 1 : 0];
  if (int n = slot.load(std::memory_order_relaxed)) return n - 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(splits), 1, 1);
  cfg.blockDim = dim3(C::THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES) !=
          cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();  // (dealt with: K is not split)
    n = 0;
  }
  slot.store(n + 1, std::memory_order_relaxed);
  return n;
}

}  // namespace

// The kinds with their ways to add; `what` is called with both as constants.
template <class What>
auto with_kind(int kind, int add, What what) {
  constexpr std::integral_constant<int, GROUPED_ADD_NONE> none{};
  constexpr std::integral_constant<int, GROUPED_ADD_SCALED> scaled{};
  constexpr std::integral_constant<int, GROUPED_ADD_PARTS> parts{};
  switch (kind) {
    case KIND_I8: return what(std::integral_constant<int, KIND_I8>{}, none);
    case KIND_F8:
      if (add == GROUPED_ADD_SCALED) return what(std::integral_constant<int, KIND_F8>{}, scaled);
      return add == GROUPED_ADD_PARTS ? what(std::integral_constant<int, KIND_F8>{}, parts)
                                      : what(std::integral_constant<int, KIND_F8>{}, none);
    case KIND_BF16:
      return add == GROUPED_ADD_PARTS ? what(std::integral_constant<int, KIND_BF16>{}, parts)
                                      : what(std::integral_constant<int, KIND_BF16>{}, none);
    default:
      return add == GROUPED_ADD_PARTS ? what(std::integral_constant<int, KIND_F16>{}, parts)
                                      : what(std::integral_constant<int, KIND_F16>{}, none);
  }
}

int grouped_split_clusters(int kind, int add, int splits) {
  return with_kind(kind, add, [&](auto k, auto a) {
    return split_clusters<decltype(k)::value, decltype(a)::value>(splits);
  });
}

cudaError_t launch_grouped_gemm(const GroupedMaps& maps, const GroupedArgs& g, int kind, int add,
                                bool pair, int grid, cudaStream_t stream) {
  return with_kind(kind, add, [&](auto k, auto a) {
    return pair ? launch<decltype(k)::value, decltype(a)::value, true>(maps, g, grid, stream)
                : launch<decltype(k)::value, decltype(a)::value, false>(maps, g, grid, stream);
  });
}

}  // namespace m5b
