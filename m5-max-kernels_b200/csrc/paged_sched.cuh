// Work distribution of the tiled attention kernels (paged_decode.cu,
// paged_prompt.cu), and the joining of what it splits.
//
// A tile is up to ROWS packed rows of one kv head of one sequence (row r is
// new token r / G and query head kv * G + r % G, so that a group shares the
// keys) against the key blocks (BK keys each) that any of its rows sees.  All
// tiles' blocks, in the order sequence, head, row tile, block, form one line;
// every CTA takes an equal stretch of it, found from the lengths on the
// device.  Whole tiles leave finished.  Of a tile that crosses a CTA's border
// each part goes to the workspace: unnormalized fp32 sums with the row
// maximum they refer to.  A CTA has at most two such parts, one that continues
// an earlier CTA's tile (slot 2 c) and one that a later CTA continues (slot
// 2 c + 1), so the workspace does not grow with the batch; and the parts of a
// tile are added in the order of the line, whichever is finished first.
#pragma once

#include "paged.cuh"

namespace m5b {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The reference m of a row's probabilities 2^(t - m) follows the row's maximum
// when that has grown by more than 2^kGrow, so that sums are rarely rescaled.
// For fp16 it stays 2^7 below the maximum, which uses the type's range: they
// reach 2^15, and those of the many faint keys of a long cache keep their bits
// down to 2^-21 of the largest (and vanish below 2^-32, not 2^-25).
constexpr float kGrow = 8.0f;
template <typename T> constexpr float kBelow = DTypeOf<T>::value == DT_F16 ? 7.0f : 0.0f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh(y) / y for a pair of y^2 in [0, 1]: the minimax fit of the relative
// error (Remez exchange), 6e-7.
__device__ __forceinline__ float2 tanh_ratio(float2 z) {
  float2 p = make_float2(-0x1.920178p-9f, -0x1.920178p-9f);
  p = __ffma2_rn(p, z, make_float2(0x1.1251b6p-6f, 0x1.1251b6p-6f));
  p = __ffma2_rn(p, z, make_float2(-0x1.a6c0f2p-5f, -0x1.a6c0f2p-5f));
  p = __ffma2_rn(p, z, make_float2(0x1.1000f6p-3f, 0x1.1000f6p-3f));
  p = __ffma2_rn(p, z, make_float2(-0x1.554a16p-2f, -0x1.554a16p-2f));
  return __ffma2_rn(p, z, make_float2(0x1.ffffecp-1f, 0x1.ffffecp-1f));
}

struct PagedSeq {
  int row0;    // first row of the batch
  int n;       // new tokens
  int pos0;    // position of the first
  int keys;    // keys that pages can hold
  int prefix;  // keys that every row sees
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnArgs& a, int seq) {
  const int2 rows = paged_rows(a.b, seq);
  const int len = paged_len(a.b, seq);
  PagedSeq s;
  s.row0 = rows.x;
  s.n = rows.y - rows.x;
  s.pos0 = len - s.n;
  s.keys = min(len, a.b.capacity);
  s.prefix = a.prefix_lens ? max(0, min(a.prefix_lens[seq], s.keys)) : 0;
  return s;
}

// Key blocks of a row tile: [0, pre) and [from, from + blocks - pre).  A tile
// whose rows see nothing has one block all the same, hidden entirely.
struct PagedBlocks {
  int pre, from, blocks;
  __device__ __forceinline__ int at(int i) const { return i < pre ? i : from + (i - pre); }
};

template <int ROWS, int BK>
__device__ __forceinline__ PagedBlocks paged_blocks(const PagedAttnArgs& a, const PagedSeq& s,
                                                    int rt) {
  const int g = a.b.group;
  const int lo = s.pos0 + (rt * ROWS) / g;
  const int hi = s.pos0 + min(rt * ROWS + ROWS - 1, s.n * g - 1) / g;
  const int last = min(hi, s.keys - 1);
  PagedBlocks r;
  r.pre = s.prefix / BK + (s.prefix % BK != 0);
  r.from = max(r.pre, lo >= a.window ? (lo - a.window + 1) / BK : 0);
  r.blocks = max(1, r.pre + (last >= 0 ? max(0, last / BK + 1 - r.from) : 0));
  return r;
}

// The first key that a tile's rows see through their windows.  Pages between
// the prefix and there may be somebody else's by now and hold NaN, which a zero
// probability would not stop: their boxes are not loaded but filled with zeros.
// (Blanking such slots one by one in shared memory, as behind the end, took 174
// us instead of 163 for capped prompts with a window of 1024.)
template <int ROWS>
__device__ __forceinline__ int paged_window(const PagedAttnArgs& a, const PagedSeq& s, int rt) {
  const int pos = s.pos0 + rt * ROWS / a.b.group;
  return pos >= a.window ? pos - a.window + 1 : 0;
}

__device__ __forceinline__ int paged_tiles(const PagedAttnArgs& a, int n, int rows) {
  return (n * a.b.group + rows - 1) / rows;
}

// Blocks of one kv head of a sequence; all lanes of the warp pass their own.
template <int ROWS, int BK>
__device__ __forceinline__ long long paged_seq_blocks(const PagedAttnArgs& a, const PagedSeq& s) {
  constexpr int kAlone = 4;  // longer sums are shared by the warp's lanes
  const int tiles = paged_tiles(a, s.n, ROWS);
  long long sum = 0;
  if (tiles <= kAlone)
    for (int t = 0; t < tiles; ++t) sum += paged_blocks<ROWS, BK>(a, s, t).blocks;
  const int lane = threadIdx.x % 32;
  for (uint32_t left = __ballot_sync(~0u, tiles > kAlone); left; left &= left - 1) {
    const int src = __ffs(left) - 1;
    PagedSeq o;
    o.n = __shfl_sync(~0u, s.n, src);
    o.pos0 = __shfl_sync(~0u, s.pos0, src);
    o.keys = __shfl_sync(~0u, s.keys, src);
    o.prefix = __shfl_sync(~0u, s.prefix, src);
    const int all = __shfl_sync(~0u, tiles, src);
    long long part = 0;
    for (int t = lane; t < all; t += 32) part += paged_blocks<ROWS, BK>(a, o, t).blocks;
    for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(~0u, part, d);
    if (lane == src) sum = part;
  }
  return sum;
}

// One stretch of a tile: blocks [begin, end) of its `r.blocks`.
struct PagedPiece {
  int seq, head, rt, begin, end;
  long long tile_at;  // place of the tile's first block in the line
  PagedSeq s;
  PagedBlocks r;
  __device__ __forceinline__ bool whole() const { return begin == 0 && end == r.blocks; }
};

// a / b, by the short division where that does (a long one is a call).
__device__ __forceinline__ long long paged_div(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// The stretch of this CTA, piece by piece.  Every thread that walks it sees
// the same pieces.
template <int ROWS, int BK>
struct PagedWalk {
  int seq, head, rt, tiles, blk;
  long long left, share, at;  // blocks left, of an equal stretch; the next block's place in the line
  PagedSeq s;

  __device__ __forceinline__ void enter(const PagedAttnArgs& a) {  // first tile of a sequence >= seq
    while (seq < a.b.batch) {
      s = paged_seq(a, seq);
      tiles = paged_tiles(a, s.n, ROWS);
      if (tiles > 0) return;
      ++seq;
    }
    left = 0;
  }

  __device__ __forceinline__ bool next(const PagedAttnArgs& a, PagedPiece& p) {
    if (left <= 0) return false;
    p.seq = seq;
    p.head = head;
    p.rt = rt;
    p.s = s;
    p.r = paged_blocks<ROWS, BK>(a, s, rt);
    p.begin = blk;
    p.end = static_cast<int>(min(static_cast<long long>(p.r.blocks), blk + left));
    left -= p.end - p.begin;
    p.tile_at = at - p.begin;
    at += p.end - p.begin;
    if (p.end == p.r.blocks) {
      blk = 0;
      if (++rt == tiles) {
        rt = 0;
        if (++head == a.b.kv_heads) {
          head = 0;
          ++seq;
          if (left > 0) enter(a);
        }
      }
    }
    return true;
  }
};

// Shared memory of paged_walk.
template <int THREADS> struct PagedWalkScratch {
  long long sums[THREADS / 32];
  long long rest;  // blocks of the head before the stretch
  int seq, head;
  PagedSeq s;
};

// Called by all threads of the CTA (THREADS of them, whole warps).  A thread
// sums the blocks of its sequences, and the one whose sequences hold the
// stretch's first block says where; the rest of the way every warp goes alone.
template <int ROWS, int BK, int THREADS>
__device__ __forceinline__ PagedWalk<ROWS, BK> paged_walk(const PagedAttnArgs& a,
                                                          PagedWalkScratch<THREADS>& scratch) {
  constexpr int kWarps = THREADS / 32;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per = (a.b.batch + THREADS - 1) / THREADS;
  const int b0 = threadIdx.x * per;
  long long mine = 0, one = 0;
  PagedSeq s{};
  for (int i = 0; i < per; ++i) {
    s = PagedSeq{};
    if (b0 + i < a.b.batch) s = paged_seq(a, b0 + i);
    one = paged_seq_blocks<ROWS, BK>(a, s);
    mine += one * a.b.kv_heads;
  }
  long long upto = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(~0u, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) scratch.sums[warp] = upto;
  __syncthreads();
  long long before = upto - mine, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scratch.sums[w];
    total += scratch.sums[w];
  }
  PagedWalk<ROWS, BK> walk;
  walk.share = paged_div(total + gridDim.x - 1, gridDim.x);
  const long long at = walk.share * blockIdx.x;
  walk.at = at;
  walk.left = max(0ll, min(walk.share, total - at));
  // (all lanes of the warp take part in the sums of more sequences than threads)
  const bool here = walk.left > 0 && before <= at && at < before + mine;
  if (__any_sync(~0u, here)) {
    long long base = before;
    bool found = false;
    for (int i = 0; i < per; ++i) {
      if (per > 1) {
        s = PagedSeq{};
        if (b0 + i < a.b.batch) s = paged_seq(a, b0 + i);
        one = paged_seq_blocks<ROWS, BK>(a, s);
      }
      const long long all = one * a.b.kv_heads;
      if (here && !found && at < base + all) {
        found = true;
        const long long head = paged_div(at - base, one);
        scratch.seq = b0 + i;
        scratch.head = static_cast<int>(head);
        scratch.rest = at - base - head * one;
        scratch.s = s;
      }
      base += all;
    }
  }
  __syncthreads();
  walk.seq = walk.head = walk.rt = walk.blk = walk.tiles = 0;
  if (walk.left > 0) {
    walk.seq = scratch.seq;
    walk.head = scratch.head;
    walk.s = scratch.s;
    long long rest = scratch.rest;
    walk.tiles = paged_tiles(a, walk.s.n, ROWS);
    if (walk.tiles == 1) {
      walk.blk = static_cast<int>(rest);
    } else {
      for (int base = 0; base < walk.tiles; base += 32) {  // 32 row tiles at a time
        const int t = base + lane;
        const int blocks = t < walk.tiles ? paged_blocks<ROWS, BK>(a, walk.s, t).blocks : 0;
        long long sum = blocks;
        for (int d = 1; d < 32; d <<= 1) {
          const long long o = __shfl_up_sync(~0u, sum, d);
          if (lane >= d) sum += o;
        }
        const uint32_t past = __ballot_sync(~0u, sum > rest);
        if (past) {
          const int src = __ffs(past) - 1;
          walk.rt = base + src;
          walk.blk = static_cast<int>(rest - __shfl_sync(~0u, sum - blocks, src));
          break;
        }
        rest -= __shfl_sync(~0u, sum, 31);
      }
    }
  }
  return walk;
}

// Workspace of a launch of `ctas` CTAs.
struct PagedSplit {  // the tile that CTA c leaves to later ones
  int parts;         // slots: 2 c + 1, then 2 (c + 1), 2 (c + 2), ...; 0: none
  int row0, first, rows, head;  // batch row, packed rows [first, first + rows), kv head
  int pad[3];
};
template <int ROWS, int D>
struct PagedPartials {
  PagedSplit* split;  // [ctas]
  float2* ml;         // [2 ctas][ROWS]: maximum (in log2 units) and sum
  float* o;           // [2 ctas][ROWS][D], or [2 ctas][D / 4][ROWS][4]
  __host__ __device__ PagedPartials(void* ws, int ctas) {
    split = static_cast<PagedSplit*>(ws);
    ml = reinterpret_cast<float2*>(split + (ctas + 7) / 8 * 8);
    o = reinterpret_cast<float*>(ml + int64_t(2) * ctas * ROWS);
  }
  static int64_t bytes(int ctas) {
    return (ctas + 7) / 8 * 8 * int64_t(sizeof(PagedSplit)) +
           int64_t(2) * ctas * ROWS * (sizeof(float2) + D * sizeof(float));
  }
};

// Written by one thread of every CTA, after its last piece (or without any).
__device__ __forceinline__ void paged_write_split(PagedSplit* at, const PagedPiece* last,
                                                  long long share, int rows_per_tile, int group) {
  PagedSplit m{};
  if (last && last->end < last->r.blocks && last->begin == 0) {
    m.parts = 1 + static_cast<int>(paged_div(last->r.blocks - last->end + share - 1, share));
    m.row0 = last->s.row0;
    m.first = last->rt * rows_per_tile;
    m.rows = min(rows_per_tile, last->s.n * group - m.first);
    m.head = last->head;
  }
  *at = m;
}

// Joins the `parts` of a tile that CTA c began, stored by rows: the calling
// warp takes rows row, row + STEP, ... (R of them) of the tile's packed rows
// from `first` on, the lanes across the channels, four parts at a time.  (Short
// code on purpose: a launch runs it once, from a cold instruction cache.)
template <typename T, int ROWS, int D, int R, int STEP>
__device__ __forceinline__ void paged_join_rows(const PagedAttnArgs& a, const PagedPartials<ROWS, D>& w,
                                                int c, int parts, int row, int row0, int head, int first) {
  constexpr int V = D / 32, U = 4;
  const int lane = threadIdx.x % 32;
  float top[R], sum[R], o[R][V] = {};
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = -INFINITY, sum[r] = 0.0f;
#pragma unroll 1
  for (int i = 0; i < parts; i += U) {
    float2 ml[R][U], x[R][U][V / 2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(i + u, parts - 1);
      const int64_t at = int64_t(k == 0 ? 2 * c + 1 : 2 * (c + k)) * ROWS + row;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ml[r][u] = __ldcg(&w.ml[at + r * STEP]);
        const float2* po = reinterpret_cast<const float2*>(w.o + (at + r * STEP) * D + lane * V);
#pragma unroll
        for (int v = 0; v < V / 2; ++v) x[r][u][v] = __ldcg(po + v);
        if (i + u >= parts) ml[r][u].x = -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float m2 = top[r];
#pragma unroll
      for (int u = 0; u < U; ++u) m2 = fmaxf(m2, ml[r][u].x);
      const float base = m2 == -INFINITY ? 0.0f : m2, keep = ex2(top[r] - base);
      top[r] = m2;
      sum[r] *= keep;
#pragma unroll
      for (int v = 0; v < V; ++v) o[r][v] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = ex2(ml[r][u].x - base);
        sum[r] = fmaf(ml[r][u].y, f, sum[r]);
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          o[r][2 * v] = fmaf(x[r][u][v].x, f, o[r][2 * v]);
          o[r][2 * v + 1] = fmaf(x[r][u][v].y, f, o[r][2 * v + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int packed = first + row + r * STEP, h = head * a.b.group + packed % a.b.group;
    const int64_t t = row0 + packed / a.b.group;
    const bool none = sum[r] == 0.0f;  // (NaN is something)
    const float inv = none ? 0.0f : 1.0f / sum[r];
    T* out = static_cast<T*>(a.out) + t * a.o_token + h * a.o_head + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = from_f32<T>(o[r][v] * inv);
    if (a.lse && lane == 0)
      a.lse[t * a.b.q_heads + h] = none ? -INFINITY : (top[r] + log2f(sum[r])) * kLn2;
  }
}

// Joins the parts, stored by columns, [D / 4][ROWS][4], of the tiles that were
// split: CTA (c, i) takes channels 16 i .. 16 i + 15 of the one that CTA c left
// to others, a thread a row.
template <typename T, int ROWS, int D>
__global__ void __launch_bounds__(ROWS) paged_join_columns_kernel(const PagedAttnArgs a, int ctas) {
  grid_dependency_wait();
  const PagedPartials<ROWS, D> w(a.workspace, ctas);
  const int c = blockIdx.x, row = threadIdx.x;
  const PagedSplit m = w.split[c];
  if (row >= m.rows || m.parts == 0) return;
  float top = -INFINITY, sum = 0.0f, o[16] = {};
  for (int i = 0; i < m.parts; ++i)
    top = fmaxf(top, w.ml[int64_t(i == 0 ? 2 * c + 1 : 2 * (c + i)) * ROWS + row].x);
#pragma unroll 2
  for (int i = 0; i < m.parts; ++i) {
    const int64_t slot = i == 0 ? 2 * c + 1 : 2 * (c + i);
    const float2 ml = w.ml[slot * ROWS + row];
    const float4* po = reinterpret_cast<const float4*>(w.o + slot * ROWS * D) + blockIdx.y * 4 * ROWS + row;
    const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - top);
    sum = fmaf(ml.y, f, sum);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 x = po[k * ROWS];
      o[4 * k] = fmaf(x.x, f, o[4 * k]);
      o[4 * k + 1] = fmaf(x.y, f, o[4 * k + 1]);
      o[4 * k + 2] = fmaf(x.z, f, o[4 * k + 2]);
      o[4 * k + 3] = fmaf(x.w, f, o[4 * k + 3]);
    }
  }
  const int packed = m.first + row, t = m.row0 + packed / a.b.group;
  const int h = m.head * a.b.group + packed % a.b.group;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  __align__(16) T y[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) y[k] = from_f32<T>(o[k] * inv);
  uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + t * a.o_token + h * a.o_head +
                                        blockIdx.y * 16);
  out[0] = *reinterpret_cast<const uint4*>(y);
  out[1] = *reinterpret_cast<const uint4*>(y + 8);
  if (a.lse && blockIdx.y == 0)
    a.lse[int64_t(t) * a.b.q_heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// Rows outside every sequence leave as zeros; `id` of `count` threads.
template <typename T, int D>
__device__ __forceinline__ void paged_zero_outside(const PagedAttnArgs& a, int64_t id, int64_t count) {
  const int lo = max(0, min(a.b.query_start[0], a.b.tokens));
  const int hi = max(lo, min(a.b.query_start[a.b.batch], a.b.tokens));
  const int64_t per = int64_t(a.b.q_heads) * (D / 8);
  const int64_t all = (int64_t(lo) + a.b.tokens - hi) * per;
  for (int64_t i = id; i < all; i += count) {
    int64_t t = i / per;
    if (t >= lo) t += hi - lo;
    const int h = static_cast<int>(i % per) / (D / 8), c = static_cast<int>(i % (D / 8));
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + t * a.o_token + h * a.o_head + c * 8) =
        make_uint4(0u, 0u, 0u, 0u);
    if (a.lse && c == 0) a.lse[t * a.b.q_heads + h] = -INFINITY;
  }
}

}  // namespace m5b
