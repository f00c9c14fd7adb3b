// Matrix products grouped by expert and block-scaled E4M3 products: what
// grouped_api.cu and grouped_gemm.cu share.
#pragma once
#include "common.cuh"
#include "m5b_internal.h"

namespace m5b {

constexpr int kMaxGroups = 1024;  // the table of the groups' rows and tiles is in shared memory

struct GroupedArgs {
  int rows;                    // of the activations and the output
  int groups;                  // experts
  int n;                       // output channels
  int num_k_blocks;            // of 128 bytes of a row
  int tile_rows;               // most rows of a tile
  int k_splits;                // CTAs (a cluster) that share a tile's K range; 1: none
  const int32_t* group_start;  // [groups + 1], NULL: all rows are group 0's
  // Scales of the quantized kinds.  Rows and channels: a_scales[row * as_row],
  // b_scales[group * bs_group + channel * bs_n].  Blocks of 128 channels of K:
  // a_scales[row * as_row + kb * as_k], b_scales[group * bs_group +
  // (channel / 128) * bs_n + kb * bs_k].
  const float* a_scales;
  const float* b_scales;
  int64_t as_row, as_k, bs_group, bs_n, bs_k;
  void* out;
  int64_t out_row;             // elements between the output's rows
  int out_dtype;               // DT_BF16 / DT_F16 / DT_F32
  int out_vec;                 // the output's rows are whole aligned 16-byte pieces
  int zero_rest;               // rows outside every group are set to zero
  unsigned int* status;
};

// Activations [rows, K] in boxes of 128, 64 and 16 rows, weights
// [groups, N, K] in boxes of 128; all boxes 128 bytes wide, 128-byte swizzle.
struct GroupedMaps {
  CUtensorMap a128, a64, a16, b;
};

// Rows of the widest tile: 256 on CTA pairs (256 channels), 64 on one CTA (128 channels).
constexpr int kPairTileRows = 256;
constexpr int kSingleTileRows = 64;

// What is added in fp32 registers, not in the accumulator: nothing; blocks of 128
// channels of K, each by its scale (E4M3); parts of four blocks of 128 bytes (fp32
// results of other operands than INT8).  The tensor cores truncate their sums: without
// parts fp16 operands were off by 4.9e-6 (relative 2-norm) at K 16384 and 1.3e-6 at
// 4096, E4M3 ones by 1.2e-6 at 16384; with them fp16 by 3.5e-7 at any.  16-bit results
// do not show it, and INT32 sums are exact.
enum GroupedAdd : int { GROUPED_ADD_NONE = 0, GROUPED_ADD_SCALED = 1, GROUPED_ADD_PARTS = 2 };

cudaError_t launch_grouped_gemm(const GroupedMaps& maps, const GroupedArgs& g, int kind, int add,
                                bool pair, int grid, cudaStream_t stream);

// Clusters of `splits` single CTAs that the current device runs at a time; 0 on failure.
int grouped_split_clusters(int kind, int add, int splits);

struct BlockQuantArgs {
  const void* x;
  const void* gate;      // NULL, or values silu(gate) * x
  const int32_t* index;  // NULL, or output row r is x[index[r]]
  int64_t x_row, gate_row, x_batch;
  int64_t rows;          // of the output (each batch)
  int64_t x_rows;        // of x
  int64_t k;
  int64_t batch;
  uint8_t* q;            // [batch, rows, k]
  float* scales;         // [batch, rows or row blocks, ceil(k / 128)]
  int vec;               // rows on the 16-byte grid, k a multiple of 16
  int sms;
};

cudaError_t launch_block_quantize(const BlockQuantArgs& a, int dtype, bool square,
                                  cudaStream_t stream);

}  // namespace m5b
