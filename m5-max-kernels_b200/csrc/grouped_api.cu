// C-ABI entry points of the block-scaled and grouped products (declared in
// include/m5b200.h): contract checks, tile and schedule choice, launches.
// Nothing here allocates or synchronizes, and nothing throws.
#include <climits>
#include <cstdio>

#include "grouped.cuh"
#include "m5b200.h"

using namespace m5b;

namespace {

int einval(const char* msg) { return set_last_error(M5B_EINVAL, msg); }
int eunsupported(const char* msg) { return set_last_error(M5B_EUNSUPPORTED, msg); }

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return set_last_error(M5B_OK, "");
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return set_last_error(M5B_ECUDA, msg);
}

bool float_dtype(int64_t dt) { return dt == M5B_F32 || dt == M5B_F16 || dt == M5B_BF16; }
int64_t dtype_bytes(int64_t dt) { return dt == M5B_F32 ? 4 : 2; }
bool grid16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Strides of a tensor map are below 2^40 bytes.
bool map_stride(int64_t bytes) {
  return bytes > 0 && bytes < (int64_t(1) << 40) && bytes % 16 == 0;
}

struct Plan {
  bool pair;
  int tile_rows, splits, grid;
};

// Tiles and schedule.  Single CTAs take 128 channels x 64 rows, several of them
// (a cluster) sharing the K range where the tiles do not fill the GPU; CTA pairs
// take 256 channels x 256 rows.  Taken is what needs less time for its waves, a
// block of 128 bytes of K costing 0.32 us on a single CTA and 0.40 us on a pair,
// and leaving a pair's tile 0.5 us (0.56 and 2.5 where each block is scaled): fitted
// to, in us for single CTAs and pairs, block-scaled 65, 200 and 517 rows x 4096 x
// 16384 25 / 72, 38 / 73, 80 / 74; 64 experts of 2048 -> 4096, 64, 96, 128 and 192
// rows each 111 / 161, 145 / 165, 182 / 172, 246 / 191, with bf16 64 and 96 rows
// 181 / 175, 213 / 183.  (Block-scaled pairs take about 5 % less since their waits vote:
// 70 at 517 rows.)  One price for all other kinds: fp32 results that add parts take pairs
// a quarter longer, 192 us against 154 for 9914 x 5376 x 4096 in E4M3.  Of several groups'
// sizes only the sum is known here: each is taken to end in the middle of a tile, and to
// have one at least.
Plan plan_for(int64_t rows, int64_t groups, int64_t n, int64_t nkb, int kind, int add, int sms) {
  const int64_t busy = groups < rows ? groups : rows;  // groups with rows, at most
  auto waves = [&](int64_t tile_rows, int64_t ch, int64_t units, int64_t splits, double block,
                   double leave) {
    const int64_t ch_tiles = ceil_div(n, ch);
    int64_t tiles = ceil_div(rows, tile_rows);
    if (groups > 1) {
      tiles = ceil_div(2 * rows + tile_rows * busy, 2 * tile_rows);
      if (tiles < busy) tiles = busy;
    }
    return ceil_div(tiles * ch_tiles * splits, units) * (ceil_div(nkb, splits) * block + leave);
  };
  // (every group rounds its last tile up: no more tiles than these)
  const auto most_tiles = [&](int64_t tile_rows, int64_t ch) {
    return (groups == 1 ? ceil_div(rows, tile_rows) : rows / tile_rows + busy) * ceil_div(n, ch);
  };
  Plan p{};
  // a cluster has one tile, and all of them run at once
  int64_t tiles = most_tiles(kSingleTileRows, 128);
  p.splits = 1;
  while (p.splits < 8 && tiles * p.splits * 2 <= sms && nkb >= p.splits * 2 * 4 &&
         tiles <= grouped_split_clusters(kind, add, p.splits * 2))
    p.splits *= 2;
  const double single = waves(kSingleTileRows, 128, sms, p.splits, 0.32, 0.0);
  const bool scaled = add == GROUPED_ADD_SCALED;
  const double pair =
      waves(kPairTileRows, 256, sms / 2, 1, scaled ? 0.56 : 0.40, scaled ? 2.5 : 0.5);
  p.pair = pair < single;
  if (p.pair) {
    tiles = most_tiles(kPairTileRows, 256);
    p.splits = 1;
  }
  p.tile_rows = p.pair ? kPairTileRows : kSingleTileRows;
  const int64_t units = p.pair ? sms / 2 : sms;
  const int64_t used = tiles < units ? tiles : units;
  p.grid = static_cast<int>(used) * (p.pair ? 2 : p.splits);
  return p;
}

// What a call's sizes and types say; M5B_OK, or the error.
struct Product {
  int kind, add;
  int64_t elem, num_k_blocks;
  bool quantized;
};
int check_product(const m5b_grouped_gemm_args* s, Product* p) {
  if (!s) return einval("arguments are NULL");
  int kind = 0;
  int64_t elem = 1;
  bool quantized = true;
  switch (s->mode) {
    case M5B_MODE_INT8: kind = KIND_I8; break;
    case M5B_MODE_FP8: kind = KIND_F8; break;
    case M5B_MODE_BF16: kind = KIND_BF16, elem = 2, quantized = false; break;
    case M5B_MODE_FP16: kind = KIND_F16, elem = 2, quantized = false; break;
    case M5B_MODE_FP32: return eunsupported("fp32 operands are not supported by the grouped GEMM");
    default: return einval("unknown GEMM mode");
  }
  if (s->rows < 0 || s->groups < 1 || s->n < 1 || s->k < 1)
    return einval("rows, groups, n and k must be positive");
  if (s->block_scales && s->mode != M5B_MODE_FP8) return einval("block scales need FP8 operands");
  if (!float_dtype(s->out_dtype))
    return eunsupported("output dtype must be bfloat16, float16 or float32");
  if (s->groups > kMaxGroups) return eunsupported("more than 1024 groups are unsupported");
  if (kind == KIND_I8 && s->k > 133144)
    return eunsupported("INT32 worst-case overflow bound exceeded");
  // (rows and channels are rounded up to whole tiles, and tiles counted in 32 bits)
  const int64_t most = INT_MAX - 4096;
  if (s->rows > most || s->n > most || s->k > most ||
      (s->rows / 64 + s->groups) * ceil_div(s->n, 128) > most)
    return eunsupported("rows x channels exceed the index range");
  p->kind = kind;
  p->elem = elem;
  p->quantized = quantized;
  p->num_k_blocks = ceil_div(s->k * elem, 128);
  p->add = s->block_scales                                 ? GROUPED_ADD_SCALED
           : kind != KIND_I8 && s->out_dtype == M5B_F32 ? GROUPED_ADD_PARTS
                                                        : GROUPED_ADD_NONE;
  return M5B_OK;
}

}  // namespace

extern "C" {

int m5b_block_quantize(const m5b_block_quantize_args* s, void* stream) {
  if (!s) return einval("arguments are NULL");
  if (!float_dtype(s->x_dtype)) return einval("input dtype must be float16, bfloat16 or float32");
  if (s->block_rows != 1 && s->block_rows != 128) return einval("block_rows must be 1 or 128");
  if (s->rows < 0 || s->k < 1 || s->batch < 1 || s->x_rows < 0)
    return einval("rows, k and batch must be positive");
  if (s->block_rows == 1 && s->batch != 1) return einval("a batch needs block_rows 128");
  if (s->block_rows != 1 && (s->gate || s->row_index))
    return einval("gate and row_index need block_rows 1");
  if (!s->row_index && s->rows != s->x_rows) return einval("rows must be x's without row_index");
  // (rows of blocks are counted in 32 bits, and rounded up to whole CTAs)
  const int64_t most = INT_MAX - (1 << 20);
  if (s->rows > most || s->x_rows > most || s->k > most || s->batch > most ||
      ceil_div(s->rows, s->block_rows) * ceil_div(s->k, 128) > most / s->batch)
    return eunsupported("rows x k exceed the index range");
  if (s->rows == 0) return set_last_error(M5B_OK, "");
  if (!s->q || !s->scales || (!s->x && s->x_rows > 0)) return einval("x, q and scales are required");
  BlockQuantArgs a{};
  a.x = s->x;
  a.gate = s->gate;
  a.index = s->row_index;
  a.x_row = s->x_row_stride;
  a.gate_row = s->gate_row_stride;
  a.x_batch = s->x_batch_stride;
  a.rows = s->rows;
  a.x_rows = s->x_rows;
  a.k = s->k;
  a.batch = s->batch;
  a.q = s->q;
  a.scales = s->scales;
  const int64_t size = dtype_bytes(s->x_dtype);
  a.vec = s->k % 16 == 0 && grid16(s->x) && grid16(s->gate) && (s->x_row_stride * size) % 16 == 0 &&
          (s->gate_row_stride * size) % 16 == 0 && (s->x_batch_stride * size) % 16 == 0 &&
          grid16(s->q);
  int rc = current_device_state(nullptr, &a.sms);
  if (rc) return rc;
  return launched(launch_block_quantize(a, static_cast<int>(s->x_dtype), s->block_rows == 128,
                                        static_cast<cudaStream_t>(stream)),
                  "block quantize launch");
}

int m5b_grouped_gemm(const m5b_grouped_gemm_args* s, void* stream) {
  Product product{};
  int rc = check_product(s, &product);
  if (rc) return rc;
  if (!s->group_start && s->groups != 1) return einval("group_start is required");
  const int kind = product.kind, add = product.add;
  const int64_t elem = product.elem;
  if (s->rows == 0) return set_last_error(M5B_OK, "");
  if (!s->a || !s->b || !s->out) return einval("a, b and out are required");
  if (product.quantized && (!s->a_scales || !s->b_scales)) return einval("scales required");
  // (every element is stored by a thread of its own)
  if (s->rows > 1 && s->out_row_stride < s->n && s->out_row_stride > -s->n)
    return einval("out's rows must not overlap");
  const int64_t row_bytes = ceil_div(s->k * elem, 16) * 16;
  const int64_t a_row = s->rows > 1 ? s->a_row_stride * elem : row_bytes;
  const int64_t b_row = s->n > 1 ? s->b_row_stride * elem : row_bytes;
  const int64_t b_group = s->groups > 1 ? s->b_group_stride * elem : row_bytes;
  if (!grid16(s->a) || !grid16(s->b) || !map_stride(a_row) || !map_stride(b_row) ||
      !map_stride(b_group))
    return eunsupported("operand rows must start on 16-byte boundaries for TMA");

  GroupedArgs g{};
  g.rows = static_cast<int>(s->rows);
  g.groups = static_cast<int>(s->groups);
  g.n = static_cast<int>(s->n);
  g.num_k_blocks = static_cast<int>(product.num_k_blocks);
  g.group_start = s->group_start;
  g.a_scales = s->a_scales;
  g.b_scales = s->b_scales;
  g.as_row = s->a_scale_row_stride;
  g.as_k = s->a_scale_block_stride;
  g.bs_group = s->b_scale_group_stride;
  g.bs_n = s->b_scale_row_stride;
  g.bs_k = s->b_scale_block_stride;
  g.out = s->out;
  g.out_row = s->out_row_stride;
  g.out_dtype = static_cast<int>(s->out_dtype);
  const int64_t piece = 16 / dtype_bytes(s->out_dtype);
  g.out_vec = s->n % piece == 0 && s->out_row_stride % piece == 0 && grid16(s->out);
  g.zero_rest = s->zero_rest ? 1 : 0;
  int sms = 0;
  rc = current_device_state(&g.status, &sms);
  if (rc) return rc;
  const Plan p = plan_for(s->rows, s->groups, s->n, g.num_k_blocks, kind, add, sms);
  g.tile_rows = p.tile_rows;
  g.k_splits = p.splits;

  GroupedMaps m{};
  const uint64_t a_dims[2] = {uint64_t(s->k), uint64_t(s->rows)};
  const uint64_t a_strides[1] = {uint64_t(a_row)};
  const uint64_t b_dims[3] = {uint64_t(s->k), uint64_t(s->n), uint64_t(s->groups)};
  const uint64_t b_strides[2] = {uint64_t(b_row), uint64_t(b_group)};
  const uint32_t wide = static_cast<uint32_t>(128 / elem);
  const uint32_t box128[3] = {wide, 128, 1}, box64[2] = {wide, 64}, box16[2] = {wide, 16};
  const int bytes = static_cast<int>(elem);
  // (only those that the tiles use)
  const auto rows_map = [&](CUtensorMap* map, const uint32_t* box) {
    return make_swizzled_map(map, bytes, 2, s->a, a_dims, a_strides, box);
  };
  const bool rows_m = p.pair && add == GROUPED_ADD_SCALED;
  if (!make_swizzled_map(&m.b, bytes, 3, s->b, b_dims, b_strides, box128) ||
      (p.pair && !rows_map(&m.a128, box128)) || (!rows_m && !rows_map(&m.a64, box64)) ||
      (!p.pair && !rows_map(&m.a16, box16)))
    return set_last_error(M5B_ECUDA, "cuTensorMapEncodeTiled failed");
  return launched(launch_grouped_gemm(m, g, kind, add, p.pair, p.grid,
                                      static_cast<cudaStream_t>(stream)),
                  "grouped GEMM launch");
}

int m5b_grouped_gemm_plan(const m5b_grouped_gemm_args* s, int64_t* plan) {
  Product product{};
  int rc = check_product(s, &product);
  if (rc) return rc;
  if (!plan) return einval("plan is NULL");
  if (s->rows == 0) return einval("rows must be positive");
  int sms = 0;
  rc = current_device_state(nullptr, &sms);
  if (rc) return rc;
  const Plan p = plan_for(s->rows, s->groups, s->n, product.num_k_blocks, product.kind,
                          product.add, sms);
  plan[0] = p.pair ? 2 : 1;
  plan[1] = p.tile_rows;
  plan[2] = p.splits;
  plan[3] = p.grid;
  return set_last_error(M5B_OK, "");
}

}  // extern "C"
