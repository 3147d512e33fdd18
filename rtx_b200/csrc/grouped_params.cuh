// What the host side of the row quantizer passes to it (grouped.cuh); used by the grouped linear (grouped.cu) and by the
// linear with an epilogue (api.cu).
#pragma once

#include "common.cuh"

namespace rtxb {

struct GroupList {
  const int* offsets;   // [groups + 1]
  int groups;
  int rows;             // rows of the operand; offsets are held inside [0, rows] and non-decreasing
};

// What the quantizer leaves for the GEMM behind it (global memory, written by block 0).
struct GroupPlan {
  int* row_tiles;    // [0] = number of row tiles over all groups
  int4* tiles;       // per row tile: {first row, live rows, first 128-row scale tile, group | (32-row offset in it) << 16}
  int* k_tiles;      // [groups + 1] = GroupScan::tile
  int tile_rows;     // 64, 128 or 256
};

struct RowsOperand {
  const __nv_bfloat16* src;   // nullptr = absent
  int64_t ld;
  uint8_t* q;                 // [.., kp], 32-byte aligned
  uint8_t* scales;            // 128-row tiles
  int rows;                   // per matrix (x: all groups)
  int align;                  // of src and its pitch: 2 = 32 bytes, 1 = 16 bytes, 0 = neither
  const __nv_bfloat16* end;   // behind the last value of all matrices
};
struct RowsParams {
  RowsOperand x, w;
  GroupList list;             // offsets nullptr: x is one group of all its rows, no plan, no rows to zero
  int batches;                // matrices of w
  int k, kp, chunks;          // chunks = 512-byte scale tiles per 128 rows
  int lanes;                  // lanes that share a row: 4, 8, 16 or 32; then 32 / lanes rows share a warp
  int stacked;
  int segs;                   // units side by side along a row
  int per_tile;               // units of one 128-row tile
  int w_row_tiles;            // 128-row tiles of one matrix of w
  int round_to_infinity;
  GroupPlan plan;
  __nv_bfloat16* out;         // result whose rows of no group become zero
  int out_cols;
  int64_t ldo;
  int* status;
};
// fills in the fields that follow from k and enqueues the quantizer; x_tiles: the most 128-row tiles x can have
int launch_quantize_rows(RowsParams& p, int64_t x_tiles, int64_t k, int rounding, cudaStream_t stream);   // grouped.cu

// Operand of the transposed quantizer: matrices [rows, cols] quantized in blocks of 32 along their rows, the payload
// [cols, pitch] K-major per matrix.
struct TransposedOperand {
  const __nv_bfloat16* src;   // nullptr = absent
  int64_t ld;
  int rows, cols;             // per matrix (x: all groups)
  uint8_t* q;                 // per matrix [cols, pitch], 32-byte aligned
  int64_t pitch;              // bytes; also where the payload ends
  uint8_t* scales;            // per matrix [ceil(cols / 128)][chunks][512]
  int chunks;
};
struct TransposedParams {
  TransposedOperand x, w;
  GroupList list;             // with the gradient only; else x is one group of all its rows
  int batches;                // matrices of w
  int x_col_units, w_col_units, w_row_tiles;
  const float* partial;       // column sums [row_tiles][n] left by the launch before this one; nullptr = none
  int row_tiles, n;
  __nv_bfloat16* dbias;       // their sum over the row tiles
  // with the gradient, whose groups are those of x: q null = no columns (dW), dy_rows null = no rows (dX)
  TransposedOperand dy;
  int dy_col_units;
  uint8_t* dy_rows;           // [rows, round_up(cols, 32)]
  uint8_t* dy_row_scales;     // 128-row tiles counted per group
  GroupPlan plan;
  __nv_bfloat16* dx;          // result whose rows of no group become zero; nullptr = none
  int dx_cols;
  int* status;
};
// enqueues the transposed quantizer as a programmatic dependent that may run beside the launch before it (none of whose
// results it reads but `partial`) and ends after that launch has, or, with a gradient, as the first launch of its chain;
// x_tiles: the most 128-row tiles x can have
int launch_quantize_transposed(TransposedParams& p, int64_t x_tiles, cudaStream_t stream);   // grouped.cu

}  // namespace rtxb
