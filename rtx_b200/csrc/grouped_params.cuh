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
  int* row_tiles;    // [0] = number of 256-row tiles over all groups
  int4* tiles;       // per 256-row tile: {first row, live rows, first scale tile, group}
  int* k_tiles;      // [groups + 1] = GroupScan::tile
};

struct RowsOperand {
  const __nv_bfloat16* src;   // nullptr = absent
  int64_t ld;
  uint8_t* q;                 // [.., kp], 32-byte aligned
  uint8_t* scales;            // 128-row tiles
  int rows;                   // per matrix (x: all groups)
  int align;                  // of src and its pitch: 2 = 32 bytes, 1 = 16 bytes, 0 = neither
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

}  // namespace rtxb
