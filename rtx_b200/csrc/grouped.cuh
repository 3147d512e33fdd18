// Operands split into groups of consecutive rows (the experts of a mixture): the list of groups, and the MXFP8
// quantizers that lay a grouped operand out for the grouped GEMM (gemm_grouped.cuh).
//
// Group g holds rows offsets[g] .. offsets[g + 1] - 1.  Two things have to start on a 128-row boundary for the
// block-scaled MMA: the 512-byte scale tiles (128 rows each) when the rows are an MMA operand's rows, and the K steps
// (128 bytes) when the rows are the contraction (dW).  The payload of a row operand needs no such boundary, because a
// TMA box may start at any row.  So
//   rows        payload stays in place, [rows, kp]; scale tiles are counted per group: tile[g] .. tile[g + 1] - 1;
//   transposed  payload and scales are [columns, 128 * tiles], group g at columns 128 * tile[g], zero behind its end:
//               one 128-byte K step is one 128-row tile, one 512-byte scale tile belongs to it.
// Rows of no group are never read; the kernels here set them to zero in the result.
#pragma once

#include "grouped_params.cuh"
#include "quant_tiles.cuh"

namespace rtxb {

constexpr int kMaxGroups = 512;   // the list is scanned in shared memory beside the staged tiles (4 KB at 512)

struct GroupScan {
  int start[kMaxGroups + 1];   // first row of the group; [groups] = end of the last one
  int tile[kMaxGroups + 1];    // 128-row tiles of the groups before it
  int warp_part[8];
};

__device__ __forceinline__ int block_scan_max(int v, int* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v = max(v, o);
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v = max(v, part[w]);
  __syncthreads();
  return v;   // inclusive
}
__device__ __forceinline__ int block_scan_sum(int v, int* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v += part[w];
  __syncthreads();
  return v;   // inclusive
}

__device__ __forceinline__ int warp_scan_sum(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;   // inclusive
}

// All kQuantThreads threads of a block: the list from memory into `s`.  Fewer than 32 groups take one warp and one barrier
// instead of the block-wide scans' six: a small batch's quantizer is little more than this (forward in a graph, without and
// with it: 16 rows, 8 groups of 1024 x 1024 9.7 and 8.8 us; 777 rows, 12 groups of 776 x 520 13.0 and 12.4).  Offsets outside [0, rows] or below an earlier
// one are brought back inside (and reported in the status word), so that no list makes a kernel leave its buffers.
__device__ __forceinline__ void scan_groups(const GroupList& l, GroupScan& s, int* status) {
  if (l.groups < 32) {
    if (threadIdx.x < 32) {
      const int g = threadIdx.x;
      const int raw = g <= l.groups ? l.offsets[g] : 0;
      int run = max(min(raw, l.rows), 0);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, run, d);
        if (g >= d) run = max(run, o);
      }
      const int next = __shfl_down_sync(0xffffffffu, run, 1);
      const int n = g < l.groups ? (next - run + 127) >> 7 : 0;
      const int incl = warp_scan_sum(n);
      if (g <= l.groups) {
        s.start[g] = run;
        s.tile[g] = incl - n;
        if (run != raw && status && blockIdx.x == 0) atomicCAS(status, 0, kStatusGroupOffsets);
      }
    }
    __syncthreads();
    return;
  }
  constexpr int kPer = (kMaxGroups + 1 + kQuantThreads - 1) / kQuantThreads;
  const int first = threadIdx.x * kPer;
  int v[kPer], m = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int raw = first + i <= l.groups ? l.offsets[first + i] : 0;
    v[i] = raw;
    m = max(m, min(raw, l.rows));
  }
  const int incl = block_scan_max(m, s.warp_part);
  const int lane = threadIdx.x & 31;
  // exclusive value of this thread: the inclusive one of the thread before it
  __shared__ int edge[kQuantThreads / 32];
  if (lane == 31) edge[threadIdx.x >> 5] = incl;
  int run = __shfl_up_sync(0xffffffffu, incl, 1);
  __syncthreads();
  if (lane == 0) run = threadIdx.x ? edge[(threadIdx.x >> 5) - 1] : 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    run = max(run, min(v[i], l.rows));
    if (first + i <= l.groups) {
      s.start[first + i] = run;
      bad |= run != v[i];
    }
  }
  if (bad && status && blockIdx.x == 0) atomicCAS(status, 0, kStatusGroupOffsets);
  __syncthreads();
  int n[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    n[i] = first + i < l.groups ? (s.start[first + i + 1] - s.start[first + i] + 127) >> 7 : 0;
    sum += n[i];
  }
  int before = block_scan_sum(sum, s.warp_part) - sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (first + i <= l.groups) s.tile[first + i] = before;
    before += n[i];
  }
  __syncthreads();
}

// the last group g with before[g] <= t, where before[] counts the tiles of the groups ahead of each group: the one
// that holds tile t
__device__ __forceinline__ int group_before(const int* before, int groups, int t) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The plan for the GEMM behind the quantizer, written by one block; `wide` is shared scratch of kMaxGroups + 1 ints.
__device__ __forceinline__ void write_group_plan(const GroupList& l, GroupScan& s, const GroupPlan& plan, int* wide) {
  auto tiles_of = [&](int g) {
    return g < l.groups ? (s.start[g + 1] - s.start[g] + plan.tile_rows - 1) / plan.tile_rows : 0;
  };
  if (l.groups < 32) {
    if (threadIdx.x < 32) {
      const int g = threadIdx.x, n = tiles_of(g), incl = warp_scan_sum(n);
      if (g <= l.groups) {
        wide[g] = incl - n;
        plan.k_tiles[g] = s.tile[g];
      }
    }
  } else {
    constexpr int kPer = (kMaxGroups + 1 + kQuantThreads - 1) / kQuantThreads;
    const int first = threadIdx.x * kPer;
    int n[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      n[i] = tiles_of(first + i);
      sum += n[i];
    }
    int before = block_scan_sum(sum, s.warp_part) - sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (first + i <= l.groups) {
        wide[first + i] = before;
        plan.k_tiles[first + i] = s.tile[first + i];
      }
      before += n[i];
    }
  }
  __syncthreads();
  const int total = wide[l.groups];
  if (threadIdx.x == 0) plan.row_tiles[0] = total;
  for (int t = threadIdx.x; t < total; t += kQuantThreads) {
    const int g = group_before(wide, l.groups, t);
    const int off = (t - wide[g]) * plan.tile_rows, row = s.start[g] + off;
    plan.tiles[t] = make_int4(row, min(plan.tile_rows, s.start[g + 1] - row), s.tile[g] + (off >> 7),
                              g | ((off & 127) >> 5) << 16);
  }
  __syncthreads();
}

// rows of no group: zero in `out` [rows, cols]
__device__ __forceinline__ void zero_rows_of_no_group(const GroupList& l, const GroupScan& s, __nv_bfloat16* out,
                                                      int cols, int64_t ldo) {
  const int head = s.start[0], dead = head + l.rows - s.start[l.groups];
  const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ldo % 8 == 0;
  for (int i = blockIdx.x; i < dead; i += gridDim.x) {
    const int row = i < head ? i : s.start[l.groups] + i - head;
    __nv_bfloat16* dst = out + static_cast<int64_t>(row) * ldo;
    const int vecs = vec ? cols / 8 : 0;
    for (int c = threadIdx.x; c < vecs; c += blockDim.x) reinterpret_cast<uint4*>(dst)[c] = make_uint4(0, 0, 0, 0);
    for (int c = vecs * 8 + threadIdx.x; c < cols; c += blockDim.x) dst[c] = __float2bfloat16_rn(0.0f);
  }
}

// ---------------------------------------------------------------------------
// Row quantizer of the grouped forward and of the linear with an epilogue, both operands in one launch: the rows of x
// (by group), then the `batches` weight matrices [w.rows, k], each with scale tiles of its own.
//
// One lane owns one block of 32 values (two 32-byte loads, one 32-byte store), so a block's maximum needs no exchange
// between lanes and its scale is computed once: 7 instructions a value, where eight values per lane (quant_mxfp8_rows_tile)
// take 17, and those bound that form (70 % issue at 4.3 TB/s).  HBM bound: 16384 x 4096 rows and 8 weights of 4096 x 4096
// (403 MB read, 205 MB written) in 96 to 101 us, 6.0 to 6.3 TB/s, 0.92 to 0.96 of the copy rate; 138 us before.  A warp takes 32 blocks of the four rows r, r + 32, r + 64,
// r + 96 of a 128-row tile: their scale bytes are whole 16-byte segments of the scale tiles, put together by four
// shuffles; no shared memory, no barrier.  Narrow rows (fewer than 32 blocks) share a warp.
// Rows of a tile behind the operand's last row: payload and scales stay unwritten; they reach only accumulator entries
// that are never stored.
// ---------------------------------------------------------------------------
constexpr int kRowsOccupancy = 4;

// 32 values of a row (zero from `valid` on).  align: 2 = 32-byte, 1 = 16-byte aligned rows, 0 = neither; [lo, hi): the operand
__device__ __forceinline__ void load_block32(const __nv_bfloat16* src, int valid, int align, const void* lo, const void* hi,
                                             uint32_t (&w)[16]) {
  if (valid >= 32 && align == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
          : "=r"(w[8 * h]), "=r"(w[8 * h + 1]), "=r"(w[8 * h + 2]), "=r"(w[8 * h + 3]), "=r"(w[8 * h + 4]),
            "=r"(w[8 * h + 5]), "=r"(w[8 * h + 6]), "=r"(w[8 * h + 7])
          : "l"(src + 16 * h));
  } else if (align != 0 && (valid >= 32 || valid % 8 == 0)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 v = 8 * j < valid ? __ldg(reinterpret_cast<const uint4*>(src) + j) : make_uint4(0, 0, 0, 0);
      w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
    }
  } else {
    // 16-byte pieces around the block, shifted into place (3666 rows, 6 groups, 1003 x 2181: 17.5 us, value by value 48.7).
    // A piece that reaches beyond the operand is not read: the ends of its first and last rows are loaded value by value.
    const uintptr_t from = reinterpret_cast<uintptr_t>(src);
    const uint4* piece = reinterpret_cast<const uint4*>(from & ~uintptr_t(15));
    const int pieces = static_cast<int>((from & 15) + 2 * min(valid, 32) + 15) >> 4;
    if (valid > 0 && piece >= reinterpret_cast<const uint4*>(lo) && piece + pieces <= reinterpret_cast<const uint4*>(hi)) {
      uint32_t t[20];
#pragma unroll
      for (int j = 0; j < 5; ++j) {
        const uint4 v = j < pieces ? __ldg(piece + j) : make_uint4(0, 0, 0, 0);
        t[4 * j] = v.x; t[4 * j + 1] = v.y; t[4 * j + 2] = v.z; t[4 * j + 3] = v.w;
      }
      const bool by2 = from & 8, by1 = from & 4;
      const uint32_t half = (from & 2) * 8;
#pragma unroll
      for (int e = 0; e < 18; ++e) t[e] = by2 ? t[e + 2] : t[e];
#pragma unroll
      for (int e = 0; e < 17; ++e) t[e] = by1 ? t[e + 1] : t[e];
#pragma unroll
      for (int e = 0; e < 16; ++e) w[e] = __funnelshift_r(t[e], t[e + 1], half);
      if (valid < 32) {
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] &= 2 * e + 1 < valid ? 0xFFFFFFFFu : 2 * e < valid ? 0xFFFFu : 0u;
      }
    } else {
      const uint16_t* bits = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t a = 2 * e < valid ? bits[2 * e] : 0u, b = 2 * e + 1 < valid ? bits[2 * e + 1] : 0u;
        w[e] = a | (b << 16);
      }
    }
  }
}

// one unit of a warp: rows r, r + 32, r + 64, r + 96 (r = this lane's) of a 128-row tile with `rows` live rows, block b
__device__ __forceinline__ void quant_mxfp8_rows_unit(const RowsOperand& o, const RowsParams& p, const __nv_bfloat16* src,
                                                      uint8_t* q, uint8_t* scales, int rows, int r, int b, int align) {
  const int lane = threadIdx.x & 31;
  const int valid = p.k - 32 * b;            // values of this block inside the row; <= 0: padding of the scale tile
  const bool in_row = 32 * b < p.kp;
  uint32_t word = 0;                         // scale bytes of the four rows
#pragma unroll
  for (int pair = 0; pair < 2; ++pair) {
    uint32_t w[2][16];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r + 32 * (2 * pair + i);
      if (row < rows && in_row) {
        load_block32(src + row * o.ld + 32 * b, valid, align, o.src, o.end, w[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) w[i][e] = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r + 32 * (2 * pair + i);
      uint32_t m2 = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) m2 = absmax_bf16x2(m2, w[i][e]);
      const uint32_t code = e8m0_from_amax(fmax_nan(bf16_lo(m2), bf16_hi(m2)), p.round_to_infinity != 0);
      const f32x2 recip = both(e8m0_reciprocal(code));
      if (row < rows && in_row) {
        uint32_t c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = cvt_e4m3x4_bf16(w[i][2 * e], w[i][2 * e + 1], recip);
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(q + static_cast<int64_t>(row) * p.kp + 32 * b),
                     "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]), "r"(c[4]), "r"(c[5]), "r"(c[6]), "r"(c[7])
                     : "memory");
        word |= code << (8 * (2 * pair + i));
      }
    }
  }
  // four lanes with the blocks of one scale tile: lane j collects the bytes of row group j
  const int j = lane & 3;
  uint32_t seg = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) seg |= ((__shfl_sync(0xffffffffu, word, (lane & ~3) | i) >> (8 * j)) & 0xFFu) << (8 * i);
  if ((b >> 2) < p.chunks) *reinterpret_cast<uint32_t*>(scales + static_cast<size_t>(b >> 2) * 512 + r * 16 + j * 4) = seg;
}

__global__ void __launch_bounds__(kQuantThreads, kRowsOccupancy) quant_mxfp8_rows_units_kernel(const RowsParams p) {
  __shared__ GroupScan scan;
  griddep_launch_dependents();
  const bool grouped = p.list.offsets != nullptr;
  if (grouped) {
    scan_groups(p.list, scan, p.status);
    if (blockIdx.x == 0) {
      __shared__ int wide[kMaxGroups + 1];
      write_group_plan(p.list, scan, p.plan, wide);
    }
    zero_rows_of_no_group(p.list, scan, p.out, p.out_cols, p.ldo);
  }
  const int lane = threadIdx.x & 31;
  const uint32_t x_units = (grouped ? scan.tile[p.list.groups] : (p.x.rows + 127) / 128) * p.per_tile;
  const uint32_t units = x_units + (p.w.src ? p.batches * p.w_row_tiles * p.per_tile : 0u);   // < 2^31, checked by the host
  const uint32_t warps = gridDim.x * (kQuantThreads / 32);
  for (uint32_t u = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    const bool is_x = u < x_units;
    const uint32_t v = is_x ? u : u - x_units;
    const uint32_t rt = v / p.per_tile;                      // 128-row tile (of all matrices)
    const uint32_t in_tile = v - rt * p.per_tile;
    const uint32_t first_r = in_tile / p.segs * p.stacked;
    const int r = first_r + lane / p.lanes;
    const int b = in_tile % p.segs * p.lanes + lane % p.lanes;
    int64_t row0;
    int rows;
    if (!is_x) {
      const uint32_t e = rt / p.w_row_tiles;
      const int first = (rt - e * p.w_row_tiles) * 128;
      row0 = static_cast<int64_t>(e) * p.w.rows + first;
      rows = min(128, p.w.rows - first);
    } else if (grouped) {
      const int g = group_before(scan.tile, p.list.groups, rt);
      row0 = scan.start[g] + 128ll * (rt - scan.tile[g]);
      rows = min(128, scan.start[g + 1] - static_cast<int>(row0));
    } else {
      row0 = 128ll * rt;
      rows = min(128, p.x.rows - static_cast<int>(row0));
    }
    if (static_cast<int>(first_r) >= rows) continue;         // warp-uniform: no live row
    const RowsOperand& o = is_x ? p.x : p.w;
    quant_mxfp8_rows_unit(o, p, o.src + row0 * o.ld, o.q + row0 * p.kp, o.scales + static_cast<size_t>(rt) * p.chunks * 512,
                          rows, r, b, o.align);
  }
}

// ---------------------------------------------------------------------------
// Quantizer of the backward's operands, in one launch: the gradient (by group; blocks along the columns for dX and along
// the rows for dW, from one read), x (by group, along the rows, for dW) and the weight matrices (along the rows, for dX).
// A warp takes 64 columns of a 128-row tile.  Along the rows, one lane owns two neighbouring columns and walks down 32 rows
// at a time, so that a block is in its registers and its maximum needs no exchange; along the columns a lane owns a row.
// The blocks come through shared memory, two ahead of the one at work (with loads into the registers themselves 96 KB are
// in flight per SM only while nothing is computed), and the columns' payload leaves through it, because a lane holds 32
// bytes of a column whose K step is 128.  No barrier but the warp's own.
// Bound by memory and, with 16 warps per SM, by instruction latency (56 % issue): 8192 x 4096 gradient and x, 4 weights of
// 4096 x 4096 (268 MB read, 168 MB written) in 79 us, 5.5 TB/s, 0.84 of the copy rate.  On the way, 8192 rows, 32 groups,
// 2048 x 4096 (a launch for the gradient on staged 128 x 128 tiles and one for the rest, together): 253 us with direct loads
// and stores, 225 with staged stores, 195 with blocks fetched ahead too; one launch 196, without register spills 187.
// ---------------------------------------------------------------------------
constexpr int kTransposedOccupancy = 2;
constexpr int kTransposedFetchBytes = 32 * 128;   // a block of 64 columns
constexpr int kTransposedStageBytes = 64 * 64;    // 64 bytes of each column's payload
constexpr int kTransposedLastBytes = 16 * 4;      // last values of rows that come shifted
constexpr int kTransposedWarpBytes = 2 * (kTransposedFetchBytes + kTransposedLastBytes) + kTransposedStageBytes;
constexpr int kTransposedSmemBytes = kQuantThreads / 32 * kTransposedWarpBytes;

// What one warp does at a time: 64 columns of a 128-row tile, four blocks of 32 rows.  Two of these live in registers, and
// pointers are formed where they are used: a register too many is a load from L2 where shared memory leaves L1 nothing.
struct TransposedUnit {
  int operand;      // 0 = w, 1 = x, 2 = gradient
  int row0, live;   // first row (over all matrices) and rows
  int rt, matrix;   // 128-row tile, of its matrix
  int col0;
};

// the block at `src` value by value or by words, where rows or columns are no 16-byte pieces (quant_mxfp8_transposed_fetch); a
// call, so that it costs the common path no registers
__device__ __noinline__ void quant_mxfp8_transposed_fetch_words(const uint16_t* src, const void* none, int64_t ld, int row0, int live,
                                                                int cols, int by, uint8_t* buf, uint8_t* last) {
  const int lane = threadIdx.x & 31, left = cols - 2 * lane;   // columns from this lane's first one on
  const uint16_t* at = src + 2 * lane;
  auto slot = [&](int e) { return buf + e * 128 + (((lane >> 2) ^ (e & 7)) << 4) + 4 * (lane & 3); };
  if (by == 1) {
    // with an odd pitch every other row starts between two words: it comes one value early (shift_odd_rows puts it right)
    const int odd = static_cast<int>(ld & 1);
#pragma unroll 8
    for (int e = 0; e < 32; ++e) {
      const int early = odd & (row0 + e), have = e < live ? left + early : 0;
      cp_async_4(slot(e), have > 0 ? static_cast<const void*>(at + e * ld - early) : none, have >= 2 ? 4 : have == 1 ? 2 : 0);
    }
    if (odd && lane < 16) {   // the last value of each of those rows
      const int e = 2 * lane + (~row0 & 1);
      const bool have = e < live && cols >= 64;
      cp_async_4(last + 4 * lane, have ? static_cast<const void*>(src + e * ld + 63) : none, have ? 2 : 0);
    }
  } else {
#pragma unroll 8
    for (int e = 0; e < 32; ++e) {
      const bool row = e < live;
      const uint32_t a = row && left >= 1 ? at[e * ld] : 0u, b = row && left >= 2 ? at[e * ld + 1] : 0u;
      *reinterpret_cast<uint32_t*>(slot(e)) = a | (b << 16);
    }
  }
}

// Block j of the unit into `buf` [32 rows][64 columns]; what lies outside the operand is zero.  16-byte chunk i of row r
// lies at chunk i ^ (r % 8): eight lanes that read one chunk of eight rows meet in no bank, nor do 32 that read a row.
// `by`: 2 = 16-byte pieces (rows and columns are multiples of them), 1 = words (the operand starts at one), 0 = values.
// 3666 rows, 6 groups: 1024 x 2176 by pieces 21 us, 1004 x 2180 by words 33, 1003 x 2181 by words shifted 38, by values 113.
__device__ __forceinline__ void quant_mxfp8_transposed_fetch(const TransposedUnit& f, const TransposedOperand& o, int by, int j,
                                                             uint8_t* buf, uint8_t* last) {
  const int lane = threadIdx.x & 31;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(o.src) + static_cast<int64_t>(f.row0) * o.ld + f.col0;
  const int cols = o.cols - f.col0;
  if (by == 2) {
    const int c8 = (lane & 7) * 8, r0 = 32 * j + (lane >> 3);
    const uint16_t* at = src + r0 * o.ld + c8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool valid = r0 + 4 * i < f.live && c8 < cols;   // cols is a multiple of 8 here
      const int r = 4 * i + (lane >> 3);
      cp_async_16(buf + r * 128 + (((lane & 7) ^ (r & 7)) << 4), valid ? at + 4 * i * o.ld : src, valid);
    }
  } else {
    quant_mxfp8_transposed_fetch_words(src + 32 * j * o.ld, o.src, o.ld, f.row0, f.live - 32 * j, cols, by, buf, last);
  }
  cp_async_commit();
}

__device__ __noinline__ void shift_odd_rows(int row0, uint8_t* buf, const uint8_t* last) {
  const int lane = threadIdx.x & 31;
#pragma unroll 8
  for (int i = 0; i < 16; ++i) {
    const int e = 2 * i + (~row0 & 1);
    uint32_t* at = reinterpret_cast<uint32_t*>(buf + e * 128 + (((lane >> 2) ^ (e & 7)) << 4) + 4 * (lane & 3));
    const uint32_t word = *at;
    uint32_t next = __shfl_down_sync(0xffffffffu, word, 1);
    if (lane == 31) next = *reinterpret_cast<const uint32_t*>(last + 4 * i);
    *at = __byte_perm(word, next, 0x5432);   // the second value of this lane's word, the first of the next one's
  }
  __syncwarp();
}

// The rows of a gradient block in `buf`, a lane each: two blocks of 32 values along the columns
__device__ __forceinline__ void quant_mxfp8_gradient_rows(const TransposedUnit& f, const TransposedParams& p, int j,
                                                          const uint8_t* buf) {
  const int lane = threadIdx.x & 31, row = 32 * j + lane;
  const int np = (p.dy.cols + 31) / 32 * 32;
  uint32_t codes = 0;
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    if (f.col0 + 32 * blk >= np) break;   // warp-uniform
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(buf + lane * 128 + (((4 * blk + i) ^ (lane & 7)) << 4));
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    uint32_t m2 = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) m2 = absmax_bf16x2(m2, w[e]);
    const uint32_t code = e8m0_from_amax(fmax_nan(bf16_lo(m2), bf16_hi(m2)), true);
    const f32x2 recip = both(e8m0_reciprocal(code));
    codes |= code << (8 * blk);
    if (row < f.live) {
      uint32_t c[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = cvt_e4m3x4_bf16(w[2 * e], w[2 * e + 1], recip);
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p.dy_rows + static_cast<int64_t>(f.row0 + row) * np + f.col0 + 32 * blk),
                   "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]), "r"(c[4]), "r"(c[5]), "r"(c[6]), "r"(c[7])
                   : "memory");
    }
  }
  if (row < f.live) {
    // 64 columns are half a word of a row's four codes; the last ones fill theirs with zeros
    uint8_t* at = p.dy_row_scales + (static_cast<size_t>(f.rt) * ((np + 127) / 128) + (f.col0 >> 7)) * 512 + lane * 16 + j * 4 +
                  ((f.col0 >> 5) & 3);
    if ((f.col0 & 64) == 0 && f.col0 + 64 >= np) *reinterpret_cast<uint32_t*>(at) = codes;
    else *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(codes);
  }
}

// GRADIENT (the grouped backward): the gradient's units come first, in both orientations from one read, its rows and x's
// are split into groups, and the kernel is the first of its chain (it leaves the plan and sets the result's rows of no
// group to zero).  Else x is one group of all its rows.
template <bool GRADIENT>
__global__ void __launch_bounds__(kQuantThreads, kTransposedOccupancy)
quant_mxfp8_transposed_units_kernel(const TransposedParams p) {
  extern __shared__ __align__(128) uint8_t qt_smem[];
  uint8_t* buf = qt_smem + (threadIdx.x >> 5) * kTransposedWarpBytes;
  uint8_t* stage = buf + 2 * kTransposedFetchBytes;
  uint8_t* last = stage + kTransposedStageBytes;
  __shared__ GroupScan scan;
  griddep_launch_dependents();
  if (GRADIENT) {
    scan_groups(p.list, scan, p.status);
    if (blockIdx.x == 0) write_group_plan(p.list, scan, p.plan, reinterpret_cast<int*>(qt_smem));
    if (p.dx) zero_rows_of_no_group(p.list, scan, p.dx, p.dx_cols, p.dx_cols);
  }
  const uint32_t x_tiles = GRADIENT ? scan.tile[p.list.groups] : (p.x.rows + 127) / 128;
  const uint32_t dy_units = GRADIENT ? x_tiles * p.dy_col_units : 0;
  const uint32_t x_end = dy_units + (p.x.src ? x_tiles * p.x_col_units : 0);
  const uint32_t units = x_end + (p.w.src ? p.batches * p.w_row_tiles * p.w_col_units : 0u);   // < 2^31 (host)
  auto operand = [&](int i) -> const TransposedOperand& { return GRADIENT && i == 2 ? p.dy : i ? p.x : p.w; };
  auto locate = [&](uint32_t u) {
    TransposedUnit f;
    f.operand = GRADIENT && u < dy_units ? 2 : u < x_end ? 1 : 0;
    const TransposedOperand& o = operand(f.operand);
    const uint32_t v = u - (f.operand == 2 ? 0 : f.operand ? dy_units : x_end);
    const uint32_t col_units = f.operand == 2 ? p.dy_col_units : f.operand ? p.x_col_units : p.w_col_units;
    f.rt = v / col_units;
    f.matrix = 0;
    f.col0 = (v - f.rt * col_units) * 64;
    if (f.operand == 0) {
      f.matrix = f.rt / p.w_row_tiles;
      f.rt -= f.matrix * p.w_row_tiles;
      f.row0 = f.matrix * o.rows + 128 * f.rt;
      f.live = o.rows - 128 * f.rt;
    } else if (GRADIENT) {
      const int g = group_before(scan.tile, p.list.groups, f.rt);
      f.row0 = scan.start[g] + 128 * (f.rt - scan.tile[g]);
      f.live = scan.start[g + 1] - f.row0;
    } else {
      f.row0 = 128 * f.rt;
      f.live = o.rows - f.row0;
    }
    f.live = min(128, f.live);
    return f;
  };
  auto by_of = [](const TransposedOperand& o) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(o.src);
    return o.ld % 8 == 0 && o.cols % 8 == 0 && from % 16 == 0 ? 2 : from % 4 == 0 ? 1 : 0;
  };
  const int by = by_of(p.w) | by_of(p.x) << 2 | (GRADIENT ? by_of(p.dy) << 4 : 0);
  auto fetch = [&](const TransposedUnit& f, int j) {
    quant_mxfp8_transposed_fetch(f, operand(f.operand), by >> 2 * f.operand & 3, j, buf + (j & 1) * kTransposedFetchBytes,
                                 last + (j & 1) * kTransposedLastBytes);
  };
  const int lane = threadIdx.x & 31;
  const uint32_t stride = gridDim.x * (kQuantThreads / 32);
  uint32_t u = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  TransposedUnit f, ahead;
  if (u < units) {
    f = ahead = locate(u);
    fetch(f, 0);
    fetch(f, 1);
  }
  for (; u < units; u += stride, f = ahead) {
    const TransposedOperand& o = operand(f.operand);
    const int bytes = static_cast<int>(min(static_cast<int64_t>(128), o.pitch - static_cast<int64_t>(128 * f.rt)));   // of a column
    const bool columns = !GRADIENT || f.operand != 2 || p.dy.q != nullptr;
    const bool shifted = (o.ld & 1) && (by >> 2 * f.operand & 3) == 1;
    uint32_t word0 = 0, word1 = 0;   // the four scale bytes of either column
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      cp_async_wait<1>();            // everything but the newest group: block j is here
      __syncwarp();
      uint8_t* rows = buf + (j & 1) * kTransposedFetchBytes;
      if (shifted) shift_odd_rows(f.row0, rows, last + (j & 1) * kTransposedLastBytes);
      if (GRADIENT && f.operand == 2 && p.dy_rows && 32 * j < f.live) quant_mxfp8_gradient_rows(f, p, j, rows);
      uint32_t w[32];
#pragma unroll
      for (int e = 0; e < 32; ++e)
        w[e] = *reinterpret_cast<const uint32_t*>(rows + e * 128 + (((lane >> 2) ^ (e & 7)) << 4) + 4 * (lane & 3));
      __syncwarp();
      // the buffer takes the block after the next one
      if (j == 2 && u + stride < units) ahead = locate(u + stride);
      if (j < 2) fetch(f, j + 2);
      else if (u + stride < units) fetch(ahead, j - 2);
      else cp_async_commit();
      if (!columns || 32 * j >= bytes) continue;
      uint32_t m2 = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) m2 = absmax_bf16x2(m2, w[e]);
      const uint32_t code0 = e8m0_from_amax(bf16_lo(m2), true), code1 = e8m0_from_amax(bf16_hi(m2), true);
      const f32x2 recip = pack2(e8m0_reciprocal(code0), e8m0_reciprocal(code1));
      word0 |= code0 << (8 * j);
      word1 |= code1 << (8 * j);
      // the stage holds 64 bytes of each column as four 16-byte chunks: chunk i of column c at chunk i ^ (c / 2 % 4) of row
      // c ^ (c / 8 % 2): no two of eight lanes meet in a bank, here or below
      uint8_t* at0 = stage + ((2 * lane) ^ ((lane >> 2) & 1)) * 64;
      uint8_t* at1 = stage + ((2 * lane + 1) ^ ((lane >> 2) & 1)) * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t o0[4], o1[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f32x2 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = mul2(unpack_bf16x2(w[16 * h + 4 * e + i]), recip);
          o0[e] = cvt_e4m3x2(lo(v[0]), lo(v[1])) | (cvt_e4m3x2(lo(v[2]), lo(v[3])) << 16);
          o1[e] = cvt_e4m3x2(hi(v[0]), hi(v[1])) | (cvt_e4m3x2(hi(v[2]), hi(v[3])) << 16);
        }
        const int chunk = ((2 * (j & 1) + h) ^ (lane & 3)) << 4;
        *reinterpret_cast<uint4*>(at0 + chunk) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
        *reinterpret_cast<uint4*>(at1 + chunk) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
      }
      if ((j & 1) == 0 && 32 * j + 32 < bytes) continue;
      __syncwarp();
      const int first = 64 * (j >> 1), part = lane & 3;
      uint8_t* q = o.q + (static_cast<int64_t>(f.matrix) * o.cols + f.col0) * o.pitch + 128ll * f.rt + first + 16 * part;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = 8 * i + (lane >> 2);
        if (f.col0 + col < o.cols && first + 16 * part < bytes)
          *reinterpret_cast<uint4*>(q + col * o.pitch) = *reinterpret_cast<const uint4*>(
              stage + (col ^ ((col >> 3) & 1)) * 64 + ((part ^ ((col >> 1) & 3)) << 4));
      }
      __syncwarp();   // the stage is free again
    }
    if (columns) {
      const int c = (f.col0 & 127) + 2 * lane;   // within its 128 columns; even: both columns in one scale tile
      uint8_t* at = o.scales + ((static_cast<size_t>(f.matrix) * ((o.cols + 127) / 128) + (f.col0 >> 7)) * o.chunks + f.rt) * 512;
      if (f.col0 + 2 * lane < o.cols) *reinterpret_cast<uint32_t*>(at + (c & 31) * 16 + (c >> 5) * 4) = word0;
      if (f.col0 + 2 * lane + 1 < o.cols) *reinterpret_cast<uint32_t*>(at + ((c + 1) & 31) * 16 + (c >> 5) * 4) = word1;
    }
  }
  cp_async_wait<0>();
  if (GRADIENT) return;
  griddep_wait();   // the launch before this one is complete: whoever waits for this grid has waited for that one too
  if (p.partial == nullptr) return;
  __shared__ float part[8][33];
  // dbias[c] = bf16( sum over the row tiles of partial[t][c] ): eight threads per column add every eighth tile, the eight
  // sums are added in a fixed order
  const int k = threadIdx.x >> 5;
  for (int c = blockIdx.x; c < (p.n + 31) / 32; c += gridDim.x) {
    const int col = c * 32 + lane;
    float s = 0.0f;
    if (col < p.n)
      for (int t = k; t < p.row_tiles; t += 8) s += __ldcg(p.partial + static_cast<int64_t>(t) * p.n + col);
    part[k][lane] = s;
    __syncthreads();
    if (k == 0 && col < p.n) {
#pragma unroll
      for (int i = 1; i < 8; ++i) s += part[i][lane];
      p.dbias[col] = __float2bfloat16_rn(s);
    }
    __syncthreads();
  }
}

}  // namespace rtxb
