// Tile bodies of the MXFP8 quantizers (rows, transposed, both from one staged read): what one block does to one
// 128 x 128 tile.  The kernels that walk the tiles are in quant.cuh (dense operands) and grouped.cuh (operands
// split into groups of rows).
#pragma once

#include "common.cuh"

namespace rtxb {

enum ScaleLayout : int { kScaleRowMajor = 0, kScaleMma64 = 1, kScaleMma128 = 2 };

constexpr int kQuantThreads = 256;

// ---------------------------------------------------------------------------
// MXFP8 rows: src bf16 [rows, k] (pitch ld elements) -> q e4m3 [rows, kp],
// scales e8m0.
// ---------------------------------------------------------------------------
struct QuantMxParams {
  const __nv_bfloat16* src;
  uint8_t* q;
  uint8_t* scales;
  int rows, k, kp;       // kp = k rounded up to 32
  int64_t ld;            // source row pitch (elements)
  int nb;                // kp / 32 scale blocks per row
  int sf_chunks;         // 512-byte scale tiles per 128 rows (ceil(nb / 4))
  int layout;            // ScaleLayout
  int round_to_infinity; // 1 = default, 0 = OCP floor ablation
};

__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) a = fmax_nan(a, fabsf(v[e]));
  return a;
}

// write one 128-row x (4*chunks) block tile of scale bytes held in shared
// memory as tile[row][blocks_in_tile] to global in the requested layout
template <int BLOCKS>
__device__ __forceinline__ void store_scale_tile(const uint8_t (*tile)[BLOCKS], uint8_t* scales, int layout, int row0,
                                                 int blk0, int rows, int nb, int sf_chunks) {
  if (layout == kScaleMma128) {
    // BLOCKS/4 tiles of 512 bytes; one 16-byte segment per (tile, row % 32)
    for (int t = threadIdx.x; t < (BLOCKS / 4) * 32; t += blockDim.x) {
      const int chunk = t >> 5, r32 = t & 31;
      if ((blk0 >> 2) + chunk >= sf_chunks) continue;
      uint32_t w[4];
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const uint8_t* s = tile[rg * 32 + r32] + chunk * 4;
        w[rg] = s[0] | (s[1] << 8) | (s[2] << 16) | (static_cast<uint32_t>(s[3]) << 24);
      }
      uint8_t* dst = scales + (static_cast<size_t>(row0 >> 7) * sf_chunks + (blk0 >> 2) + chunk) * 512 + r32 * 16;
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    for (int t = threadIdx.x; t < 128 * BLOCKS; t += blockDim.x) {
      const int r = t / BLOCKS, b = t % BLOCKS;
      if (row0 + r < rows && blk0 + b < nb) scales[static_cast<size_t>(row0 + r) * nb + blk0 + b] = tile[r][b];
    }
  }
}

// raw 16-byte load of 8 BF16 values (zero beyond k); scalar path for ragged or unaligned rows
__device__ __forceinline__ uint4 load8_raw(const __nv_bfloat16* row_ptr, int col, int k, bool vec_ok) {
  if (vec_ok && col + 8 <= k) return __ldg(reinterpret_cast<const uint4*>(row_ptr + col));
  const uint16_t* s = reinterpret_cast<const uint16_t*>(row_ptr);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = (col + 2 * e < k) ? s[col + 2 * e] : 0u;
    const uint32_t hi = (col + 2 * e + 1 < k) ? s[col + 2 * e + 1] : 0u;
    w[e] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void unpack8(const uint4 raw, float (&v)[8]) {
  v[0] = bf16_lo(raw.x); v[1] = bf16_hi(raw.x); v[2] = bf16_lo(raw.y); v[3] = bf16_hi(raw.y);
  v[4] = bf16_lo(raw.z); v[5] = bf16_hi(raw.z); v[6] = bf16_lo(raw.w); v[7] = bf16_hi(raw.w);
}

// One 128 x 128 tile of the row quantizer (see quant_mxfp8_rows_kernel); ends with a block-wide barrier.
__device__ __forceinline__ void quant_mxfp8_rows_tile(const QuantMxParams& p, int tile, uint8_t (*tile_scales)[4]) {
  const int sub = threadIdx.x & 15, rsel = threadIdx.x >> 4;
  const int col_tiles = (p.kp + 127) / 128;
  const bool vec_ok = (p.ld % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.src) & 15) == 0);
  const bool q_vec_ok = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0;  // kp % 32 == 0 keeps rows 8-byte aligned
  const bool rinf = p.round_to_infinity != 0;
  const int row0 = (tile / col_tiles) * 128;
  const int col = (tile % col_tiles) * 128 + sub * 8;
  const bool col_ok = col < p.kp;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + rsel + 16 * (half * 4 + j);
      raw[j] = (row < p.rows && col_ok) ? load8_raw(p.src + static_cast<int64_t>(row) * p.ld, col, p.k, vec_ok)
                                        : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = rsel + 16 * (half * 4 + j);
      const int row = row0 + r;
      const bool live = row < p.rows && col_ok;
      // |max| of the block on packed pairs; 4 lanes hold its 32 values
      uint32_t m2 = absmax_bf16x2(absmax_bf16x2(0u, raw[j].x), raw[j].y);
      m2 = absmax_bf16x2(absmax_bf16x2(m2, raw[j].z), raw[j].w);
      m2 = absmax_bf16x2(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
      m2 = absmax_bf16x2(m2, __shfl_xor_sync(0xffffffffu, m2, 2));
      const uint32_t code = e8m0_from_amax(fmax_nan(bf16_lo(m2), bf16_hi(m2)), rinf);
      const f32x2 recip = both(e8m0_reciprocal(code));
      if ((sub & 3) == 0) tile_scales[r][sub >> 2] = live ? static_cast<uint8_t>(code) : 0;
      if (live) {
        const uint32_t lo = cvt_e4m3x4_bf16(raw[j].x, raw[j].y, recip);
        const uint32_t hi = cvt_e4m3x4_bf16(raw[j].z, raw[j].w, recip);
        uint8_t* dst = p.q + static_cast<int64_t>(row) * p.kp + col;
        if (q_vec_ok) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
        } else {
          for (int e = 0; e < 4; ++e) { dst[e] = lo >> (8 * e); dst[4 + e] = hi >> (8 * e); }
        }
      }
    }
  }
  __syncthreads();
  store_scale_tile<4>(tile_scales, p.scales, p.layout, row0, (tile % col_tiles) * 4, p.rows, p.nb, p.sf_chunks);
  __syncthreads();
}

// ---------------------------------------------------------------------------
// MXFP8 transposed: src bf16 stored [k, rows] (pitch ld) -> q e4m3 [rows, kp]
// K-major with blocks of 32 along the stored row index k; equal to quantising
// src^T.contiguous() by rows.  Tile = 128 output rows x 128 k: the CTA reads
// 128 source rows of 128 values (coalesced), keeps them in shared memory and
// each thread then walks one output row's 32-value blocks down a column.
// ---------------------------------------------------------------------------
struct QuantMxTParams {
  const __nv_bfloat16* src;  // [k, rows]
  uint8_t* q;                // [rows, kp]
  uint8_t* scales;
  int rows, k, kp;
  int64_t ld;
  int nb, sf_chunks, layout, round_to_infinity;
  // dual form: the same staged tile is also quantized along the source rows (blocks of 32 source columns),
  // i.e. the plain row quantization of src, so that src is read from memory once for both
  uint8_t* q_rows;           // [k, np], np = source columns rounded up to 32
  uint8_t* s_rows;
  int np, nb_rows, chunks_rows;
};

// Staged tile: [k_local][row_local] BF16 bits, pitch 136 halfwords (272 bytes: 16-byte aligned rows for the
// asynchronous 16-byte copies; a warp reading one k with 32 consecutive row pairs is conflict free).
constexpr int kQtPitch = 136;
constexpr int kQtTileBytes = 128 * kQtPitch * 2;
constexpr int kQtSmemBytes = 2 * kQtTileBytes;   // two tiles: the next one is fetched while this one is quantized

// Pitch of the output staging rows (128 payload bytes + 16): the staged input tile is re-used, once every
// thread has read it, to collect the tile's output bytes so that they leave the SM as whole 128-byte rows.
constexpr int kQtOutPitch = 144;

// Column pass over a staged 128 x 128 tile `tile[k_local][row_local]` (BF16 bits, pitch kQtPitch halfwords):
// thread -> two adjacent output rows (source columns) x one block of 32 along k, so every
// shared-memory read is one 32-bit word holding both rows' values; consecutive lanes read consecutive
// words (conflict free).  Returns the two rows' 32 payload bytes in `o` (o[h][0..7]) and writes the
// 128 x 4 scale codes to `tile_scales`; the payload is stored by quant_mxfp8_tile_columns_store.
__device__ __forceinline__ void quant_mxfp8_tile_columns(const uint16_t (*tile)[kQtPitch], uint8_t (*tile_scales)[4],
                                                         uint32_t (&o)[2][8], int kp, int rows, int row0, int k0,
                                                         bool round_to_infinity) {
  const int rp = threadIdx.x & 63, j = threadIdx.x >> 6;   // 64 row pairs x 4 blocks = 256 threads
  uint32_t w[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) w[e] = *reinterpret_cast<const uint32_t*>(&tile[j * 32 + e][2 * rp]);
  const int kcol = k0 + j * 32;
  uint32_t m2 = 0;   // |max| of both rows at once
#pragma unroll
  for (int e = 0; e < 32; ++e) m2 = absmax_bf16x2(m2, w[e]);
  const uint32_t code0 = e8m0_from_amax(bf16_lo(m2), round_to_infinity), code1 = e8m0_from_amax(bf16_hi(m2), round_to_infinity);
  const f32x2 recip = pack2(e8m0_reciprocal(code0), e8m0_reciprocal(code1));
  const int row = row0 + 2 * rp;
  tile_scales[2 * rp][j] = row < rows && kcol < kp ? static_cast<uint8_t>(code0) : 0;
  tile_scales[2 * rp + 1][j] = row + 1 < rows && kcol < kp ? static_cast<uint8_t>(code1) : 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f32x2 v[4];   // four values of k, both rows
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul2(unpack_bf16x2(w[4 * e + i]), recip);
    o[0][e] = cvt_e4m3x2(lo(v[0]), lo(v[1])) | (cvt_e4m3x2(lo(v[2]), lo(v[3])) << 16);
    o[1][e] = cvt_e4m3x2(hi(v[0]), hi(v[1])) | (cvt_e4m3x2(hi(v[2]), hi(v[3])) << 16);
  }
}

// Second half of the column pass, after every thread has finished reading the staged tile: the payload goes
// into the tile's own storage as [row_local][128 bytes] and leaves as whole rows — eight lanes write one
// 128-byte row of q, a warp four rows per instruction (the direct form wrote 16 bytes to 32 different rows
// per instruction).
__device__ __forceinline__ void quant_mxfp8_tile_columns_store(uint8_t* stage, const uint32_t (&o)[2][8], uint8_t* q,
                                                               int kp, int rows, int row0, int k0) {
  const int rp = threadIdx.x & 63, j = threadIdx.x >> 6;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4* dst = reinterpret_cast<uint4*>(stage + (2 * rp + h) * kQtOutPitch + j * 32);
    dst[0] = make_uint4(o[h][0], o[h][1], o[h][2], o[h][3]);
    dst[1] = make_uint4(o[h][4], o[h][5], o[h][6], o[h][7]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = threadIdx.x + kQuantThreads * i;
    const int r = c >> 3, part = c & 7;
    const int row = row0 + r, col = k0 + part * 16;
    if (row < rows && col < kp)
      *reinterpret_cast<uint4*>(q + static_cast<int64_t>(row) * kp + col) =
          *reinterpret_cast<const uint4*>(stage + r * kQtOutPitch + part * 16);
  }
}

// Row pass over the same staged tile (dual form): eight lanes cover one source row of the tile (16 values each,
// two lanes per MX block), so a warp writes four whole 128-byte rows of the row-quantized payload per pass.
__device__ __forceinline__ void quant_mxfp8_tile_rows(const uint16_t (*tile)[kQtPitch], uint8_t (*tile_scales)[4],
                                                      uint8_t* q, int np, int k_rows, int cols, int k0, int col0,
                                                      bool round_to_infinity) {
  const int part = threadIdx.x & 7;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int r = (threadIdx.x >> 3) + 32 * pass;
    uint32_t w[8];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint4 v = *reinterpret_cast<const uint4*>(&tile[r][part * 16 + 8 * c]);
      w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
    }
    uint32_t m2 = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m2 = absmax_bf16x2(m2, w[e]);
    m2 = absmax_bf16x2(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
    const uint32_t code = e8m0_from_amax(fmax_nan(bf16_lo(m2), bf16_hi(m2)), round_to_infinity);
    const f32x2 recip = both(e8m0_reciprocal(code));
    const int row = k0 + r, col = col0 + part * 16;
    const bool live = row < k_rows && col < np;
    if ((part & 1) == 0) tile_scales[r][part >> 1] = live ? static_cast<uint8_t>(code) : 0;
    if (live) {
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = cvt_e4m3x4_bf16(w[2 * e], w[2 * e + 1], recip);
      *reinterpret_cast<uint4*>(q + static_cast<int64_t>(row) * np + col) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

constexpr int kQtOccupancy = 3;   // resident CTAs per SM the transposed quantizer is compiled for (registers, 70 KB of tiles)
__device__ __forceinline__ void cp_async_16(void* smem_dst, const void* gmem_src, bool valid) {
  // copies 16 bytes, or writes 16 zero bytes when !valid (source size 0)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem_dst)), "l"(gmem_src),
               "r"(valid ? 16 : 0)
               : "memory");
}
// the first `bytes` (0, 2 or 4) of a word, zeros behind them
__device__ __forceinline__ void cp_async_4(void* smem_dst, const void* gmem_src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(smem_dst)), "l"(gmem_src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// fetch tile t (128 source rows x 128 source columns) into `tile`; aligned full-width tiles asynchronously
__device__ __forceinline__ void quant_mxfp8_t_fetch(const QuantMxTParams& p, uint16_t (*tile)[kQtPitch], int row0, int k0,
                                                    bool vec_ok) {
  const uint16_t* src = reinterpret_cast<const uint16_t*>(p.src);
  if (vec_ok && row0 + 128 <= p.rows) {
    const int c8 = (threadIdx.x & 15) * 8, kr = threadIdx.x >> 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int gk = k0 + kr + 16 * j;
      const bool valid = gk < p.k;
      cp_async_16(&tile[kr + 16 * j][c8], src + static_cast<int64_t>(valid ? gk : 0) * p.ld + row0 + c8, valid);
    }
  } else {
    for (int i = threadIdx.x; i < 128 * 64; i += kQuantThreads) {
      const int kk = i >> 6, c2 = (i & 63) * 2;
      const int gk = k0 + kk, gc = row0 + c2;
      uint16_t a = 0, b = 0;
      if (gk < p.k) {
        const uint16_t* rp = src + static_cast<int64_t>(gk) * p.ld;
        if (gc < p.rows) a = rp[gc];
        if (gc + 1 < p.rows) b = rp[gc + 1];
      }
      tile[kk][c2] = a;
      tile[kk][c2 + 1] = b;
    }
  }
  cp_async_commit();
}

}  // namespace rtxb
