// Backward of the linear with an epilogue, its elementwise half fused with the quantizers:
//   dz = dy act'(z)                          [m, n], FP32, rounded once to BF16 (the gradient autograd would carry)
//   q_rows  MXFP8 of dz, blocks along n      (A operand of dX = dz W)
//   q_t     MXFP8 of dz^T, blocks along m    (A operand of dW = dz^T X)
//   partial[m / 128][n] = sum of 128 rows of dz in FP32, before the rounding   (dbias, finished by quant_mxfp8_transposed_units_kernel)
// dy and z are read once (4 bytes per value), 2 bytes of payload leave: without the fusion dz is written and read again
// (4 more).  One 128 x 128 tile per block step; three blocks per SM overlap one another's loads, arithmetic and stores.
// Measured, gelu, 8192 x 8192 (409 MB): 93 us at 1965 MHz (4.4 TB/s, 0.67 of the copy rate), 126 us at 1390 MHz, where the
// GEMMs of a training step hold the power cap.  The time goes with the clock, because instructions bound it (63 % issue): 29
// a value, 17 of them before the quantization.  Evaluating the slopes instead of looking them up takes a third longer.
#pragma once

#include "activation.cuh"
#include "quant_tiles.cuh"

namespace rtxb {

struct QuantActParams {
  const __nv_bfloat16* dy;   // [m, n], pitch lddy
  const __nv_bfloat16* z;    // [m, n], pitch n; nullptr when act is none
  int m, n, act;
  int64_t lddy;
  uint8_t* q_rows;           // [m, np] or nullptr
  uint8_t* s_rows;
  uint8_t* q_t;              // [n, mp] or nullptr
  uint8_t* s_t;
  float* partial;            // [ceil(m / 128)][n] or nullptr
};

constexpr int kActOccupancy = 3;                  // resident blocks per SM (registers)
constexpr int kActSumRows = kQuantThreads / 32;   // partial column sums per tile before the last step, one per warp

// z has eight significant bits, so between 2^-21 and 128 it takes 28 x 128 magnitudes: the slopes of silu and the gelus are
// looked up.  For each of them act'(z) = 1 - act'(-z) (f(z) - f(-z) = z), so the table holds the slopes of negative z, which
// keep their relative accuracy however small, and a positive z takes 1 less its entry.  Below 2^-21 the slope is within
// 8e-7 of 1/2, beyond +-128 it is 1 or 0.  That is a third of the instructions of an evaluation, and instructions are what
// bounds the pass.  A second table for positive z saves three instructions a pair and is a quarter slower (for relu too, which
// reads no table): three blocks with 31 KB of tables each leave L1 too little.
constexpr int kSlopeLow = 106 << 7, kSlopeHigh = 134 << 7;     // BF16 magnitudes of 2^-21 and 128
constexpr int kSlopeEntries = kSlopeHigh - kSlopeLow + 1;
constexpr int act_smem_bytes(bool lookup) { return kQtTileBytes + (lookup ? (kSlopeEntries * 4 + 15) / 16 * 16 : 0); }

// Eight gradients dy act'(z) as four pairs.  LOOKUP: from the table; else relu, relu2 or none by `act`.
template <bool LOOKUP>
__device__ __forceinline__ void act_gradient8(const float* table, int act, const uint4 dy, const uint4 z, f32x2 (&v)[4]) {
  const uint32_t g[4] = {dy.x, dy.y, dy.z, dy.w}, w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = unpack_bf16x2(g[e]);
  if (LOOKUP) {
    uint32_t m2 = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t mag = __vminu2(__vmaxu2(w[e] & 0x7FFF7FFFu, kSlopeLow * 0x10001u), kSlopeHigh * 0x10001u);
      // t for z < 0, 1 - t for z >= 0: sign t + (1 - sign) / 2 with sign = -1 for z >= 0
      const f32x2 sign = pack2(__uint_as_float((~(w[e] << 16) & 0x80000000u) | 0x3F800000u),
                               __uint_as_float((~w[e] & 0x80000000u) | 0x3F800000u));
      v[e] = mul2(v[e], fma2(pack2(table[mag & 0xFFFFu], table[mag >> 16]), sign, fma2(sign, both(-0.5f), both(0.5f))));
      m2 = absmax_bf16x2(m2, w[e]);
    }
    if (bf16_lo(m2) != bf16_lo(m2) || bf16_hi(m2) != bf16_hi(m2)) {   // a NaN among them: it goes on to dz
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z0 = bf16_lo(w[e]), z1 = bf16_hi(w[e]);
        v[e] = pack2(z0 != z0 ? z0 : lo(v[e]), z1 != z1 ? z1 : hi(v[e]));
      }
    }
  } else if (act != kActNone) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = lo(v[e]), b = hi(v[e]);
      if (act == kActRelu) relu_slope2<kActRelu>(a, b, bf16_lo(w[e]), bf16_hi(w[e]));
      else relu_slope2<kActRelu2>(a, b, bf16_lo(w[e]), bf16_hi(w[e]));
      v[e] = pack2(a, b);
    }
  }
}

template <bool LOOKUP>
__global__ void __launch_bounds__(kQuantThreads, kActOccupancy) quant_mxfp8_act_backward_kernel(const QuantActParams p) {
  extern __shared__ __align__(16) uint8_t qt_smem[];
  uint16_t (*tile)[kQtPitch] = reinterpret_cast<uint16_t (*)[kQtPitch]>(qt_smem);
  float* slopes = reinterpret_cast<float*>(qt_smem + kQtTileBytes) - kSlopeLow;   // indexed by magnitude
  __shared__ __align__(16) uint8_t scales_t[128][4];
  __shared__ __align__(16) uint8_t scales_rows[128][4];
  __shared__ float sums[kActSumRows][128];
  griddep_launch_dependents();
  if (LOOKUP) {
    for (int i = kSlopeLow + threadIdx.x; i <= kSlopeHigh; i += kQuantThreads)
      slopes[i] = slope_at_minus(p.act, __uint_as_float(static_cast<uint32_t>(i) << 16));
    __syncthreads();
  }
  const int col_tiles = (p.n + 127) / 128, row_tiles = (p.m + 127) / 128;
  const int np = (p.n + 31) / 32 * 32, mp = (p.m + 31) / 32 * 32;
  const bool vec_dy = (p.lddy % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.dy) & 15) == 0);
  const bool vec_z = p.z == nullptr || ((p.n % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.z) & 15) == 0));
  const int c8 = (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4;
  const int64_t total = static_cast<int64_t>(row_tiles) * col_tiles;
  // tile (rt, ct); the grid's stride in both, so that no tile costs a division
  int rt = blockIdx.x / col_tiles, ct = blockIdx.x - rt * col_tiles;
  const int step_r = gridDim.x / col_tiles, step_c = gridDim.x - step_r * col_tiles;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x, rt += step_r, ct += step_c) {
    if (ct >= col_tiles) { ct -= col_tiles; ++rt; }
    const int row0 = rt * 128, col0 = ct * 128;
    const int col = col0 + c8;
    f32x2 sum[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = both(0.0f);
    const bool whole = vec_dy && vec_z && row0 + 128 <= p.m && col0 + 128 <= p.n;
    const __nv_bfloat16* gp = p.dy + static_cast<int64_t>(row0 + r0) * p.lddy + col;
    const __nv_bfloat16* zp = p.z + static_cast<int64_t>(row0 + r0) * p.n + col;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      uint4 g[4], z[4];
      if (whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          g[j] = __ldg(reinterpret_cast<const uint4*>(gp));
          z[j] = p.z ? __ldg(reinterpret_cast<const uint4*>(zp)) : make_uint4(0, 0, 0, 0);
          gp += 16 * p.lddy;
          zp += 16 * static_cast<int64_t>(p.n);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t row = row0 + r0 + 16 * (half * 4 + j);
          const bool live = row < p.m && col < p.n;
          g[j] = live ? load8_raw(p.dy + row * p.lddy, col, p.n, vec_dy) : make_uint4(0, 0, 0, 0);
          z[j] = live && p.z ? load8_raw(p.z + row * p.n, col, p.n, vec_z) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x2 v[4];
        act_gradient8<LOOKUP>(slopes, p.act, g[j], z[j], v);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[e] = add2(sum[e], v[e]);
          __nv_bfloat162 b = __floats2bfloat162_rn(lo(v[e]), hi(v[e]));
          w[e] = *reinterpret_cast<uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(&tile[r0 + 16 * (half * 4 + j)][c8]) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (p.partial) {
      // the two row halves of a warp, then one row of sums per warp
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = lo(sum[e]), b = hi(sum[e]);
        const float sa = a + __shfl_xor_sync(0xffffffffu, a, 16), sb = b + __shfl_xor_sync(0xffffffffu, b, 16);
        if ((threadIdx.x & 16) == 0) {
          sums[threadIdx.x >> 5][c8 + 2 * e] = sa;
          sums[threadIdx.x >> 5][c8 + 2 * e + 1] = sb;
        }
      }
    }
    __syncthreads();
    uint32_t o[2][8];
    if (p.q_t) quant_mxfp8_tile_columns(tile, scales_t, o, mp, p.n, col0, row0, true);
    if (p.q_rows) quant_mxfp8_tile_rows(tile, scales_rows, p.q_rows, np, p.m, p.n, row0, col0, true);
    if (p.partial && threadIdx.x < 128 && col0 + threadIdx.x < p.n) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kActSumRows; ++w) s += sums[w][threadIdx.x];
      p.partial[static_cast<int64_t>(rt) * p.n + col0 + threadIdx.x] = s;
    }
    __syncthreads();   // every thread has read the staged tile: its storage now collects the transposed payload
    if (p.q_t) {
      quant_mxfp8_tile_columns_store(qt_smem, o, p.q_t, mp, p.n, col0, row0);
      store_scale_tile<4>(scales_t, p.s_t, kScaleMma128, col0, row0 / 32, p.n, mp / 32, (mp / 32 + 3) / 4);
    }
    if (p.q_rows)
      store_scale_tile<4>(scales_rows, p.s_rows, kScaleMma128, row0, col0 / 32, p.m, np / 32, (np / 32 + 3) / 4);
    __syncthreads();   // the staged tile, the sums and the scale tiles are free again
  }
}

}  // namespace rtxb
