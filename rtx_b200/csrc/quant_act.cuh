// Backward of the linear with an epilogue, its elementwise half fused with the quantizers:
//   dz = dy act'(z)                          [m, n], FP32, rounded once to BF16 (the gradient autograd would carry)
//   q_rows  MXFP8 of dz, blocks along n      (A operand of dX = dz W)
//   q_t     MXFP8 of dz^T, blocks along m    (A operand of dW = dz^T X)
//   partial[m / 128][n] = sum of 128 rows of dz in FP32, before the rounding   (dbias, finished by the kernel below)
// dy and z are read once (4 bytes per value), 2 bytes of payload leave: without the fusion dz is written and read again
// (4 more).  HBM bound; one 128 x 128 tile per block step, the next one
// is fetched asynchronously while this one is quantized.
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

constexpr int kActOccupancy = 2;                  // resident blocks per SM (three staged tiles each)
constexpr int kActSumRows = kQuantThreads / 32;   // partial column sums per tile before the last step, one per warp
constexpr int kActSmemBytes = 3 * kQtTileBytes;   // raw dy, raw z, dz

// Raw tile of dy or z into `raw`: thread t copies the 8 columns (t & 15) of the rows (t >> 4) + 16 j, the ones it will
// read back itself, so no barrier stands between the copy and its use.
__device__ __forceinline__ void act_fetch(const __nv_bfloat16* src, int64_t ld, bool vec_ok, int m, int n, int row0, int col0,
                                          uint16_t (*raw)[kQtPitch]) {
  const int c8 = (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4;
  const int col = col0 + c8;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = row0 + r0 + 16 * j;
    const bool live = row < m && col < n;
    if (vec_ok && (!live || col + 8 <= n)) {
      cp_async_16(&raw[r0 + 16 * j][c8], src + (live ? row * ld + col : 0), live);
    } else {
      *reinterpret_cast<uint4*>(&raw[r0 + 16 * j][c8]) = live ? load8_raw(src + row * ld, col, n, false) : make_uint4(0, 0, 0, 0);
    }
  }
}

__global__ void __launch_bounds__(kQuantThreads, kActOccupancy) quant_mxfp8_act_backward_kernel(const QuantActParams p) {
  extern __shared__ __align__(16) uint8_t qt_smem[];
  uint16_t (*raw_g)[kQtPitch] = reinterpret_cast<uint16_t (*)[kQtPitch]>(qt_smem);
  uint16_t (*raw_z)[kQtPitch] = reinterpret_cast<uint16_t (*)[kQtPitch]>(qt_smem + kQtTileBytes);
  uint8_t* stage = qt_smem + 2 * kQtTileBytes;
  uint16_t (*tile)[kQtPitch] = reinterpret_cast<uint16_t (*)[kQtPitch]>(stage);
  __shared__ __align__(16) uint8_t scales_t[128][4];
  __shared__ __align__(16) uint8_t scales_rows[128][4];
  __shared__ float sums[kActSumRows][128];
  const int col_tiles = (p.n + 127) / 128, row_tiles = (p.m + 127) / 128;
  const int np = (p.n + 31) / 32 * 32, mp = (p.m + 31) / 32 * 32;
  const bool vec_dy = (p.lddy % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.dy) & 15) == 0);
  const bool vec_z = (p.n % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.z) & 15) == 0);
  const int c8 = (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4;
  const int64_t total = static_cast<int64_t>(row_tiles) * col_tiles;
  auto fetch = [&](int64_t t) {
    const int rt = static_cast<int>(t / col_tiles), ct = static_cast<int>(t - static_cast<int64_t>(rt) * col_tiles);
    act_fetch(p.dy, p.lddy, vec_dy, p.m, p.n, rt * 128, ct * 128, raw_g);
    if (p.z) act_fetch(p.z, p.n, vec_z, p.m, p.n, rt * 128, ct * 128, raw_z);
    cp_async_commit();
  };
  if (blockIdx.x < total) fetch(blockIdx.x);
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int rt = static_cast<int>(t / col_tiles);
    const int row0 = rt * 128, col0 = static_cast<int>(t - static_cast<int64_t>(rt) * col_tiles) * 128;
    cp_async_wait<0>();
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < 8; ++j) {
      float v[8];
      unpack8(*reinterpret_cast<const uint4*>(&raw_g[r0 + 16 * j][c8]), v);
      if (p.z) {
        float z[8];
        unpack8(*reinterpret_cast<const uint4*>(&raw_z[r0 + 16 * j][c8]), z);
        with_activation(p.act, [&](auto tag) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) act_slope2<decltype(tag)::value>(v[e], v[e + 1], z[e], z[e + 1]);
        });
      }
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum[2 * e] += v[2 * e];
        sum[2 * e + 1] += v[2 * e + 1];
        __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        w[e] = *reinterpret_cast<uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(&tile[r0 + 16 * j][c8]) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // this thread's part of the raw tiles is read: the next tile's may come in while this one is quantized
    if (t + gridDim.x < total) fetch(t + gridDim.x);
    if (p.partial) {
      // the two row halves of a warp, then one row of sums per warp
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
      if ((threadIdx.x & 16) == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[threadIdx.x >> 5][c8 + e] = sum[e];
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
      quant_mxfp8_tile_columns_store(stage, o, p.q_t, mp, p.n, col0, row0);
      store_scale_tile<4>(scales_t, p.s_t, kScaleMma128, col0, row0 / 32, p.n, mp / 32, (mp / 32 + 3) / 4);
    }
    if (p.q_rows)
      store_scale_tile<4>(scales_rows, p.s_rows, kScaleMma128, row0, col0 / 32, p.m, np / 32, (np / 32 + 3) / 4);
    __syncthreads();   // the staged tile, the sums and the scale tiles are free again
  }
}

// dbias[c] = bf16( sum over the row tiles of partial[t][c] ): eight threads per column add every eighth tile, the eight
// sums are added in a fixed order
__global__ void __launch_bounds__(256) bias_grad_kernel(const float* __restrict__ partial, int row_tiles, int n,
                                                        __nv_bfloat16* __restrict__ out) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (col < n)
    for (int t = k; t < row_tiles; t += 8) s += partial[static_cast<int64_t>(t) * n + col];
  part[k][lane] = s;
  __syncthreads();
  if (k == 0 && col < n) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    out[col] = __float2bfloat16_rn(s);
  }
}

}  // namespace rtxb
