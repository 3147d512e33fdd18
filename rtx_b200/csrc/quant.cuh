// HBM-bound quantizers for sm_100a: BF16 -> MXFP8 (rows and transposed) and
// BF16 -> NVFP4, plus the per-tensor |max| reduction that feeds the NVFP4
// outer scale.  They replace the reference's MXFP8QuantKernel /
// MXFP8TransposedQuantKernel (rtx/kernels/mxfp8_quant.py:52-395, :526-1019)
// and NVFP4QuantKernel (rtx/kernels/nvfp4_quant.py:32-349).
//
// Every kernel walks 128-row tiles with a grid-stride loop, reads 16 bytes per
// thread per load, and stages the tile's scale factors in shared memory so
// that the 128-row scale tiles (the layout tcgen05.cp consumes) leave the SM
// as whole 16-byte segments.
#pragma once

#include "quant_tiles.cuh"

namespace rtxb {

// Tile = 128 rows x 128 columns (exactly one 512-byte scale tile).  Thread t owns 8 columns
// (t & 15) of row (t >> 4) + 16 i; four neighbouring lanes share a block of 32.  Four row loads
// are issued before any is consumed so that each thread keeps 64 bytes in flight.
__global__ void __launch_bounds__(kQuantThreads, 6) quant_mxfp8_rows_kernel(const QuantMxParams p) {
  __shared__ __align__(16) uint8_t tile_scales[128][4];
  const int tiles = ((p.kp + 127) / 128) * ((p.rows + 127) / 128);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) quant_mxfp8_rows_tile(p, tile, tile_scales);
}

// Two tensors in one launch (the reference's dual quantizer, rtx/kernels/mxfp8_quant.py:398-1399: activations and
// weight of a dynamic forward): the tiles of `a`, then the tiles of `b`.  On small layers a launch costs more than
// the quantization, and the GEMM launched behind this kernel as a programmatic dependent can set up meanwhile.
__global__ void __launch_bounds__(kQuantThreads, 6) quant_mxfp8_rows2_kernel(const QuantMxParams a, const QuantMxParams b) {
  __shared__ __align__(16) uint8_t tile_scales[128][4];
  griddep_launch_dependents();
  const int tiles_a = ((a.kp + 127) / 128) * ((a.rows + 127) / 128);
  const int tiles_b = ((b.kp + 127) / 128) * ((b.rows + 127) / 128);
  for (int tile = blockIdx.x; tile < tiles_a + tiles_b; tile += gridDim.x) {
    if (tile < tiles_a) quant_mxfp8_rows_tile(a, tile, tile_scales);
    else quant_mxfp8_rows_tile(b, tile - tiles_a, tile_scales);
  }
}

template <bool DUAL>
__global__ void __launch_bounds__(kQuantThreads, kQtOccupancy) quant_mxfp8_transposed_kernel(const QuantMxTParams p) {
  extern __shared__ __align__(16) uint8_t qt_smem[];
  uint16_t (*tiles[2])[kQtPitch] = {reinterpret_cast<uint16_t (*)[kQtPitch]>(qt_smem),
                                    reinterpret_cast<uint16_t (*)[kQtPitch]>(qt_smem + kQtTileBytes)};
  __shared__ __align__(16) uint8_t tile_scales[128][4];
  __shared__ __align__(16) uint8_t tile_scales_rows[DUAL ? 128 : 1][4];
  const int row_tiles = (p.rows + 127) / 128;
  const int k_tiles = (p.kp + 127) / 128;
  const int total = row_tiles * k_tiles;
  const bool vec_ok = (p.ld % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.src) & 15) == 0);
  int buf = 0;
  if (static_cast<int>(blockIdx.x) < total)
    quant_mxfp8_t_fetch(p, tiles[0], (blockIdx.x % row_tiles) * 128, (blockIdx.x / row_tiles) * 128, vec_ok);
  for (int t = blockIdx.x; t < total; t += gridDim.x) {
    const int row0 = (t % row_tiles) * 128;  // output rows = source columns
    const int k0 = (t / row_tiles) * 128;
    const int tn = t + gridDim.x;
    if (tn < total) {
      quant_mxfp8_t_fetch(p, tiles[buf ^ 1], (tn % row_tiles) * 128, (tn / row_tiles) * 128, vec_ok);
      cp_async_wait<1>();   // everything but the newest group (the next tile) has landed
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    uint32_t o[2][8];
    quant_mxfp8_tile_columns(tiles[buf], tile_scales, o, p.kp, p.rows, row0, k0, p.round_to_infinity != 0);
    if (DUAL)
      quant_mxfp8_tile_rows(tiles[buf], tile_scales_rows, p.q_rows, p.np, p.k, p.rows, k0, row0,
                            p.round_to_infinity != 0);
    __syncthreads();   // every thread has read the staged tile: its storage now collects the transposed payload
    quant_mxfp8_tile_columns_store(reinterpret_cast<uint8_t*>(tiles[buf]), o, p.q, p.kp, p.rows, row0, k0);
    store_scale_tile<4>(tile_scales, p.scales, p.layout, row0, k0 / 32, p.rows, p.nb, p.sf_chunks);
    if (DUAL) store_scale_tile<4>(tile_scales_rows, p.s_rows, p.layout, k0, row0 / 32, p.k, p.nb_rows, p.chunks_rows);
    __syncthreads();   // the scale tiles and this buffer are free again
    buf ^= 1;
  }
}

// ---------------------------------------------------------------------------
// per-tensor |max| (NaN-propagating) of a BF16 matrix, accumulated with an
// integer atomic max on the FP32 bit pattern (non-negative floats order like
// integers and every NaN pattern is larger than infinity)
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) amax_bf16_kernel(const __nv_bfloat16* src, int64_t rows, int64_t k, int64_t ld,
                                                        uint32_t* amax_bits) {
  uint32_t m = 0;
  const bool vec_ok = (ld % 8 == 0) && (k % 8 == 0) && ((reinterpret_cast<uintptr_t>(src) & 15) == 0);
  if (vec_ok && ld == k) {
    // contiguous tensor: plain linear indexing (no division per load), eight 16-byte loads in flight per thread
    const uint4* base = reinterpret_cast<const uint4*>(src);
    const int64_t total = rows * (k / 8);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i0 = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i0 < total; i0 += 8 * stride) {
      uint4 raw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = i0 + j * stride < total ? __ldg(base + i0 + j * stride) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m = max(m, (w[e] << 16) & 0x7FFFFFFFu);
          m = max(m, w[e] & 0x7FFF0000u);
        }
      }
    }
  } else if (vec_ok) {
    // four 16-byte loads in flight per thread
    const int64_t vec_per_row = k / 8;
    const int64_t total = rows * vec_per_row;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i0 = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i0 < total; i0 += 4 * stride) {
      uint4 raw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t i = i0 + j * stride;
        raw[j] = i < total ? __ldg(reinterpret_cast<const uint4*>(src + (i / vec_per_row) * ld + (i % vec_per_row) * 8))
                           : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m = max(m, (w[e] << 16) & 0x7FFFFFFFu);
          m = max(m, w[e] & 0x7FFF0000u);
        }
      }
    }
  } else {
    const int64_t total = rows * k;
    const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
      m = max(m, (static_cast<uint32_t>(s[(i / k) * ld + (i % k)]) << 16) & 0x7FFFFFFFu);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m != 0) atomicMax(amax_bits, m);
}

// Outer (per tensor / per region) decode scale from a |max| given as FP32 bits.
// mode 0: exact amax / (448 * 6); mode 1: the power of two 2^ceil(log2(max(amax / 2688, 2^-126))).
// 1.0 when amax is zero or NaN (the reference selects with `amax > 0`, rtx/fp4.py:343-365).
// The reference forms the quotient in two ways and both are kept bit for bit:
//   kernel_form = false  division, as its PyTorch functions do for the `current` policy and for
//                        quantize_nvfp4 (rtx/fp4.py:346, 361);
//   kernel_form = true   multiplication by the FP32 constant 1/2688, as its quantizer kernels do for
//                        the delayed and row-region policies (rtx/kernels/nvfp4_quant.py:117-143).
// The power of two comes from the exponent-bump rule of those kernels; on every BF16 magnitude it
// equals the PyTorch exp2(ceil(log2(t))) form (checked exhaustively against the reference's function).
__device__ __forceinline__ float nvfp4_scale_from_amax_bits(uint32_t amax_bits, int mode, bool kernel_form = false) {
  const float amax = __uint_as_float(amax_bits);
  const float quotient = kernel_form ? __fmul_rn(amax, 1.0f / 2688.0f) : __fdiv_rn(amax, 2688.0f);
  float s;
  if (mode == 0) {
    s = quotient;
  } else {
    const float target = fmax_nan(quotient, 1.17549435e-38f);
    const uint32_t bits = __float_as_uint(target);
    uint32_t ebits = bits & 0x7F800000u;
    if (bits & 0x007FFFFFu) ebits += 1u << 23;
    s = __uint_as_float(ebits);
  }
  if (!(amax > 0.0f)) s = 1.0f;
  return s;
}

__global__ void nvfp4_tensor_scale_kernel(const uint32_t* amax_bits, int mode, float* scale, const float* other_scale,
                                          float* out_scale, bool kernel_form) {
  const float s = nvfp4_scale_from_amax_bits(*amax_bits, mode, kernel_form);
  *scale = s;
  if (out_scale) *out_scale = s * *other_scale;
}

// ---------------------------------------------------------------------------
// NVFP4: src bf16 [rows, k] -> packed e2m1 [rows, kp/2] (kp = k rounded up to
// 32), E4M3 block scale per 16 values; a thread owns one whole block of 16
// values (two 16-byte loads, one 8-byte store).
// ---------------------------------------------------------------------------
struct QuantNvParams {
  const __nv_bfloat16* src;
  uint8_t* q;
  uint8_t* scales;
  const float* tensor_scale;  // device scalar, nullptr = 1.0 (block policy)
  const float* region_scales; // row-region policy: outer scale of rows [i * region_rows, (i + 1) * region_rows)
  int region_rows;            // 0 = one scale for the tensor (tensor_scale)
  int rows, k, kp;
  int64_t ld;
  int nb;         // kp / 16
  int sf_chunks;  // 512-byte tiles per 128 rows
  int layout;
};

// Tile = 128 rows x 256 columns (16 blocks = four 512-byte scale tiles).  Thread t owns the
// block (t & 15) of row (t >> 4) + 16 i; the loads of two rows (four 16-byte loads) are issued
// before the first is consumed.
struct QuantNvTileCtx {
  int sub, rsel, col_tiles, row_bytes;
  bool vec_ok;
  float six_st, inv_st;
};

__device__ __forceinline__ QuantNvTileCtx quant_nvfp4_ctx(const QuantNvParams& p, float st) {
  QuantNvTileCtx c;
  c.sub = threadIdx.x & 15;
  c.rsel = threadIdx.x >> 4;
  c.col_tiles = (p.kp + 255) / 256;
  c.row_bytes = p.kp / 2;
  c.vec_ok = (p.ld % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.src) & 15) == 0);
  c.six_st = 6.0f * st;
  c.inv_st = __fdiv_rn(1.0f, st);
  return c;
}

// one 128 x 256 tile: payload bytes and the tile's scale bytes (block-wide: ends with a barrier).
// REGION: the outer scale is looked up per row (row-region policy) instead of being one per tensor.
template <bool REGION = false, bool OBSERVE = false>
__device__ __forceinline__ void quant_nvfp4_tile(const QuantNvParams& p, const QuantNvTileCtx& c, int tile,
                                                 uint8_t (*tile_scales)[16], const float2* row_factors = nullptr,
                                                 float* observed = nullptr) {
  // OBSERVE: *observed accumulates the |max| of everything this thread quantizes (delayed policy)
  // row_factors (REGION): per row of the tile {6 * scale, 1 / scale} of the row's region, in shared memory
  const int row0 = (tile / c.col_tiles) * 128;
  const int col = (tile % c.col_tiles) * 256 + c.sub * 16;
  const bool col_ok = col < p.kp;
#pragma unroll
  for (int pair = 0; pair < 4; ++pair) {
    uint4 raw[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = row0 + c.rsel + 16 * (pair * 2 + j);
      if (row < p.rows && col_ok) {
        const __nv_bfloat16* rp = p.src + static_cast<int64_t>(row) * p.ld;
        raw[j][0] = load8_raw(rp, col, p.k, c.vec_ok);
        raw[j][1] = load8_raw(rp, col + 8, p.k, c.vec_ok);
      } else {
        raw[j][0] = raw[j][1] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = c.rsel + 16 * (pair * 2 + j);
      const int row = row0 + r;
      const bool live = row < p.rows && col_ok;
      float v[16];
      unpack8(raw[j][0], *reinterpret_cast<float(*)[8]>(&v[0]));
      unpack8(raw[j][1], *reinterpret_cast<float(*)[8]>(&v[8]));
      float a = fabsf(v[0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) a = fmax_nan(a, fabsf(v[e]));
      if (OBSERVE) *observed = fmax_nan(*observed, a);
      float six_st = c.six_st, inv_st = c.inv_st;
      if (REGION) {
        const float2 f = row_factors[r];
        six_st = f.x;
        inv_st = f.y;
      }
      float rawscale = __fdiv_rn(a, six_st);
      rawscale = fmin_nan(fmax_nan(rawscale, 0.015625f), 448.0f);
      const uint32_t sb = cvt_e4m3x2(rawscale, rawscale) & 0xFF;
      const float recip = __fdiv_rn(inv_st, e4m3_to_float(sb));
      tile_scales[r][c.sub] = live ? static_cast<uint8_t>(sb) : 0;
      if (live) {
        uint32_t w0 = 0, w1 = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w0 |= cvt_e2m1x2(v[2 * e] * recip, v[2 * e + 1] * recip) << (8 * e);
          w1 |= cvt_e2m1x2(v[8 + 2 * e] * recip, v[8 + 2 * e + 1] * recip) << (8 * e);
        }
        *reinterpret_cast<uint2*>(p.q + static_cast<int64_t>(row) * c.row_bytes + col / 2) = make_uint2(w0, w1);
      }
    }
  }
  __syncthreads();
  store_scale_tile<16>(tile_scales, p.scales, p.layout, row0, (tile % c.col_tiles) * 16, p.rows, p.nb, p.sf_chunks);
  __syncthreads();
}

__global__ void __launch_bounds__(kQuantThreads, 4) quant_nvfp4_rows_kernel(const QuantNvParams p) {
  __shared__ __align__(16) uint8_t tile_scales[128][16];
  const float st = p.tensor_scale ? __ldg(p.tensor_scale) : 1.0f;
  const QuantNvTileCtx c = quant_nvfp4_ctx(p, st);
  const int row_tiles = (p.rows + 127) / 128;
  for (int tile = blockIdx.x; tile < c.col_tiles * row_tiles; tile += gridDim.x) quant_nvfp4_tile(p, c, tile, tile_scales);
}

// ---------------------------------------------------------------------------
// Delayed policy (NVFP4DelayedDualQuantKernel, rtx/kernels/nvfp4_quant.py:473-664): the outer scale
// comes from the |max| history of earlier steps (history[0] = most recent; the window maximum or only
// the most recent entry), and the same single read of the tensor both quantizes it with that scale
// and observes its |max|, published as next_history[0]; next_history[i] = history[i - 1].  No
// reduction over the current tensor stands before the quantization.  next_history[0] must be zero
// when the kernel starts (the entry point clears it).
// ---------------------------------------------------------------------------
struct QuantNvDelayedParams {
  QuantNvParams q;            // q.tensor_scale / region fields are not read
  const float* history;       // [history_len]
  float* next_history;        // [history_len]
  int history_len, entries;   // entries read for the scale: history_len (window_max) or 1 (most_recent)
  int mode;
  float* scale_out;           // [1] the scale used
  const float* other_scale;   // nullptr or [1]
  float* out_scale;           // nullptr or [1] = scale * other_scale
};

__global__ void __launch_bounds__(kQuantThreads, 4) quant_nvfp4_delayed_kernel(const QuantNvDelayedParams dp) {
  __shared__ __align__(16) uint8_t tile_scales[128][16];
  __shared__ uint32_t prior_bits;
  const QuantNvParams& p = dp.q;
  if (threadIdx.x < 32) {
    uint32_t m = 0;
    for (int i = threadIdx.x; i < dp.entries; i += 32) m = max(m, __float_as_uint(__ldg(dp.history + i)) & 0x7FFFFFFFu);
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x == 0) prior_bits = m;
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x + 1; i < dp.history_len; i += 32) dp.next_history[i] = __ldg(dp.history + i - 1);
    }
  }
  __syncthreads();
  const float st = nvfp4_scale_from_amax_bits(prior_bits, dp.mode, true);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *dp.scale_out = st;
    if (dp.out_scale) *dp.out_scale = st * *dp.other_scale;
  }
  const QuantNvTileCtx c = quant_nvfp4_ctx(p, st);
  const int row_tiles = (p.rows + 127) / 128;
  float observed = 0.0f;
  for (int tile = blockIdx.x; tile < c.col_tiles * row_tiles; tile += gridDim.x)
    quant_nvfp4_tile<false, true>(p, c, tile, tile_scales, nullptr, &observed);
  uint32_t obs = __float_as_uint(observed) & 0x7FFFFFFFu;   // NaN keeps a pattern above infinity
  obs = __reduce_max_sync(0xffffffffu, obs);
  if ((threadIdx.x & 31) == 0 && obs != 0) atomicMax(reinterpret_cast<uint32_t*>(dp.next_history), obs);
}

// ---------------------------------------------------------------------------
// Row-region policy (the reference's default NVFP4 scaling, NVFP4JITRegionDualQuantKernel,
// rtx/kernels/nvfp4_quant.py:667-1000): one FP32 outer scale per region of `region_rows` consecutive
// rows, from the region's current |max|.  Here: one warp reduces a region and applies the scale rule
// (amax_regions_kernel), then the tiled quantizer looks the scale up per row.
// ---------------------------------------------------------------------------
// |max| bits of one region (region_rows rows of k values), reduced by one warp
__device__ __forceinline__ uint32_t amax_region_warp(const __nv_bfloat16* src, int k, int64_t ld, int region_rows, int region,
                                                     int lane, bool vec_ok) {
  uint32_t m = 0;
  if (vec_ok && ld == k) {
    // contiguous region: one flat range, eight 16-byte loads in flight per lane (a region of a small layer is a few
    // tens of kilobytes read by ONE warp: the number of dependent load rounds is its whole cost)
    const uint4* base = reinterpret_cast<const uint4*>(src + static_cast<int64_t>(region) * region_rows * ld);
    const int vecs = region_rows * (k / 8);
    for (int i0 = lane; i0 < vecs; i0 += 256) {
      uint4 raw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = i0 + 32 * j < vecs ? __ldg(base + i0 + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m = max(m, (w[e] << 16) & 0x7FFFFFFFu);
          m = max(m, w[e] & 0x7FFF0000u);
        }
      }
    }
    return __reduce_max_sync(0xffffffffu, m);
  }
  for (int r = 0; r < region_rows; ++r) {
    const __nv_bfloat16* rp = src + static_cast<int64_t>(region * region_rows + r) * ld;
    if (vec_ok) {
      const int vecs = k / 8;
      for (int i0 = lane; i0 < vecs; i0 += 128) {   // four 16-byte loads in flight per lane
        uint4 raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          raw[j] = i0 + 32 * j < vecs ? __ldg(reinterpret_cast<const uint4*>(rp) + i0 + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            m = max(m, (w[e] << 16) & 0x7FFFFFFFu);
            m = max(m, w[e] & 0x7FFF0000u);
          }
        }
      }
    } else {
      const uint16_t* sp = reinterpret_cast<const uint16_t*>(rp);
      for (int i = lane; i < k; i += 32) m = max(m, (static_cast<uint32_t>(sp[i]) << 16) & 0x7FFFFFFFu);
    }
  }
  return __reduce_max_sync(0xffffffffu, m);
}

__global__ void __launch_bounds__(256) amax_regions_kernel(const __nv_bfloat16* src, int rows, int k, int64_t ld,
                                                           int region_rows, int mode, float* region_scales) {
  const int regions = rows / region_rows;
  const int lane = threadIdx.x & 31;
  const int warps = (gridDim.x * blockDim.x) >> 5;
  const bool vec_ok = (ld % 8 == 0) && (k % 8 == 0) && ((reinterpret_cast<uintptr_t>(src) & 15) == 0);
  for (int region = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; region < regions; region += warps) {
    const uint32_t m = amax_region_warp(src, k, ld, region_rows, region, lane, vec_ok);
    if (lane == 0) region_scales[region] = nvfp4_scale_from_amax_bits(m, mode, true);
  }
}

// Region scales of two tensors with the same k (activations and weight of a dynamic forward) in one launch: on
// small layers the launches cost more than the reductions.
struct RegionScaleJob {
  const __nv_bfloat16* src;
  float* region_scales;
  int rows, region_rows;
  int64_t ld;
};
__global__ void __launch_bounds__(256) amax_regions2_kernel(const RegionScaleJob a, const RegionScaleJob b, int k, int mode) {
  griddep_launch_dependents();
  const int regions_a = a.rows / a.region_rows, regions_b = b.rows / b.region_rows;
  const int lane = threadIdx.x & 31;
  const int warps = (gridDim.x * blockDim.x) >> 5;
  for (int idx = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; idx < regions_a + regions_b; idx += warps) {
    const RegionScaleJob& j = idx < regions_a ? a : b;
    const int region = idx < regions_a ? idx : idx - regions_a;
    const bool vec_ok = (j.ld % 8 == 0) && (k % 8 == 0) && ((reinterpret_cast<uintptr_t>(j.src) & 15) == 0);
    const uint32_t m = amax_region_warp(j.src, k, j.ld, j.region_rows, region, lane, vec_ok);
    if (lane == 0) j.region_scales[region] = nvfp4_scale_from_amax_bits(m, mode, true);
  }
}

// The same reduction with a whole CTA per region, for regions large enough to keep 256 threads busy
// (a region is contiguous when ld == k: the threads then stride over it as one flat range).
__global__ void __launch_bounds__(256) amax_regions_cta_kernel(const __nv_bfloat16* src, int rows, int k, int64_t ld,
                                                               int region_rows, int mode, float* region_scales) {
  __shared__ uint32_t warp_max[8];
  const int regions = rows / region_rows;
  const bool flat = (ld == k) && (k % 8 == 0) && ((reinterpret_cast<uintptr_t>(src) & 15) == 0);
  for (int region = blockIdx.x; region < regions; region += gridDim.x) {
    uint32_t m = 0;
    if (flat) {
      const uint4* base = reinterpret_cast<const uint4*>(src + static_cast<int64_t>(region) * region_rows * ld);
      const int vecs = region_rows * (k / 8);
      for (int i0 = threadIdx.x; i0 < vecs; i0 += 4 * 256) {
        uint4 raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = i0 + 256 * j < vecs ? __ldg(base + i0 + 256 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            m = max(m, (w[e] << 16) & 0x7FFFFFFFu);
            m = max(m, w[e] & 0x7FFF0000u);
          }
        }
      }
    } else {
      const uint16_t* sp = reinterpret_cast<const uint16_t*>(src);
      const int64_t total = static_cast<int64_t>(region_rows) * k;
      for (int64_t i = threadIdx.x; i < total; i += 256) {
        const int64_t row = region * static_cast<int64_t>(region_rows) + i / k;
        m = max(m, (static_cast<uint32_t>(sp[row * ld + i % k]) << 16) & 0x7FFFFFFFu);
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
      uint32_t v = threadIdx.x < 8 ? warp_max[threadIdx.x] : 0u;
      v = __reduce_max_sync(0xffffffffu, v);
      if (threadIdx.x == 0) region_scales[region] = nvfp4_scale_from_amax_bits(v, mode, true);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kQuantThreads, 4) quant_nvfp4_regions_kernel(const QuantNvParams p) {
  __shared__ __align__(16) uint8_t tile_scales[128][16];
  __shared__ float2 row_factors[128];
  const QuantNvTileCtx c = quant_nvfp4_ctx(p, 1.0f);
  const int row_tiles = (p.rows + 127) / 128;
  int table_row0 = -1;
  for (int tile = blockIdx.x; tile < c.col_tiles * row_tiles; tile += gridDim.x) {
    const int row0 = (tile / c.col_tiles) * 128;
    if (row0 != table_row0) {
      // the 128 rows of this tile: look the region scale up once per row, not once per block of 16 values
      if (threadIdx.x < 128) {
        const int row = row0 + threadIdx.x;
        const float st = row < p.rows ? __ldg(p.region_scales + row / p.region_rows) : 1.0f;
        row_factors[threadIdx.x] = make_float2(6.0f * st, __fdiv_rn(1.0f, st));
      }
      table_row0 = row0;
      __syncthreads();
    }
    quant_nvfp4_tile<true>(p, c, tile, tile_scales, row_factors);   // ends with a block-wide barrier
  }
}

// Two tensors in one launch (tiles of `a`, then tiles of `b`), launched as a programmatic dependent of
// amax_regions2_kernel: it waits for that grid before it reads a region scale.
__global__ void __launch_bounds__(kQuantThreads, 4) quant_nvfp4_regions2_kernel(const QuantNvParams a, const QuantNvParams b) {
  __shared__ __align__(16) uint8_t tile_scales[128][16];
  __shared__ float2 row_factors[128];
  griddep_launch_dependents();
  const QuantNvTileCtx ca = quant_nvfp4_ctx(a, 1.0f), cb = quant_nvfp4_ctx(b, 1.0f);
  const int tiles_a = ca.col_tiles * ((a.rows + 127) / 128), tiles_b = cb.col_tiles * ((b.rows + 127) / 128);
  griddep_wait();
  int table_key = -1;
  for (int idx = blockIdx.x; idx < tiles_a + tiles_b; idx += gridDim.x) {
    const bool first = idx < tiles_a;
    const QuantNvParams& p = first ? a : b;
    const QuantNvTileCtx& c = first ? ca : cb;
    const int tile = first ? idx : idx - tiles_a;
    const int row0 = (tile / c.col_tiles) * 128;
    const int key = 2 * row0 + (first ? 0 : 1);
    if (key != table_key) {
      if (threadIdx.x < 128) {
        const int row = row0 + threadIdx.x;
        const float st = row < p.rows ? __ldg(p.region_scales + row / p.region_rows) : 1.0f;
        row_factors[threadIdx.x] = make_float2(6.0f * st, __fdiv_rn(1.0f, st));
      }
      table_key = key;
      __syncthreads();
    }
    quant_nvfp4_tile<true>(p, c, tile, tile_scales, row_factors);   // ends with a block-wide barrier
  }
}

// ---------------------------------------------------------------------------
// Small tensors (decode activations): the outer scale from the tensor's own |max| and the
// quantization as two launches chained by programmatic dependent launch, with no memset and no
// one-thread finalize launch in between:
//   amax_partials_kernel     CTA p writes the |max| bits of tiles p, p + P, ... to partials[p]
//   quant_nvfp4_dynamic_kernel  every CTA reduces the P partials itself, applies the scale rule
//                            (all CTAs get the same bits), CTA 0 publishes the scale(s), then the
//                            tiles are quantized with the code of the two-pass path.
// Both let their dependents start early (griddepcontrol.launch_dependents first thing) and wait
// for their own predecessor before touching global memory that it may still use.
// Replaces, for small M, the reference's torch reductions of `_outer_tensor_scale`
// (rtx/fp4.py:343-365) followed by compile_nvfp4_quant (rtx/kernels/nvfp4_quant.py:32-349).
// ---------------------------------------------------------------------------
constexpr int kDynamicMaxPartials = 64;

__global__ void __launch_bounds__(kQuantThreads) amax_partials_kernel(const QuantNvParams p, uint32_t* partials) {
  __shared__ uint32_t cta_amax;
  griddep_launch_dependents();
  if (threadIdx.x == 0) cta_amax = 0;
  griddep_wait();   // src may be the output of the kernel before this one; partials may still be read by it
  __syncthreads();
  const QuantNvTileCtx c = quant_nvfp4_ctx(p, 1.0f);
  const int tiles = c.col_tiles * ((p.rows + 127) / 128);
  uint32_t m = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int row0 = (tile / c.col_tiles) * 128;
    const int col = (tile % c.col_tiles) * 256 + c.sub * 16;
    if (col >= p.kp) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + c.rsel + 16 * i;
      if (row >= p.rows) continue;
      const __nv_bfloat16* rp = p.src + static_cast<int64_t>(row) * p.ld;
      const uint4 a = load8_raw(rp, col, p.k, c.vec_ok), b = load8_raw(rp, col + 8, p.k, c.vec_ok);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m = max(m, (w[e] << 16) & 0x7FFFFFFFu);
        m = max(m, w[e] & 0x7FFF0000u);
      }
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m != 0) atomicMax(&cta_amax, m);
  __syncthreads();
  if (threadIdx.x == 0) partials[blockIdx.x] = cta_amax;
}

struct QuantNvDynamicParams {
  QuantNvParams q;           // q.tensor_scale is not read
  int mode;                  // 0 exact, 1 power of two
  const uint32_t* partials;  // [n_partials] |max| bits
  int n_partials;            // <= kDynamicMaxPartials
  float* scale_out;          // [1]
  const float* other_scale;  // nullptr or [1]
  float* out_scale;          // nullptr or [1] = scale * other_scale
};

__global__ void __launch_bounds__(kQuantThreads, 4) quant_nvfp4_dynamic_kernel(const QuantNvDynamicParams dp) {
  __shared__ __align__(16) uint8_t tile_scales[128][16];
  __shared__ uint32_t warp_amax[2];
  griddep_launch_dependents();
  griddep_wait();
  const QuantNvParams& p = dp.q;
  if (threadIdx.x < 64) {
    uint32_t v = threadIdx.x < dp.n_partials ? dp.partials[threadIdx.x] : 0u;
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) warp_amax[threadIdx.x >> 5] = v;
  }
  __syncthreads();
  const float st = nvfp4_scale_from_amax_bits(max(warp_amax[0], warp_amax[1]), dp.mode);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *dp.scale_out = st;
    if (dp.out_scale) *dp.out_scale = st * *dp.other_scale;
  }
  const QuantNvTileCtx c = quant_nvfp4_ctx(p, st);
  const int tiles = c.col_tiles * ((p.rows + 127) / 128);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) quant_nvfp4_tile(p, c, tile, tile_scales);
}

}  // namespace rtxb
