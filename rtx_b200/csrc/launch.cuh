// Host-side launch support shared by the library's translation units: error detail, tensor-map encoding,
// launch attributes, SM count, workspace carving.
#pragma once

#include "../../include/rtxb.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <vector>

namespace rtxb {

int set_last_error(int code, const char* msg);   // api.cu: the text behind rtxb_last_cuda_error()

inline int fail_msg(int code, const char* msg) { return set_last_error(code, msg); }
inline int fail_cuda(cudaError_t e, const char* where) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", where, cudaGetErrorString(e));
  return set_last_error(RTXB_E_CUDA, msg);
}

#define RTXB_CHECK_LAUNCH(where)                                \
  do {                                                          \
    cudaError_t e__ = cudaGetLastError();                       \
    if (e__ != cudaSuccess) return fail_cuda(e__, where);       \
  } while (0)

inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// ---- driver entry point for tensor-map encoding (no link-time libcuda) ----
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// ---- tensor maps --------------------------------------------------------------------------------
// A tensor map is a pure function of the base address, extents, strides and box, so encoded maps are
// kept in a small per-thread table and re-used by later launches on the same buffers (a decode step
// launches in microseconds; two to four driver encodes per launch were a visible part of that).
struct MapKey {
  const void* base;
  uint64_t dim[3];
  uint64_t stride[2];   // bytes, dimensions 1 and 2
  uint32_t box[3];
  uint32_t rank;        // 2 or 3
  uint32_t words;       // 0: bytes with the 128-byte swizzle (payload); 1: 32-bit words, no swizzle (scale tiles);
                        // 2 / 3: 16-bit / 32-bit elements with the 64-byte swizzle (output tiles of the epilogue)
};

struct MapSlot {
  MapKey key;
  CUtensorMap map;
  bool valid;
};

constexpr int kMapSlots = 256;
inline thread_local MapSlot t_map_cache[kMapSlots];

inline int encode_map(CUtensorMap* out, const MapKey& key, const char* what) {
  // every word of the key (blank_key cleared its padding) enters the slot number: the maps of one launch differ in the
  // box height or the base alone, and two of them in one slot would be encoded anew at every call
  static_assert(sizeof(MapKey) % 8 == 0, "the key is hashed in 64-bit words");
  uint64_t words[sizeof(MapKey) / 8], h = 0;
  memcpy(words, &key, sizeof(MapKey));
  for (uint64_t w : words) {
    h = (h ^ w) * 0x9E3779B97F4A7C15ull;
    h ^= h >> 29;
  }
  MapSlot& slot = t_map_cache[(h >> 32) % kMapSlots];
  if (slot.valid && memcmp(&slot.key, &key, sizeof(MapKey)) == 0) {
    *out = slot.map;
    return RTXB_OK;
  }
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail_msg(RTXB_E_DRIVER, "cuTensorMapEncodeTiled entry point not available");
  cuuint64_t gdim[3] = {key.dim[0], key.dim[1], key.dim[2]};
  cuuint64_t gstride[2] = {key.stride[0], key.stride[1]};
  cuuint32_t box[3] = {key.box[0], key.box[1], key.box[2]};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  static const CUtensorMapDataType kTypes[5] = {CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_DATA_TYPE_UINT32,
                                               CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_DATA_TYPE_UINT32,
                                               CU_TENSOR_MAP_DATA_TYPE_UINT32};
  static const CUtensorMapSwizzle kSwizzles[5] = {CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_SWIZZLE_NONE,
                                                  CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_SWIZZLE_64B,
                                                  CU_TENSOR_MAP_SWIZZLE_128B};
  const int kind = key.words < 5 ? key.words : 0;
  CUresult r = fn(out, kTypes[kind], key.rank, const_cast<void*>(key.base), gdim, gstride, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, kSwizzles[kind], CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char msg[128];
    snprintf(msg, sizeof(msg), "cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, static_cast<int>(r));
    return fail_msg(RTXB_E_DRIVER, msg);
  }
  slot.key = key;
  slot.map = *out;
  slot.valid = true;
  return RTXB_OK;
}

inline MapKey blank_key(const void* base) {
  MapKey k;
  memset(&k, 0, sizeof(k));   // padding bytes too: keys are compared with memcmp
  k.base = base;
  return k;
}

// byte matrix [rows, row_bytes] (pitch row_bytes), boxes of 128 bytes x box_rows, 128-byte swizzle,
// out-of-range elements read as zero
inline int make_payload_map(CUtensorMap* map, const void* base, int64_t rows, int64_t row_bytes, int box_rows) {
  if (!aligned(base, 16) || row_bytes % 16 != 0) return fail_msg(RTXB_E_ALIGNMENT, "payload must be 16-byte aligned");
  MapKey k = blank_key(base);
  k.rank = 2;
  k.dim[0] = static_cast<uint64_t>(row_bytes);
  k.dim[1] = static_cast<uint64_t>(rows);
  k.stride[0] = static_cast<uint64_t>(row_bytes);
  k.box[0] = 128u;
  k.box[1] = static_cast<uint32_t>(box_rows);
  return encode_map(map, k, "payload");
}

// the same byte matrix viewed as [row_bytes / 128][rows][128]: boxes of `box_k` consecutive 128-byte
// K chunks x box_rows rows, each chunk landing as its own swizzled tile.  Needs row_bytes % 128 == 0
// (otherwise the last chunk of a row would run into the next row instead of reading zeros).
inline int make_payload_map_ksteps(CUtensorMap* map, const void* base, int64_t rows, int64_t row_bytes, int box_rows,
                            int box_k) {
  if (!aligned(base, 16) || row_bytes % 128 != 0) return fail_msg(RTXB_E_ALIGNMENT, "payload rows must be 128-byte multiples");
  MapKey k = blank_key(base);
  k.rank = 3;
  k.dim[0] = 128u;
  k.dim[1] = static_cast<uint64_t>(rows);
  k.dim[2] = static_cast<uint64_t>(row_bytes / 128);
  k.stride[0] = static_cast<uint64_t>(row_bytes);
  k.stride[1] = 128u;
  k.box[0] = 128u;
  k.box[1] = static_cast<uint32_t>(box_rows);
  k.box[2] = static_cast<uint32_t>(box_k);
  return encode_map(map, k, "payload K steps");
}

// scale tiles as a matrix of 512-byte rows (128 x uint32), boxes of `box_rows` consecutive tiles
inline int make_scale_map(CUtensorMap* map, const void* base, int64_t total_tiles, int box_rows) {
  MapKey k = blank_key(base);
  k.rank = 2;
  k.words = 1;
  k.dim[0] = 128u;
  k.dim[1] = static_cast<uint64_t>(total_tiles);
  k.stride[0] = 512u;
  k.box[0] = 128u;
  k.box[1] = static_cast<uint32_t>(box_rows);
  return encode_map(map, k, "scales");
}

// scale tiles of B for the pair kernel: [2 halves][rows = 512-byte tiles][128 words], the second half
// `delta_tiles` tiles after the first, so one box brings the tiles of both 128-row blocks behind a
// 256-wide accumulator tile.  Rows are limited to those whose second half lies inside the buffer.
inline int make_scale_map_halves(CUtensorMap* map, const void* base, int64_t total_tiles, int box_rows, int64_t delta_tiles) {
  MapKey k = blank_key(base);
  k.rank = 3;
  k.words = 1;
  k.dim[0] = 128u;
  k.dim[1] = static_cast<uint64_t>(total_tiles - delta_tiles);
  k.dim[2] = 2u;
  k.stride[0] = 512u;
  k.stride[1] = static_cast<uint64_t>(delta_tiles) * 512u;
  k.box[0] = 128u;
  k.box[1] = static_cast<uint32_t>(box_rows);
  k.box[2] = 2u;
  return encode_map(map, k, "scale halves");
}

// output matrix [rows, cols] of 2- or 4-byte elements, row pitch ldo elements; one box = the 32 rows x 32 columns an
// epilogue warp stages per store: 64-byte rows with the 64-byte swizzle (BF16), 128-byte rows with the 128-byte
// swizzle (FP32: whole 128-byte lines, also over NVLink); stores are clipped at the edges
inline int make_out_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ldo, int elem_bytes) {
  MapKey k = blank_key(base);
  k.rank = 2;
  k.words = elem_bytes == 2 ? 2 : 4;
  k.dim[0] = static_cast<uint64_t>(cols);
  k.dim[1] = static_cast<uint64_t>(rows);
  k.stride[0] = static_cast<uint64_t>(ldo) * elem_bytes;
  k.box[0] = 32u;
  k.box[1] = 32u;
  return encode_map(map, k, "output");
}

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per kernel and device instead of per launch
inline cudaError_t ensure_dynamic_smem(const void* kernel, int bytes) {
  struct Done { const void* kernel; int device; int bytes; };
  static std::mutex mu;
  static std::vector<Done> done;
  thread_local Done last = {nullptr, -1, 0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (last.kernel == kernel && last.device == dev && last.bytes >= bytes) return cudaSuccess;
  {
    std::lock_guard<std::mutex> lock(mu);
    for (const Done& d : done)
      if (d.kernel == kernel && d.device == dev && d.bytes >= bytes) {
        last = d;
        return cudaSuccess;
      }
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    done.push_back({kernel, dev, bytes});
    last = done.back();
  }
  return cudaSuccess;
}

// SMs the persistent kernels leave free (for a collective that runs beside them); process-wide
inline std::atomic<int> g_sm_margin{0};

inline int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  int n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) {
    if (cached[dev] == 0) {
      int q = 0;
      if (cudaDeviceGetAttribute(&q, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || q <= 0) q = 148;
      cached[dev] = q;
    }
    n = cached[dev];
  }
  const int usable = n - g_sm_margin.load(std::memory_order_relaxed);
  return usable < 2 ? 2 : usable;
}

// launch `kernel` so that it may start while the kernel before it on the stream is still running
// (both sides use griddepcontrol to order their memory accesses)
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t stream,
                             bool dependent, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// grid-stride kernels: one wave of resident CTAs (per_sm = CTAs that fit one SM).  Fewer CTAs with equal tile
// counts (no straggler round) were measured slower: these kernels are bound by the loads in flight, and 8 %
// fewer CTAs cost 8 % of the rate (row quantizer 41.5 against 37.6 us on 16384 x 4096).
inline int quant_grid(int64_t tiles, int per_sm) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(tiles < cap ? (tiles > 0 ? tiles : 1) : cap);
}

struct Carver {
  uint8_t* base;
  size_t off = 0;
  explicit Carver(void* p) : base(static_cast<uint8_t*>(p)) {}
  uint8_t* take(size_t bytes) {
    uint8_t* r = base ? base + off : nullptr;
    off += static_cast<size_t>(round_up(static_cast<int64_t>(bytes), 256));
    return r;
  }
};

}  // namespace rtxb
