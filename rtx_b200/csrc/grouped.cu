// extern "C" entry points of the grouped (experts') MXFP8 linear: argument checks, workspace layout, launches.
#include "launch.cuh"
#include "gemm_grouped.cuh"
#include "grouped.cuh"

using namespace rtxb;

namespace rtxb {

int launch_quantize_rows(RowsParams& p, int64_t x_tiles, int64_t k, int rounding, cudaStream_t stream) {
  p.k = static_cast<int>(k);
  p.kp = static_cast<int>(round_up(k, 32));
  p.chunks = static_cast<int>((p.kp / 32 + 3) / 4);
  p.lanes = 4;
  while (p.lanes < 32 && p.lanes < p.kp / 32) p.lanes *= 2;
  p.round_to_infinity = rounding != RTXB_ROUND_FLOOR;
  p.stacked = 32 / p.lanes;
  p.segs = (4 * p.chunks + p.lanes - 1) / p.lanes;
  p.per_tile = p.lanes * p.segs;
  p.w_row_tiles = (p.w.rows + 127) / 128;
  for (RowsOperand* o : {&p.x, &p.w}) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(o->src) | static_cast<uintptr_t>(o->ld * 2);
    o->align = a % 32 == 0 ? 2 : a % 16 == 0 ? 1 : 0;
    const int64_t rows = o == &p.w ? static_cast<int64_t>(p.batches) * o->rows : o->rows;
    o->end = o->src ? o->src + (rows - 1) * o->ld + k : nullptr;
  }
  const int64_t w_tiles = p.w.src ? static_cast<int64_t>(p.batches) * p.w_row_tiles : 0;
  const int64_t units = (x_tiles + w_tiles) * p.per_tile;
  if (units > INT32_MAX) return fail_msg(RTXB_E_UNSUPPORTED, "operand exceeds the 32-bit unit count of the quantizer");
  quant_mxfp8_rows_units_kernel<<<quant_grid((units + 7) / 8, kRowsOccupancy), kQuantThreads, 0, stream>>>(p);
  RTXB_CHECK_LAUNCH("quant_mxfp8_rows_units_kernel");
  return RTXB_OK;
}

int launch_quantize_transposed(TransposedParams& p, int64_t x_tiles, cudaStream_t stream) {
  p.x_col_units = (p.x.cols + 63) / 64;
  p.w_col_units = (p.w.cols + 63) / 64;
  p.w_row_tiles = (p.w.rows + 127) / 128;
  const bool gradient = p.dy.src != nullptr;
  p.dy_col_units = (p.dy.cols + 63) / 64;
  const int64_t units = (gradient ? x_tiles * p.dy_col_units : 0) + (p.x.src ? x_tiles * p.x_col_units : 0) +
                        (p.w.src ? static_cast<int64_t>(p.batches) * p.w_row_tiles * p.w_col_units : 0);
  if (units > INT32_MAX) return fail_msg(RTXB_E_UNSUPPORTED, "operand exceeds the 32-bit unit count of the quantizer");
  int64_t blocks = (units + 7) / 8;
  if (p.partial && blocks < (p.n + 31) / 32) blocks = (p.n + 31) / 32;
  auto kernel = gradient ? quant_mxfp8_transposed_units_kernel<true> : quant_mxfp8_transposed_units_kernel<false>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kTransposedSmemBytes);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(transposed quantizer)");
  e = launch_dependent(kernel, quant_grid(blocks, kTransposedOccupancy), kQuantThreads, kTransposedSmemBytes, stream, !gradient, p);
  if (e != cudaSuccess) return fail_cuda(e, "quant_mxfp8_transposed_units_kernel launch");
  return RTXB_OK;
}

}  // namespace rtxb

namespace {

// output [groups][rows][cols] of BF16, row pitch ldo and group pitch `group_elems` elements; boxes of 32 rows x 32
// columns in the 64-byte swizzle the epilogue stages
int make_out_map_groups(CUtensorMap* map, const void* base, int64_t groups, int64_t rows, int64_t cols, int64_t ldo,
                        int64_t group_elems) {
  MapKey k = blank_key(base);
  k.rank = 3;
  k.words = 2;
  k.dim[0] = static_cast<uint64_t>(cols);
  k.dim[1] = static_cast<uint64_t>(rows);
  k.dim[2] = static_cast<uint64_t>(groups);
  k.stride[0] = static_cast<uint64_t>(ldo) * 2;
  k.stride[1] = static_cast<uint64_t>(group_elems) * 2;
  k.box[0] = 32u;
  k.box[1] = 32u;
  k.box[2] = 1u;
  return encode_map(map, k, "grouped output");
}

// most 128-row (256-row) tiles that `groups` groups of `rows` rows in all can have: a started tile per group that has
// rows, beside the full ones
int64_t most_tiles(int64_t rows, int64_t groups, int64_t tile) { return rows / tile + (groups < rows ? groups : rows); }

// Rows per tile of the rows form.  A 256-row tile does the most per byte of A it fetches, but a small batch has too few of
// them to occupy the CTA pairs.  The host knows rows and groups, not the list: half a tile is counted for what is left of
// each group.  256 while those tiles fill three quarters of the pairs, 128 while its own fill half of them, else 64.
// Measured, microseconds per forward at 256 / 128 / 64 rows (packed weights where n allows):
//   256 rows, 1 group, 1024 x 4096        19.9 / 16.1 / 14.8       1003 rows, 7 groups, 1238 x 1000    19.0 / 16.4 / 16.6
//   512 rows, 4 groups, 1024 x 2048       16.1 / 13.6 / 13.1       2048 rows, 8 groups, 1024 x 1024    14.6 / 14.2 / 14.0
//   1024 rows, 1 group, 4096 x 4096       21.8 / 23.5 / 32.2       4096 rows, 8 groups, 2048 x 4096    44.9 / 48.4 / 67.5
int rows_per_tile(int64_t rows, int64_t groups, int64_t a_rows) {
  const int64_t pairs = sm_count() / 2, a_tiles = (a_rows + 255) / 256;
  auto tiles2 = [&](int64_t tile) { return (2 * rows / tile + (groups < rows ? groups : rows)) * a_tiles; };   // twice
  if (4 * tiles2(256) >= 6 * pairs) return 256;
  return tiles2(128) >= pairs ? 128 : 64;
}

struct Operand {
  const void* q;
  const void* s;
  int64_t rows;        // rows of its tensor map
  int64_t sf_tiles;    // 512-byte scale tiles in all
};

int launch_grouped(GroupedGemmParams p, const Operand& a, const Operand& b, int64_t row_bytes_a, int64_t row_bytes_b,
                   int64_t out_groups, int64_t out_rows, int64_t most, cudaStream_t stream) {
  using P = PairTraits<kKindMxfp8>;
  constexpr int KS = P::kStepsPerBarrierP;
  CUtensorMap map_a, map_sfa, map_sfb, map_out;
  GroupedMapsB maps_b;
  int rc;
  p.map3d = row_bytes_a % 128 == 0 && row_bytes_b % 128 == 0;
  if (p.map3d) rc = make_payload_map_ksteps(&map_a, a.q, a.rows, row_bytes_a, 128, KS);
  else rc = make_payload_map(&map_a, a.q, a.rows, row_bytes_a, 128);
  for (int i = 0; i < 4 && !rc; ++i) {
    if (p.map3d) rc = make_payload_map_ksteps(&maps_b.m[i], b.q, b.rows, row_bytes_b, 128 >> i, KS);
    else rc = make_payload_map(&maps_b.m[i], b.q, b.rows, row_bytes_b, 128 >> i);
  }
  if (rc || (rc = make_scale_map(&map_sfa, a.s, a.sf_tiles, KS)) || (rc = make_scale_map(&map_sfb, b.s, b.sf_tiles, KS)))
    return rc;
  p.tma_out = aligned(p.out, 16) && (p.ldo * 2) % 16 == 0;
  memset(&map_out, 0, sizeof(map_out));
  if (p.tma_out && (rc = make_out_map_groups(&map_out, p.out, out_groups, out_rows, p.out_cols, p.ldo,
                                             out_groups > 1 ? p.out_group : p.ldo * out_rows)))
    return rc;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(gemm_grouped_pair_kernel), P::kSmemBytes);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(grouped gemm)");
  const int64_t max_pairs = sm_count() / 2;
  const int pairs = static_cast<int>(most < max_pairs ? most : max_pairs);
  e = launch_dependent(gemm_grouped_pair_kernel, 2 * pairs, kGroupedThreads, P::kSmemBytes, stream, true, map_a, maps_b, map_sfa,
                       map_sfb, map_out, p);
  if (e != cudaSuccess) return fail_cuda(e, "gemm_grouped_pair_kernel launch");
  return RTXB_OK;
}

int check_grouped(const int* offsets, int64_t rows, int64_t n, int64_t k, int64_t groups) {
  if (!offsets) return fail_msg(RTXB_E_INVALID_ARGUMENT, "null offsets");
  if (!aligned(offsets, 4)) return fail_msg(RTXB_E_ALIGNMENT, "offsets must be int32 aligned");
  if (rows <= 0 || n <= 0 || k <= 0 || groups <= 0) return fail_msg(RTXB_E_INVALID_ARGUMENT, "rows, n, k, groups must be positive");
  if (groups > kMaxGroups) return fail_msg(RTXB_E_UNSUPPORTED, "at most 512 groups");
  // tile numbers, rows of the tensor maps and columns of the transposed operands are 32-bit
  const int64_t lim = INT32_MAX / 2;
  const int64_t rt = most_tiles(rows, groups, 128), nt = (n + 127) / 128, kt = (k + 127) / 128;
  if (rows > lim || n > lim || k > lim || groups * n > lim || groups * k > lim || rt * 128 > lim || rt * nt > lim ||
      rt * kt > lim || groups * nt * kt > lim)
    return fail_msg(RTXB_E_UNSUPPORTED, "grouped operand exceeds the 32-bit tile count");
  return RTXB_OK;
}

size_t scale_tiles_bytes(int64_t row_tiles, int64_t k) { return static_cast<size_t>(row_tiles * ((round_up(k, 32) / 32 + 3) / 4) * 512); }

// the plan in a workspace
struct PlanMemory {
  GroupPlan plan;
  PlanMemory(Carver& c, int64_t rows, int64_t groups) {
    plan.row_tiles = reinterpret_cast<int*>(c.take(16));
    plan.tiles = reinterpret_cast<int4*>(c.take(most_tiles(rows, groups, 64) * sizeof(int4)));   // the smallest tiles
    plan.k_tiles = reinterpret_cast<int*>(c.take((groups + 1) * sizeof(int)));
    plan.tile_rows = 256;
  }
};

struct FwdMemory {
  PlanMemory plan;
  uint8_t *qx, *sx, *qw, *sw;
  FwdMemory(Carver& c, int64_t rows, int64_t n, int64_t k, int64_t groups, bool dynamic_w) : plan(c, rows, groups) {
    qx = c.take(rows * round_up(k, 32));
    sx = c.take(scale_tiles_bytes(most_tiles(rows, groups, 128), k));
    qw = dynamic_w ? c.take(groups * n * round_up(k, 32)) : nullptr;
    sw = dynamic_w ? c.take(scale_tiles_bytes(groups * ((n + 127) / 128), k)) : nullptr;
  }
};

struct BwdMemory {
  PlanMemory plan;
  uint8_t *q_dy = nullptr, *s_dy = nullptr, *q_wt = nullptr, *s_wt = nullptr;   // dX
  uint8_t *q_dyt = nullptr, *s_dyt = nullptr, *q_xt = nullptr, *s_xt = nullptr; // dW
  BwdMemory(Carver& c, int64_t rows, int64_t n, int64_t k, int64_t groups, bool need_dx, bool need_dw)
      : plan(c, rows, groups) {
    const int64_t tiles = most_tiles(rows, groups, 128);
    if (need_dx) {
      q_dy = c.take(rows * round_up(n, 32));
      s_dy = c.take(scale_tiles_bytes(tiles, n));
      q_wt = c.take(groups * k * round_up(n, 32));
      s_wt = c.take(scale_tiles_bytes(groups * ((k + 127) / 128), n));
    }
    if (need_dw) {
      q_dyt = c.take(n * tiles * 128);
      s_dyt = c.take((n + 127) / 128 * tiles * 512);
      q_xt = c.take(k * tiles * 128);
      s_xt = c.take((k + 127) / 128 * tiles * 512);
    }
  }
};

GroupedGemmParams gemm_params(const GroupPlan& plan, void* out, int64_t ldo, int64_t out_cols, int* status) {
  GroupedGemmParams g = {};
  g.plan_rows = plan.row_tiles;
  g.plan_tiles = plan.tiles;
  g.plan_k = plan.k_tiles;
  g.out = static_cast<__nv_bfloat16*>(out);
  g.ldo = ldo;
  g.out_cols = static_cast<int>(out_cols);
  g.status = status;
  return g;
}

// D[r, a] = sum_k B[r, k] A_g[a, k]
int launch_rows_form(const GroupPlan& plan, const void* q_rows, const void* s_rows, int64_t rows, const void* qa,
                     const void* sa, int64_t a_rows, int64_t k, int64_t groups, void* out, int64_t ldo, int* status,
                     cudaStream_t stream) {
  const int64_t kp = round_up(k, 32), chunks = (kp / 32 + 3) / 4, a_sf = (a_rows + 127) / 128;
  GroupedGemmParams g = gemm_params(plan, out, ldo, a_rows, status);
  g.a_rows = static_cast<int>(a_rows);
  g.a_tiles = static_cast<int>((a_rows + 255) / 256);
  g.a_sf_tiles = static_cast<int>(a_sf);
  g.groups = static_cast<int>(groups);
  g.k_tiles = static_cast<int>((kp + 127) / 128);
  g.sf_chunks_a = g.sf_chunks_b = static_cast<int>(chunks);
  const Operand a{qa, sa, groups * a_rows, groups * a_sf * chunks};
  const Operand b{q_rows, s_rows, rows, most_tiles(rows, groups, 128) * chunks};
  g.tile_rows = plan.tile_rows;
  return launch_grouped(g, a, b, kp, kp, 1, rows, most_tiles(rows, groups, plan.tile_rows) * g.a_tiles, stream);
}

int grouped_fwd(const void* x, int64_t ldx, const void* w, const void* qw, const void* sw, const int* offsets,
                int64_t groups, void* out, int64_t ldo, int64_t rows, int64_t n, int64_t k, int rounding, void* workspace,
                size_t workspace_bytes, void* stream, int* status) {
  int rc = check_grouped(offsets, rows, n, k, groups);
  if (rc) return rc;
  if (!x || !out || !(w || (qw && sw))) return fail_msg(RTXB_E_INVALID_ARGUMENT, "null operand");
  if (ldx < k || ldo < n) return fail_msg(RTXB_E_INVALID_ARGUMENT, "row pitch smaller than the row");
  if (!aligned(x, 2) || !aligned(out, 2) || (w && !aligned(w, 2)))
    return fail_msg(RTXB_E_ALIGNMENT, "pointer is not element aligned");
  Carver c(workspace);
  FwdMemory mem(c, rows, n, k, groups, w != nullptr);
  if (!workspace || workspace_bytes < c.off) return fail_msg(RTXB_E_WORKSPACE, "workspace too small for the grouped forward");
  if (!aligned(workspace, 256)) return fail_msg(RTXB_E_ALIGNMENT, "workspace must be 256-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RowsParams q = {};
  q.x = RowsOperand{static_cast<const __nv_bfloat16*>(x), ldx, mem.qx, mem.sx, static_cast<int>(rows)};
  q.list = GroupList{offsets, static_cast<int>(groups), static_cast<int>(rows)};
  if (w) {
    q.w = RowsOperand{static_cast<const __nv_bfloat16*>(w), k, mem.qw, mem.sw, static_cast<int>(n)};
    q.batches = static_cast<int>(groups);
    qw = mem.qw;
    sw = mem.sw;
  }
  mem.plan.plan.tile_rows = rows_per_tile(rows, groups, n);
  q.plan = mem.plan.plan;
  q.out = static_cast<__nv_bfloat16*>(out);
  q.out_cols = static_cast<int>(n);
  q.ldo = ldo;
  q.status = status;
  if ((rc = launch_quantize_rows(q, most_tiles(rows, groups, 128), k, rounding, s))) return rc;
  return launch_rows_form(mem.plan.plan, mem.qx, mem.sx, rows, qw, sw, n, k, groups, out, ldo, status, s);
}

}  // namespace

extern "C" {

size_t rtxb_mxfp8_grouped_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int64_t groups, int dynamic_w) {
  Carver c(nullptr);
  FwdMemory mem(c, rows, n, k, groups, dynamic_w != 0);
  return c.off;
}

int rtxb_mxfp8_grouped_linear_fwd(const void* x, int64_t ldx, const void* w, const int* offsets, int64_t groups, void* out,
                                  int64_t ldo, int64_t rows, int64_t n, int64_t k, int rounding, void* workspace,
                                  size_t workspace_bytes, void* stream, int* status) {
  if (!w) return fail_msg(RTXB_E_INVALID_ARGUMENT, "null operand");
  return grouped_fwd(x, ldx, w, nullptr, nullptr, offsets, groups, out, ldo, rows, n, k, rounding, workspace, workspace_bytes,
                     stream, status);
}

int rtxb_mxfp8_grouped_linear_fwd_prequant_w(const void* x, int64_t ldx, const void* qw, const void* sw, const int* offsets,
                                             int64_t groups, void* out, int64_t ldo, int64_t rows, int64_t n, int64_t k,
                                             int rounding, void* workspace, size_t workspace_bytes, void* stream,
                                             int* status) {
  if (!qw || !sw) return fail_msg(RTXB_E_INVALID_ARGUMENT, "null operand");
  if (groups > 1 && n % 128 != 0)
    return fail_msg(RTXB_E_UNSUPPORTED, "packed group weights need n % 128 == 0 (scale tiles of 128 rows per group)");
  if (!aligned(qw, 16) || !aligned(sw, 16)) return fail_msg(RTXB_E_ALIGNMENT, "packed operands must be 16-byte aligned");
  return grouped_fwd(x, ldx, nullptr, qw, sw, offsets, groups, out, ldo, rows, n, k, rounding, workspace, workspace_bytes,
                     stream, status);
}

size_t rtxb_mxfp8_grouped_backward_workspace_bytes(int64_t rows, int64_t n, int64_t k, int64_t groups, int need_dx,
                                                   int need_dw) {
  Carver c(nullptr);
  BwdMemory mem(c, rows, n, k, groups, need_dx != 0, need_dw != 0);
  return c.off;
}

int rtxb_mxfp8_grouped_linear_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w,
                                  const int* offsets, int64_t groups, void* dx, void* dw, int64_t rows, int64_t n, int64_t k,
                                  void* workspace, size_t workspace_bytes, void* stream, int* status) {
  int rc = check_grouped(offsets, rows, n, k, groups);
  if (rc) return rc;
  if (!dy || (!dx && !dw) || (dx && !w) || (dw && !x)) return fail_msg(RTXB_E_INVALID_ARGUMENT, "null operand");
  if (lddy < n || (dw && ldx < k)) return fail_msg(RTXB_E_INVALID_ARGUMENT, "row pitch smaller than the row");
  if (!aligned(dy, 2) || !aligned(x, 2) || !aligned(w, 2) || !aligned(dx, 2) || !aligned(dw, 2))
    return fail_msg(RTXB_E_ALIGNMENT, "pointer is not element aligned");
  Carver c(workspace);
  BwdMemory mem(c, rows, n, k, groups, dx != nullptr, dw != nullptr);
  if (!workspace || workspace_bytes < c.off) return fail_msg(RTXB_E_WORKSPACE, "workspace too small for the grouped backward");
  if (!aligned(workspace, 256)) return fail_msg(RTXB_E_ALIGNMENT, "workspace must be 256-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t tiles128 = most_tiles(rows, groups, 128), nt = (n + 127) / 128, kt = (k + 127) / 128;
  TransposedParams t = {};
  t.dy = TransposedOperand{static_cast<const __nv_bfloat16*>(dy), lddy, static_cast<int>(rows), static_cast<int>(n), mem.q_dyt,
                           tiles128 * 128, mem.s_dyt, static_cast<int>(tiles128)};
  t.dy_rows = mem.q_dy;
  t.dy_row_scales = mem.s_dy;
  t.list = GroupList{offsets, static_cast<int>(groups), static_cast<int>(rows)};
  mem.plan.plan.tile_rows = rows_per_tile(rows, groups, k);
  t.plan = mem.plan.plan;
  t.dx = static_cast<__nv_bfloat16*>(dx);
  t.dx_cols = static_cast<int>(k);
  t.status = status;
  if (dw)
    t.x = TransposedOperand{static_cast<const __nv_bfloat16*>(x), ldx, static_cast<int>(rows), static_cast<int>(k), mem.q_xt,
                            tiles128 * 128, mem.s_xt, static_cast<int>(tiles128)};
  if (dx) {
    t.w = TransposedOperand{static_cast<const __nv_bfloat16*>(w), k, static_cast<int>(n), static_cast<int>(k), mem.q_wt,
                            round_up(n, 32), mem.s_wt, static_cast<int>(nt)};
    t.batches = static_cast<int>(groups);
  }
  if ((rc = launch_quantize_transposed(t, tiles128, s))) return rc;
  if (dx && (rc = launch_rows_form(mem.plan.plan, mem.q_dy, mem.s_dy, rows, mem.q_wt, mem.s_wt, k, n, groups, dx, k, status, s)))
    return rc;
  if (dw) {
    // dW_g[n, k] = sum over the rows of g: operand A = X^T (output columns), operand B = dY^T (output rows)
    GroupedGemmParams g = gemm_params(mem.plan.plan, dw, k, k, status);
    g.contraction = 1;
    g.a_rows = static_cast<int>(k);
    g.a_tiles = static_cast<int>((k + 255) / 256);
    g.b_rows = static_cast<int>(n);
    // dW has groups * n rows to spread over the pairs: tiles of 128 or 64 of them gain at most 1 us (300 rows, 4 groups,
    // 512 x 512: 16.7 / 16.2 / 15.6 us) and lose 3 to 75 % elsewhere (16384 rows, 8 groups, 4096 x 4096: 289 / 356 / 507)
    g.tile_rows = 256;
    g.b_tiles = static_cast<int>((n + 255) / 256);
    g.groups = static_cast<int>(groups);
    g.sf_chunks_a = g.sf_chunks_b = static_cast<int>(tiles128);
    g.out_group = n * k;
    const Operand a{mem.q_xt, mem.s_xt, k, kt * tiles128};
    const Operand b{mem.q_dyt, mem.s_dyt, n, nt * tiles128};
    return launch_grouped(g, a, b, tiles128 * 128, tiles128 * 128, groups, n, groups * g.a_tiles * g.b_tiles, s);
  }
  return RTXB_OK;
}

}  // extern "C"
