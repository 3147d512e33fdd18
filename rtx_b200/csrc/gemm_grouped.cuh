// Grouped MXFP8 GEMM: one launch for the products of all groups (experts).
//
//   rows         D[r, n] = sum_k X[r, k] W_g[n, k]        group g = the rows offsets[g] .. offsets[g + 1] - 1
//   contraction  D_g[n, k] = sum_r Y[r, n] X[r, k]        summed over the rows r of group g
//
// Both are tiles D^T[a, b] of a CTA pair (tcgen05 cta_group::2): the MMA's 256 rows are 256 consecutive output
// COLUMNS (weights, or the columns of dW), its N dimension runs over output ROWS (tokens, or the rows of dW).  The
// ragged extent is then the MMA's N, which may be any multiple of 32 up to 256: the last tile of a group costs what its
// rows cost (a tile of 40 tokens runs N = 64, a quarter of a full one), and one decode step streams its weights through
// the 256-row operand while a handful of tokens sits on the 32-wide side.  With the ragged extent on the MMA's rows
// every started tile costs 256 rows.  Small batches take tiles of 128 or 64 rows (rows_per_tile in grouped.cu).
//
// What bounds it.  Large batches: the tensor pipe, 81 to 83 % of active cycles (8192 rows, 4 groups, 4096 x 4096: 93 us,
// 2.95 PFLOP/s in a burst; in a longer run the 1 kW power cap, at 1.43 GHz).  The rest of the cycles is the hand-over
// between tiles: 2 x 256 accumulator columns and the scale sets do not fit TMEM, so a tile's MMAs wait for the shared
// chunk of the tile before.  Decode: HBM, every weight read once (128 rows, 32 groups of 4096 x 4096: 84 us, 6.6 TB/s).
// In between, the weights of groups with one partial tile each: 8192 rows in 32 uneven groups of 2048 x 4096 take 79 us
// where weights and rows are 51 us of HBM and the MMAs 46: pairs are 88 to 120 k cycles busy, since tiles of unlike size
// are dealt out in turn.  Dealing the full tiles first and the partial ones by size was no faster (86 us): groups of
// several tiles lose their weights from L2 in between, 413 MB read instead of 312.  Handing tiles out as pairs come free (a
// counter in memory, drawn ahead by an idle warp and passed on through shared memory) was slower everywhere: whole forward
// 96.6 -> 98.9 us, backward with its short dW tiles 476 -> 529, however many tiles were drawn ahead.
//
// Roles, TMEM plan and ring as in gemm_blockscaled_pair_kernel; what differs: tiles come from the plan the quantizer
// left, N and the number of K steps are per tile, and the epilogue holds one output column per lane, so a chunk of 32
// accumulator columns is 32 output rows of 64 bytes, staged and stored as one TMA box where all 32 rows belong to the
// tile, and written row by row (64-byte segments) where they do not.
#pragma once

#include "gemm_blockscaled.cuh"

namespace rtxb {

struct GroupedGemmParams {
  int contraction;         // 0: rows form, 1: contraction form
  int a_rows;              // rows of operand A per group (= output columns)
  int a_tiles;             // 256-row tiles of A per group
  int a_sf_tiles;          // 128-row scale tiles of A per group (rows form)
  int b_rows, b_tiles;     // contraction form: output rows per group and their tiles
  int tile_rows;           // most rows of B per tile (64, 128 or 256)
  int groups;
  int k_tiles;             // rows form: K steps; contraction form: read per group from plan_k
  int sf_chunks_a, sf_chunks_b;   // 512-byte scale tiles per 128 rows
  int map3d;               // payload maps are [K / 128][rows][128]
  const int* plan_rows;    // [0] = number of row tiles (rows form)
  const int4* plan_tiles;  // {first row, live rows, first scale tile, group}
  const int* plan_k;       // [groups + 1] first K step of each group (contraction form)
  __nv_bfloat16* out;
  int64_t ldo;             // elements
  int out_cols;
  int64_t out_group;       // contraction form: elements between the results of two groups
  int tma_out;
  int* status;
};

// boxes of operand B for 128, 64, 32 and 16 rows per CTA: a small tile fetches what it needs
struct GroupedMapsB {
  CUtensorMap m[4];
};

struct GroupedTile {
  int a_row, a_sf;         // first row of operand A (in its tensor map) and its first 128-row scale tile
  int b_row, b_sf, live;   // the same of operand B; rows of it that belong to the tile
  int sf_shift;            // 32-row groups of that scale tile before b_row (the scales of 32 rows are one TMEM column)
  int kt0, k_steps;
  int out_row, out_col, out_g;
};

__device__ __forceinline__ int grouped_total_tiles(const GroupedGemmParams& p) {
  return p.contraction ? p.groups * p.a_tiles * p.b_tiles : __ldcg(p.plan_rows) * p.a_tiles;
}

__device__ __forceinline__ GroupedTile grouped_tile(const GroupedGemmParams& p, int tile) {
  GroupedTile t;
  if (p.contraction) {
    const int per = p.a_tiles * p.b_tiles;
    const int g = tile / per, r = tile - g * per;
    const int bt = r / p.a_tiles, at = r - bt * p.a_tiles;
    t.kt0 = __ldcg(p.plan_k + g);
    t.k_steps = __ldcg(p.plan_k + g + 1) - t.kt0;
    t.a_row = at * 256;
    t.a_sf = at * 2;
    t.b_row = bt * p.tile_rows;
    t.b_sf = t.b_row >> 7;
    t.sf_shift = (t.b_row & 127) >> 5;
    t.live = min(p.tile_rows, p.b_rows - t.b_row);
    t.out_row = t.b_row;
    t.out_col = at * 256;
    t.out_g = g;
  } else {
    const int m = tile / p.a_tiles, at = tile - m * p.a_tiles;
    const int4 e = __ldcg(p.plan_tiles + m);
    t.kt0 = 0;
    t.k_steps = p.k_tiles;
    const int g = e.w & 0xFFFF;
    t.a_row = g * p.a_rows + at * 256;
    t.a_sf = g * p.a_sf_tiles + at * 2;
    t.sf_shift = e.w >> 16;
    t.b_row = e.x;
    t.b_sf = e.z;
    t.live = e.y;
    t.out_row = e.x;
    t.out_col = at * 256;
    t.out_g = 0;
  }
  return t;
}
__device__ __forceinline__ int grouped_mma_n(int live) { return (live + 31) & ~31; }

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* smem_src, int32_t c0, int32_t c1,
                                             int32_t c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

// Eight epilogue warps, two per TMEM lane quadrant, take the 32-column chunks in turn: where a pair has only one or two
// tiles the epilogue is not hidden behind MMAs, and half of it is half of that time.
constexpr int kGroupedEpiWarps = 8;
constexpr int kGroupedThreads = 64 + 32 * kGroupedEpiWarps;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGroupedThreads, 1)
gemm_grouped_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ GroupedMapsB maps_b,
                         const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfb,
                         const __grid_constant__ CUtensorMap map_out, const GroupedGemmParams p) {
  using T = PairTraits<kKindMxfp8>;
  using TP = TmemPlan<kKindMxfp8>;
  constexpr int S = T::kStagesP;
  constexpr int KS = T::kStepsPerBarrierP;
  constexpr int GROUPS = S / KS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::kOffBars);
  uint64_t* full_bar = bars;              // [GROUPS] used in the rank-0 CTA: both CTAs' loads land
  uint64_t* empty_bar = bars + S;         // [GROUPS] in each CTA
  uint64_t* acc_full_bar = bars + 2 * S;  // in each CTA: tile accumulated
  uint64_t* acc_overlap_bar = acc_full_bar + 1;  // rank 0: shared columns drained (one arrival per epilogue warp)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_overlap_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;

  griddep_launch_dependents();   // the second product of a backward sets up beside this one's tail
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(acc_full_bar, 1);
    mbar_init(acc_overlap_bar, 2 * kGroupedEpiWarps);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();   // the peer's barriers exist before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();   // operands and plan come from the quantizer launched just before this kernel
  const int total_tiles = grouped_total_tiles(p);

  if (warp == 0) {
    // ------------------------------ TMA producer (both CTAs) ------------------------------
    const bool leader = elect_one_sync();
    if (leader) {
      prefetch_tensormap(&map_a);
      prefetch_tensormap(&map_sfa);
      prefetch_tensormap(&map_sfb);
    }
    int group = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair_id; tile < total_tiles && ok; tile += num_pairs) {
      const GroupedTile t = grouped_tile(p, tile);
      const int mma_n = grouped_mma_n(t.live);
      const int half = mma_n >> 1;   // rows of B this CTA fetches
      const int box = half > 64 ? 0 : half > 32 ? 1 : half > 16 ? 2 : 3;
      const uint32_t b_bytes = (128u >> box) * kBlockKBytes;
      const bool two_sfb = mma_n > 128;
      const CUtensorMap* map_b = &maps_b.m[box];
      const uint32_t tx = 2 * KS * (T::kABytes + b_bytes + T::kSfaBytes + (two_sfb ? 2 : 1) * T::kSfaBytes);
      const int a_row = t.a_row + rank * 128, b_row = t.b_row + rank * half;
      const int k_groups = (t.k_steps + KS - 1) / KS;
      for (int kg = 0; kg < k_groups; ++kg) {
        if (!mbar_wait(&empty_bar[group], phase ^ 1, abort_flag)) {
          if (p.status && leader) atomicCAS(p.status, 0, kStatusWaitProducer);
          *abort_flag = 1;
          ok = false;
          break;
        }
        if (leader) {
          const uint32_t full_addr = mapa_shared(smem_u32(&full_bar[group]), 0);
          if (rank == 0) mbar_expect_tx(&full_bar[group], tx);
          const int slot0 = group * KS;
          const int kt = t.kt0 + kg * KS;   // steps past the tile's last are loaded but never issued
          uint8_t* sa = smem + slot0 * T::kABytes;
          // the KS steps of B lie behind one another, b_bytes apart
          uint8_t* sb = smem + T::kOffB + slot0 * T::kBBytes;
          if (p.map3d) {
            tma_load_3d_pair(sa, &map_a, full_addr, 0, a_row, kt);
            tma_load_3d_pair(sb, map_b, full_addr, 0, b_row, kt);
          } else {
#pragma unroll
            for (int sub = 0; sub < KS; ++sub) {
              tma_load_2d_pair(sa + sub * T::kABytes, &map_a, full_addr, (kt + sub) * kBlockKBytes, a_row);
              tma_load_2d_pair(sb + sub * b_bytes, map_b, full_addr, (kt + sub) * kBlockKBytes, b_row);
            }
          }
          tma_load_2d_pair(smem + T::kOffSfa + slot0 * T::kSfaBytes, &map_sfa, full_addr, 0,
                           (t.a_sf + rank) * p.sf_chunks_a + kt);
          uint8_t* ssfb = smem + T::kOffSfb + slot0 * T::kSfbBytes;
          tma_load_2d_pair(ssfb, &map_sfb, full_addr, 0, t.b_sf * p.sf_chunks_b + kt);
          if (two_sfb)
            tma_load_2d_pair(ssfb + KS * T::kSfaBytes, &map_sfb, full_addr, 0, (t.b_sf + 1) * p.sf_chunks_b + kt);
        }
        __syncwarp();
        if (++group == GROUPS) { group = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer (rank 0 only) ------------------------------
    if (rank == 0) {
      const uint32_t smem_base = smem_u32(smem);
      const bool leader = elect_one_sync();
      int group = 0;
      uint32_t phase = 0, local_tile = 0, step = 0;
      bool ok = true;
      for (int tile = pair_id; tile < total_tiles && ok; tile += num_pairs) {
        const GroupedTile t = grouped_tile(p, tile);
        if (t.k_steps == 0) continue;   // a group without rows: the epilogue writes its zeros
        const int mma_n = grouped_mma_n(t.live);
        const int half = mma_n >> 1;
        const uint32_t b_bytes = (half > 64 ? 128u : half > 32 ? 64u : half > 16 ? 32u : 16u) * kBlockKBytes;
        const uint32_t idesc = idesc_block_scaled(256, mma_n, 0u, 1u);
        const uint32_t acc_col = (local_tile & 1) ? TP::kAccWindow1 : 0;
        if (local_tile > 0) {
          // previous tile's epilogue has drained the columns both windows share
          if (!mbar_wait(acc_overlap_bar, (local_tile - 1) & 1, abort_flag)) {
            if (p.status) atomicCAS(p.status, 0, kStatusWaitMma);
            *abort_flag = 1;
            break;
          }
          tc_fence_after_sync();
        }
        const int k_groups = (t.k_steps + KS - 1) / KS;
        for (int kg = 0; kg < k_groups; ++kg) {
          if (!mbar_wait(&full_bar[group], phase, abort_flag)) {
            if (p.status) atomicCAS(p.status, 0, kStatusWaitMma);
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (leader) {
#pragma unroll
            for (int sub = 0; sub < KS; ++sub) {
              if (kg * KS + sub >= t.k_steps) break;
              const int slot = group * KS + sub;
              const int set = step & 1;
              ++step;
              const uint32_t ssfb = smem_base + T::kOffSfb + group * KS * T::kSfbBytes + sub * T::kSfaBytes;
              // the second half of a tile of at most 128 columns holds whatever the slot held: it is copied and not read
              issue_scale_copy<kKindMxfp8, true>(tmem_base, smem_base + T::kOffSfa + slot * T::kSfaBytes, ssfb,
                                                 ssfb + KS * T::kSfaBytes, set);
              issue_k_step<kKindMxfp8, true>(tmem_base, acc_col, smem_base + slot * T::kABytes,
                                             smem_base + T::kOffB + group * KS * T::kBBytes + sub * b_bytes, set, idesc,
                                             kg == 0 && sub == 0, t.sf_shift);
            }
            tc_commit_pair(&empty_bar[group], 3);
          }
          __syncwarp();
          if (++group == GROUPS) { group = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (leader) tc_commit_pair(acc_full_bar, 3);
        __syncwarp();
        ++local_tile;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue (both CTAs) ------------------------------
    const int quad = warp & 3, turn = (warp - 2) >> 2;   // this warp's lane quadrant; chunks turn, turn + 2, ...
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t overlap_addr = mapa_shared(smem_u32(acc_overlap_bar), 0);
    uint8_t* buf = smem + T::kOffStage + (warp - 2) * kEpiStageBufBytes;
    uint32_t local_tile = 0;
    for (int tile = pair_id; tile < total_tiles; tile += num_pairs) {
      const GroupedTile t = grouped_tile(p, tile);
      const int mma_n = grouped_mma_n(t.live);
      const int col0 = t.out_col + rank * 128 + quad * 32;   // first output column of this warp
      __nv_bfloat16* out = p.out + t.out_g * p.out_group + static_cast<int64_t>(t.out_row) * p.ldo + col0 + lane;
      const bool col_ok = col0 + lane < p.out_cols;
      // 32 accumulator columns = 32 output rows from c on
      auto emit = [&](const int c, const uint32_t (&r)[32]) {
        if (col0 >= p.out_cols) return;   // warp-uniform: nothing of this warp's columns exists
        if (p.tma_out && c + 32 <= t.live) {
          if (lane == 0) tma_store_wait_read<0>();   // the last store has read the buffer
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            *reinterpret_cast<__nv_bfloat16*>(buf + j * 64 + (((lane >> 3) ^ ((j >> 1) & 3)) << 4) + (lane & 7) * 2) =
                __float2bfloat16_rn(__uint_as_float(r[j]));
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&map_out, buf, col0, t.out_row + c, t.out_g);
            tma_store_commit();
          }
        } else if (col_ok) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < t.live) out[(c + j) * p.ldo] = __float2bfloat16_rn(__uint_as_float(r[j]));
        }
      };
      if (t.k_steps == 0) {
        uint32_t zero[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) zero[j] = 0;
#pragma unroll 1
        for (int c = 32 * turn; c < mma_n; c += 64) emit(c, zero);
        continue;
      }
      const bool odd = (local_tile & 1) != 0;
      const uint32_t tacc = tmem_base + lane_base + (odd ? TP::kAccWindow1 : 0);
      if (!mbar_wait(acc_full_bar, local_tile & 1, abort_flag)) {
        if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusWaitEpilogue);
        *abort_flag = 1;
        break;
      }
      ++local_tile;
      tc_fence_after_sync();
      // The 32 columns both windows share (the last of an even window, the first of an odd one) are read first by the
      // warps whose turn they are; with them in registers the next tile's MMAs may start.  All warps signal, and only
      // after they have seen this tile accumulated, so that no signal can count for the tile before it.
      static_assert(TP::kOverlapChunks == 1, "one shared chunk");
      const int shared0 = odd ? 0 : TP::kAccWindow1;
      const bool holder = turn == (odd ? 0 : 1) && shared0 < mma_n;
      uint32_t r[32];
      if (holder) {
        tmem_ld_32x32(tacc + shared0, r);
        tmem_ld_wait();
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(overlap_addr);
      if (holder) emit(shared0, r);
#pragma unroll 1
      for (int c = 32 * turn; c < mma_n; c += 64) {
        if (c == shared0) continue;
        tmem_ld_32x32(tacc + c, r);
        tmem_ld_wait();
        emit(c, r);
      }
    }
    if (p.tma_out && lane == 0) tma_store_wait_all<0>();   // shared memory outlives the last store's reads
    __syncwarp();
  }

  // ------------------------------ teardown ------------------------------
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();   // neither CTA frees TMEM or leaves while the pair may still touch it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace rtxb
