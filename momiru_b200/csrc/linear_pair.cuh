// linear_pair.cuh -- the 16-bit product on CTA pairs (tcgen05 cta_group::2):
//   out = epilogue(A B), A m x k, B k x n, both bf16 or both f16, f32 sums.
//
// A pair computes a 256 x 256 tile with one 256 x 256 x 16 instruction per
// k-step: each CTA stages its 128 rows of A and its 128 columns of B in
// 64-wide k-blocks (128-byte swizzled rows, 32 KiB a stage), and keeps two
// 128 x 256 f32 accumulators in tensor memory, so that the epilogue of one
// tile runs under the MMAs of the next.
//
// RAG 0: one product; tiles walk in groups of LP_GROUP row tiles so that the
//        pairs running together share panels in L2.
// RAG 1: ragged rows, the experts' products: expert e multiplies rows
//        [offsets[e], offsets[e] + counts[e]) of A by its own B (the tensor
//        map's batch). Tiles start at the segment, rows past its tokens are
//        stored as zeros up to the segment's end, and so are the rows after
//        the last segment.
// RAG 2: ragged contraction, the experts' weight gradients: out[e] = A_e^T B_e
//        over the segment's rows. Segments are multiples of 64 rows whose pad
//        rows are zero, so a k-block never meets another expert's rows; an
//        expert without tokens gets zeros.
//
// Bound: the tensor pipe. 128 cycles per instruction; the issuing thread only
// adds fixed offsets to precomputed descriptors.
//
// Warps: 0-7 epilogue (TMEM lane quarter x column half), 8 TMA producer, 9 MMA
// issuer (even CTA), 10-11 idle.
#pragma once
#include <type_traits>

#include "linear_epi.cuh"
#include "ptx.cuh"

namespace mmr {

constexpr int LP_THREADS = 384;
constexpr int LP_BN = 256;
constexpr int LP_BK = 64;
constexpr int LP_A_BYTES = 128 * LP_BK * 2;
constexpr int LP_STAGE_BYTES = 2 * LP_A_BYTES;
constexpr int LP_CSTAGE_BYTES = 4096;  // per epilogue warp: 32 rows x 32 f32
constexpr int LP_GROUP = 8;
constexpr int LP_MAX_EXPERTS = 1024;

constexpr int lp_stages(int rag) { return rag ? 5 : 6; }
// ragged: every expert's first tile and first row (and the ends), and its token count
constexpr int lp_table_bytes(int rag) { return rag ? (3 * LP_MAX_EXPERTS + 2) * 4 : 0; }
constexpr int lp_smem_bytes(int rag) {
  return lp_stages(rag) * LP_STAGE_BYTES + 8 * LP_CSTAGE_BYTES + lp_table_bytes(rag) + 256 + 1024;
}
static_assert(lp_smem_bytes(0) <= 232448 && lp_smem_bytes(1) <= 232448, "shared memory of one SM");

struct PairParams {
  int m = 0, n = 0;
  int tiles_m = 0, tiles_n = 0, tiles_total = 0;  // RAG 1: tiles_n only
  int k_blocks = 0;                               // RAG 2: from the counts
  int experts = 0;
  const int* offsets = nullptr;
  const int* counts = nullptr;
  long long rows = 0;
  EpiParams epi;
  int* err = nullptr;
  unsigned long long timeout_ns = 0;
};

// One tile of work, found from its index.
struct LpTile {
  int row0, row_end, zero_end;  // output rows: [row0, row_end) computed, up to zero_end zeroed
  int a_row;                    // row coordinate of A's tile
  int col0;
  int batch;                    // expert
  int kb, k_row;                // k-blocks, and the row where the contraction starts (RAG 2)
};

template <int RAG>
struct LpWalk {
  const PairParams& p;
  const int *first, *off, *cnt;  // shared-memory tables (RAG 1, 2)
  int t, step, total, e;
  __device__ __forceinline__ LpWalk(const PairParams& p_, const int* table, int t0, int step_)
      : p(p_), first(table), off(table + LP_MAX_EXPERTS + 1), cnt(table + 2 * LP_MAX_EXPERTS + 2), t(t0), step(step_),
        total(RAG == 1 ? table[p_.experts] : p_.tiles_total), e(0) {}
  __device__ __forceinline__ bool next(LpTile& w) {
    if (t >= total) return false;
    int mt, nt;
    if (RAG == 1) {
      while (first[e + 1] <= t) ++e;
      const int local = t - first[e], tm = (cnt[e] + 255) >> 8;
      mt = local % tm;
      nt = local / tm;
      w.row0 = w.a_row = off[e] + mt * 256;
      w.row_end = off[e] + cnt[e];
      w.zero_end = off[e + 1];
      w.batch = e;
      w.kb = p.k_blocks;
      w.k_row = 0;
    } else {
      int r = t;
      w.batch = 0;
      w.kb = p.k_blocks;
      w.k_row = 0;
      if (RAG == 2) {
        const int per = p.tiles_m * p.tiles_n;
        w.batch = t / per;
        r = t - w.batch * per;
        w.kb = (cnt[w.batch] + LP_BK - 1) / LP_BK;
        w.k_row = off[w.batch];
      }
      const int span = LP_GROUP * p.tiles_n, group = r / span, first_m = group * LP_GROUP;
      const int size = min(p.tiles_m - first_m, LP_GROUP), q = r - group * span;
      mt = first_m + q % size;
      nt = q / size;
      w.row0 = w.a_row = mt * 256;
      w.row_end = p.m;
      w.zero_end = 0;
    }
    w.col0 = nt * LP_BN;
    t += step;
    return true;
  }
};

template <typename T, bool A_MN, bool B_MN, int RAG>
__global__ void __launch_bounds__(LP_THREADS, 1)
    mmr_linear_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                           const PairParams p) {
  constexpr int S = lp_stages(RAG);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ops = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* cstage = ops + S * LP_STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(cstage + 8 * LP_CSTAGE_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* acc_full = bars + 2 * S;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* table = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
  const WaitCtl ctl{p.err, p.timeout_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 16);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 9) {
    tmem_alloc_2sm(tmem_slot, 512);
    tmem_relinquish_2sm();
  }
  griddep_wait();
  if (RAG && warp == 0) {
    int* first = table;
    int* off = table + LP_MAX_EXPERTS + 1;
    int* cnt = table + 2 * LP_MAX_EXPERTS + 2;
    int base = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < p.experts ? p.counts[e] : 0;
      int incl = ((c + 255) >> 8) * p.tiles_n;
      const int own = incl;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      if (e < p.experts) {
        first[e] = base + incl - own;
        off[e] = p.offsets[e];
        cnt[e] = c;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      first[p.experts] = base;
      off[p.experts] = p.offsets[p.experts];
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barrier inits and both TMEM allocations visible to the pair
  tc_fence_after();
  griddep_release();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    // ------------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = warp >> 2;
    uint8_t* buf = cstage + warp * LP_CSTAGE_BYTES;
    const uint32_t acc_empty_leader = mapa_shared(smem_u32(acc_empty), 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    LpWalk<RAG> walk(p, table, pair, npairs);
    LpTile w;
    while (walk.next(w)) {
      if (w.kb > 0) {
        if (!mbar_wait_cluster(&acc_full[acc], acc_phase, ctl, kDevTimeoutAcc)) break;
        tc_fence_after();
      }
      const int row0 = w.row0 + static_cast<int>(rank) * 128 + quarter * 32;
      const uint32_t tb = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * LP_BN + half * 128;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        const int col0 = w.col0 + half * 128 + j * 32;
        uint32_t r[32];
        if (w.kb > 0) {
          tmem_ld_32x32b_x32(tb + j * 32, r);
          tmem_ld_wait();
          if (j == 3) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty_leader + 8u * acc);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        if (col0 >= p.n || row0 >= max(w.row_end, w.zero_end)) continue;
        // row `lane`: 16-byte chunk q at q ^ (lane & 7)
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4)) =
              make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
        __syncwarp();
        const int c2 = (lane & 3) * 2, col = col0 + (lane & 3) * 8;
        float bias[8];
        load_bias8<T>(p.epi, w.batch, col, bias);
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int rr = it * 8 + (lane >> 2), row = row0 + rr;
          const float4 x = *reinterpret_cast<const float4*>(buf + rr * 128 + ((c2 ^ (rr & 7)) << 4));
          const float4 y = *reinterpret_cast<const float4*>(buf + rr * 128 + (((c2 + 1) ^ (rr & 7)) << 4));
          float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          if (col >= p.n) continue;
          if (row < w.row_end) epi_store8<T>(p.epi, RAG == 2 ? w.batch : 0, row, col, v, bias);
          else if (RAG == 1 && row < w.zero_end) epi_zero8<T>(p.epi, row, col);
        }
        __syncwarp();
      }
      if (w.kb > 0 && ++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    if (RAG == 1) {
      const int g = static_cast<int>(blockIdx.x) * 8 + warp, gn = static_cast<int>(gridDim.x) * 8;
      for (long long row = table[LP_MAX_EXPERTS + 1 + p.experts] + static_cast<long long>(g); row < p.rows; row += gn)
        for (int col = lane * 8; col < p.n; col += 256) epi_zero8<T>(p.epi, row, col);
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------- producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int last[S];
#pragma unroll
      for (int s = 0; s < S; ++s) last[s] = -1;
      bool ok = true;
      const uint32_t full_leader = mapa_shared(smem_u32(full), 0);
      LpWalk<RAG> walk(p, table, pair, npairs);
      LpTile w;
      while (ok && walk.next(w)) {
        const int m0 = w.a_row + static_cast<int>(rank) * 128, n0 = w.col0 + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < w.kb; ++kb) {
          if (!mbar_wait_cluster(&empty[stage], phase ^ 1u, ctl, kDevTimeoutEmpty)) { ok = false; break; }
          uint8_t* sa = ops + stage * LP_STAGE_BYTES;
          uint8_t* sb = sa + LP_A_BYTES;
          const uint32_t bar = full_leader + 8u * stage;
          const int k0 = w.k_row + kb * LP_BK, bb = RAG == 1 ? w.batch : 0;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * LP_STAGE_BYTES);
          if (A_MN) {
            tma_load_3d_pair(sa, &tmA, bar, m0, k0, 0);
            tma_load_3d_pair(sa + LP_A_BYTES / 2, &tmA, bar, m0 + 64, k0, 0);
          } else {
            tma_load_3d_pair(sa, &tmA, bar, k0, m0, 0);
          }
          if (B_MN) {
            tma_load_3d_pair(sb, &tmB, bar, n0, k0, bb);
            tma_load_3d_pair(sb + LP_A_BYTES / 2, &tmB, bar, n0 + 64, k0, bb);
          } else {
            tma_load_3d_pair(sb, &tmB, bar, k0, n0, bb);
          }
          last[stage] = static_cast<int>(phase);
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
      // Every load of the pair (they count on the even CTA's barriers) lands
      // before either CTA leaves: the closing cluster barrier waits for this.
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (rank != 0 || last[s] < 0) continue;
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait_cluster(smem_u32(&full[s]), static_cast<uint32_t>(last[s])))
          if (globaltimer_ns() - t0 > p.timeout_ns) { atomicCAS(p.err, 0, kDevTimeoutDrain); break; }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------ MMA issuer (pair)
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_f16(256, LP_BN, std::is_same<T, __nv_bfloat16>::value, A_MN, B_MN);
      // K-major: 128-byte rows, 8-row groups 1024 bytes apart, 32 bytes a
      // k-step. MN-major: 64-element atoms 8 KiB apart (the 64 K rows of a
      // box), 8-row K groups 1024 bytes apart, two groups a k-step.
      constexpr uint32_t a_lbo = A_MN ? 8192u : 16u, b_lbo = B_MN ? 8192u : 16u;
      constexpr uint32_t a_step = A_MN ? 2048u : 32u, b_step = B_MN ? 2048u : 32u;
      const uint64_t a_desc0 = smem_desc(smem_u32(ops), a_lbo, 1024u, 2u);
      const uint64_t b_desc0 = smem_desc(smem_u32(ops) + LP_A_BYTES, b_lbo, 1024u, 2u);
      const uint32_t empty_peer = mapa_shared(smem_u32(empty), 1), acc_full_peer = mapa_shared(smem_u32(acc_full), 1);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true, issued = false;
      LpWalk<RAG> walk(p, table, pair, npairs);
      LpTile w;
      while (ok && walk.next(w)) {
        if (w.kb == 0) continue;
        if (!mbar_wait_cluster(&acc_empty[acc], acc_phase ^ 1u, ctl, kDevTimeoutAcc)) break;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(acc * LP_BN);
        uint32_t accumulate = 0;
        for (int kb = 0; kb < w.kb; ++kb) {
          if (!mbar_wait_cluster(&full[stage], phase, ctl, kDevTimeoutFull)) { ok = false; break; }
          tc_fence_after();
          const uint64_t so = static_cast<uint64_t>(stage) * (LP_STAGE_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < LP_BK / 16; ++kk) {
            umma_f16_2sm(d, a_desc0 + so + ((a_step * kk) >> 4), b_desc0 + so + ((b_step * kk) >> 4), idesc, accumulate);
            accumulate = 1u;
          }
          issued = true;
          umma_commit_2sm(smem_u32(&empty[stage]));
          umma_commit_2sm(empty_peer + 8u * stage);
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_2sm(smem_u32(&acc_full[acc]));
        umma_commit_2sm(acc_full_peer + 8u * acc);
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
      if (issued) {
        // The pair's MMAs are done before either CTA's memory goes: this wait
        // holds the even CTA, whose cluster barrier holds the odd one.
        umma_commit_2sm(smem_u32(drain));
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait_cluster(smem_u32(drain), 0u))
          if (globaltimer_ns() - t0 > p.timeout_ns) { atomicCAS(p.err, 0, kDevTimeoutDrain); break; }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc_2sm(tmem, 512);
  }
}

}  // namespace mmr
