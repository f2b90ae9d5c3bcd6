// linear_pair.cuh -- the 16-bit product on CTA pairs (tcgen05 cta_group::2):
//   out = epilogue(A B), A m x k, B k x n, both bf16 or both f16, f32 sums.
//
// A pair computes a tile of 256 columns by up to 256 rows with one instruction
// per 16 of K: the columns (B, the weights) are the instruction's 256 rows, 128 a
// CTA, and the rows of A its columns, any multiple of 32, half a CTA. So a tile
// costs what its rows need: 300 rows are two tiles of 160, an expert's last tile
// ends with its tokens. Each CTA stages its 128 columns of B and its half of the
// rows of A in 64-wide k-blocks (128-byte swizzled rows, 32 KiB a stage), and
// keeps two 128 x 256 f32 accumulators in tensor memory, so that the epilogue of
// one tile runs under the MMAs of the next.
//
// RAG 0: one product; tiles walk in groups of LP_GROUP row tiles so that the
//        pairs running together share panels in L2 (4 or 16 lost 1 to 7 %).
// RAG 1: ragged rows, the experts' products: expert e multiplies rows
//        [offsets[e], offsets[e] + counts[e]) of A by its own B (the tensor
//        map's batch). Tiles start at the segment; the rows past its tokens, up
//        to the segment's end, are stored as zeros, and so are the rows after the
//        last segment.
// RAG 2: ragged contraction, the experts' weight gradients: out[e] = A_e^T B_e
//        over the segment's rows. Segments are multiples of 64 rows whose pad
//        rows are zero, so a k-block never meets another expert's rows; an
//        expert without tokens gets zeros.
//
// Work split: whole rounds of tiles, one a pair. Where the tiles of the last
// round fill at most half the pairs, each is cut into two of half its rows, so
// the round ends after half the MMAs and a product of few tiles reaches twice the
// SMs: 512 x 4096 x 4096 22.5 us against 29 uncut; 4096^3 (3.46 rounds) 96 us.
// Dividing those tiles along K instead, with parts parked in memory and joined by
// the last to finish, cost more than it saved (104 and 36 us): a part's 256 KB
// go out and come back.
//
// Bound: the tensor pipe. A tile of 4096 k takes 33.3 thousand cycles against
// 32.8 of MMAs; the clock under that load is the power cap's. 4096 x 11008 x
// 4096: 1.52 PFLOP/s in a short run, 1.31 after a second of it (the library's
// product 1.55 and 1.34 on the same box).
//
// Warps: 0-7 epilogue (TMEM lane quarter = 32 columns, every second box of 32
// rows), 8 TMA producer, 9 MMA
// issuer (even CTA), 10-11 idle.
#pragma once
#include <type_traits>

#include "linear_epi.cuh"
#include "ptx.cuh"

namespace mmr {

constexpr int LP_THREADS = 384;
constexpr int LP_LAUNCH_REGS = 168, LP_EPI_REGS = 208, LP_OTHER_REGS = 80;
static_assert(256 * LP_EPI_REGS + 128 * LP_OTHER_REGS <= LP_THREADS * LP_LAUNCH_REGS, "register split exceeds the launch");
constexpr int LP_BK = 64;
constexpr int LP_A_BYTES = 128 * LP_BK * 2;
constexpr int LP_CSTAGE_BYTES = 4096;  // per epilogue warp: 32 rows x 32 f32
constexpr int LP_GROUP = 8;
constexpr int LP_MAX_EXPERTS = 1024;

constexpr int LP_STAGE_BYTES = 2 * LP_A_BYTES;

constexpr int lp_stages(int rag) { return rag ? 5 : 6; }
// ragged: every expert's first tile and first row (and the ends), and its token count
constexpr int lp_table_bytes(int rag) { return rag ? (3 * LP_MAX_EXPERTS + 2) * 4 : 0; }
constexpr int lp_smem_bytes(int rag) {
  return lp_stages(rag) * LP_STAGE_BYTES + 8 * LP_CSTAGE_BYTES + lp_table_bytes(rag) + 256 + 1024;
}
static_assert(lp_smem_bytes(0) <= 232448 && lp_smem_bytes(1) <= 232448, "shared memory of one SM");

struct PairParams {
  int m = 0, n = 0;
  int tiles_m = 0, tiles_n = 0, tiles_total = 0;  // RAG 1: tiles_n, and the most tiles any layout has
  int tile_rows = 256;                            // rows of a tile, a multiple of 32 (RAG 1: by expert)
  int k_blocks = 0;                               // RAG 2: from the counts
  int experts = 0;
  const int* offsets = nullptr;
  const int* counts = nullptr;
  long long rows = 0;
  EpiParams epi;
  int* err = nullptr;
  unsigned long long timeout_ns = 0;
};

// Rows of each of `tiles` equal tiles of `rows` rows; tiles = ceil(rows / 256),
// so every tile but the last is full and the last has at least one row. No sum
// passes 32 bits at the largest extent admitted, 2^31 - 1024 rows.
__host__ __device__ constexpr int lp_tile_rows(int rows, int tiles) { return ((rows - 1) / tiles + 32) / 32 * 32; }
static_assert(lp_tile_rows(2147482624, 8388604) == 256 && lp_tile_rows(300, 2) == 160 && lp_tile_rows(1, 1) == 32,
              "rows of a tile");

// One piece of work, found from its index.
struct LpTile {
  int row0, rows;         // first row, and the instruction's columns: a multiple of 32
  int row_end, zero_end;  // rows from row_end on are not stored; [row_end, zero_end) are zeroed
  int col0;
  int batch;              // expert
  int kb, k_row;          // k-blocks, and the row where the contraction starts (RAG 2)
};

template <int RAG>
struct LpWalk {
  const PairParams& p;
  const int *first, *off, *cnt;  // shared-memory tables (RAG 1, 2)
  int t, step, e;
  int whole, end;                // pieces before `whole` are tiles, up to `end` half tiles
  __device__ __forceinline__ LpWalk(const PairParams& p_, const int* table, int pair, int npairs)
      : p(p_), first(table), off(table + LP_MAX_EXPERTS + 1), cnt(table + 2 * LP_MAX_EXPERTS + 2), t(pair), step(npairs), e(0) {
    const int total = RAG == 1 ? table[p_.experts] : p_.tiles_total;
    const int rem = total % npairs;
    whole = 2 * rem <= npairs ? total - rem : total;
    end = total + (total - whole);
  }
  __device__ __forceinline__ bool next(LpTile& w) {
    if (t >= end) return false;
    int tile = t, part = -1;
    if (t >= whole) {
      tile = whole + ((t - whole) >> 1);
      part = (t - whole) & 1;
    }
    t += step;
    int mt, nt, per, m;
    w.batch = 0;
    w.kb = p.k_blocks;
    w.k_row = 0;
    w.row0 = 0;
    w.zero_end = 0;
    if (RAG == 1) {
      while (first[e + 1] <= tile) ++e;
      const int local = tile - first[e], tm = (cnt[e] + 255) >> 8;
      mt = local % tm;
      nt = local / tm;
      m = cnt[e];
      per = lp_tile_rows(m, tm);
      w.row0 = off[e];
      w.batch = e;
      if (mt == tm - 1 && part != 0) w.zero_end = off[e + 1];
    } else {
      int r = tile;
      if (RAG == 2) {
        const int each = p.tiles_m * p.tiles_n;
        w.batch = tile / each;
        r = tile - w.batch * each;
        w.kb = (cnt[w.batch] + LP_BK - 1) / LP_BK;
        w.k_row = off[w.batch];
      }
      const int span = LP_GROUP * p.tiles_n, group = r / span, first_m = group * LP_GROUP;
      const int size = min(p.tiles_m - first_m, LP_GROUP), q = r - group * span;
      mt = first_m + q % size;
      nt = q / size;
      m = p.m;
      per = p.tile_rows;
    }
    w.row_end = w.row0 + m;
    w.row0 += mt * per;
    w.rows = min(per, (w.row_end - w.row0 + 31) / 32 * 32);
    if (part >= 0) {
      const int left = (w.rows / 2 + 31) / 32 * 32;
      if (part == 0) {
        w.rows = left;
      } else {
        w.row0 += left;
        w.rows -= left;
      }
      if (w.rows <= 0) w.kb = 0;  // a tile of 32 rows has no second half
    }
    w.col0 = nt * 256;
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
      // (the layout is data: whatever it says, nothing outside the rows is touched)
      int c = 0, o = 0;
      if (e < p.experts) {
        o = static_cast<int>(min(static_cast<long long>(max(p.offsets[e], 0)), p.rows));
        c = static_cast<int>(min(static_cast<long long>(max(p.counts[e], 0)), p.rows - o));
      }
      int incl = ((c + 255) >> 8) * p.tiles_n;
      const int own = incl;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      if (e < p.experts) {
        first[e] = min(base + incl - own, p.tiles_total);
        off[e] = o;
        cnt[e] = c;
      }
      base = min(base + __shfl_sync(0xffffffffu, incl, 31), p.tiles_total);  // no layout of a sort has more tiles
    }
    if (lane == 0) {
      first[p.experts] = base;
      off[p.experts] = static_cast<int>(min(static_cast<long long>(max(p.offsets[p.experts], 0)), p.rows));
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barrier inits and both TMEM allocations visible to the pair
  tc_fence_after();
  griddep_release();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) reg_alloc<LP_EPI_REGS>();
  else reg_dealloc<LP_OTHER_REGS>();
  if (warp < 8) {
    // ------------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = warp >> 2;
    uint8_t* buf = cstage + warp * LP_CSTAGE_BYTES;
    const uint32_t acc_empty_leader = mapa_shared(smem_u32(acc_empty), 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    LpWalk<RAG> walk(p, table, pair, npairs);
    LpTile w;
    const bool vec = epi_vec(p.epi);
    // The bias eight columns at a time: n and the experts' rows multiples of 8.
    const bool vec_bias = vec && p.epi.bias && p.epi.bias_s == 1 && (p.n & 7) == 0 && (p.epi.bias_bs & 7) == 0 &&
                          (reinterpret_cast<uintptr_t>(p.epi.bias) & 15) == 0;
    auto load_bias16 = [&](const LpTile& w, int col0) {
      const int col = col0 + (lane & 3) * 8;
      const T* q = static_cast<const T*>(p.epi.bias) + w.batch * p.epi.bias_bs + col;
      return vec_bias && col < p.n ? *(reinterpret_cast<const uint4*>(q)) : make_uint4(0, 0, 0, 0);
    };
    // The residual of one 32 x 32 box, in the layout it is added in: vector `it`
    // of lane l is row 8 it + l / 4, columns 8 (l % 4) of the box.
    auto load_residual = [&](const LpTile& w, int row0, int col0, uint4 (&res)[4]) {
      const int row = row0 + (lane >> 2), col = col0 + (lane & 3) * 8;
      const T* q = static_cast<const T*>(p.epi.residual.p) + row * p.epi.residual.ld + col;
#pragma unroll
      for (int it = 0; it < 4; ++it)
        if (row + 8 * it < w.row_end && col + 8 <= p.n)
          res[it] = *reinterpret_cast<const uint4*>(q + 8 * it * p.epi.residual.ld);
    };
    // Stores one staged 32 x 32 box (row r: 16-byte chunk q at q ^ (r & 7)). All
    // 32 of a lane's values go through each step together: with two warps a
    // scheduler, their independence is what hides the latencies.
    auto store_box = [&](const LpTile& w, int row0, int col0, const uint4 (&res)[4], const uint4& bias16) {
      const long long batch = RAG == 2 ? w.batch : 0;
      if (vec) {
        const int c2 = (lane & 3) * 2, col = col0 + (lane & 3) * 8, r0 = lane >> 2;
        if (col >= p.n) return;
        float bias[8];
        if (vec_bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) bias[i] = 0.0f;
          add8<T>(bias, bias16);
        } else {
          load_bias8<T>(p.epi, w.batch, col, bias);
        }
        if (col + 8 <= p.n && row0 + 32 <= w.row_end) {
          float v[32];
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const uint8_t* src = buf + (it * 8 + r0) * 128;  // row & 7 == r0
            *reinterpret_cast<float4*>(v + 8 * it) = *reinterpret_cast<const float4*>(src + ((c2 ^ r0) << 4));
            *reinterpret_cast<float4*>(v + 8 * it + 4) = *reinterpret_cast<const float4*>(src + (((c2 + 1) ^ r0) << 4));
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += bias[i & 7];
          auto put = [&](const EpiMat& m) {
            T* q = static_cast<T*>(m.p) + batch * m.bs + (row0 + r0) * m.ld + col;
#pragma unroll
            for (int it = 0; it < 4; ++it)
              *reinterpret_cast<uint4*>(q + 8 * it * m.ld) = pack8<T>(*reinterpret_cast<const float(*)[8]>(v + 8 * it));
          };
          if (p.epi.pre.p) put(p.epi.pre);
          lact_apply(p.epi.act, v);
          if (p.epi.residual.p) {
#pragma unroll
            for (int it = 0; it < 4; ++it) add8<T>(*reinterpret_cast<float(*)[8]>(v + 8 * it), res[it]);
          }
          put(p.epi.out);
          return;
        }
#pragma unroll 1
        for (int it = 0; it < 4; ++it) {
          const int rr = it * 8 + r0, row = row0 + rr;
          const float4 x = *reinterpret_cast<const float4*>(buf + rr * 128 + ((c2 ^ r0) << 4));
          const float4 y = *reinterpret_cast<const float4*>(buf + rr * 128 + (((c2 + 1) ^ r0) << 4));
          float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          if (row < w.row_end) epi_store8<T>(p.epi, batch, row, col, v, bias);
        }
      } else {
        // a lane a column, so that any pitch is stored in whole segments
        const int col = col0 + lane;
        if (col >= p.n) return;
        const float bias =
            p.epi.bias ? to_f32<T>(static_cast<const T*>(p.epi.bias)[w.batch * p.epi.bias_bs + col * p.epi.bias_s]) : 0.0f;
        const int rows = min(w.row_end - row0, 32);
        float add[32];
        if (p.epi.residual.p) {
          const T* q = static_cast<const T*>(p.epi.residual.p) + row0 * p.epi.residual.ld + col * p.epi.residual.cs;
#pragma unroll
          for (int r = 0; r < 32; ++r) {
            add[r] = r < rows ? to_f32<T>(*q) : 0.0f;
            q += p.epi.residual.ld;
          }
        }
        float v[32];
#pragma unroll
        for (int r = 0; r < 32; ++r)
          v[r] = bias + *reinterpret_cast<const float*>(buf + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
        auto put = [&](const EpiMat& m) {
          T* q = static_cast<T*>(m.p) + batch * m.bs + row0 * m.ld + col * m.cs;
#pragma unroll
          for (int r = 0; r < 32; ++r) {
            if (r < rows) *q = from_f32<T>(v[r]);
            q += m.ld;
          }
        };
        if (p.epi.pre.p) put(p.epi.pre);
        lact_apply(p.epi.act, v);
        if (p.epi.residual.p) {
#pragma unroll
          for (int r = 0; r < 32; ++r) v[r] += add[r];
        }
        put(p.epi.out);
      }
    };
    while (walk.next(w)) {
      const bool sums = w.kb > 0;
      // This warp's 32 columns, and every second box of 32 rows.
      const int col0 = w.col0 + static_cast<int>(rank) * 128 + quarter * 32;
      const int boxes = w.rows / 32;
      const bool adds = vec && p.epi.residual.p && col0 < p.n;
      uint4 res[2][4];
      // under the MMAs: the residual to L2, its first box to registers
      if (p.epi.residual.p && col0 < p.n) {
        for (int r = w.row0 + half * 32 + lane; r < min(w.row0 + w.rows, w.row_end); r += 64)
          prefetch_l2(static_cast<const T*>(p.epi.residual.p) + r * p.epi.residual.ld + col0 * p.epi.residual.cs);
      }
      if (adds && half < boxes) load_residual(w, w.row0 + half * 32, col0, res[0]);
      const uint4 bias16 = load_bias16(w, col0);
      if (sums) {
        if (!mbar_wait_cluster(&acc_full[acc], acc_phase, ctl, kDevTimeoutAcc)) break;
        tc_fence_after();
      }
      const uint32_t tb = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * 256;
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty_leader + 8u * acc);
      };
#pragma unroll 1
      for (int j2 = half; j2 < boxes; j2 += 4) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int j = j2 + 2 * b, row0 = w.row0 + j * 32;
          if (j >= boxes) continue;
          if (adds && j + 2 < boxes) load_residual(w, row0 + 64, col0, res[b ^ 1]);
          uint32_t r[32];
          if (sums) {
            tmem_ld_32x32b_x32(tb + j * 32, r);
            tmem_ld_wait();
            if (j + 2 >= boxes) release();  // the last of this warp's boxes is in registers
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = 0u;
          }
          if (col0 >= p.n || row0 >= w.row_end) continue;
          // a lane holds a column: transposed on the way in, so that row i's
          // 16-byte chunk q lies at q ^ (i & 7)
          __syncwarp();  // the box before has been read
#pragma unroll
          for (int i = 0; i < 32; ++i)
            *reinterpret_cast<uint32_t*>(buf + i * 128 + ((((lane >> 2) ^ (i & 7)) << 4) | ((lane & 3) << 2))) = r[i];
          __syncwarp();
          store_box(w, row0, col0, res[b], bias16);
        }
      }
      if (sums) {
        if (half >= boxes) release();  // 32 rows: nothing for the second four warps
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
      if (RAG == 1) {
        // the segment's rows past its tokens, this CTA's 128 columns of them
        for (int c = static_cast<int>(threadIdx.x); w.row_end + c / 16 < w.zero_end; c += 256) {
          const int col = w.col0 + static_cast<int>(rank) * 128 + (c % 16) * 8;
          if (col < p.n) epi_zero8<T>(p.epi, w.row_end + c / 16, col);
        }
      }
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
        // this CTA's 128 columns and its half of the rows, in boxes of 64
        const int n0 = w.col0 + static_cast<int>(rank) * 128, r0 = w.row0 + static_cast<int>(rank) * (w.rows / 2);
        const bool two = w.rows > 128;
        for (int kb = 0; kb < w.kb; ++kb) {
          if (!mbar_wait_cluster(&empty[stage], phase ^ 1u, ctl, kDevTimeoutEmpty)) { ok = false; break; }
          uint8_t* sw = ops + stage * LP_STAGE_BYTES;
          uint8_t* sr = sw + LP_A_BYTES;
          const uint32_t bar = full_leader + 8u * stage;
          const int k0 = w.k_row + kb * LP_BK, bb = RAG == 1 ? w.batch : 0;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], two ? 4 * LP_A_BYTES : 3 * LP_A_BYTES);
          if (B_MN) {
            tma_load_3d_pair(sw, &tmB, bar, n0, k0, bb);
            tma_load_3d_pair(sw + LP_A_BYTES / 2, &tmB, bar, n0 + 64, k0, bb);
          } else {
            tma_load_3d_pair(sw, &tmB, bar, k0, n0, bb);
          }
          if (A_MN) {
            tma_load_3d_pair(sr, &tmA, bar, r0, k0, 0);
            if (two) tma_load_3d_pair(sr + LP_A_BYTES / 2, &tmA, bar, r0 + 64, k0, 0);
          } else {
            tma_load_3d_pair(sr, &tmA, bar, k0, r0, 0);
            if (two) tma_load_3d_pair(sr + LP_A_BYTES / 2, &tmA, bar, k0, r0 + 64, 0);
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
    // The whole warp walks the loop and one elected lane issues, so that the
    // descriptors stay in uniform registers: with a single lane in the branch
    // an MMA took ~65 cycles to issue and a k-block, its two commits
    // included, ~620, against 512 cycles of MMAs (a clock64 trace).
    if (rank == 0) {
      constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
      // all but the instruction's columns
      constexpr uint32_t idesc0 = idesc_f16(256, 0, kBf16, B_MN, A_MN);
      // K-major: 128-byte rows, 8-row groups 1024 bytes apart, 32 bytes a
      // k-step. MN-major: 64-element atoms 8 KiB apart (the 64 K rows of a
      // box), 8-row K groups 1024 bytes apart, two groups a k-step.
      constexpr uint32_t w_lbo = B_MN ? 8192u : 16u, r_lbo = A_MN ? 8192u : 16u;
      constexpr uint32_t w_step = B_MN ? 2048u : 32u, r_step = A_MN ? 2048u : 32u;
      const uint64_t w_desc0 = smem_desc(smem_u32(ops), w_lbo, 1024u, 2u);
      const uint64_t r_desc0 = smem_desc(smem_u32(ops) + LP_A_BYTES, r_lbo, 1024u, 2u);
      const bool leader = elect_one();
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true, issued = false;
      LpWalk<RAG> walk(p, table, pair, npairs);
      LpTile w;
      while (ok && walk.next(w)) {
        if (w.kb == 0) continue;
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[acc], acc_phase ^ 1u, ctl, kDevTimeoutAcc))) break;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(acc * 256);
        const uint32_t idesc = idesc0 | (static_cast<uint32_t>(w.rows >> 3) << 17);
        bool ready = mbar_test_wait(smem_u32(&full[stage]), phase);
        for (int kb = 0; kb < w.kb; ++kb) {
          if (!__all_sync(0xffffffffu, ready))
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(&full[stage], phase, ctl, kDevTimeoutFull));
          if (!ok) break;
          tc_fence_after();
          const int now = stage;
          if (++stage == S) { stage = 0; phase ^= 1u; }
          // asked before this block's MMAs, so that the answer's latency is theirs
          ready = mbar_test_wait(smem_u32(&full[stage]), phase);
          const uint64_t so = static_cast<uint64_t>(now) * (LP_STAGE_BYTES >> 4);
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < LP_BK / 16; ++kk)
              umma_f16_2sm(d, w_desc0 + so + ((w_step * kk) >> 4), r_desc0 + so + ((r_step * kk) >> 4), idesc,
                           kk > 0 || kb > 0 ? 1u : 0u);
            umma_commit_2sm_both(&empty[now]);
          }
          __syncwarp();
          issued = true;
        }
        if (!ok) break;
        if (leader) umma_commit_2sm_both(&acc_full[acc]);
        __syncwarp();
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
      if (issued) {
        // The pair's MMAs are done before either CTA's memory goes: this wait
        // holds the even CTA, whose cluster barrier holds the odd one.
        if (leader) umma_commit_2sm(smem_u32(drain));
        __syncwarp();
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
