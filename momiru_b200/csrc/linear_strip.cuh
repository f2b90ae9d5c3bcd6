// linear_strip.cuh -- the 16-bit product for few rows per weight matrix:
//   out[m, n] = epilogue(sum_k x[m, k] w[k, n])
// with the weights as the tensor core's M operand: a 128-column strip of w is
// the 128 MMA rows, up to `mt` rows of x are its N. One CTA accumulates
// D[n, m] of a strip over its slice of K; the CTAs of a cluster split K. Each
// owns an equal share of the strip's columns, the others push it their parts of
// those (st.async: distributed shared-memory stores counted by the owner's
// barrier), and it adds them in rank order, so the result does not depend on
// timing. Pulling the parts between two cluster barriers instead took 5 us of
// the 10 at 16 x 4096 x 4096.
//
// Bound: the weights' bytes. Nothing of the tensor core is wasted on absent
// tokens, and the split over K is what puts every SM on the stream when the
// strips are fewer than the SMs (strip_shape in ops.cu).
//
// Ragged rows (expert products): a unit is (expert, mt rows of its segment,
// strip); each CTA finds its expert from the counts. The rows of a segment's
// last unit past its tokens, and the rows after the last segment, are written
// as zeros.
//
// Warps: 0-3 read the accumulators (TMEM lane quarters), 4 TMA producer, 5 MMA
// issuer; all six run the epilogue.
#pragma once
#include <type_traits>

#include "linear_epi.cuh"
#include "ptx.cuh"

namespace mmr {

constexpr int LS_COLS = 128;  // strip width: MMA rows
constexpr int LS_BK = 64;     // k-block: one 128-byte swizzled row
constexpr int LS_THREADS = 192;
constexpr int LS_W_BYTES = LS_COLS * LS_BK * 2;
constexpr int LS_MAX_STAGES = 8;
constexpr int LS_MAX_SPLIT = 8;

struct StripParams {
  int m = 0, n = 0;
  int k_blocks = 0;
  int mt = 16;             // rows of x per unit (MMA N), a multiple of 16 up to 128
  int strips = 0, m_units = 0;
  int split = 1;           // CTAs of a cluster: K slices
  int stages = 0;
  uint32_t tmem_cols = 32;
  int experts = 0;         // 0: plain rows
  const int* offsets = nullptr;
  const int* counts = nullptr;
  long long rows = 0;      // rows of the sorted buffers
  EpiParams epi;
  int* err = nullptr;
  unsigned long long timeout_ns = 0;
};

// Pushed parts: [slice][four rows][column of this CTA's share] as float4, so
// that a warp pushes whole 256-byte runs and reads them back conflict-free.
constexpr int strip_parts_bytes(int mt, int split) { return split > 1 ? LS_COLS * mt * 4 : 0; }
constexpr int strip_smem_bytes(int mt, int stages, int split) {
  return stages * (LS_W_BYTES + mt * 128) + 256 + strip_parts_bytes(mt, split) + 1024;
}

// Four floats into the shared memory of a CTA of the cluster, their 16 bytes
// counted on that CTA's barrier.
__device__ __forceinline__ void st_async_f4(uint32_t addr, uint32_t bar, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(addr),
               "r"(bar), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// Expert and first row of unit `unit` when each expert with c tokens has
// ceil(c / mt) units; false when there are fewer units. One warp. The counts are
// data: sums stop at LS_UNITS_END, above every unit's number, so that none wraps.
constexpr int LS_UNITS_END = 1 << 29;
__device__ __forceinline__ bool find_expert_unit(const int* counts, int experts, int mt, int unit, int lane, int* expert,
                                                 int* local) {
  int base = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int c = e0 + lane < experts ? max(counts[e0 + lane], 0) : 0;
    int incl = c > 0 ? (c - 1) / mt + 1 : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl = min(incl + up, LS_UNITS_END);
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + incl > unit);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const int before = __shfl_sync(0xffffffffu, incl, max(l - 1, 0));
      *expert = e0 + l;
      *local = unit - base - (l ? before : 0);
      return true;
    }
    base = min(base + __shfl_sync(0xffffffffu, incl, 31), LS_UNITS_END);
  }
  return false;
}

template <typename T, bool W_MN>
__global__ void __launch_bounds__(LS_THREADS, 3)
    mmr_linear_strip_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                            const StripParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ops = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = LS_W_BYTES + p.mt * 128;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ops + p.stages * stage_bytes);
  uint64_t* full = bars;
  uint64_t* empty = bars + LS_MAX_STAGES;
  uint64_t* acc_full = bars + 2 * LS_MAX_STAGES;
  uint64_t* parts_bar = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(parts_bar + 1);
  int* unit_info = reinterpret_cast<int*>(tmem_slot + 1);  // expert, local unit
  float4* parts = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(bars) + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = static_cast<int>(blockIdx.x) / p.split;
  const int strip = unit % p.strips, mu = unit / p.strips;
  const WaitCtl ctl{p.err, p.timeout_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(parts_bar, 1);
    fence_mbar_init();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  // The first k-blocks of plain weights start towards L2 while the previous
  // kernel drains (an expert's are known only after it).
  if (warp == 4 && lane == 0 && !p.experts) {
    const int b0 = static_cast<int>(static_cast<long long>(p.k_blocks) * rank / p.split);
    const int b1 = static_cast<int>(static_cast<long long>(p.k_blocks) * (rank + 1) / p.split);
    for (int kb = b0; kb < min(b1, b0 + p.stages); ++kb) {
      if (W_MN) {
        tma_prefetch_l2_3d(&tmW, strip * LS_COLS, kb * LS_BK, 0);
        tma_prefetch_l2_3d(&tmW, strip * LS_COLS + 64, kb * LS_BK, 0);
      } else {
        tma_prefetch_l2_3d(&tmW, kb * LS_BK, strip * LS_COLS, 0);
      }
    }
  }
  if (p.split > 1) {
    __syncthreads();
    cluster_arrive_release();  // this CTA's barriers stand; waited for before the first push
  }
  griddep_wait();
  if (p.experts && warp == 0) {
    int e = -1, local = 0;
    if (!find_expert_unit(p.counts, p.experts, p.mt, mu, lane, &e, &local)) e = -1;
    if (lane == 0) {
      unit_info[0] = e;
      unit_info[1] = local;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_release();
  const uint32_t tmem = *tmem_slot;

  // This unit's rows: [row0, row0 + valid) computed, up to zero_end zeroed.
  int expert = 0;
  long long row0 = static_cast<long long>(mu) * p.mt, zero_end = 0;
  int valid = static_cast<int>(min(static_cast<long long>(p.mt), p.m - row0));
  if (p.experts) {
    expert = unit_info[0];
    valid = 0;
    if (expert >= 0) {
      // (the layout is data: whatever it says, nothing outside the rows is touched)
      const int local = unit_info[1], count = p.counts[expert];
      row0 = max(p.offsets[expert], 0) + static_cast<long long>(local) * p.mt;
      valid = static_cast<int>(max(0ll, min(static_cast<long long>(min(p.mt, count - local * p.mt)), p.rows - row0)));
      if (count - local * p.mt <= p.mt) zero_end = min(static_cast<long long>(p.offsets[expert + 1]), p.rows);
    }
  }
  const int kb0 = static_cast<int>(static_cast<long long>(p.k_blocks) * rank / p.split);
  const int kb1 = static_cast<int>(static_cast<long long>(p.k_blocks) * (rank + 1) / p.split);
  const bool work = valid > 0 && kb1 > kb0;

  if (warp == 4) {
    if (lane == 0 && work) {
      int stage = 0;
      uint32_t phase = 0;
      int last[LS_MAX_STAGES];
#pragma unroll
      for (int s = 0; s < LS_MAX_STAGES; ++s) last[s] = -1;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, ctl, kDevTimeoutEmpty)) { ok = false; break; }
        uint8_t* sw = ops + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], stage_bytes);
        if (W_MN) {
          tma_load_3d(sw, &tmW, &full[stage], strip * LS_COLS, kb * LS_BK, expert);
          tma_load_3d(sw + LS_W_BYTES / 2, &tmW, &full[stage], strip * LS_COLS + 64, kb * LS_BK, expert);
        } else {
          tma_load_3d(sw, &tmW, &full[stage], kb * LS_BK, strip * LS_COLS, expert);
        }
        tma_load_3d(sw + LS_W_BYTES, &tmX, &full[stage], kb * LS_BK, static_cast<int>(row0), 0);
        last[stage] = static_cast<int>(phase);
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
      // Copies in flight must land before this CTA's shared memory goes; on the
      // normal path the MMAs have consumed them all.
      if (!ok) {
        for (int s = 0; s < p.stages; ++s) {
          if (last[s] < 0) continue;
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(smem_u32(&full[s]), static_cast<uint32_t>(last[s])))
            if (globaltimer_ns() - t0 > p.timeout_ns) break;
        }
      }
    }
  } else if (warp == 5) {
    if (work) {  // the whole warp, one elected lane issuing (linear_pair.cuh says why)
      const uint32_t idesc = idesc_f16(LS_COLS, p.mt, std::is_same<T, __nv_bfloat16>::value, W_MN, false);
      constexpr uint32_t w_lbo = W_MN ? 64u * 128u : 16u, w_step = W_MN ? 2048u : 32u;
      const uint64_t w_desc0 = smem_desc(smem_u32(ops), w_lbo, 1024u, 2u);
      const uint64_t x_desc0 = smem_desc(smem_u32(ops) + LS_W_BYTES, 16u, 1024u, 2u);
      const bool leader = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, ctl, kDevTimeoutFull))) break;
        tc_fence_after();
        const uint64_t so = static_cast<uint64_t>(stage * stage_bytes) >> 4;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < LS_BK / 16; ++kk)
            umma_f16(tmem, w_desc0 + so + ((w_step * kk) >> 4), x_desc0 + so + ((32u * kk) >> 4), idesc,
                     kk > 0 || kb > kb0 ? 1u : 0u);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
      if (leader) umma_commit(acc_full);  // also after a failed wait: covers whatever was issued
      __syncwarp();
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(smem_u32(acc_full), 0u))  // no MMA in flight past here
        if (globaltimer_ns() - t0 > p.timeout_ns) { atomicCAS(p.err, 0, kDevTimeoutDrain); break; }
    }
  }

  __syncwarp();
  if (p.split > 1) cluster_wait_acquire();

  // This CTA's share of the strip's columns.
  const int width = LS_COLS / p.split, col0 = strip * LS_COLS + rank * width;
  const int slice = p.mt / 4 * width;  // float4 of one slice's parts
  // One slice: the accumulators go to shared memory transposed, red[m][n] (a
  // lane holds one n, so each store of a warp is 32 neighbouring floats); the
  // operand stages are free once the MMAs are done. Several: every lane pushes
  // its column's rows to the column's owner.
  float* red = reinterpret_cast<float*>(ops);
  const bool vec = epi_vec(p.epi);
  if (warp < 4 && valid > 0) {
    const int n = static_cast<int>(threadIdx.x);
    if (p.split > 1 && n == 0) mbar_arrive_expect_tx(parts_bar, LS_COLS * ((valid + 3) / 4) * 16);
    if (p.epi.residual.p) {  // on its way to L2 until the sums are there
      const T* res = static_cast<const T*>(p.epi.residual.p) + row0 * p.epi.residual.ld;
      for (int m = n; m < valid; m += 128)
        for (int c = col0; c < min(col0 + width, p.n); c += 64)
          prefetch_l2(res + m * p.epi.residual.ld + c * p.epi.residual.cs);
    }
    if (work) {
      mbar_wait(acc_full, 0u, ctl, kDevTimeoutAcc);
      tc_fence_after();
    }
    const int owner = n / width;
    const uint32_t to = p.split > 1 ? mapa_shared(smem_u32(parts + rank * slice + n - owner * width), owner) : 0u;
    const uint32_t bar = p.split > 1 ? mapa_shared(smem_u32(parts_bar), owner) : 0u;
    for (int c = 0; c < valid; c += 16) {
      uint32_t r[16];
      if (work) {
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;
      }
      if (p.split > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          if (c + i < valid) st_async_f4(to + (c + i) / 4 * width * 16, bar, r[i], r[i + 1], r[i + 2], r[i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) red[(c + i) * LS_COLS + n] = __uint_as_float(r[i]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // All parts arrive, whatever went wrong elsewhere: nobody leaves before its
  // own have (their stores must find this CTA's memory).
  if (p.split > 1 && valid > 0) mbar_wait_acquire_cluster(parts_bar, 0u, ctl, kDevTimeoutReduce);

  const int tid = static_cast<int>(threadIdx.x);
  if (p.split > 1) {
    // four rows of one column a thread (of two, where the outputs take pairs),
    // slices in order; the loop stays rolled: this runs once, from a cold
    // instruction cache
    auto quads = [&](auto columns) {
      constexpr int C = decltype(columns)::value;
      const int across = width / C;
      for (int u = tid; u < (valid + 3) / 4 * across; u += LS_THREADS) {
        const int q = u / across, lc = (u - q * across) * C, col = col0 + lc;
        if (col >= p.n) continue;
        float v[4 * C];
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) v[i] = 0.0f;
        const float4* at = parts + q * width + lc;
#pragma unroll 2
        for (int r = 0; r < p.split; ++r) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float4 x = at[c];
            v[4 * c] += x.x; v[4 * c + 1] += x.y; v[4 * c + 2] += x.z; v[4 * c + 3] += x.w;
          }
          at += slice;
        }
        epi_store_quad<T, C>(p.epi, expert, row0 + 4 * q, valid - 4 * q, col, v);
      }
    };
    if (vec && p.n % 2 == 0) quads(std::integral_constant<int, 2>());
    else quads(std::integral_constant<int, 1>());
  } else if (vec) {
    constexpr int pieces = LS_COLS / 8;  // of eight columns
    for (int c = tid; c < valid * pieces; c += LS_THREADS) {
      const int m = c / pieces, lc = (c % pieces) * 8, col = col0 + lc;
      if (col >= p.n) continue;
      const float4 x = *reinterpret_cast<const float4*>(red + m * LS_COLS + lc);
      const float4 y = *reinterpret_cast<const float4*>(red + m * LS_COLS + lc + 4);
      float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      float bias[8];
      load_bias8<T>(p.epi, expert, col, bias);
      epi_store8<T>(p.epi, 0, row0 + m, col, v, bias);
    }
  } else {
    // neighbouring lanes on neighbouring columns, four rows a thread
    for (int u = tid; u < (valid + 3) / 4 * LS_COLS; u += LS_THREADS) {
      const int q = u / LS_COLS, lc = u % LS_COLS, col = col0 + lc;
      if (col >= p.n) continue;
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = red[(4 * q + r) * LS_COLS + lc];
      epi_store_quad<T, 1>(p.epi, expert, row0 + 4 * q, valid - 4 * q, col, v);
    }
  }
  if (p.experts) {
    // pad rows of the segment, then this unit's share of the rows after the last segment
    const int pieces = width / 8;
    for (int pass = 0; pass < 2; ++pass) {
      const long long from = pass ? max(p.offsets[p.experts], 0) + static_cast<long long>(mu) : row0 + valid;
      const long long to = pass ? p.rows : zero_end, step = pass ? p.m_units : 1;
      for (long long c = tid; from + (c / pieces) * step < to; c += LS_THREADS) {
        const int col = col0 + static_cast<int>(c % pieces) * 8;
        if (col < p.n) epi_zero8<T>(p.epi, from + (c / pieces) * step, col);
      }
    }
  }
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

}  // namespace mmr
