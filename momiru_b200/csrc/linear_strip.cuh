// linear_strip.cuh -- the 16-bit product for few rows per weight matrix:
//   out[m, n] = epilogue(sum_k x[m, k] w[k, n])
// with the weights as the tensor core's M operand: a 128-column strip of w is
// the 128 MMA rows, up to `mt` rows of x are its N. One CTA accumulates
// D[n, m] of a strip over its slice of K; the CTAs of a cluster split K and
// add their partial sums over distributed shared memory, in rank order, so the
// result does not depend on timing.
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
  int mt = 16;             // rows of x per unit (MMA N), a multiple of 16 up to 256
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

constexpr int strip_smem_bytes(int mt, int stages) { return stages * (LS_W_BYTES + mt * 128) + 256 + 1024; }

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Expert and first row of unit `unit` when each expert with c tokens has
// ceil(c / mt) units; false when there are fewer units. One warp.
__device__ __forceinline__ bool find_expert_unit(const int* counts, int experts, int mt, int unit, int lane, int* expert,
                                                 int* local) {
  int base = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int c = e0 + lane < experts ? counts[e0 + lane] : 0;
    const int units = (c + mt - 1) / mt;
    int incl = units;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + incl > unit);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *expert = e0 + l;
      *local = unit - base - __shfl_sync(0xffffffffu, incl - units, l);
      return true;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
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
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  int* unit_info = reinterpret_cast<int*>(tmem_slot + 1);  // expert, local unit

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
      const int local = unit_info[1], count = p.counts[expert];
      row0 = p.offsets[expert] + static_cast<long long>(local) * p.mt;
      valid = min(p.mt, count - local * p.mt);
      if ((local + 1) * p.mt >= count) zero_end = p.offsets[expert + 1];
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
    if (lane == 0 && work) {
      const uint32_t idesc = idesc_f16(LS_COLS, p.mt, std::is_same<T, __nv_bfloat16>::value, W_MN, false);
      constexpr uint32_t w_lbo = W_MN ? 64u * 128u : 16u, w_step = W_MN ? 2048u : 32u;
      int stage = 0;
      uint32_t phase = 0, accumulate = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, ctl, kDevTimeoutFull)) break;
        tc_fence_after();
        const uint32_t sw = smem_u32(ops + stage * stage_bytes);
        const uint64_t wd = smem_desc(sw, w_lbo, 1024u, 2u), xd = smem_desc(sw + LS_W_BYTES, 16u, 1024u, 2u);
#pragma unroll
        for (int kk = 0; kk < LS_BK / 16; ++kk) {
          umma_f16(tmem, wd + ((w_step * kk) >> 4), xd + ((32u * kk) >> 4), idesc, accumulate);
          accumulate = 1u;
        }
        umma_commit(&empty[stage]);
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
      umma_commit(acc_full);  // also after a failed wait: covers whatever was issued
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(smem_u32(acc_full), 0u))  // no MMA in flight past here
        if (globaltimer_ns() - t0 > p.timeout_ns) { atomicCAS(p.err, 0, kDevTimeoutDrain); break; }
    }
  }

  // The accumulators to shared memory, transposed to red[m][n]: a lane holds
  // one n, so each store of a warp is 32 neighbouring floats. The operand
  // stages are free once the MMAs are done.
  float* red = reinterpret_cast<float*>(ops);
  const bool vec = epi_vec(p.epi);
  if (warp < 4 && valid > 0) {
    if (p.epi.residual.p) {  // on its way to L2 until the sums are there
      const T* res = static_cast<const T*>(p.epi.residual.p) + row0 * p.epi.residual.ld;
      if (vec) {
        const int c = rank * LS_THREADS + static_cast<int>(threadIdx.x), m = c / (LS_COLS / 8);
        const int col = strip * LS_COLS + (c % (LS_COLS / 8)) * 8;
        if (m < valid && col < p.n) prefetch_l2(res + m * p.epi.residual.ld + col);
      } else if ((lane & 15) == 0) {
        const int col = strip * LS_COLS + static_cast<int>(threadIdx.x);
        for (int m = rank; col < p.n && m < valid; m += p.split)
          prefetch_l2(res + m * p.epi.residual.ld + col * p.epi.residual.cs);
      }
    }
    if (work) {
      mbar_wait(acc_full, 0u, ctl, kDevTimeoutAcc);
      tc_fence_after();
    }
    for (int c = 0; c < valid; c += 16) {
      uint32_t r[16];
      if (work) {
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) red[(c + i) * LS_COLS + warp * 32 + lane] = __uint_as_float(r[i]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (p.split > 1) cluster_sync_all();

  const int g0 = rank * LS_THREADS + static_cast<int>(threadIdx.x), gstep = p.split * LS_THREADS;
  constexpr int per_row = LS_COLS / 8;  // 8-column pieces of a strip's row
  if (vec) {
    for (int c = g0; c < valid * per_row; c += gstep) {
      const int m = c / per_row, lc = (c - m * per_row) * 8;
      const int col = strip * LS_COLS + lc;
      if (col >= p.n) continue;
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      const uint32_t at = smem_u32(red + m * LS_COLS + lc);
      // four slices' parts are on their way before the first is added
      for (int r0 = 0; r0 < p.split; r0 += 4) {
        float4 part[4][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r0 + r >= p.split) break;
          const uint32_t a = p.split > 1 ? mapa_shared(at, static_cast<uint32_t>(r0 + r)) : at;
          part[r][0] = ld_cluster_f4(a);
          part[r][1] = ld_cluster_f4(a + 16);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r0 + r >= p.split) break;
          v[0] += part[r][0].x; v[1] += part[r][0].y; v[2] += part[r][0].z; v[3] += part[r][0].w;
          v[4] += part[r][1].x; v[5] += part[r][1].y; v[6] += part[r][1].z; v[7] += part[r][1].w;
        }
      }
      float bias[8];
      load_bias8<T>(p.epi, expert, col, bias);
      epi_store8<T>(p.epi, 0, row0 + m, col, v, bias);
    }
  } else {
    // one element a lane, four rows' residuals in flight; a strip's 128 columns
    // are a fixed one per thread of four warps
    constexpr int kAt = 4;
    const int lc = static_cast<int>(threadIdx.x) & (LS_COLS - 1), col = strip * LS_COLS + lc;
    const float bias = warp < 4 && p.epi.bias && col < p.n
                           ? to_f32<T>(static_cast<const T*>(p.epi.bias)[expert * p.epi.bias_bs + col * p.epi.bias_s])
                           : 0.0f;
    for (int m0 = rank; warp < 4 && col < p.n && m0 < valid; m0 += kAt * p.split) {
      float v[kAt], res[kAt];
#pragma unroll
      for (int q = 0; q < kAt; ++q) {
        const int m = m0 + q * p.split;
        v[q] = res[q] = 0.0f;
        if (m >= valid) continue;
        if (p.epi.residual.p)
          res[q] = to_f32<T>(static_cast<const T*>(p.epi.residual.p)[(row0 + m) * p.epi.residual.ld + col * p.epi.residual.cs]);
        const uint32_t at = smem_u32(red + m * LS_COLS + lc);
        for (int r = 0; r < p.split; ++r)
          v[q] += ld_cluster_f1(p.split > 1 ? mapa_shared(at, static_cast<uint32_t>(r)) : at);
      }
#pragma unroll
      for (int q = 0; q < kAt; ++q) {
        const int m = m0 + q * p.split;
        if (m < valid) epi_store1<T>(p.epi, 0, row0 + m, col, v[q], bias, res[q]);
      }
    }
  }
  if (p.experts) {
    // pad rows of the segment, then this unit's share of the rows after the last segment
    for (int pass = 0; pass < 2; ++pass) {
      const long long from = pass ? p.offsets[p.experts] + static_cast<long long>(mu) : row0 + valid;
      const long long to = pass ? p.rows : zero_end, step = pass ? p.m_units : 1;
      for (long long c = g0; from + (c / per_row) * step < to; c += gstep) {
        const int col = strip * LS_COLS + static_cast<int>(c % per_row) * 8;
        if (col < p.n) epi_zero8<T>(p.epi, from + (c / per_row) * step, col);
      }
    }
  }
  if (p.split > 1) cluster_sync_all();  // peers may still read this CTA's sums
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

}  // namespace mmr
