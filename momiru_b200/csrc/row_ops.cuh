// row_ops.cuh -- the row-wise passes around the linear products:
//   pack      a strided operand copied to rows of a 16-byte pitch, so that the
//             products reach any layout through TMA
//   act_grad  d_pre = d_out act'(pre), and the column sums of d_pre for the
//             bias gradient
// All are bound by memory: one read of each input, one write of each output.
#pragma once
#include <cstring>

#include "linear_epi.cuh"
#include "ptx.cuh"

namespace mmr {

// ----------------------------------------------------------------- pack --
struct PackParams {
  const void* src = nullptr;
  void* dst = nullptr;  // [batch][rows][pitch], columns past `cols` zeroed
  long long s_b = 0, s_r = 0, s_c = 0;  // source strides (elements, signed)
  int rows = 0, cols = 0, pitch = 0;
};

// 32 x 32 tiles through shared memory: the read runs along whichever source
// axis has the smaller stride, the write along the rows of the destination.
__global__ void __launch_bounds__(256) mmr_pack_kernel(const PackParams p) {
  __shared__ unsigned short tile[32][34];
  griddep_wait();
  griddep_release();
  const unsigned short* src = static_cast<const unsigned short*>(p.src) + blockIdx.z * p.s_b;
  unsigned short* dst = static_cast<unsigned short*>(p.dst) + static_cast<long long>(blockIdx.z) * p.rows * p.pitch;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const long long ar = p.s_r < 0 ? -p.s_r : p.s_r, ac = p.s_c < 0 ? -p.s_c : p.s_c;
  const bool along_rows = ar < ac;
  const int tiles_c = (p.pitch + 31) / 32;
  const long long tiles = static_cast<long long>(tiles_c) * ((p.rows + 31) / 32);
  for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int r0 = static_cast<int>(t / tiles_c) * 32, c0 = static_cast<int>(t % tiles_c) * 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = y + 8 * i, r = along_rows ? x : a, c = along_rows ? a : x;
      unsigned short v = 0;
      if (r0 + r < p.rows && c0 + c < p.cols) v = src[(r0 + r) * p.s_r + (c0 + c) * p.s_c];
      tile[r][c] = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = y + 8 * i;
      if (r0 + r < p.rows && c0 + x < p.pitch) dst[static_cast<long long>(r0 + r) * p.pitch + c0 + x] = tile[r][x];
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------- act_grad --
// Derivatives. 16-bit types take the fast forms of linear_epi.cuh, f32 CUDA's
// math functions. The argument is clamped to +-1e4, where every derivative has
// long reached its limit of 0 or 1 (so that infinities give the limit and not
// 0 * inf); NaN stays NaN.
template <bool FAST>
__device__ __forceinline__ float lact_grad(int act, float x) {
  if (act == ACT_NONE) return 1.0f;
  if (act == ACT_RELU) return x != x ? x : (x > 0.0f ? 1.0f : 0.0f);
  if (act == ACT_RELU6) return x != x ? x : (x > 0.0f && x < 6.0f ? 1.0f : 0.0f);
  x = x > 1e4f ? 1e4f : (x < -1e4f ? -1e4f : x);
  if (act == ACT_GELU_ERF) {
    if (FAST) {
      float g;
      const float c = normal_cdf(x, &g);
      return fmaf(0.39894228040143f * x, g, c);
    }
    return fmaf(0.39894228040143f * x, expf(-0.5f * x * x), normcdff(x));
  }
  if (act == ACT_SILU) {
    const float s = FAST ? __fdividef(1.0f, 1.0f + __expf(-x)) : 1.0f / (1.0f + expf(-x));
    return s * fmaf(x, 1.0f - s, 1.0f);
  }
  // gelu_tanh: with s = (1 + tanh u) / 2, d(x s) = s + 2 x s (1 - s) u'
  const float u2 = x * fmaf(0.0713548162726f, x * x, 1.5957691216057f);
  const float s = FAST ? __fdividef(1.0f, 1.0f + __expf(-u2)) : 1.0f / (1.0f + expf(-u2));
  const float du2 = fmaf(0.2140644488178f, x * x, 1.5957691216057f);
  return fmaf(x * s * (1.0f - s), du2, s);
}

constexpr int AG_ROWS = 64;   // rows of one block: a chunk of the column sums
constexpr int AG_COLS = 256;  // columns of one block: 32 threads x 8

struct ActGradParams {
  EpiMat d_out, pre, d_pre;  // d_pre.p null: only the column sums
  float* partial = nullptr;  // [chunks][n] column sums of 64-row chunks, or null
  long long rows = 0;
  int n = 0, act = 0;
  const int* sources = nullptr;  // sorted rows: a row without a token counts as zero
};

template <typename T>
__device__ __forceinline__ void ag_load8(const EpiMat& m, long long row, int col, int n, float (&v)[8]) {
  const T* q = static_cast<const T*>(m.p) + row * m.ld + col * m.cs;
  if (m.vec && col + 8 <= n) {
    constexpr int kVec = sizeof(T) == 4 ? 2 : 1;
    uint4 w[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(q) + i);
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < n ? to_f32<T>(q[i * m.cs]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void ag_store8(const EpiMat& m, long long row, int col, int n, const float (&v)[8]) {
  T* q = static_cast<T*>(m.p) + row * m.ld + col * m.cs;
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(v[i]);
  if (m.vec && col + 8 <= n) {
    constexpr int kVec = sizeof(T) == 4 ? 2 : 1;
    uint4 w[kVec];
    memcpy(w, t, sizeof w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) reinterpret_cast<uint4*>(q)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < n) q[i * m.cs] = t[i];
  }
}

// Grid (column strips, row chunks). The sums are of the f32 values, before
// d_pre is rounded. Chunk sums go out in f32 and are added in chunk order by
// mmr_col_sum_kernel, so the result does not depend on which block ran first.
template <typename T>
__global__ void __launch_bounds__(256) mmr_act_grad_kernel(const ActGradParams p) {
  __shared__ float sums[8][AG_COLS];
  griddep_wait();
  griddep_release();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = static_cast<int>(blockIdx.x) * AG_COLS + tx * 8;
  for (long long chunk = blockIdx.y; chunk * AG_ROWS < p.rows; chunk += gridDim.y) {
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = 0; i < AG_ROWS / 8; ++i) {
      const long long row = chunk * AG_ROWS + i * 8 + ty;
      if (row >= p.rows || col >= p.n) continue;
      float d[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (!p.sources || p.sources[row] >= 0) {
        ag_load8<T>(p.d_out, row, col, p.n, d);
        if (p.act != ACT_NONE) {
          float x[8];
          ag_load8<T>(p.pre, row, col, p.n, x);
#pragma unroll
          for (int q = 0; q < 8; ++q) d[q] *= lact_grad<sizeof(T) == 2>(p.act, x[q]);
        }
      }
      if (p.d_pre.p) ag_store8<T>(p.d_pre, row, col, p.n, d);
#pragma unroll
      for (int q = 0; q < 8; ++q) s[q] += d[q];
    }
    if (p.partial) {
#pragma unroll
      for (int q = 0; q < 8; ++q) sums[ty][tx * 8 + q] = s[q];
      __syncthreads();
      const int c = static_cast<int>(blockIdx.x) * AG_COLS + static_cast<int>(threadIdx.x);
      float t = 0.0f;
#pragma unroll
      for (int y = 0; y < 8; ++y) t += sums[y][threadIdx.x];
      if (c < p.n) p.partial[chunk * p.n + c] = t;
      __syncthreads();
    }
  }
}

struct ColSumParams {
  const float* partial = nullptr;
  void* out = nullptr;
  long long out_bs = 0, out_s = 0;
  int n = 0, chunks = 0;
  const int* offsets = nullptr;  // experts: chunks offsets[e] / 64 .. offsets[e + 1] / 64
};

// Grid (columns / 32, experts or 1), 256 threads: eight threads a column, each
// over every eighth chunk, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) mmr_col_sum_kernel(const ColSumParams p) {
  __shared__ float sums[8][32];
  griddep_wait();
  griddep_release();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = static_cast<int>(blockIdx.x) * 32 + tx, e = static_cast<int>(blockIdx.y);
  const int c0 = p.offsets ? p.offsets[e] / AG_ROWS : 0, c1 = p.offsets ? p.offsets[e + 1] / AG_ROWS : p.chunks;
  float s = 0.0f;
  if (c < p.n) {
#pragma unroll 4
    for (int i = c0 + ty; i < c1; i += 8) s += p.partial[static_cast<long long>(i) * p.n + c];
  }
  sums[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < p.n) {
    float t = 0.0f;
#pragma unroll
    for (int y = 0; y < 8; ++y) t += sums[y][tx];
    static_cast<T*>(p.out)[e * p.out_bs + c * p.out_s] = from_f32<T>(t);
  }
}

// ---------------------------------------------- activation and residual --
// out = act(pre) + residual over an f32 product that was left in `out` or kept
// in `pre` (the f32 linear node with a residual or a kept pre).
struct ActResParams {
  const float* pre = nullptr;
  const float* residual = nullptr;
  float* out = nullptr;
  long long pre_ld = 0, res_ld = 0, res_cs = 0, out_ld = 0, out_cs = 0, pre_cs = 0;
  int m = 0, n = 0, act = 0;
};

__global__ void __launch_bounds__(256) mmr_act_res_kernel(const ActResParams p) {
  griddep_wait();
  griddep_release();
  const long long total = static_cast<long long>(p.m) * p.n;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / p.n, c = i - r * p.n;
    float x = act_apply(p.act, p.pre[r * p.pre_ld + c * p.pre_cs]);
    if (p.residual) x += p.residual[r * p.res_ld + c * p.res_cs];
    p.out[r * p.out_ld + c * p.out_cs] = x;
  }
}

}  // namespace mmr
