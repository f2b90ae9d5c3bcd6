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
  void* dst = nullptr;  // [batch][rows_out][pitch], columns past `cols` zeroed
  long long s_b = 0, s_r = 0, s_c = 0;  // source strides (elements, signed)
  int rows = 0, cols = 0, pitch = 0, batch = 1;
  int rows_out = 0;  // rows written; those from `rows` on are zeros
};
struct PackList {
  PackParams p[2];
  int n = 0;
};

// Eight 16-bit elements from `src`, which may lie on any element: whole 32-bit
// words, shifted by a half word where they straddle. The words read are inside
// src[0, 8) and, when they straddle, src[-1, 9): the caller has those.
__device__ __forceinline__ uint4 pack_load8(const unsigned short* src) {
  uint4 v;
  if ((reinterpret_cast<uintptr_t>(src) & 2) == 0) {
    const unsigned int* w = reinterpret_cast<const unsigned int*>(src);
    v = make_uint4(*(w), *(w + 1), *(w + 2), *(w + 3));
  } else {
    const unsigned int* w = reinterpret_cast<const unsigned int*>(src - 1);
    const unsigned int a = *(w), b = *(w + 1), c = *(w + 2), d = *(w + 3), e = *(w + 4);
    v = make_uint4(__funnelshift_r(a, b, 16), __funnelshift_r(b, c, 16), __funnelshift_r(c, d, 16),
                   __funnelshift_r(d, e, 16));
  }
  return v;
}

// Grid (blocks, operands, matrices). E: the element's bits. Rows that are
// contiguous in the source: one 16-byte vector of the destination a thread, 4
// TB/s (element by element it ran at a sixth of that). Other strides: 32 x 32
// tiles through shared memory, the read running along whichever source axis has
// the smaller stride.
template <typename E>
__global__ void __launch_bounds__(256) mmr_pack_kernel(const PackList list) {
  constexpr int kPer = 16 / sizeof(E);
  __shared__ E tile[32][33 + (sizeof(E) == 2)];
  griddep_wait();
  griddep_release();
  const PackParams p = blockIdx.y ? list.p[1] : list.p[0];
  if (static_cast<int>(blockIdx.z) >= p.batch) return;
  const E* src = static_cast<const E*>(p.src) + blockIdx.z * p.s_b;
  E* dst = static_cast<E*>(p.dst) + static_cast<long long>(blockIdx.z) * p.rows_out * p.pitch;
  if (p.s_c == 1) {
    const unsigned int vecs = p.pitch / kPer;
    const long long total = static_cast<long long>(p.rows_out) * vecs, step = gridDim.x * 256ll;
    for (long long i0 = blockIdx.x * 256ll + threadIdx.x; i0 < total; i0 += 4 * step) {
      uint4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long long i = i0 + q * step;
        if (i >= total) continue;
        const long long r = i / vecs;
        const int c = static_cast<int>(i - r * vecs) * kPer;
        const E* s = src + r * p.s_r + c;
        bool done = false;
        if constexpr (sizeof(E) == 2) {
          if (r < p.rows && c > 0 && c + 9 <= p.cols) {
            v[q] = pack_load8(s);
            done = true;
          }
        }
        if (!done) {
          E t[kPer];
#pragma unroll
          for (int x = 0; x < kPer; ++x) t[x] = r < p.rows && c + x < p.cols ? s[x] : E(0);
          memcpy(&v[q], t, 16);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + q * step < total) reinterpret_cast<uint4*>(dst)[i0 + q * step] = v[q];
    }
    return;
  }
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const long long ar = p.s_r < 0 ? -p.s_r : p.s_r, ac = p.s_c < 0 ? -p.s_c : p.s_c;
  const bool along_rows = ar < ac;
  const int tiles_c = (p.pitch + 31) / 32;
  const long long tiles = static_cast<long long>(tiles_c) * ((p.rows_out + 31) / 32);
  for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int r0 = static_cast<int>(t / tiles_c) * 32, c0 = static_cast<int>(t % tiles_c) * 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = y + 8 * i, r = along_rows ? x : a, c = along_rows ? a : x;
      E v = 0;
      if (r0 + r < p.rows && c0 + c < p.cols) v = src[(r0 + r) * p.s_r + (c0 + c) * p.s_c];
      tile[r][c] = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = y + 8 * i;
      if (r0 + r < p.rows_out && c0 + x < p.pitch) dst[static_cast<long long>(r0 + r) * p.pitch + c0 + x] = tile[r][x];
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
      float g;  // Phi(x) + x phi(x), which is 1 less its value at -|x| for x > 0
      const float w = normal_tail(x, &g), left = fmaf(-0.39894228040143f * fabsf(x), g, w);
      return x < 0.0f ? left : 1.0f - left;
    }
    return fmaf(0.39894228040143f * x, expf(-0.5f * x * x), normcdff(x));
  }
  if (act == ACT_SILU) {
    const float s = FAST ? fast_sigmoid(x) : 1.0f / (1.0f + expf(-x));
    return s * fmaf(x, 1.0f - s, 1.0f);
  }
  // gelu_tanh: with s = (1 + tanh u) / 2, d(x s) = s + 2 x s (1 - s) u'
  const float s =
      FAST ? gelu_gate(x) : 1.0f / (1.0f + expf(-x * fmaf(0.0713548162726f, x * x, 1.5957691216057f)));
  const float du2 = fmaf(0.2140644488178f, x * x, 1.5957691216057f);
  return fmaf(x * s * (1.0f - s), du2, s);
}

constexpr int AG_ROWS = 64;   // rows of one block: a chunk of the column sums
constexpr int AG_COLS = 256;  // columns of one block: 32 threads x 8

struct ActGradParams {
  EpiMat d_out, pre, d_pre;  // without an activation only the column sums are made
  float* partial = nullptr;  // [chunks][n] column sums of 64-row chunks, or null
  long long rows = 0;
  int n = 0, act = 0;
  const int* sources = nullptr;  // sorted rows: a row without a token counts as zero
};

// Grid (column strips, row chunks). A thread has eight columns of a strip: with
// VEC neighbouring ones, one 16-byte vector (two in f32) a row, several rows'
// loads in flight together; without, every 32nd, so that a warp's accesses stay
// contiguous for any pitch. The sums are of the f32 values, before d_pre is
// rounded. Chunk sums go out in f32 and are added in chunk order by
// mmr_col_sum_kernel, so the result does not depend on which block ran first.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) mmr_act_grad_kernel(const ActGradParams p) {
  constexpr int kRows = VEC ? (sizeof(T) == 2 ? 4 : 2) : 1;
  constexpr int kVec = sizeof(T) / 2;
  union Raw {
    uint4 w[kVec];
    T t[8];
    __device__ Raw() {}
  };
  __shared__ float sums[8][AG_COLS];
  griddep_wait();
  griddep_release();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = static_cast<int>(blockIdx.x) * AG_COLS;
  auto col = [&](int i) { return VEC ? tx * 8 + i : tx + 32 * i; };
  auto load = [&](const T* q, const EpiMat& m, Raw& r) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) r.w[i] = __ldcg(reinterpret_cast<const uint4*>(q + tx * 8) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.t[i] = c0 + col(i) < p.n ? q[col(i) * m.cs] : from_f32<T>(0.0f);
    }
  };
  for (long long chunk = blockIdx.y; chunk * AG_ROWS < p.rows; chunk += gridDim.y) {
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (!VEC || c0 + tx * 8 < p.n) {
      const long long row0 = chunk * AG_ROWS + ty;
      const int left = static_cast<int>(min(p.rows - row0, static_cast<long long>(AG_ROWS)));  // rows 0, 8, .. below this
      const T* dq = static_cast<const T*>(p.d_out.p) + row0 * p.d_out.ld + c0 * p.d_out.cs;
      const T* xq = static_cast<const T*>(p.pre.p) + row0 * p.pre.ld + c0 * p.pre.cs;
      T* oq = static_cast<T*>(p.d_pre.p) + row0 * p.d_pre.ld + c0;  // the workspace: dense rows
#pragma unroll 1
      for (int i = 0; i < AG_ROWS; i += 8 * kRows) {
        Raw d[kRows], x[kRows];
        bool held[kRows];
#pragma unroll
        for (int q = 0; q < kRows; ++q) {
          held[q] = i + 8 * q < left && (!p.sources || p.sources[row0 + i + 8 * q] >= 0);
          if (held[q]) {
            load(dq + 8 * q * p.d_out.ld, p.d_out, d[q]);
            if (ACT != ACT_NONE) load(xq + 8 * q * p.pre.ld, p.pre, x[q]);
          }
        }
#pragma unroll
        for (int q = 0; q < kRows; ++q) {
          float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
          if (held[q]) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              v[c] = to_f32<T>(d[q].t[c]);
              if (ACT != ACT_NONE) v[c] *= lact_grad<sizeof(T) == 2>(ACT, to_f32<T>(x[q].t[c]));
              s[c] += v[c];
            }
          }
          if (ACT != ACT_NONE && i + 8 * q < left) {
            T* to = oq + 8 * q * p.d_pre.ld;
            if constexpr (VEC && sizeof(T) == 2) {
              *reinterpret_cast<uint4*>(to + tx * 8) = pack8<T>(v);
            } else if (VEC) {
#pragma unroll
              for (int c = 0; c < 8; c += 4)
                *reinterpret_cast<float4*>(to + tx * 8 + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
            } else {
#pragma unroll
              for (int c = 0; c < 8; ++c)
                if (c0 + col(c) < p.n) to[col(c)] = from_f32<T>(v[c]);
            }
          }
        }
        dq += 8 * kRows * p.d_out.ld;
        xq += 8 * kRows * p.pre.ld;
        oq += 8 * kRows * p.d_pre.ld;
      }
    }
    if (p.partial) {
#pragma unroll
      for (int q = 0; q < 8; ++q) sums[ty][col(q)] = s[q];
      __syncthreads();
      const int c = c0 + static_cast<int>(threadIdx.x);
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
  const int c0 = p.offsets ? max(p.offsets[e], 0) / AG_ROWS : 0;
  const int c1 = p.offsets ? min(p.offsets[e + 1] / AG_ROWS, p.chunks) : p.chunks;
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

// ------------------------------------- bias, activation and residual (f32) --
// pre = x + bias; out = act(pre) + residual over a bare f32 product x, which may
// lie in pre's or out's own storage (each element is read and written by one
// thread) or in the parts of a divided K, added in order. Bound by memory.
struct ActResParams {
  EpiMat x, pre, residual, out;  // pre.p and residual.p may be null
  int parts = 1;                 // x.bs apart
  const float* bias = nullptr;
  long long bias_s = 0;
  int m = 0, n = 0;
};

// The activations in f32, inlined (the matmul node's epilogue calls them out of
// line): the formulas of linear_epi.cuh on CUDA's expf and normcdff and correctly
// rounded divisions. EXACT: the node's own, step by step (act_apply).
template <int ACT, bool EXACT = false>
__device__ __forceinline__ float act_f32(float x) {
  if (EXACT) return act_apply(ACT, x);
  if (ACT == ACT_RELU) return act_relu(x);
  if (ACT == ACT_RELU6) return x != x ? x : fminf(fmaxf(x, 0.0f), 6.0f);
  if (ACT == ACT_SILU) return no_inf(x, __fdiv_rn(x, 1.0f + expf(-x)));
  if (ACT == ACT_GELU_TANH) return no_inf(x, __fdiv_rn(x, 1.0f + expf(-x * fmaf(0.0713548162726f, x * x, 1.5957691216057f))));
  if (ACT == ACT_GELU_ERF) return no_inf(x, x * normcdff(x));
  return x;
}

// A warp takes 128 columns of a row, four columns a thread where everything is
// 16-byte vectors.
template <int ACT, bool EXACT>
__global__ void __launch_bounds__(256) mmr_act_res_kernel(const ActResParams p) {
  griddep_wait();
  griddep_release();
  const int lane = threadIdx.x & 31;
  const unsigned int pieces = (p.n + 127) / 128;
  const long long units = static_cast<long long>(p.m) * pieces, step = static_cast<long long>(gridDim.x) * 8;
  const bool vec = p.x.vec && p.out.vec && (!p.residual.p || p.residual.vec) && (!p.pre.p || p.pre.vec);
  const float *x = static_cast<const float*>(p.x.p), *res = static_cast<const float*>(p.residual.p);
  float *out = static_cast<float*>(p.out.p), *pre = static_cast<float*>(p.pre.p);
  for (long long u = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); u < units; u += step) {
    const long long row = u / pieces;
    const int c0 = static_cast<int>(u - row * pieces) * 128;
    if (vec && c0 + 128 <= p.n) {
      const int c = c0 + lane * 4;
      float4 v = *reinterpret_cast<const float4*>(x + row * p.x.ld + c);
#pragma unroll 4
      for (int q = 1; q < p.parts; ++q) {
        const float4 y = *reinterpret_cast<const float4*>(x + q * p.x.bs + row * p.x.ld + c);
        v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
      }
      float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (res) r = *reinterpret_cast<const float4*>(res + row * p.residual.ld + c);
      if (p.bias) {
        v.x = __fadd_rn(v.x, p.bias[c * p.bias_s]);
        v.y = __fadd_rn(v.y, p.bias[(c + 1) * p.bias_s]);
        v.z = __fadd_rn(v.z, p.bias[(c + 2) * p.bias_s]);
        v.w = __fadd_rn(v.w, p.bias[(c + 3) * p.bias_s]);
      }
      if (pre) *reinterpret_cast<float4*>(pre + row * p.pre.ld + c) = v;
      v = make_float4(act_f32<ACT, EXACT>(v.x), act_f32<ACT, EXACT>(v.y), act_f32<ACT, EXACT>(v.z), act_f32<ACT, EXACT>(v.w));
      if (res) v = make_float4(v.x + r.x, v.y + r.y, v.z + r.z, v.w + r.w);
      *reinterpret_cast<float4*>(out + row * p.out.ld + c) = v;
    } else {
      for (int c = c0 + lane; c < min(c0 + 128, p.n); c += 32) {
        float v = x[row * p.x.ld + c * p.x.cs];
        for (int q = 1; q < p.parts; ++q) v += x[q * p.x.bs + row * p.x.ld + c * p.x.cs];
        if (p.bias) v = __fadd_rn(v, p.bias[c * p.bias_s]);
        if (pre) pre[row * p.pre.ld + c * p.pre.cs] = v;
        v = act_f32<ACT, EXACT>(v);
        if (res) v += res[row * p.residual.ld + c * p.residual.cs];
        out[row * p.out.ld + c * p.out.cs] = v;
      }
    }
  }
}

// ------------------------------------------------ f32 products of few rows --
// pre = a b^T + bias; out = act(pre) + residual, b contiguous along k and a of at
// most eight rows: a warp takes a row of b, read once, against all rows of a
// (which stay in L1), and lane i finishes row i. Bound by b's bytes: 1 x 16384 x
// 4096 42 to 45 us by the box, 6.0 to 6.4 TB/s. The MatMul node's streaming kernels want b row-major;
// its tensor-core kernel took 184 us at 1 x 4096 x 4096.
struct DotParams {
  const float *a = nullptr, *b = nullptr;
  long long a_m = 0, a_k = 0, b_n = 0;
  int k = 0, act = ACT_NONE;
  ActResParams post;  // what follows the product; its x is not used
};

__device__ __forceinline__ float act_f32_any(int act, float x) {
  switch (act) {
    case ACT_RELU: return act_f32<ACT_RELU>(x);
    case ACT_RELU6: return act_f32<ACT_RELU6>(x);
    case ACT_SILU: return act_f32<ACT_SILU>(x);
    case ACT_GELU_TANH: return act_f32<ACT_GELU_TANH>(x);
    case ACT_GELU_ERF: return act_f32<ACT_GELU_ERF>(x);
    default: return x;
  }
}

// VEC: every row of a and b is 16-byte vectors (k a multiple of 4).
template <int M, bool VEC>
__global__ void __launch_bounds__(256) mmr_dot_kernel(const DotParams p) {
  constexpr int kStep = VEC ? 4 : 1;  // k a lane takes at a time
  constexpr int kFly = M <= 2 ? 4 : 2;
  griddep_wait();
  griddep_release();
  const int lane = threadIdx.x & 31;
  const ActResParams& e = p.post;
  for (long long n = blockIdx.x * 8ll + (threadIdx.x >> 5); n < e.n; n += gridDim.x * 8ll) {
    const float* b = p.b + n * p.b_n;
    float s[M];
#pragma unroll
    for (int i = 0; i < M; ++i) s[i] = 0.0f;
    for (int k0 = lane * kStep; k0 < p.k; k0 += 32 * kStep * kFly) {
      float w[kFly][kStep];
#pragma unroll
      for (int q = 0; q < kFly; ++q) {
        const int k = k0 + 32 * kStep * q;
#pragma unroll
        for (int c = 0; c < kStep; ++c) w[q][c] = 0.0f;
        if (k >= p.k) continue;
        if constexpr (VEC) *reinterpret_cast<float4*>(w[q]) = __ldcg(reinterpret_cast<const float4*>(b + k));
        else w[q][0] = __ldcg(b + k);
      }
#pragma unroll
      for (int q = 0; q < kFly; ++q) {
        const int k = k0 + 32 * kStep * q;
        if (k >= p.k) continue;
#pragma unroll
        for (int i = 0; i < M; ++i) {
          if (i >= e.m) continue;
          if constexpr (VEC) {
            const float4 a = *reinterpret_cast<const float4*>(p.a + i * p.a_m + k);
            s[i] = fmaf(a.x, w[q][0], s[i]);
            s[i] = fmaf(a.y, w[q][1], s[i]);
            s[i] = fmaf(a.z, w[q][2], s[i]);
            s[i] = fmaf(a.w, w[q][3], s[i]);
          } else {
            s[i] = fmaf(p.a[i * p.a_m + k * p.a_k], w[q][0], s[i]);
          }
        }
      }
    }
    float v = 0.0f;  // lane i: row i
#pragma unroll
    for (int i = 0; i < M; ++i) {
#pragma unroll
      for (int d = 16; d; d >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
      if (lane == i) v = s[i];
    }
    if (lane < e.m) {
      if (e.bias) v = __fadd_rn(v, e.bias[n * e.bias_s]);
      if (e.pre.p) static_cast<float*>(e.pre.p)[lane * e.pre.ld + n * e.pre.cs] = v;
      v = act_f32_any(p.act, v);
      if (e.residual.p) v += static_cast<const float*>(e.residual.p)[lane * e.residual.ld + n * e.residual.cs];
      static_cast<float*>(e.out.p)[lane * e.out.ld + n * e.out.cs] = v;
    }
  }
}

}  // namespace mmr
