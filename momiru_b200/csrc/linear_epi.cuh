// linear_epi.cuh -- what the linear and expert products do to an accumulator
// on its way out:
//   pre = acc + bias[col];  out = act(pre) + residual
// in f32, rounded once to the output's 16-bit type (pre is rounded on its own).
//
// The accumulators are staged in shared memory as f32 first and handled here
// eight neighbouring columns at a time, so that every global access of a warp
// is a 16-byte vector on a 64-byte row segment, whatever the kernel's tile
// shape, and the residual joins before the only rounding.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "epilogue.cuh"

namespace mmr {



template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Activations for 16-bit results. Each is written so that one exponential and
// one division carry it: their approximate forms are good to about 2^-21,
// against the 2^-12 of an f16 rounding.
//   silu       x / (1 + e^-x)
//   gelu_tanh  x (1 + tanh u) / 2 = x / (1 + e^-2u), u = sqrt(2/pi)(x + 0.044715 x^3):
//              no 1 + tanh, which cancels for x < 0
//   gelu_erf   x Phi(x) with erfc by Abramowitz & Stegun 7.1.26 (absolute
//              error below 1.5e-7)
// As in the f32 epilogue, -inf gives -0 (not inf / inf) and NaN stays NaN.
__device__ __forceinline__ float lact_silu(float x) {
  return x == -__int_as_float(0x7f800000) ? -0.0f : __fdividef(x, 1.0f + __expf(-x));
}
__device__ __forceinline__ float lact_gelu_tanh(float x) {
  const float u2 = x * fmaf(0.0713548162726f, x * x, 1.5957691216057f);  // 2 sqrt(2/pi) (0.044715, 1)
  return x == -__int_as_float(0x7f800000) ? -0.0f : __fdividef(x, 1.0f + __expf(-u2));
}
// Phi(x) and e^(-x^2/2).
__device__ __forceinline__ float normal_cdf(float x, float* gauss) {
  const float z = fabsf(x) * 0.70710678118655f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
  const float g = __expf(-z * z);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float half_erfc = 0.5f * p * t * g;
  *gauss = g;
  return x < 0.0f ? half_erfc : 1.0f - half_erfc;
}
__device__ __forceinline__ float lact_gelu_erf(float x) {
  float g;
  const float c = normal_cdf(x, &g);
  return x == -__int_as_float(0x7f800000) ? -0.0f : x * c;
}

template <int N>
__device__ __forceinline__ void lact_apply(int act, float (&v)[N]) {
  switch (act) {
    case ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (v[i] != v[i] || v[i] > 0.0f) ? v[i] : 0.0f;
      break;
    case ACT_RELU6:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] != v[i] ? v[i] : fminf(fmaxf(v[i], 0.0f), 6.0f);
      break;
    case ACT_GELU_ERF:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lact_gelu_erf(v[i]);
      break;
    case ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lact_gelu_tanh(v[i]);
      break;
    case ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lact_silu(v[i]);
      break;
    default: break;
  }
}

// A strided matrix of the epilogue: element (row, col) of batch b (an expert's
// weight gradient) at p + b * bs + row * ld + col * cs. vec: 8 columns starting
// at a multiple of 8 are one aligned 16-byte vector.
struct EpiMat {
  void* p = nullptr;
  long long bs = 0, ld = 0, cs = 0;
  int vec = 0;
};

struct EpiParams {
  EpiMat out, pre, residual;
  const void* bias = nullptr;
  long long bias_bs = 0, bias_s = 0;
  int act = 0;
  int n = 0;
};

union Pack8 {
  uint4 u;
  unsigned short h[8];
};

template <typename T>
__device__ __forceinline__ void store8(const EpiMat& m, long long b, long long row, int col, int n,
                                       const float (&v)[8]) {
  T* q = static_cast<T*>(m.p) + b * m.bs + row * m.ld + col * m.cs;
  if (m.vec && col + 8 <= n) {
    Pack8 w;
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<T*>(&w.h[i]) = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(q) = w.u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < n) q[i * m.cs] = from_f32<T>(v[i]);
  }
}

// The bias of columns col .. col + 7 (zero past the edge or without a bias).
template <typename T>
__device__ __forceinline__ void load_bias8(const EpiParams& e, int batch, int col, float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    b[i] = e.bias && col + i < e.n
               ? to_f32<T>(static_cast<const T*>(e.bias)[batch * e.bias_bs + (col + i) * e.bias_s])
               : 0.0f;
}

// The epilogue of (row, col .. col + 7): v holds the accumulators. The residual
// may be the output's own storage: each element is read before it is written,
// by the thread that writes it (so it is not read through the read-only path).
template <typename T>
__device__ __forceinline__ void epi_store8(const EpiParams& e, long long batch, long long row, int col, float (&v)[8],
                                           const float (&bias)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  if (e.pre.p) store8<T>(e.pre, batch, row, col, e.n, v);
  lact_apply(e.act, v);
  if (e.residual.p) {
    const T* q = static_cast<const T*>(e.residual.p) + row * e.residual.ld + col * e.residual.cs;
    if (e.residual.vec && col + 8 <= e.n) {
      Pack8 w;
      w.u = *reinterpret_cast<const uint4*>(q);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += to_f32<T>(*reinterpret_cast<T*>(&w.h[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < e.n) v[i] += to_f32<T>(q[i * e.residual.cs]);
    }
  }
  store8<T>(e.out, batch, row, col, e.n, v);
}

template <typename T>
__device__ __forceinline__ void epi_zero8(const EpiParams& e, long long row, int col) {
  const float z[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (e.pre.p) store8<T>(e.pre, 0, row, col, e.n, z);
  store8<T>(e.out, 0, row, col, e.n, z);
}

}  // namespace mmr
