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

// 2^x and 1 / x by the special function unit: about 2 and 1 units in the last
// place, subnormals flushed.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Activations for 16-bit results, each of one exponential and one reciprocal:
// relative error below 2^-17 plus 2^-22 for every unit of the exponent (an
// argument rounded in f32), against the 2^-12 of an f16 rounding.
//   silu       x / (1 + e^-x)
//   gelu_tanh  x (1 + tanh u) / 2 = x / (1 + e^-2u), u = sqrt(2/pi)(x + 0.044715 x^3):
//              no 1 + tanh, which cancels for x < 0
//   gelu_erf   x Phi(x), by the tail Phi(-|x|) below
// As in the f32 epilogue, -inf gives -0 (not inf times 0) and NaN stays NaN.
constexpr float kLog2e = 1.4426950408890f;
__device__ __forceinline__ float no_inf(float x, float y) { return x == -__int_as_float(0x7f800000) ? -0.0f : y; }
__device__ __forceinline__ float fast_sigmoid(float x) { return fast_rcp(1.0f + fast_exp2(-kLog2e * x)); }
// sigmoid(2u): the coefficients 2 sqrt(2/pi) (0.044715, 1)
__device__ __forceinline__ float gelu_gate(float x) {
  return fast_rcp(1.0f + fast_exp2(x * fmaf(-0.0713548162726f * kLog2e, x * x, -1.5957691216057f * kLog2e)));
}
__device__ __forceinline__ float lact_silu(float x) { return no_inf(x, x * fast_sigmoid(x)); }
__device__ __forceinline__ float lact_gelu_tanh(float x) { return no_inf(x, x * gelu_gate(x)); }
// Phi(-|x|) and e^(-x^2/2). With z = |x| / sqrt 2 and t = 1 / (1 + 0.38 z),
//   erfc(z) = t P(t) e^(-z^2),
// P of degree 6 with the least largest relative error on 0 <= z <= 9.5, 1.0e-6
// (found by linear programming over 6000 points): relative, so that x Phi(x)
// keeps its bits where it runs out to the left. The coefficients are P's halves.
__device__ __forceinline__ float normal_tail(float x, float* gauss) {
  const float t = fast_rcp(fmaf(0.38f * 0.70710678118655f, fabsf(x), 1.0f));
  const float g = fast_exp2(-0.5f * kLog2e * x * x);
  float p = fmaf(-0.0625223433007686f, t, 0.1673000517084580f);
  p = fmaf(p, t, -0.0338413079234745f);
  p = fmaf(p, t, 0.1230267267987761f);
  p = fmaf(p, t, 0.0906809299674027f);
  p = fmaf(p, t, 0.1082044550110211f);
  p = fmaf(p, t, 0.1071509821877172f);
  *gauss = g;
  return p * t * g;
}
// x Phi(x) = max(x, 0) - |x| Phi(-|x|); of an infinity the first term alone.
__device__ __forceinline__ float lact_gelu_erf(float x) {
  float g;
  const float tail = normal_tail(x, &g), rest = fmaxf(x, -0.0f);
  return fabsf(x) == __int_as_float(0x7f800000) ? rest : fmaf(-fabsf(x), tail, rest);
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

// Eight f32 to eight 16-bit values, two a conversion, and back.
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float2 unpack2(__nv_bfloat16, uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
__device__ __forceinline__ float2 unpack2(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2(T(), v[0], v[1]), pack2(T(), v[2], v[3]), pack2(T(), v[4], v[5]), pack2(T(), v[6], v[7]));
}
template <typename T>
__device__ __forceinline__ void add8(float (&v)[8], const uint4& w) {
  const float2 a = unpack2(T(), w.x), b = unpack2(T(), w.y), c = unpack2(T(), w.z), d = unpack2(T(), w.w);
  v[0] += a.x; v[1] += a.y; v[2] += b.x; v[3] += b.y;
  v[4] += c.x; v[5] += c.y; v[6] += d.x; v[7] += d.y;
}

template <typename T>
__device__ __forceinline__ void store8(const EpiMat& m, long long b, long long row, int col, int n,
                                       const float (&v)[8]) {
  T* q = static_cast<T*>(m.p) + b * m.bs + row * m.ld + col * m.cs;
  if (m.vec && col + 8 <= n) {
    *reinterpret_cast<uint4*>(q) = pack8<T>(v);
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
  for (int i = 0; i < 8; ++i) b[i] = 0.0f;
  if (!e.bias) return;
  const T* q = static_cast<const T*>(e.bias) + batch * e.bias_bs + col * e.bias_s;
  if (e.bias_s == 1 && col + 8 <= e.n && (reinterpret_cast<uintptr_t>(q) & 15) == 0) {
    add8<T>(b, *(reinterpret_cast<const uint4*>(q)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < e.n) b[i] = to_f32<T>(q[i * e.bias_s]);
  }
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
      add8<T>(v, *reinterpret_cast<const uint4*>(q));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < e.n) v[i] += to_f32<T>(q[i * e.residual.cs]);
    }
  }
  store8<T>(e.out, batch, row, col, e.n, v);
}

// Four rows of C neighbouring columns: v[4 c + r]. C 2 wants every view's pairs
// of columns on one 32-bit word (n even, and epi_vec). Rows from `rows` on are left out.
template <typename T, int C>
__device__ __forceinline__ void epi_store_quad(const EpiParams& e, int expert, long long row, int rows, int col,
                                               float (&v)[4 * C]) {
  float add[4 * C];
  if (e.residual.p) {
    const T* q = static_cast<const T*>(e.residual.p) + row * e.residual.ld + col * e.residual.cs;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r < rows) {
        if (C == 2) {
          const float2 w = unpack2(T(), *reinterpret_cast<const uint32_t*>(q));
          add[r] = w.x;
          add[4 * (C - 1) + r] = w.y;
        } else {
          add[r] = to_f32<T>(*q);
        }
      }
      q += e.residual.ld;
    }
  }
  if (e.bias) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float b = to_f32<T>(static_cast<const T*>(e.bias)[expert * e.bias_bs + (col + c) * e.bias_s]);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[4 * c + r] += b;
    }
  }
  auto put = [&](const EpiMat& m) {
    T* q = static_cast<T*>(m.p) + row * m.ld + col * m.cs;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r < rows) {
        if (C == 2) *reinterpret_cast<uint32_t*>(q) = pack2(T(), v[r], v[4 * (C - 1) + r]);
        else *q = from_f32<T>(v[r]);
      }
      q += m.ld;
    }
  };
  if (e.pre.p) put(e.pre);
  lact_apply(e.act, v);
  if (e.residual.p) {
#pragma unroll
    for (int r = 0; r < 4 * C; ++r) v[r] += (r & 3) < rows ? add[r] : 0.0f;
  }
  put(e.out);
}
__device__ __forceinline__ bool epi_vec(const EpiParams& e) {
  return e.out.vec && (!e.pre.p || e.pre.vec) && (!e.residual.p || e.residual.vec);
}

template <typename T>
__device__ __forceinline__ void epi_zero8(const EpiParams& e, long long row, int col) {
  const float z[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (e.pre.p) store8<T>(e.pre, 0, row, col, e.n, z);
  store8<T>(e.out, 0, row, col, e.n, z);
}

}  // namespace mmr
