// linear_pair_launch.cuh -- launch and preparation of the CTA-pair product for
// one element type. Included by exactly one translation unit per type.
#pragma once
#include "launch.cuh"
#include "linear_launch.h"

namespace mmr {

using PairKernel = void (*)(const CUtensorMap, const CUtensorMap, const PairParams);

template <typename T>
PairKernel pair_kernel(const PairShape& sh) {
  const bool a_mn = sh.a_mn, b_mn = sh.b_mn;
  const int rag = sh.rag;
  if (rag == 0) {
    if (a_mn) return b_mn ? mmr_linear_pair_kernel<T, true, true, 0> : mmr_linear_pair_kernel<T, true, false, 0>;
    return b_mn ? mmr_linear_pair_kernel<T, false, true, 0> : mmr_linear_pair_kernel<T, false, false, 0>;
  }
  if (rag == 1 && !a_mn)
    return b_mn ? mmr_linear_pair_kernel<T, false, true, 1> : mmr_linear_pair_kernel<T, false, false, 1>;
  if (rag == 2 && a_mn && b_mn) return mmr_linear_pair_kernel<T, true, true, 2>;
  return nullptr;
}
template <typename T>
cudaError_t pair_launch_t(const PairShape& sh, cudaStream_t s, const CUtensorMap& tm_a, const CUtensorMap& tm_b,
                          const PairParams& p) {
  const PairKernel k = pair_kernel<T>(sh);
  if (!k) return cudaErrorInvalidValue;
  return launch_kernel(k, dim3(sh.grid), dim3(LP_THREADS), lp_smem_bytes(sh.rag), s, dim3(2, 1, 1), tm_a, tm_b, p);
}

template <typename T>
cudaError_t pair_prepare_t(const PairShape& sh) {
  const PairKernel k = pair_kernel<T>(sh);
  if (!k) return cudaErrorInvalidValue;
  // setmaxnreg.inc waits for registers that the launch has to have: a build
  // compiled with fewer is refused here instead of launched.
  cudaFuncAttributes fa;
  const cudaError_t e = cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(k));
  if (e != cudaSuccess) return e;
  if (fa.numRegs * LP_THREADS < 256 * LP_EPI_REGS + 128 * LP_OTHER_REGS) return cudaErrorInvalidConfiguration;
  return cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeMaxDynamicSharedMemorySize,
                              lp_smem_bytes(sh.rag));
}

}  // namespace mmr
