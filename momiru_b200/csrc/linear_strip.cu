// linear_strip.cu -- the few-row products of both 16-bit types.
#include "launch.cuh"
#include "linear_launch.h"

namespace mmr {

using StripKernel = void (*)(const CUtensorMap, const CUtensorMap, const StripParams);

static StripKernel strip_kernel(bool bf16, bool w_mn) {
  if (bf16) return w_mn ? mmr_linear_strip_kernel<__nv_bfloat16, true> : mmr_linear_strip_kernel<__nv_bfloat16, false>;
  return w_mn ? mmr_linear_strip_kernel<__half, true> : mmr_linear_strip_kernel<__half, false>;
}

cudaError_t strip_launch(bool bf16, bool w_mn, int grid, int smem, cudaStream_t s, const CUtensorMap& tm_w,
                         const CUtensorMap& tm_x, const StripParams& p) {
  return launch_kernel(strip_kernel(bf16, w_mn), dim3(grid), dim3(LS_THREADS), smem, s, dim3(p.split, 1, 1), tm_w, tm_x,
                       p);
}

// The limit belongs to the function, which handles of many sizes share: always
// all that a block may have.
cudaError_t strip_prepare(bool bf16, bool w_mn) {
  return cudaFuncSetAttribute(reinterpret_cast<const void*>(strip_kernel(bf16, w_mn)),
                              cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
}

}  // namespace mmr
