// linear_launch.h -- host-side entry points of the 16-bit products, each
// instantiated in a unit of its own so that they compile in parallel.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "linear_pair.cuh"
#include "linear_strip.cuh"

namespace mmr {

// w_mn: the weights are contiguous along n (row-major k x n).
cudaError_t strip_launch(bool bf16, bool w_mn, int grid, int smem, cudaStream_t s, const CUtensorMap& tm_w,
                         const CUtensorMap& tm_x, const StripParams& p);
cudaError_t strip_prepare(bool bf16, bool w_mn);

// a_mn / b_mn: the operand is contiguous along m / n. RAG 1 takes a K-major A,
// RAG 2 both operands MN-major (cudaErrorInvalidValue otherwise).
struct PairShape {
  int rag = 0, grid = 2;
  bool bf16 = true, a_mn = false, b_mn = false;
};
cudaError_t pair_launch_bf16(const PairShape& sh, cudaStream_t s, const CUtensorMap& tm_a, const CUtensorMap& tm_b,
                             const PairParams& p);
cudaError_t pair_launch_f16(const PairShape& sh, cudaStream_t s, const CUtensorMap& tm_a, const CUtensorMap& tm_b,
                            const PairParams& p);
cudaError_t pair_prepare_bf16(const PairShape& sh);
cudaError_t pair_prepare_f16(const PairShape& sh);

inline cudaError_t pair_launch(const PairShape& sh, cudaStream_t s, const CUtensorMap& tm_a, const CUtensorMap& tm_b,
                               const PairParams& p) {
  return sh.bf16 ? pair_launch_bf16(sh, s, tm_a, tm_b, p) : pair_launch_f16(sh, s, tm_a, tm_b, p);
}
inline cudaError_t pair_prepare(const PairShape& sh) { return sh.bf16 ? pair_prepare_bf16(sh) : pair_prepare_f16(sh); }

}  // namespace mmr
