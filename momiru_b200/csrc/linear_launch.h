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
cudaError_t strip_prepare(bool bf16, bool w_mn, int smem);

// a_mn / b_mn: the operand is contiguous along m / n. RAG 1 takes a K-major A,
// RAG 2 both operands MN-major (cudaErrorInvalidValue otherwise).
cudaError_t pair_launch_bf16(bool a_mn, bool b_mn, int rag, int grid, cudaStream_t s, const CUtensorMap& tm_a,
                             const CUtensorMap& tm_b, const PairParams& p);
cudaError_t pair_launch_f16(bool a_mn, bool b_mn, int rag, int grid, cudaStream_t s, const CUtensorMap& tm_a,
                            const CUtensorMap& tm_b, const PairParams& p);
cudaError_t pair_prepare_bf16(bool a_mn, bool b_mn, int rag);
cudaError_t pair_prepare_f16(bool a_mn, bool b_mn, int rag);

}  // namespace mmr
