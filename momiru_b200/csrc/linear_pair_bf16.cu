// linear_pair_bf16.cu -- the CTA-pair products of bf16 operands.
#include "linear_pair_launch.cuh"

namespace mmr {

cudaError_t pair_launch_bf16(bool a_mn, bool b_mn, int rag, int grid, cudaStream_t s, const CUtensorMap& tm_a,
                             const CUtensorMap& tm_b, const PairParams& p) {
  return pair_launch_t<__nv_bfloat16>(a_mn, b_mn, rag, grid, s, tm_a, tm_b, p);
}
cudaError_t pair_prepare_bf16(bool a_mn, bool b_mn, int rag) { return pair_prepare_t<__nv_bfloat16>(a_mn, b_mn, rag); }

}  // namespace mmr
