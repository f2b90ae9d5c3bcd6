// linear_pair_bf16.cu -- the CTA-pair products of bf16 operands.
#include "linear_pair_launch.cuh"

namespace mmr {

cudaError_t pair_launch_bf16(const PairShape& sh, cudaStream_t s, const CUtensorMap& tm_a, const CUtensorMap& tm_b,
                             const PairParams& p) {
  return pair_launch_t<__nv_bfloat16>(sh, s, tm_a, tm_b, p);
}
cudaError_t pair_prepare_bf16(const PairShape& sh) { return pair_prepare_t<__nv_bfloat16>(sh); }

}  // namespace mmr
