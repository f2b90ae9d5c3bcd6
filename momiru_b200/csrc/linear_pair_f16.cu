// linear_pair_f16.cu -- the CTA-pair products of f16 operands.
#include "linear_pair_launch.cuh"

namespace mmr {

cudaError_t pair_launch_f16(const PairShape& sh, cudaStream_t s, const CUtensorMap& tm_a, const CUtensorMap& tm_b,
                             const PairParams& p) {
  return pair_launch_t<__half>(sh, s, tm_a, tm_b, p);
}
cudaError_t pair_prepare_f16(const PairShape& sh) { return pair_prepare_t<__half>(sh); }

}  // namespace mmr
