// f16 streams: the post-norm + mix-write kernels.
#include "block_norm.cuh"

namespace hc {

int write_norm_launch_f16(bool bwd, NormGeometry& g, const NormArgs& a, cudaStream_t s) {
  return norm_launch<__half, true>(bwd, g, a, s);
}

}  // namespace hc
