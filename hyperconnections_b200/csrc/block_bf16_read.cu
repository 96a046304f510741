// bf16 streams: the read + pre-norm kernels, and dropout.
#include "block_norm.cuh"
#include "dropout.cuh"

namespace hc {

int read_norm_launch_bf16(bool bwd, NormGeometry& g, const NormArgs& a, cudaStream_t s) {
  return norm_launch<__nv_bfloat16, false>(bwd, g, a, s);
}

int dropout_launch_bf16(const void* x, void* y, int64_t N, const DropArgs& d, cudaStream_t s) {
  return dropout_launch<__nv_bfloat16>(x, y, N, d, s);
}

}  // namespace hc
