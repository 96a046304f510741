// block_inst.cuh — instantiates the norm and dropout kernels for one stream
// dtype. Included by block_<dtype>.cu with HC_T (the element type) and
// HC_SUFFIX (the entry-point suffix) defined.
#include "block_elem.cuh"
#include "dropout.cuh"

#define HC_CAT2(a, b) a##b
#define HC_CAT(a, b) HC_CAT2(a, b)

namespace hc {

int HC_CAT(norm_launch_, HC_SUFFIX)(bool write, bool bwd, const NormGeometry& g, const NormArgs& a, cudaStream_t s) {
  return norm_launch_elem<HC_T>(write, bwd, g, a, s);
}

int HC_CAT(dropout_launch_, HC_SUFFIX)(const void* x, void* y, int64_t N, const DropArgs& d, cudaStream_t s) {
  return dropout_launch<HC_T>(x, y, N, d, s);
}

}  // namespace hc
