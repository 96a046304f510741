// bf16 streams: the norm and dropout kernels of a block.
#define HC_T __nv_bfloat16
#define HC_SUFFIX bf16
#include "block_inst.cuh"
