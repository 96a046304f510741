// f16 streams: the norm and dropout kernels of a block.
#define HC_T __half
#define HC_SUFFIX f16
#include "block_inst.cuh"
