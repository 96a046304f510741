// f32 streams: the norm and dropout kernels of a block.
#define HC_T float
#define HC_SUFFIX f32
#include "block_inst.cuh"
