// r4c_distill_tile_bf16.cu — distillation of short rows, bf16 logits.
#include "r4c_distill_tile.cuh"

template cudaError_t r4c::distill::launch_tiles<__nv_bfloat16>(r4c::distill::Args&, bool, int*, cudaStream_t);
