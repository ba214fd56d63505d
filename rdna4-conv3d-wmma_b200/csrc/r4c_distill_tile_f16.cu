// r4c_distill_tile_f16.cu — distillation of short rows, f16 logits.
#include "r4c_distill_tile.cuh"

template cudaError_t r4c::distill::launch_tiles<__half>(r4c::distill::Args&, bool, int*, cudaStream_t);
