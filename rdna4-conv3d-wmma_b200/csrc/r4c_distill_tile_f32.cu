// r4c_distill_tile_f32.cu — distillation of short rows, f32 logits.
#include "r4c_distill_tile.cuh"

template cudaError_t r4c::distill::launch_tiles<float>(r4c::distill::Args&, bool, int*, cudaStream_t);
