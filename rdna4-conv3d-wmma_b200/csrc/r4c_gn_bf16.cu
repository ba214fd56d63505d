// r4c_gn_bf16.cu — group normalisation kernels for bf16 activations.
#include "r4c_gn_launch.cuh"

namespace r4c {
namespace gn {
R4C_GN_INSTANCE(__nv_bfloat16)
}  // namespace gn
}  // namespace r4c
