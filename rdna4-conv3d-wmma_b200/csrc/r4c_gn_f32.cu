// r4c_gn_f32.cu — group normalisation kernels for f32 activations.
#include "r4c_gn_launch.cuh"

namespace r4c {
namespace gn {
R4C_GN_INSTANCE(float)
}  // namespace gn
}  // namespace r4c
