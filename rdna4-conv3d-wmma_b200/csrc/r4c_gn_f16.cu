// r4c_gn_f16.cu — group normalisation kernels for f16 activations.
#include "r4c_gn_launch.cuh"

namespace r4c {
namespace gn {
R4C_GN_INSTANCE(__half)
}  // namespace gn
}  // namespace r4c
