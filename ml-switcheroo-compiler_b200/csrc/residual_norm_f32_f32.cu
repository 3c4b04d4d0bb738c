// The residual sum's kernels for a stream of fp32 and blocks of fp32.
#include "residual_norm.cuh"

namespace b200 {
namespace rnorm {
B200_RESIDUAL_NORM(float, float)
}  // namespace rnorm
}  // namespace b200
