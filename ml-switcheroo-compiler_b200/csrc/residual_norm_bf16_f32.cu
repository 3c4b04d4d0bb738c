// The residual sum's kernels for a stream of bf16 and blocks of fp32.
#include "residual_norm.cuh"

namespace b200 {
namespace rnorm {
B200_RESIDUAL_NORM(__nv_bfloat16, float)
}  // namespace rnorm
}  // namespace b200
