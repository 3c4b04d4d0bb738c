// The residual sum's kernels for a stream of fp32 and blocks of bf16.
#include "residual_norm.cuh"

namespace b200 {
namespace rnorm {
B200_RESIDUAL_NORM(float, __nv_bfloat16)
}  // namespace rnorm
}  // namespace b200
