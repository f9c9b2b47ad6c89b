// Layer norm, forward pass (layer_norm.cuh)
#include "layer_norm.cuh"

namespace attn {
namespace layer {

cudaError_t launch_norm_forward(const NormPlan& p, const NormArgs& a, int dtype, unsigned ctas, cudaStream_t stream) {
  return launch_typed<0>(p, a, dtype, ctas, stream);
}

}  // namespace layer
}  // namespace attn
