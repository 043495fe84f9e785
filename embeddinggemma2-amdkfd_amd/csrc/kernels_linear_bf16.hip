// eg2_hip_linear and eg2_hip_linear_gated of bf16 activations (linear_device.hpp).
#include "linear_device.hpp"

namespace eg2 {
namespace block {

hipError_t launch_linear_bf16(const Linear& p, unsigned weight_type, bool gated, hipStream_t st) {
  return launch_linear_type<__bf16>(p, weight_type, gated, st);
}

}  // namespace block
}  // namespace eg2
