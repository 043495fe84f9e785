// eg2_hip_linear and eg2_hip_linear_gated of f32 activations (linear_device.hpp).
#include "linear_device.hpp"

namespace eg2 {
namespace block {

hipError_t launch_linear_f32(const Linear& p, unsigned weight_type, bool gated, hipStream_t st) {
  return launch_linear_type<float>(p, weight_type, gated, st);
}

}  // namespace block
}  // namespace eg2
