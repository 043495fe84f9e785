// Launchers of the block operators (include/eg2_hip.h). The records have been
// checked (block_ops.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "eg2_hip.h"

namespace eg2 {
namespace block {

// One product's operands in the kernels: of a gated pair w[0] is the gate.
struct Linear {
  void* y;
  const void* x;
  const void* w[2];
  const float* bias[2];
  const void* residual;
  uint64_t ldx, ldw, ldy, ldr;
  unsigned n, k, m, act;
};

// By the type of the activations (kernels_linear_*.hip).
hipError_t launch_linear_f32(const Linear& p, unsigned weight_type, bool gated, hipStream_t st);
hipError_t launch_linear_f16(const Linear& p, unsigned weight_type, bool gated, hipStream_t st);
hipError_t launch_linear_bf16(const Linear& p, unsigned weight_type, bool gated, hipStream_t st);

hipError_t launch_heads_norm_rope(const eg2_heads_norm_rope_args& a, hipStream_t st);
uint64_t window_attention_workspace(const eg2_window_attention_args& a);
hipError_t launch_window_attention(const eg2_window_attention_args& a, hipStream_t st);

}  // namespace block
}  // namespace eg2
