// Launchers of the block operators (include/eg2_hip.h). The records have been
// checked (block_ops.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include "eg2_hip.h"

namespace eg2 {
namespace block {

hipError_t launch_linear(const eg2_linear_args& a, hipStream_t st);
hipError_t launch_linear_gated(const eg2_linear_gated_args& a, hipStream_t st);
hipError_t launch_heads_norm_rope(const eg2_heads_norm_rope_args& a, hipStream_t st);
uint64_t window_attention_workspace(const eg2_window_attention_args& a);
hipError_t launch_window_attention(const eg2_window_attention_args& a, hipStream_t st);

}  // namespace block
}  // namespace eg2
