// Element types, activations and lane reductions of the block operators
// (include/eg2_hip.h, "block operators").
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "eg2_device.hpp"
#include "eg2_hip.h"

namespace eg2 {
namespace block {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

// The GELU and SiLU as z / (1 + exp(-t)): no difference of two numbers near 1,
// so the result keeps its relative precision where it is small. exp2 and the
// reciprocal are the hardware's (1 ulp each); past their range the quotient is
// -0, as the limit is.
__device__ __forceinline__ float over_one_plus_exp(float z, float t) {
  return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * t));
}
__device__ __forceinline__ float activate(float z, unsigned act) {
  switch (act) {
    case EG2_ACT_GELU:
      return over_one_plus_exp(z, 2.0f * gelu_inner(z));
    case EG2_ACT_SILU:
      return over_one_plus_exp(z, z);
    case EG2_ACT_RELU:
      return z < 0.0f ? 0.0f : z;
    default:
      return z;
  }
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// Q8_0: 34-byte blocks of an fp16 scale and 32 int8 values, on 2 bytes.
constexpr int kBlockBytes = 34;
struct Q8 {};

template <class W>
__device__ __forceinline__ float weight_value(const void* w, size_t row, uint64_t ld, unsigned k) {
  if constexpr (__is_same(W, Q8)) {
    const unsigned char* b = static_cast<const unsigned char*>(w) + (row * (ld / 32) + k / 32) * kBlockBytes;
    return fp16_bits_to_fp32(*reinterpret_cast<const uint16_t*>(b)) * (float)(int8_t)b[2 + k % 32];
  } else {
    return to_float(static_cast<const W*>(w)[row * ld + k]);
  }
}

// Calls f with a value of the C++ type of an EG2_TYPE_ id of activations.
template <class F>
auto with_type(unsigned type, F f) {
  switch (type) {
    case EG2_TYPE_F32:
      return f(float{});
    case EG2_TYPE_F16:
      return f(_Float16{});
    default:
      return f(__bf16{});
  }
}

}  // namespace block
}  // namespace eg2
