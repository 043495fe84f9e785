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
template <unsigned ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == EG2_ACT_GELU) return over_one_plus_exp(z, 2.0f * gelu_inner(z));
  if constexpr (ACT == EG2_ACT_SILU) return over_one_plus_exp(z, z);
  if constexpr (ACT == EG2_ACT_RELU) return z < 0.0f ? 0.0f : z;
  return z;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// Q8_0: 34-byte blocks of an fp16 scale and 32 int8 values, on 2 bytes.
constexpr int kBlockBytes = 34;
struct Q8 {};

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfloatx8 __attribute__((ext_vector_type(8)));

// Values in 16 bytes.
template <class T>
constexpr int kPer16 = 16 / (int)sizeof(T);

// c += a . b over 16 bytes of each lane: 32 values deep (16-bit types), 16 (fp32).
template <class T>
__device__ __forceinline__ floatx4 mfma16(uintx4 a, uintx4 b, floatx4 c) {
  if constexpr (__is_same(T, float)) {
    const floatx4 fa = __builtin_bit_cast(floatx4, a), fb = __builtin_bit_cast(floatx4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[e], fb[e], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0,
                                                  0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloatx8, a), __builtin_bit_cast(bfloatx8, b), c,
                                                   0, 0, 0);
  }
}

template <int N>
struct Const {
  static constexpr int value = N;
};

// Calls f with the Const of an activation id: one branch around a whole epilogue.
template <class F>
__device__ __forceinline__ void with_activation(unsigned act, F f) {
  switch (act) {
    case EG2_ACT_GELU:
      return f(Const<EG2_ACT_GELU>{});
    case EG2_ACT_SILU:
      return f(Const<EG2_ACT_SILU>{});
    case EG2_ACT_RELU:
      return f(Const<EG2_ACT_RELU>{});
    default:
      return f(Const<EG2_ACT_NONE>{});
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
