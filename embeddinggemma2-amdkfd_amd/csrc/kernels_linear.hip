// Products with an epilogue, and the gated pair of products
// (eg2_hip_linear, eg2_hip_linear_gated).
//
//   y = act(x W^T + b) + r            y = act(x Wg^T + bg) * (x Wu^T + bu)
#include <hip/hip_runtime.h>

#include "block_device.hpp"
#include "eg2_block.hpp"

namespace eg2 {
namespace block {
namespace {

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

// What becomes of an output's sums.
template <class X, bool GATED>
__device__ __forceinline__ void finish(const Linear& p, unsigned row, unsigned col, float a, float b) {
  float z = p.bias[0] ? a + p.bias[0][col] : a;
  z = activate(z, p.act);
  if constexpr (GATED) z = z * (p.bias[1] ? b + p.bias[1][col] : b);
  if (!GATED && p.residual) z = z + to_float(static_cast<const X*>(p.residual)[row * p.ldr + col]);
  static_cast<X*>(p.y)[row * p.ldy + col] = (X)z;
}

// Any sizes, strides and alignment: 64 x 64 outputs per workgroup of four
// waves, fp32 MFMA on 32-deep slices of both operands in LDS as fp32, zeros
// past the edges. The MFMA's k index is a permutation of the slice: lane group
// g feeds the elements 8 g .. 8 g + 7, one per MFMA.
constexpr int kTile = 64, kSlice = 32, kPitch = kSlice + 4;
template <class X, class W, bool GATED>
__global__ void __launch_bounds__(256) linear_kernel(Linear p) {
  constexpr int G = GATED ? 2 : 1;
  __shared__ float xs[kTile * kPitch], ws[G][kTile * kPitch];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, r = lane & 15;
  const unsigned across = (p.m + kTile - 1) / kTile;
  const unsigned row0 = blockIdx.x / across * kTile, col0 = blockIdx.x % across * kTile;
  const int rbase = 32 * (wave >> 1), cbase = 32 * (wave & 1);
  floatx4 acc[G][2][2] = {};
  for (unsigned k0 = 0; k0 < p.k; k0 += kSlice) {
    for (int i = tid; i < kTile * kSlice; i += 256) {
      const int rr = i / kSlice, kk = i % kSlice;
      const unsigned k = k0 + kk;
      xs[rr * kPitch + kk] = row0 + rr < p.n && k < p.k ? to_float(static_cast<const X*>(p.x)[(row0 + rr) * p.ldx + k]) : 0.0f;
#pragma unroll
      for (int z = 0; z < G; ++z)
        ws[z][rr * kPitch + kk] = col0 + rr < p.m && k < p.k ? weight_value<W>(p.w[z], col0 + rr, p.ldw, k) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) a[i] = xs[(rbase + 16 * i + r) * kPitch + 8 * g + e];
#pragma unroll
      for (int z = 0; z < G; ++z)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float b = ws[z][(cbase + 16 * j + r) * kPitch + 8 * g + e];
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[z][i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b, acc[z][i][j], 0, 0, 0);
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const unsigned row = row0 + rbase + 16 * i + 4 * g + v, col = col0 + cbase + 16 * j + r;
        if (row < p.n && col < p.m) finish<X, GATED>(p, row, col, acc[0][i][j][v], acc[G - 1][i][j][v]);
      }
}

template <bool GATED>
hipError_t launch(const Linear& p, unsigned type, unsigned weight_type, hipStream_t st) {
  return with_type(type, [&](auto x) {
    using X = decltype(x);
    auto go = [&](auto w) {
      using W = decltype(w);
      const unsigned tiles = (p.m + kTile - 1) / kTile * ((p.n + kTile - 1) / kTile);  // n m <= 2^32: at most 2^20 + 2^19
      linear_kernel<X, W, GATED><<<tiles, 256, 0, st>>>(p);
      return hipGetLastError();
    };
    if (weight_type == EG2_TYPE_Q8_0) return go(Q8{});
    if constexpr (__is_same(X, float)) {
      if (weight_type == EG2_TYPE_F16) return go(_Float16{});
      if (weight_type == EG2_TYPE_BF16) return go(__bf16{});
    }
    return go(X{});
  });
}

}  // namespace

hipError_t launch_linear(const eg2_linear_args& a, hipStream_t st) {
  return launch<false>(Linear{a.y, a.x, {a.weight, nullptr}, {a.bias, nullptr}, a.residual, a.ldx, a.ldw, a.ldy, a.ldr,
                              a.n, a.k, a.m, a.act},
                       a.type, a.weight_type, st);
}
hipError_t launch_linear_gated(const eg2_linear_gated_args& a, hipStream_t st) {
  return launch<true>(Linear{a.y, a.x, {a.gate, a.up}, {a.gate_bias, a.up_bias}, nullptr, a.ldx, a.ldw, a.ldy, 0, a.n,
                             a.k, a.m, a.act},
                      a.type, a.weight_type, st);
}

}  // namespace block
}  // namespace eg2
