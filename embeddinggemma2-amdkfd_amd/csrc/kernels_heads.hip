// The norms of queries and keys for each head with the position rotation, in
// one pass (eg2_hip_heads_norm_rope).
//
//   u = x / sqrt(mean(x^2) + eps) * w
//   (u_i, u_i+R/2) -> (u_i c - u_i+R/2 s, u_i s + u_i+R/2 c),  i < R/2
//
// Every value is read once and written once; the kernel is bound by those
// bytes. A group of L lanes takes H heads of a row, whose loads are all on their
// way at once and share the row's angles. A lane holds both halves of its pairs (V
// values of each, a 16-byte load where V allows), so that the rotation needs no
// other lane and the sum of squares one reduction over the group; the values
// past `rotary` are pairs as well, turned by no angle.
#include <hip/hip_runtime.h>

#include "block_device.hpp"
#include "eg2_block.hpp"

namespace eg2 {
namespace block {
namespace {

template <class T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Values {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ Values<T, V> load(const T* p) {
  return *reinterpret_cast<const Values<T, V>*>(p);
}

// C: pieces of V pairs per lane.
template <class T, int V, int L, int C, int H>
__global__ void __launch_bounds__(256) heads_norm_rope_kernel(eg2_heads_norm_rope_args p) {
  const unsigned heads = p.q_heads + p.k_heads, runs = (heads + H - 1) / H;
  const unsigned at = blockIdx.x * (256 / L) + threadIdx.x / L, lane = threadIdx.x % L;
  const unsigned row = at / runs, head0 = at % runs * H;
  if (row >= p.rows) return;  // whole groups
  const unsigned turned = p.rotary / 2, pairs = p.d / 2;  // pairs in all, the first `turned` of them rotated
  // Pair i < turned: values i and i + turned; others: i + turned and i + pairs.
  auto first = [&](unsigned i) { return i < turned ? i : i + turned; };
  auto second = [&](unsigned i) { return i < turned ? i + turned : i + pairs; };
  Values<T, V> a[H][C], b[H][C];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const unsigned head = min(head0 + h, heads - 1);
    const bool is_q = head < p.q_heads;
    const T* x = is_q ? static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head
                      : static_cast<const T*>(p.k) + row * p.k_row + (head - p.q_heads) * p.k_head;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const unsigned i = V * (lane + L * c);
      if (i >= pairs) continue;
      a[h][c] = load<T, V>(x + first(i));
      b[h][c] = load<T, V>(x + second(i));
    }
  }
  int pos = 0;
  if (p.rotary) pos = p.pos[row];
  const bool known = !p.rotary || (pos >= 0 && (unsigned)pos < p.table_rows);
  const float* table = p.table + (size_t)(known ? pos : 0) * p.rotary;
  Values<float, V> co[C], si[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const unsigned i = V * (lane + L * c);
    if (i >= turned) continue;
    co[c] = load<float, V>(table + i);
    si[c] = load<float, V>(table + turned + i);
  }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const unsigned head = head0 + h;
    if (head >= heads) break;
    const bool is_q = head < p.q_heads;
    const float* w = is_q ? p.q_weight : p.k_weight;
    T* out = is_q ? static_cast<T*>(p.q_out) + row * p.q_out_row + head * p.q_out_head
                  : static_cast<T*>(p.k_out) + row * p.k_out_row + (head - p.q_heads) * p.k_out_head;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (V * (lane + L * c) >= pairs) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float f = to_float(a[h][c].v[e]), g = to_float(b[h][c].v[e]);
        ss = __builtin_fmaf(f, f, ss);
        ss = __builtin_fmaf(g, g, ss);
      }
    }
#pragma unroll
    for (int m = 1; m < L; m <<= 1) ss = ss + __shfl_xor(ss, m, 64);
    float inv = rms_inverse(ss, (int)p.d, p.eps);
    if (!known) inv = __builtin_nanf("");
    const float scale = is_q ? p.q_scale : 1.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const unsigned i = V * (lane + L * c);
      if (i >= pairs) continue;
      Values<float, V> wa, wb;
      if (w) {
        wa = load<float, V>(w + first(i));
        wb = load<float, V>(w + second(i));
      }
      Values<T, V> ra, rb;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float f = to_float(a[h][c].v[e]) * inv, g = to_float(b[h][c].v[e]) * inv;
        if (w) f = f * wa.v[e], g = g * wb.v[e];
        if (i < turned) {
          const float fc = f * co[c].v[e], gs = g * si[c].v[e], fs = f * si[c].v[e], gc = g * co[c].v[e];
          f = fc - gs;
          g = fs + gc;
        }
        ra.v[e] = (T)(f * scale);
        rb.v[e] = (T)(g * scale);
      }
      *reinterpret_cast<Values<T, V>*>(out + first(i)) = ra;
      *reinterpret_cast<Values<T, V>*>(out + second(i)) = rb;
    }
  }
}

template <class T, int V, int L, int C, int H>
hipError_t go(const eg2_heads_norm_rope_args& a, hipStream_t st) {
  const unsigned runs = (a.q_heads + a.k_heads + H - 1) / H, groups = a.rows * runs;  // at most 2^25
  heads_norm_rope_kernel<T, V, L, C, H><<<(groups + 256 / L - 1) / (256 / L), 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_heads_norm_rope(const eg2_heads_norm_rope_args& a, hipStream_t st) {
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    // Whole 16-byte loads of both halves, or single values.
    auto on16 = [](const void* p, uint64_t r, uint64_t h) {
      return reinterpret_cast<uintptr_t>(p) % 16 == 0 && r % V == 0 && h % V == 0;
    };
    const bool wide = a.rotary / 2 % V == 0 && (a.d - a.rotary) / 2 % V == 0 && on16(a.q, a.q_row, a.q_head) &&
                      on16(a.q_out, a.q_out_row, a.q_out_head) &&
                      (a.k_heads == 0 || (on16(a.k, a.k_row, a.k_head) && on16(a.k_out, a.k_out_row, a.k_out_head))) &&
                      on16(a.q_weight, 0, 0) && on16(a.k_weight, 0, 0) && on16(a.table, 0, 0);
    if (!wide) return go<T, 1, 64, 4, 1>(a, st);
    const unsigned chunks = a.d / 2 / V;  // of each half, at most 64
    // Four heads to a group where that leaves a wave for every SIMD: 8192 rows of 16 + 4 x 128 bf16 20 us, 4.3 TB/s
    // (one head: 55 us); with fewer rows one (2011 of 3 + 1 x 256 fp32: 5.3 us).
    auto by = [&](auto lanes) {
      constexpr int L = decltype(lanes)::value;
      const uint64_t heads = (uint64_t)a.rows * (a.q_heads + a.k_heads);
      if (heads * L / 64 >= 4 * 1024) return go<T, V, L, 1, 4>(a, st);
      return go<T, V, L, 1, 1>(a, st);
    };
    if (chunks <= 4) return by(Const<4>{});
    if (chunks <= 8) return by(Const<8>{});
    if (chunks <= 16) return by(Const<16>{});
    if (chunks <= 32) return by(Const<32>{});
    if constexpr (V == 4) return by(Const<64>{});
    return hipErrorInvalidValue;  // d above 512
  });
}

}  // namespace block
}  // namespace eg2
