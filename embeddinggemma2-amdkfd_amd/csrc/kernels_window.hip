// Attention over a sliding window and a few first keys
// (eg2_hip_window_attention).
//
// A row's visible keys are at most two ranges, [0, sinks') and [lo, hi), walked
// once with the running maximum and sum of the softmax.
#include <hip/hip_runtime.h>

#include "block_device.hpp"
#include "eg2_block.hpp"

namespace eg2 {
namespace block {
namespace {

struct Sequence {
  int64_t q0, k0;  // first rows
  int nq, nk;      // queries and keys
};
__device__ __forceinline__ Sequence sequence(const eg2_window_attention_args& p, unsigned b) {
  auto clip = [](int v, unsigned top) { return v < 0 ? 0 : ((unsigned)v < top ? v : (int)top); };
  const int q0 = clip(p.q_offsets[b], p.rows), q1 = clip(p.q_offsets[b + 1], p.rows);
  const int k0 = clip(p.k_offsets[b], p.key_rows), k1 = clip(p.k_offsets[b + 1], p.key_rows);
  int nk = k1 > k0 ? k1 - k0 : 0;
  if (p.k_lengths) nk = clip(p.k_lengths[b], (unsigned)nk);
  return Sequence{q0, k0, q1 > q0 ? q1 - q0 : 0, nk};
}

// The keys [lo, hi) of query i, and of the first keys those below `first`
// (first <= lo).
struct Range {
  int first, lo, hi;
};
__device__ __forceinline__ Range visible(const eg2_window_attention_args& p, const Sequence& s, int i) {
  const int64_t pos = (int64_t)s.nk - s.nq + i;
  int64_t hi = s.nk, lo = 0;
  if (p.right >= 0 && pos + p.right + 1 < hi) hi = pos + p.right + 1 > 0 ? pos + p.right + 1 : 0;
  if (p.left >= 0 && pos - p.left > 0) lo = pos - p.left < hi ? pos - p.left : hi;
  return Range{(int64_t)p.sinks < lo ? (int)p.sinks : (int)lo, (int)lo, (int)hi};
}

// One wave per (row, head): 64 keys at a time, one per lane for the scores,
// then every lane owns dimensions of the output.
constexpr int kMostD = 256;
template <class T>
__global__ void __launch_bounds__(64) window_attention_kernel(eg2_window_attention_args p) {
  __shared__ float qs[kMostD], ps[64];
  const unsigned lane = threadIdx.x, h = blockIdx.x % p.heads, g = h / (p.heads / p.kv_heads);
  const unsigned row = blockIdx.x / p.heads;
  // The last sequence whose first row is at most `row`.
  unsigned lo_b = 0, hi_b = p.batch;
  while (hi_b - lo_b > 1) {
    const unsigned mid = (lo_b + hi_b) / 2;
    (p.q_offsets[mid] <= (int)row ? lo_b : hi_b) = mid;
  }
  const Sequence s = sequence(p, lo_b);
  if ((int64_t)row < s.q0 || (int64_t)row >= s.q0 + s.nq) return;
  const Range rg = visible(p, s, (int)(row - s.q0));
  const T* q = static_cast<const T*>(p.q) + row * p.q_row + h * p.q_head;
  for (unsigned e = lane; e < p.d; e += 64) qs[e] = to_float(q[e]);
  __syncthreads();
  const T* kb = static_cast<const T*>(p.k) + s.k0 * p.k_row + g * p.k_head;
  const T* vb = static_cast<const T*>(p.v) + s.k0 * p.v_row + g * p.v_head;
  float top = -__builtin_inff(), den = 0.0f, acc[4] = {};
  const int total = rg.first + (rg.hi - rg.lo);
  for (int c0 = 0; c0 < total; c0 += 64) {
    const int at = c0 + (int)lane, key = at < rg.first ? at : rg.lo + at - rg.first;
    float score = -__builtin_inff();
    if (at < total) {
      const T* k = kb + key * p.k_row;
      float sum = 0.0f;
      for (unsigned e = 0; e < p.d; ++e) sum = __builtin_fmaf(qs[e], to_float(k[e]), sum);
      score = sum * p.scale;
    }
    float next = score;
    for (int m = 32; m > 0; m >>= 1) next = fmaxf(next, __shfl_xor(next, m, 64));
    next = fmaxf(next, top);
    const float alpha = top == -__builtin_inff() ? 0.0f : libm::expf(top - next);
    const float w = score == -__builtin_inff() ? 0.0f : libm::expf(score - next);
    float sum = w;
    for (int m = 32; m > 0; m >>= 1) sum = sum + __shfl_xor(sum, m, 64);
    den = den * alpha + sum;
    top = next;
    ps[lane] = w;
    __syncthreads();
    for (int j = 0; j < 4; ++j) acc[j] = acc[j] * alpha;
    for (int i = 0; i < 64 && c0 + i < total; ++i) {
      const int ka = c0 + i, kk = ka < rg.first ? ka : rg.lo + ka - rg.first;
      for (int j = 0; j < 4; ++j)
        if (lane + 64u * j < p.d) acc[j] = __builtin_fmaf(ps[i], to_float(vb[kk * p.v_row + lane + 64 * j]), acc[j]);
    }
    __syncthreads();
  }
  T* out = static_cast<T*>(p.out) + row * p.out_row + h * p.out_head;
  for (int j = 0; j < 4; ++j)
    if (lane + 64u * j < p.d) out[lane + 64 * j] = (T)(total > 0 ? acc[j] / den : 0.0f);
}

}  // namespace

uint64_t window_attention_workspace(const eg2_window_attention_args&) { return 0; }

hipError_t launch_window_attention(const eg2_window_attention_args& a, hipStream_t st) {
  return with_type(a.type, [&](auto t) {
    window_attention_kernel<decltype(t)><<<a.rows * a.heads, 64, 0, st>>>(a);
    return hipGetLastError();
  });
}

}  // namespace block
}  // namespace eg2
