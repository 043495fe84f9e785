// Attention over a sliding window and a few first keys
// (eg2_hip_window_attention).
//
//   out = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q . k_s - max),  s visible
//
// in one pass over a row's keys with the running maximum and sum. The query
// heads of a KV head go together: a tile has rows (token, head of the group),
// 16 QB to a wave. A wave forms the transposed scores K Q^T of 16 keys x 16 rows at a
// time (mfma16, 32-bit sums), so that a lane holds one row's scores of keys
// 4 g .. 4 g + 3: the softmax is lane by lane, with two exchanges for the
// maximum, and the weights already lie as the second operand of V^T P^T, keys
// in that order. Keys and values come straight to LDS, a tile ahead; the 16-bit
// values are transposed on their way out of it (ds_read_b64_tr_b16).
//
// The softmax weights of 16-bit attention are rounded to the type, at most half
// a step each, as the matrix unit takes them; their sum is formed from the
// 32-bit ones. The running maximum moves only when a score exceeds it by 2^8
// (weights up to 2^8 lose nothing in any type), which spares most of the
// rescaling of the sums.
//
// A key that a row does not see has weight 0, but 0 times an infinite or NaN
// value is NaN: where some row of the wave does not see a tile's keys, the values
// are looked at first, and a tile with such a value goes key by key (add_by_key).
#include <hip/hip_runtime.h>

#include "block_device.hpp"
#include "eg2_block.hpp"

namespace eg2 {
namespace block {
namespace {

typedef eg2_window_attention_args Args;
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct Sequence {
  int q0, k0;  // first rows
  int nq, nk;  // queries and keys
};
__device__ __forceinline__ int clip(int v, unsigned top) { return v < 0 ? 0 : ((unsigned)v < top ? v : (int)top); }
__device__ __forceinline__ Sequence sequence(const Args& p, unsigned b) {
  const int q0 = clip(p.q_offsets[b], p.rows), q1 = clip(p.q_offsets[b + 1], p.rows);
  const int k0 = clip(p.k_offsets[b], p.key_rows), k1 = clip(p.k_offsets[b + 1], p.key_rows);
  int nk = k1 > k0 ? k1 - k0 : 0;
  if (p.k_lengths) nk = clip(p.k_lengths[b], (unsigned)nk);
  return Sequence{q0, k0, q1 > q0 ? q1 - q0 : 0, nk};
}

// Query i sees the keys below hi that are at least lo or below p.sinks. Both grow with i.
struct Range {
  int lo, hi;
};
__device__ __forceinline__ Range visible(const Args& p, const Sequence& s, int i) {
  const int64_t pos = (int64_t)s.nk - s.nq + i;
  int64_t hi = s.nk, lo = 0;
  if (p.right >= 0 && pos + p.right + 1 < hi) hi = pos + p.right + 1 > 0 ? pos + p.right + 1 : 0;
  if (p.left >= 0 && pos - p.left > 0) lo = pos - p.left;
  return Range{(int)lo, (int)hi};
}
__device__ __forceinline__ bool sees_any(const Args& p, const Range& r) { return r.hi > r.lo || (p.sinks > 0 && r.hi > 0); }

// The last b < n with first(b) <= at, first growing with b (0 if none): 64 at a time.
template <class F>
__device__ __forceinline__ unsigned last_at_most(unsigned n, unsigned at, F first) {
  unsigned lo = 0;
  while (n > 1) {
    const unsigned step = (n + 63) / 64, b = (threadIdx.x & 63) * step;
    const int count = __popcll(__ballot(b < n && first(lo + b) <= at));
    const unsigned skip = count > 1 ? (count - 1) * step : 0;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// 16 bytes a lane from its own address to LDS at `lds` + 16 bytes a lane (see dma16).
__device__ __forceinline__ void dma16_each(const void* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}

// Whether a 16-byte piece holds an infinity or NaN, as nonzero bits.
template <class T>
__device__ __forceinline__ uint32_t non_finite_bits(uintx4 v) {
  constexpr uint32_t exponent = __is_same(T, float) ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = __is_same(T, float) ? 0x00800000u : __is_same(T, _Float16) ? 0x04000400u : 0x00800080u;
  constexpr uint32_t top = __is_same(T, float) ? 0x80000000u : 0x80008000u;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= ((v[i] & exponent) + one) & top;
  return any;
}

// DP: head size padded to a multiple of 64. WM x WK waves: WM row groups, each
// with every key of its share, and WK shares of the keys, joined at the end. BN keys to a tile.
template <class T, int DP, int QB, int WM, int WK, int BN>
__global__ void __launch_bounds__(64 * WM * WK)
window_attention_kernel(Args p, unsigned slots, unsigned splits, float* part_out, float2* part_ml, float c) {
  constexpr bool k32 = __is_same(T, float);
  constexpr int RB = DP * (int)sizeof(T), CH = RB / 16, KK = RB / 64;  // bytes, 16-byte chunks, MFMA steps of a row
  constexpr int KB = BN / 16, OB = DP / 16, BM = 16 * QB * WM, N = kPer16<T>;
  constexpr int kLoads = BN * RB / 1024 / WM;  // per wave, of keys and of values
  static_assert(BN * RB % (1024 * WM) == 0 && (k32 || BN % 32 == 0) && (WM == 1 || WK == 1), "tile shape");
  constexpr int kTile = BN * RB;
  constexpr int kPart = WK > 1 ? WK * BM * DP * 4 : 0;
  constexpr int kLds = WK * 2 * 2 * kTile > kPart ? WK * 2 * 2 * kTile : kPart;
  __shared__ alignas(16) unsigned char lds[kLds];
  __shared__ float2 lds_ml[WK > 1 ? WK * BM : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15, wm = wave % WM, wk = wave / WM;
  const unsigned group = p.heads / p.kv_heads, kvh = blockIdx.x % p.kv_heads;
  const unsigned split = blockIdx.x / p.kv_heads % splits;
  const unsigned slot = slots - 1 - blockIdx.x / p.kv_heads / splits;  // the longest rows of a causal prompt first

  // Sequence b's tiles start at slot q_offsets[b] group / BM + b: at least as
  // many slots as it has tiles, found without a sum over the sequences.
  auto first_slot = [&](unsigned b) {
    return (unsigned)((uint64_t)clip(p.q_offsets[b], p.rows) * group / BM) + b;
  };
  const unsigned b = __builtin_amdgcn_readfirstlane(last_at_most(p.batch, slot, first_slot));
  const Sequence s = sequence(p, b);
  const int64_t pairs = (int64_t)s.nq * group, pair0 = (int64_t)(slot - first_slot(b)) * BM;
  if (slot < first_slot(b) || pair0 >= pairs) return;  // the whole workgroup

  // The keys that the tile's rows see: [0, first) and [start, stop), in tiles of BN.
  auto token = [&](int64_t pair) { return (int)(pair / group); };
  const Range top = visible(p, s, token(pair0)), bottom = visible(p, s, token(min(pair0 + BM, pairs) - 1));
  const int stop = bottom.hi;
  int start = min(top.lo, stop), first = (int)min((unsigned)start, p.sinks);
  if (start < BN) start = first = 0;
  const int tiles_a = (first + BN - 1) / BN, tiles_b = (stop - start + BN - 1) / BN, tiles = tiles_a + tiles_b;
  const int t0 = (int)((int64_t)tiles * split / splits), t1 = (int)((int64_t)tiles * (split + 1) / splits);
  auto tile_start = [&](int t) { return t < tiles_a ? t * BN : start + (t - tiles_a) * BN; };
  auto tile_end = [&](int t) { return t < tiles_a ? min(first, t * BN + BN) : min(stop, start + (t - tiles_a) * BN + BN); };

  // The wave's rows and the lane's: row 16 qb + r.
  const int64_t wave_pair = pair0 + 16 * QB * wm;
  const bool active = wave_pair < pairs;
  const Range wave_top = visible(p, s, token(min(wave_pair, pairs - 1)));
  const Range wave_bottom = visible(p, s, token(min(wave_pair + 16 * QB, pairs) - 1));
  Range range[QB];
  uintx4 q[QB][KK];
  const uint32_t flip = p.scale < 0.0f ? (k32 ? 0x80000000u : 0x80008000u) : 0u;  // the scale's sign
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int64_t pair = min(wave_pair + 16 * i + r, pairs - 1);
    const int t = token(pair);
    range[i] = visible(p, s, t);
    const T* row = static_cast<const T*>(p.q) + (size_t)(s.q0 + t) * p.q_row + (kvh * group + pair % group) * p.q_head;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const unsigned at = N * (4 * kk + g);
      q[i][kk] = at < p.d ? *reinterpret_cast<const uintx4*>(row + at) : uintx4{};
#pragma unroll
      for (int e = 0; e < 4; ++e) q[i][kk][e] ^= flip;
    }
  }

  unsigned char* const mine = lds + wk * 4 * kTile;  // the share's two buffers of keys and values
  const T* kbase = static_cast<const T*>(p.k) + (size_t)s.k0 * p.k_row + kvh * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + (size_t)s.k0 * p.v_row + kvh * p.v_head;
  // Chunks of a row are swizzled: the keys for 16 rows of one chunk column, the
  // values (16-bit) for 16 rows of two.
  auto key_swizzle = [](int row) { return row & 7; };
  auto value_swizzle = [](int row) { return 2 * (row & ((CH / 2 < 8 ? CH / 2 : 8) - 1)); };
  if (p.d < DP) {  // the padding of the head size stays zero
    for (int i = tid; i < WK * 4 * kTile / 16; i += 64 * WM * WK) reinterpret_cast<uintx4*>(lds)[i] = uintx4{};
    __syncthreads();
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)mine;
  auto stage = [&](int buf, int t) {
    const int from = tile_start(t), last = tile_end(t) - 1;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = kLoads * wm + i, at = 64 * piece + lane, row = at / CH, to = at % CH;
      const size_t key = min(from + row, last);
      const uint32_t lds_k = __builtin_amdgcn_readfirstlane(lds0 + buf * 2 * kTile + 1024 * piece);
      const int ck = to ^ key_swizzle(row), cv = to ^ value_swizzle(row);
      if (N * ck < (int)p.d) dma16_each(kbase + key * p.k_row + N * ck, lds_k);
      if (N * cv < (int)p.d) dma16_each(vbase + key * p.v_row + N * cv, lds_k + kTile);
    }
  };

  floatx4 acc[QB][OB];
  float m[QB], l[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    m[i] = -__builtin_inff();
    l[i] = 0.0f;
#pragma unroll
    for (int o = 0; o < OB; ++o) acc[i][o] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  auto compute = [&](const unsigned char* ks, int from, int end) {
    const unsigned char* vs = ks + kTile;
    floatx4 sc[QB][KB];
#pragma unroll
    for (int i = 0; i < QB; ++i)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) sc[i][kb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int row = 16 * kb + r;
        const uintx4 a = *reinterpret_cast<const uintx4*>(ks + row * RB + 16 * ((4 * kk + g) ^ key_swizzle(row)));
#pragma unroll
        for (int i = 0; i < QB; ++i) sc[i][kb] = mfma16<T>(a, q[i][kk], sc[i][kb]);
      }
    // Whether every row of the wave sees every key of the tile (uniform).
    const bool full = from + BN <= min(wave_top.hi, end) && (from >= wave_bottom.lo || from + BN <= (int)min(p.sinks, 0x7fffffffu));
    auto seen = [&](int i, int key) {
      return key < min(range[i].hi, end) && (key >= range[i].lo || (unsigned)key < p.sinks);
    };
    if (!full) {
#pragma unroll
      for (int i = 0; i < QB; ++i)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) sc[i][kb][v] = seen(i, from + 16 * kb + 4 * g + v) ? sc[i][kb][v] : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      float most = sc[i][0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) most = fmaxf(most, sc[i][kb][v]);
      most = rows4_max(most) * c;
      const bool grown = most > m[i] + 8.0f;
      if (__any(grown)) {
        const float next = grown ? most : m[i];
        const float alpha = grown ? __builtin_amdgcn_exp2f(m[i] - next) : 1.0f;
        m[i] = next;
        l[i] = l[i] * alpha;
#pragma unroll
        for (int o = 0; o < OB; ++o)
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[i][o][v] = acc[i][o][v] * alpha;
      }
      const float base = m[i] == -__builtin_inff() ? 0.0f : m[i];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          sc[i][kb][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][kb][v], c, -base));
          l[i] = l[i] + sc[i][kb][v];
        }
    }
    // 16-bit: chunk of values for the dimensions 16 o + lane % 16 of keys 32 kp + 4 g .. and 16 more.
    auto value16 = [&](int kp, int o) {
      union {
        uintx4 all;
        shortx4 half[2];
      } a;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int row = 32 * kp + 16 * z + 4 * g + (r >> 2);
        const unsigned char* at = vs + row * RB + 16 * ((2 * o + ((r & 3) >> 1)) ^ value_swizzle(row)) + 8 * (r & 1);
        a.half[z] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)at);
      }
      return a.all;
    };
    // fp32: dimensions 64 o + 4 (lane % 16) .. of key 16 kb + 4 g + j.
    auto value32 = [&](int kb, int j, int o) {
      const int row = 16 * kb + 4 * g + j;
      return *reinterpret_cast<const uintx4*>(vs + row * RB + 16 * ((16 * o + r) ^ value_swizzle(row)));
    };
    if (!full) {
      uint32_t odd = 0;
      if constexpr (k32) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int o = 0; o < OB / 4; ++o) odd |= non_finite_bits<T>(value32(kb, j, o));
      } else {
#pragma unroll
        for (int kp = 0; kp < KB / 2; ++kp)
#pragma unroll
          for (int o = 0; o < OB; ++o) odd |= non_finite_bits<T>(value16(kp, o));
      }
      if (__any(odd != 0)) {  // key by key
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            for (int gg = 0; gg < 4; ++gg) {
              const int row = 16 * kb + 4 * gg + v;
#pragma unroll
              for (int i = 0; i < QB; ++i) {
                const float w = __shfl(sc[i][kb][v], 16 * gg + r, 64);
                if (!seen(i, from + row)) continue;
#pragma unroll
                for (int o = 0; o < OB; ++o)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int dim = k32 ? 64 * (o / 4) + 16 * g + 4 * e + o % 4 : 16 * o + 4 * g + e;
                    const float f = to_float(
                        *reinterpret_cast<const T*>(vs + row * RB + 16 * ((dim / N) ^ value_swizzle(row)) + dim % N * sizeof(T)));
                    acc[i][o][e] = __builtin_fmaf(w, f, acc[i][o][e]);
                  }
              }
            }
        return;
      }
    }
    if constexpr (k32) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int o = 0; o < OB / 4; ++o) {
            const floatx4 f = __builtin_bit_cast(floatx4, value32(kb, j, o));
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < QB; ++i)
                acc[i][4 * o + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[e], sc[i][kb][j], acc[i][4 * o + e], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int kp = 0; kp < KB / 2; ++kp) {
        union {
          uintx4 all;
          T v[8];
        } w[QB];
#pragma unroll
        for (int i = 0; i < QB; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) w[i].v[e] = (T)sc[i][2 * kp + e / 4][e % 4];
#pragma unroll
        for (int o = 0; o < OB; ++o) {
          const uintx4 a = value16(kp, o);
#pragma unroll
          for (int i = 0; i < QB; ++i) acc[i][o] = mfma16<T>(a, w[i].all, acc[i][o]);
        }
      }
    }
  };

  const int turns = (t1 - t0 + WK - 1) / WK;
  if (t0 + wk < t1) stage(0, t0 + wk);
  for (int n = 0; n < turns; ++n) {
    const int t = t0 + wk + n * WK;
    // The tile is in LDS, and the other buffer has been read.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (WM > 1) __syncthreads();
    if (t + WK < t1) stage((n + 1) & 1, t + WK);
    if (t < t1) {
      const int from = tile_start(t), end = tile_end(t);
      if (active && from < wave_bottom.hi && (end > wave_top.lo || (unsigned)from < p.sinks))
        compute(mine + (n & 1) * 2 * kTile, from, end);
    }
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) l[i] = rows4_sum(l[i]);

  auto out_row = [&](int64_t pair) {
    return static_cast<T*>(p.out) + (size_t)(s.q0 + token(pair)) * p.out_row + (kvh * group + pair % group) * p.out_head;
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int64_t pair = wave_pair + 16 * i + r;
      if (pair >= pairs) continue;
      const float inv = sees_any(p, range[i]) ? 1.0f / l[i] : 0.0f;
      T* out = out_row(pair);
#pragma unroll
      for (int o = 0; o < OB; ++o) {
        struct alignas(4 * sizeof(T)) Four {
          T v[4];
        } f;
        if constexpr (k32) {  // acc[4 o' + e][v]: dimension 64 o' + 16 g + 4 v + e; here v = o % 4
#pragma unroll
          for (int e = 0; e < 4; ++e) f.v[e] = (T)(acc[i][o / 4 * 4 + e][o % 4] * inv);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) f.v[e] = (T)(acc[i][o][e] * inv);
        }
        const unsigned dim = k32 ? 64 * (o / 4) + 16 * g + 4 * (o % 4) : 16 * o + 4 * g;
        if (dim < p.d) *reinterpret_cast<Four*>(out + dim) = f;
      }
    }
  } else {
    // The shares brought to the rows' common maximum and added.
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < QB; ++i) lds_ml[wk * BM + 16 * (QB * wm + i) + r] = make_float2(m[i], l[i]);
    }
    __syncthreads();
    float* part = reinterpret_cast<float*>(lds);
    auto common = [&](int row) {
      float most = lds_ml[row].x;
#pragma unroll
      for (int w = 1; w < WK; ++w) most = fmaxf(most, lds_ml[w * BM + row].x);
      return most;
    };
    auto factor = [&](float own, float most) { return own == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(own - most); };
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int row = 16 * (QB * wm + i) + r;
      const float f = factor(m[i], common(row));
      float* to = part + (wk * BM + row) * DP;
#pragma unroll
      for (int o = 0; o < OB; ++o) {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (k32 ? acc[i][o / 4 * 4 + e][o % 4] : acc[i][o][e]) * f;
        *reinterpret_cast<floatx4*>(to + (k32 ? 64 * (o / 4) + 16 * g + 4 * (o % 4) : 16 * o + 4 * g)) = v;
      }
    }
    __syncthreads();
    for (int at = tid; at < BM * DP / 4; at += 64 * WM * WK) {
      const int row = at / (DP / 4), dim = at % (DP / 4) * 4;
      const int64_t pair = pair0 + row;
      if (pair >= pairs || dim >= (int)p.d) continue;
      const float most = common(row);
      floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
      float den = 0.0f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        sum = sum + *reinterpret_cast<const floatx4*>(part + (w * BM + row) * DP + dim);
        den = den + lds_ml[w * BM + row].y * factor(lds_ml[w * BM + row].x, most);
      }
      const bool any = sees_any(p, visible(p, s, token(pair)));
      if (splits == 1) {
        const float inv = any ? 1.0f / den : 0.0f;
        struct alignas(4 * sizeof(T)) Four {
          T v[4];
        } f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[e] = (T)(sum[e] * inv);
        *reinterpret_cast<Four*>(out_row(pair) + dim) = f;
      } else {
        const size_t to = ((size_t)split * p.rows + s.q0 + token(pair)) * p.heads + kvh * group + pair % group;
        *reinterpret_cast<floatx4*>(part_out + to * p.d + dim) = sum;
        if (dim == 0) part_ml[to] = make_float2(most, any ? den : -1.0f);  // -1: the row sees no key
      }
    }
  }
}

// The splits' results brought to their common maximum and added: one wave per (row, head).
template <class T>
__global__ void __launch_bounds__(256) window_join_kernel(Args p, unsigned splits, const float* part_out, const float2* part_ml) {
  const unsigned at = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const unsigned row = at / p.heads, h = at % p.heads;
  if (row >= p.rows) return;
  const unsigned b = last_at_most(p.batch, row, [&](unsigned i) { return (unsigned)clip(p.q_offsets[i], p.rows); });
  const Sequence s = sequence(p, b);
  if ((int)row < s.q0 || (int)row >= s.q0 + s.nq) return;
  const size_t stride = (size_t)p.rows * p.heads;
  const float2 own = lane < splits ? part_ml[lane * stride + at] : make_float2(-__builtin_inff(), 0.0f);
  float most = own.x;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x, 64));
  const float f = own.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(own.x - most);
  float den = own.y * f;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) den = den + __shfl_xor(den, x, 64);
  const bool none = __shfl(own.y, 0, 64) < 0.0f;
  const float inv = none ? 0.0f : 1.0f / den;
  T* out = static_cast<T*>(p.out) + row * p.out_row + h * p.out_head;
  const unsigned dim = 4 * lane;  // at most 256 of them
  floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (unsigned i = 0; i < splits; ++i) {
    const float w = __shfl(f, i, 64);
    if (dim < p.d) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(part_out + (i * stride + at) * p.d + dim);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = w == 0.0f ? sum[e] : __builtin_fmaf(w, v[e], sum[e]);
    }
  }
  if (dim < p.d) {
    struct alignas(4 * sizeof(T)) Four {
      T v[4];
    } o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = (T)(sum[e] * inv);
    *reinterpret_cast<Four*>(out + dim) = o;
  }
}

// How a call is laid out over the GPU; from the sizes alone.
struct Plan {
  bool few;         // 16 rows a tile, the keys shared among a workgroup's waves
  unsigned splits;  // of the keys over workgroups
};
constexpr unsigned kCus = 256, kFewRows = 16;
constexpr unsigned large_rows(unsigned type) { return type == EG2_TYPE_F32 ? 64 : 128; }

Plan plan(const Args& a) {
  const uint64_t group = a.heads / a.kv_heads, pairs = (uint64_t)a.rows * group;
  const uint64_t busy = a.rows < a.batch ? a.rows : a.batch;  // sequences with queries, at most
  auto groups = [&](uint64_t rows) {  // workgroups with work, about
    const uint64_t tiles = (pairs + rows - 1) / rows;
    return (tiles > busy ? tiles : busy) * a.kv_heads;
  };
  if (groups(large_rows(a.type)) >= kCus && pairs > kFewRows * busy) return Plan{false, 1};
  const uint64_t longest = a.longest ? a.longest : (uint64_t)a.key_rows / a.batch;
  uint64_t span = longest;
  if (a.left >= 0) {
    const uint64_t window = (uint64_t)a.left + a.sinks + (a.right >= 0 ? (uint64_t)a.right + 1 : longest);
    span = window < span ? window : span;
  }
  uint64_t splits = 2 * kCus / groups(kFewRows);
  if (splits > span / 256) splits = span / 256;
  if (splits > 64) splits = 64;
  return Plan{true, splits ? (unsigned)splits : 1u};
}

uint64_t join_bytes(const Args& a, unsigned splits) {  // the sums, then the maxima and denominators
  return splits > 1 ? (uint64_t)splits * a.rows * a.heads * (a.d + 2) * 4 : 0;
}

template <class T, int DP>
hipError_t go(const Args& a, hipStream_t st) {
  const Plan pl = plan(a);
  constexpr bool k32 = __is_same(T, float);
  constexpr int RB = DP * (int)sizeof(T);
  const float scale = (a.scale < 0.0f ? -a.scale : a.scale) * kLog2e;
  const float c = scale > 0x1p-100f ? scale : 0x1p-100f;  // 0: equal weights
  const unsigned group = a.heads / a.kv_heads;
  auto slots = [&](unsigned rows) { return (unsigned)((uint64_t)a.rows * group / rows) + a.batch; };
  if (!pl.few) {
    constexpr int QB = k32 ? 1 : 2, BN = RB <= 256 ? (k32 ? 32 : 64) : RB <= 512 ? 32 : 16;
    const unsigned n = slots(large_rows(a.type));
    window_attention_kernel<T, DP, QB, 4, 1, BN><<<n * a.kv_heads, 256, 0, st>>>(a, n, 1, nullptr, nullptr, c);
    return hipGetLastError();
  }
  constexpr int BN = k32 ? 16 : 32, WK = BN * RB <= 8192 ? 4 : 2;  // at most 128 KB of LDS
  const unsigned n = slots(kFewRows);
  float* sums = static_cast<float*>(a.workspace);
  float2* ml = reinterpret_cast<float2*>(sums + (uint64_t)pl.splits * a.rows * a.heads * a.d);
  window_attention_kernel<T, DP, 1, 1, WK, BN><<<n * a.kv_heads * pl.splits, 64 * WK, 0, st>>>(a, n, pl.splits, sums, ml, c);
  if (pl.splits > 1)
    window_join_kernel<T><<<(a.rows * a.heads + 3) / 4, 256, 0, st>>>(a, pl.splits, sums, ml);
  return hipGetLastError();
}

}  // namespace

uint64_t window_attention_workspace(const Args& a) {
  const Plan pl = plan(a);
  return pl.few ? join_bytes(a, pl.splits) : 0;
}

hipError_t launch_window_attention(const Args& a, hipStream_t st) {
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    if (a.d <= 64) return go<T, 64>(a, st);
    if (a.d <= 128) return go<T, 128>(a, st);
    return go<T, 256>(a, st);
  });
}

}  // namespace block
}  // namespace eg2
