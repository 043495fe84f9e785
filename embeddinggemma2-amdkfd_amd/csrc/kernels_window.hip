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
// The matrix unit takes the softmax weights of 16-bit attention in that type. Where
// a tile has up to 64 rows they go as the sum of two (PARTS: the weight rounded, and what that
// left, rounded), which costs nothing that shows there; with 128 rows, bound by the
// products, as one, rounded by at most half a step, which over many keys adds as much error
// to a result as its own rounding (rms 2.2e-3 of bf16 against 1.7e-3). The sum is
// formed from the 32-bit weights. The running maximum moves only when a score exceeds it by 2^8
// (weights up to 2^8 lose nothing in any type), which spares most of the
// rescaling of the sums.
//
// Bound: causal 8192 bf16 of 16 + 4 x 128 takes 230 to 240 us, 860 to 900 TFLOP/s; a wave's
// products, its softmax and its LDS reads each take about a third of that, and two waves a
// SIMD hide them behind each other in part (the matrix units work 42 % of the cycles). One token over caches:
// the keys' and values' bytes (24 caches of 6000 x 4 x 128 bf16 with a window of 2048: 20.8 us and 3.6
// of the join, 4.1 TB/s; 48 of 8192 x 8 x 128: 304 us, 5.3 TB/s). Short texts: the
// chain of a tile's keys and the launch (16 texts of 128 bf16, 3 + 1 x 256: 11 us).
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

// The last sequence b with first(q_offsets[b], b) <= at, first growing with b
// (0 if none), 64 at a time; of the last 64 every lane loads all that belongs
// to its own, so that the tile's sequence costs one round of loads.
template <class F>
__device__ __forceinline__ Sequence find_sequence(const Args& p, unsigned at, F first, unsigned& b) {
  const unsigned lane = threadIdx.x & 63;
  unsigned lo = 0, n = p.batch;
  while (n > 64) {
    const unsigned step = (n + 63) / 64, i = lane * step;
    const int count = __popcll(__ballot(i < n && first(clip(p.q_offsets[min(lo + i, p.batch - 1)], p.rows), lo + i) <= at));
    const unsigned skip = count > 1 ? (count - 1) * step : 0;
    lo += skip;
    n = min(step, n - skip);
  }
  const unsigned mine = lo + min(lane, n - 1);
  const int q0 = clip(p.q_offsets[mine], p.rows), q1 = clip(p.q_offsets[mine + 1], p.rows);
  const int k0 = clip(p.k_offsets[mine], p.key_rows), k1 = clip(p.k_offsets[mine + 1], p.key_rows);
  int nk = k1 > k0 ? k1 - k0 : 0;
  if (p.k_lengths) nk = clip(p.k_lengths[mine], (unsigned)nk);
  const int count = __popcll(__ballot(lane < n && first(q0, mine) <= at));
  const int pick = count > 1 ? count - 1 : 0;
  b = lo + pick;
  const int q = __builtin_amdgcn_readlane(q0, pick), end = __builtin_amdgcn_readlane(q1, pick);
  return Sequence{q, __builtin_amdgcn_readlane(k0, pick), end > q ? end - q : 0, __builtin_amdgcn_readlane(nk, pick)};
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
// with every key of its share, and WK shares of the keys, joined at the end. BN
// keys to a tile, NBUF tiles in LDS, all but one on their way.
template <class T, int DP, int QB, int WM, int WK, int BN, int NBUF, int PARTS>
__global__ void __launch_bounds__(64 * WM * WK, WM > 1 && DP * (int)sizeof(T) <= 512 ? 2 : 1)
window_attention_kernel(Args p, unsigned slots, unsigned splits, float* part_out, float2* part_ml, float c) {
  constexpr bool k32 = __is_same(T, float);
  constexpr int RB = DP * (int)sizeof(T), CH = RB / 16, KK = RB / 64;  // bytes, 16-byte chunks, MFMA steps of a row
  constexpr int KB = BN / 16, OB = DP / 16, BM = 16 * QB * WM, N = kPer16<T>;
  constexpr int kLoads = BN * RB / 1024 / WM;  // per wave, of keys and of values
  static_assert(BN * RB % (1024 * WM) == 0 && (k32 || BN % 32 == 0), "tile shape");
  constexpr int kTile = BN * RB;
  constexpr int kPart = WK > 1 ? WK * BM * DP * 4 : 0;
  constexpr int kShare = NBUF * 2 * kTile;  // a share's buffers of keys and values
  constexpr int kLds = WK * kShare > kPart ? WK * kShare : kPart;
  __shared__ alignas(16) unsigned char lds[kLds];
  __shared__ float2 lds_ml[WK > 1 ? WK * BM : 1];
  __shared__ alignas(16) float lds_w[WM * WK][16 * QB][16];  // weights, for add_by_key alone
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15, wm = wave % WM, wk = wave / WM;
  const unsigned group = p.heads / p.kv_heads, kvh = blockIdx.x % p.kv_heads;
  const unsigned split = blockIdx.x / p.kv_heads % splits;
  const unsigned slot = slots - 1 - blockIdx.x / p.kv_heads / splits;  // the longest rows of a causal prompt first

  // Sequence b's tiles start at slot q_offsets[b] group / BM + b: at least as
  // many slots as it has tiles, found without a sum over the sequences. (rows heads <= 2^27.)
  auto first_slot = [&](int q0, unsigned i) { return (unsigned)q0 * group / BM + i; };
  unsigned b;
  const Sequence s = find_sequence(p, slot, first_slot, b);
  const unsigned pairs = s.nq * group, first = first_slot(s.q0, b), pair0 = (slot - first) * BM;
  if (slot < first || slot - first >= (pairs + BM - 1) / BM) return;  // the whole workgroup

  // The keys that the tile's rows see: [0, first) and [start, stop), in tiles of BN.
  auto token = [&](unsigned pair) { return (int)(pair / group); };
  const Range top = visible(p, s, token(pair0)), bottom = visible(p, s, token(min(pair0 + BM, pairs) - 1));
  const int stop = bottom.hi;
  int start = min(top.lo, stop), sinks = (int)min((unsigned)start, p.sinks);
  if (start < BN) start = sinks = 0;
  const int tiles_a = (sinks + BN - 1) / BN, tiles_b = (stop - start + BN - 1) / BN, tiles = tiles_a + tiles_b;
  const int t0 = (int)((int64_t)tiles * split / splits), t1 = (int)((int64_t)tiles * (split + 1) / splits);
  auto tile_start = [&](int t) { return t < tiles_a ? t * BN : start + (t - tiles_a) * BN; };
  auto tile_end = [&](int t) { return t < tiles_a ? min(sinks, t * BN + BN) : min(stop, start + (t - tiles_a) * BN + BN); };

  unsigned char* const mine = lds + wk * kShare;
  const T* kbase = static_cast<const T*>(p.k) + (size_t)s.k0 * p.k_row + kvh * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + (size_t)s.k0 * p.v_row + kvh * p.v_head;
  // Chunks of a row are swizzled so that no read waits for LDS's 64 banks: the keys
  // for 16 rows of one chunk column, the 16-bit values for 8 rows of two (rows of
  // 128 bytes: two rows to the banks); fp32 values are read row by row. (Bank conflicts 0; with 8
  // rows told apart the fp32 form took 6 % longer.)
  auto key_swizzle = [](int row) { return row & (CH < 16 ? 7 : 15); };
  auto value_swizzle = [](int row) { return k32 ? 0 : 2 * (CH < 16 ? row >> 1 & 3 : row & 7); };
  if (p.d < DP) {  // the padding of the head size stays zero
    for (int i = tid; i < WK * kShare / 16; i += 64 * WM * WK) reinterpret_cast<uintx4*>(lds)[i] = uintx4{};
    __syncthreads();
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)mine;
  // A tile's loads, always 2 kLoads of them: some lane of each has a chunk below d.
  constexpr int kRows = 64 / CH > 0 ? 64 / CH : 1;  // rows of a load
  const bool near = (p.k_row | p.v_row) < 1u << 26;  // a load's rows lie within 2^32 bytes
  const uint32_t lane_k = (uint32_t)(lane / CH * p.k_row * sizeof(T)), lane_v = (uint32_t)(lane / CH * p.v_row * sizeof(T));
  const size_t step_k = kRows * p.k_row * sizeof(T), step_v = kRows * p.v_row * sizeof(T);
  const size_t wave_k = kLoads * wm * step_k, wave_v = kLoads * wm * step_v;
  auto stage = [&](int buf, int t) {
    const int from = tile_start(t), last = tile_end(t) - 1;
    uint32_t to_lds = __builtin_amdgcn_readfirstlane(lds0 + buf * 2 * kTile + 1024 * kLoads * wm);
    if (near && from + BN - 1 <= last) {
      const unsigned char* k = reinterpret_cast<const unsigned char*>(kbase + (size_t)from * p.k_row) + wave_k;
      const unsigned char* v = reinterpret_cast<const unsigned char*>(vbase + (size_t)from * p.v_row) + wave_v;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = kRows * (kLoads * wm + i) + lane / CH, to = lane % CH;
        const int ck = to ^ key_swizzle(row), cv = to ^ value_swizzle(row);
        if (p.d == DP || N * ck < (int)p.d) dma16(k, lane_k + 16 * ck, to_lds);
        if (p.d == DP || N * cv < (int)p.d) dma16(v, lane_v + 16 * cv, to_lds + kTile);
        k += step_k;
        v += step_v;
        to_lds += 1024;
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kLoads; ++i) {
        const int row = kRows * (kLoads * wm + i) + lane / CH, to = lane % CH;
        const int ck = to ^ key_swizzle(row), cv = to ^ value_swizzle(row);
        const size_t key = min(from + row, last);
        if (N * ck < (int)p.d) dma16_each(kbase + key * p.k_row + N * ck, to_lds);
        if (N * cv < (int)p.d) dma16_each(vbase + key * p.v_row + N * cv, to_lds + kTile);
        to_lds += 1024;
      }
    }
  };
#pragma unroll
  for (int i = 0; i < NBUF - 1; ++i)
    if (t0 + wk + i * WK < t1) stage(i, t0 + wk + i * WK);

  // The wave's rows and the lane's: row 16 qb + r.
  const unsigned wave_pair = pair0 + 16 * QB * wm;
  const bool active = wave_pair < pairs;
  const Range wave_top = visible(p, s, token(min(wave_pair, pairs - 1)));
  const Range wave_bottom = visible(p, s, token(min(wave_pair + 16 * QB, pairs) - 1));
  Range range[QB];
  uintx4 q[QB][KK];
  const uint32_t flip = p.scale < 0.0f ? (k32 ? 0x80000000u : 0x80008000u) : 0u;  // the scale's sign
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const unsigned pair = min(wave_pair + 16 * i + r, pairs - 1);
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
    // Adds sixteen keys from `key0` on, their weights in lds_w, their values at `rows`: each where it is seen alone.
    auto add_by_key = [&](floatx4 (&sum)[QB][OB], const unsigned char* rows, int key0) {
#pragma unroll 1
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < QB; ++i) {
          int g = lane >> 4;
          asm volatile("" : "+v"(g));  // addresses of this rare part are not kept in registers through the loop
          const float w = lds_w[wave][16 * i + r][j];
          if (!(key0 + j < min(range[i].hi, end) && (key0 + j >= range[i].lo || (unsigned)(key0 + j) < p.sinks))) continue;
#pragma unroll
          for (int o = 0; o < OB; ++o) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int dim = k32 ? 64 * (o / 4) + 16 * g + 4 * e + o % 4 : 16 * o + 4 * g + e;
              // the tile's rows go by sixteen, so row j has value_swizzle(j)
              const T f = *reinterpret_cast<const T*>(rows + j * RB + 16 * ((dim / N) ^ value_swizzle(j)) + dim % N * sizeof(T));
              sum[i][o][e] = __builtin_fmaf(w, to_float(f), sum[i][o][e]);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    };
    floatx4 sc[QB][KB];
#pragma unroll
    for (int i = 0; i < QB; ++i)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) sc[i][kb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    // Operands a step ahead of the products; the barriers keep the scheduler from taking more registers for them.
    uintx4 a[2][KB];
    auto load_keys = [&](int kk) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int row = 16 * kb + r;
        a[kk & 1][kb] = *reinterpret_cast<const uintx4*>(ks + row * RB + 16 * ((4 * kk + g) ^ key_swizzle(row)));
      }
    };
    load_keys(0);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if (kk + 1 < KK) load_keys(kk + 1);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < QB; ++i) sc[i][kb] = mfma16<T>(a[kk & 1][kb], q[i][kk], sc[i][kb]);
      __builtin_amdgcn_sched_barrier(0);
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
    auto value16 = [&](int kp, int o, int r) {
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
    auto value32 = [&](int kb, int j, int o, int r) {
      const int row = 16 * kb + 4 * g + j;
      return *reinterpret_cast<const uintx4*>(vs + row * RB + 16 * ((16 * o + r) ^ value_swizzle(row)));
    };
    if (!full) {
      uint32_t odd = 0;
      int mine_r = r;
      asm volatile("" : "+v"(mine_r));  // addresses of this rare part are not kept in registers through the loop
      if constexpr (k32) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int o = 0; o < OB / 4; ++o) odd |= non_finite_bits<T>(value32(kb, j, o, mine_r));
      } else {
#pragma unroll
        for (int kp = 0; kp < KB / 2; ++kp)
#pragma unroll
          for (int o = 0; o < OB; ++o) odd |= non_finite_bits<T>(value16(kp, o, mine_r));
      }
      asm volatile("" ::: "memory");  // read again below, not kept in registers
      if (__any(odd != 0)) {  // key by key, to sums of their own: acc is moved to no other registers behind the products
        floatx4 sum[QB][OB];
#pragma unroll
        for (int i = 0; i < QB; ++i)
#pragma unroll
          for (int o = 0; o < OB; ++o) sum[i][o] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
          for (int i = 0; i < QB; ++i) *reinterpret_cast<floatx4*>(&lds_w[wave][16 * i + r][4 * g]) = sc[i][kb];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          add_by_key(sum, vs + 16 * kb * RB, from + 16 * kb);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int i = 0; i < QB; ++i)
#pragma unroll
          for (int o = 0; o < OB; ++o) acc[i][o] = acc[i][o] + sum[i][o];
        return;
      }
    }
    if constexpr (k32) {
      constexpr int kSteps = 4 * KB;  // keys 16 kb + 4 g + j, the operands of step + 1 ahead
      uintx4 f[2][OB / 4];
      auto load_values = [&](int n) {
#pragma unroll
        for (int o = 0; o < OB / 4; ++o) f[n & 1][o] = value32(n / 4, n % 4, o, r);
      };
      load_values(0);
#pragma unroll
      for (int n = 0; n < kSteps; ++n) {
        if (n + 1 < kSteps) load_values(n + 1);
#pragma unroll
        for (int o = 0; o < OB / 4; ++o) {
          const floatx4 v = __builtin_bit_cast(floatx4, f[n & 1][o]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < QB; ++i)
              acc[i][4 * o + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], sc[i][n / 4][n % 4], acc[i][4 * o + e], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      union {
        uintx4 all;
        T v[8];
      } w[PARTS][QB][KB / 2];
#pragma unroll
      for (int i = 0; i < QB; ++i)
#pragma unroll
        for (int kp = 0; kp < KB / 2; ++kp)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = sc[i][2 * kp + e / 4][e % 4];
            w[0][i][kp].v[e] = (T)f;
            if constexpr (PARTS == 2) w[1][i][kp].v[e] = (T)(f - to_float(w[0][i][kp].v[e]));
          }
      constexpr int kSteps = KB / 2 * OB / 4;  // of four blocks of dimensions
      uintx4 f[2][4];
      auto load_values = [&](int n) {
#pragma unroll
        for (int o = 0; o < 4; ++o) f[n & 1][o] = value16(n / (OB / 4), n % (OB / 4) * 4 + o, r);
      };
      load_values(0);
#pragma unroll
      for (int n = 0; n < kSteps; ++n) {
        if (n + 1 < kSteps) load_values(n + 1);
#pragma unroll
        for (int o = 0; o < 4; ++o)
#pragma unroll
          for (int i = 0; i < QB; ++i) {
            floatx4& sum = acc[i][n % (OB / 4) * 4 + o];
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) sum = mfma16<T>(f[n & 1][o], w[part][i][n / (OB / 4)].all, sum);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  const int turns = (t1 - t0 + WK - 1) / WK;
  int buf = 0;
  for (int n = 0; n < turns; ++n) {
    const int t = t0 + wk + n * WK;
    if constexpr (NBUF == 1) {  // each wave on its own
      static_assert(NBUF > 1 || WM == 1, "one buffer is not shared");
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (t < t1) stage(0, t);
    }
    // This tile is in LDS (those behind it may be on their way), and the buffer before it has been read.
    if (NBUF > 2 && t + (NBUF - 2) * WK < t1)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NBUF > 2 ? NBUF - 2 : 0) * 2 * kLoads) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (WM > 1) __syncthreads();
    const int ahead = t + (NBUF - 1) * WK;
    if (NBUF > 1 && ahead < t1) stage(buf == 0 ? NBUF - 1 : buf - 1, ahead);
    if (t < t1) {
      const int from = tile_start(t), end = tile_end(t);
      if (active && from < wave_bottom.hi && (end > wave_top.lo || (unsigned)from < p.sinks))
        compute(mine + buf * 2 * kTile, from, end);
    }
    buf = buf + 1 < NBUF ? buf + 1 : 0;
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) l[i] = rows4_sum(l[i]);

  auto out_row = [&](unsigned pair) {
    return static_cast<T*>(p.out) + (size_t)(s.q0 + token(pair)) * p.out_row + (kvh * group + pair % group) * p.out_head;
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const unsigned pair = wave_pair + 16 * i + r;
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
    // The shares brought to the rows' common maximum and added. A row's factors
    // replace its maxima in lds_ml.
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < QB; ++i) lds_ml[wk * BM + 16 * (QB * wm + i) + r] = make_float2(m[i], l[i]);
    }
    __syncthreads();
    if (tid < BM) {
      float2 own[WK];
      float most = -__builtin_inff(), den = 0.0f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        own[w] = lds_ml[w * BM + tid];
        most = fmaxf(most, own[w].x);
      }
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        own[w].x = own[w].x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(own[w].x - most);
        den = den + own[w].y * own[w].x;
      }
      const unsigned pair = min(pair0 + tid, pairs - 1);
      const bool any = sees_any(p, visible(p, s, token(pair)));
      float scale = 1.0f;
      if (splits == 1) {
        scale = any ? 1.0f / den : 0.0f;
      } else if (pair0 + tid < pairs) {
        const size_t to = ((size_t)split * p.rows + s.q0 + token(pair)) * p.heads + kvh * group + pair % group;
        part_ml[to] = make_float2(most, any ? den : -1.0f);  // -1: the row sees no key
      }
#pragma unroll
      for (int w = 0; w < WK; ++w) lds_ml[w * BM + tid].x = own[w].x * scale;
    }
    __syncthreads();
    float* part = reinterpret_cast<float*>(lds);
    auto place = [&](int row, int dim) { return part + row * DP + (dim ^ 4 * (row & 15)); };  // for 16 rows of one column
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int row = 16 * (QB * wm + i) + r;
      const float f = lds_ml[wk * BM + row].x;
#pragma unroll
      for (int o = 0; o < OB; ++o) {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (k32 ? acc[i][o / 4 * 4 + e][o % 4] : acc[i][o][e]) * f;
        *reinterpret_cast<floatx4*>(place(wk * BM + row, k32 ? 64 * (o / 4) + 16 * g + 4 * (o % 4) : 16 * o + 4 * g)) = v;
      }
    }
    __syncthreads();
    for (int at = tid; at < BM * DP / 4; at += 64 * WM * WK) {
      const int row = at / (DP / 4), dim = at % (DP / 4) * 4;
      const unsigned pair = pair0 + row;
      if (pair >= pairs || dim >= (int)p.d) continue;
      floatx4 sum = *reinterpret_cast<const floatx4*>(place(row, dim));
#pragma unroll
      for (int w = 1; w < WK; ++w) sum = sum + *reinterpret_cast<const floatx4*>(place(w * BM + row, dim));
      if (splits == 1) {
        struct alignas(4 * sizeof(T)) Four {
          T v[4];
        } f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[e] = (T)sum[e];
        *reinterpret_cast<Four*>(out_row(pair) + dim) = f;
      } else {
        const size_t to = ((size_t)split * p.rows + s.q0 + token(pair)) * p.heads + kvh * group + pair % group;
        *reinterpret_cast<floatx4*>(part_out + to * p.d + dim) = sum;
      }
    }
  }
}

// The splits' results brought to their common maximum and added: a workgroup
// per (row, head), a thread four dimensions of every kShares-th split, all on their
// way before it is known whether the row is in a sequence.
constexpr unsigned kMostSplits = 64;
template <class T, int DP>
__global__ void __launch_bounds__(256) window_join_kernel(Args p, unsigned splits, const float* part_out, const float2* part_ml) {
  constexpr unsigned kShares = 256 / (DP / 4), kEach = kMostSplits / kShares;
  __shared__ floatx4 sums[kShares][DP / 4];
  const unsigned at = blockIdx.x, row = at / p.heads, h = at % p.heads, lane = threadIdx.x & 63;
  const unsigned dim = threadIdx.x % (DP / 4) * 4, share = threadIdx.x / (DP / 4);
  const size_t stride = (size_t)p.rows * p.heads;
  const float2 own = lane < splits ? part_ml[lane * stride + at] : make_float2(-__builtin_inff(), 0.0f);
  floatx4 v[kEach];
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i)
    if (share + kShares * i < splits && dim < p.d)
      v[i] = *reinterpret_cast<const floatx4*>(part_out + ((share + kShares * i) * stride + at) * p.d + dim);
  unsigned b;
  const Sequence s = find_sequence(p, row, [](int q0, unsigned) { return (unsigned)q0; }, b);
  if ((int)row < s.q0 || (int)row >= s.q0 + s.nq) return;  // the whole workgroup
  float most = own.x;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x, 64));
  const float f = own.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(own.x - most);
  float den = own.y * f;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) den = den + __shfl_xor(den, x, 64);
  const float inv = __shfl(own.y, 0, 64) < 0.0f ? 0.0f : 1.0f / den;  // -1: the row sees no key
  floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (unsigned i = 0; i < kEach; ++i) {
    const float w = __shfl(f, share + kShares * i, 64);
    if (share + kShares * i < splits && dim < p.d)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w, v[i][e], sum[e]);
  }
  sums[share][dim / 4] = sum;
  __syncthreads();
  if (share != 0 || dim >= p.d) return;
#pragma unroll
  for (unsigned i = 1; i < kShares; ++i) sum = sum + sums[i][dim / 4];
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  } o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o.v[e] = (T)(sum[e] * inv);
  *reinterpret_cast<Four*>(static_cast<T*>(p.out) + row * p.out_row + h * p.out_head + dim) = o;
}

// How a call is laid out over the GPU; from the sizes alone.
struct Plan {
  unsigned rows;    // of a tile; kFewRows: the keys shared among a workgroup's waves
  unsigned splits;  // of the keys over workgroups
};
constexpr unsigned kCus = 256, kFewRows = 16;

Plan plan(const Args& a) {
  const uint64_t group = a.heads / a.kv_heads, pairs = (uint64_t)a.rows * group;
  const uint64_t busy = a.rows < a.batch ? a.rows : a.batch;  // sequences with queries, at most
  auto groups = [&](uint64_t rows) {  // workgroups with work, about
    const uint64_t tiles = (pairs + rows - 1) / rows;
    return (tiles > busy ? tiles : busy) * a.kv_heads;
  };
  const uint64_t longest = a.longest ? a.longest : (uint64_t)a.key_rows / a.batch;
  uint64_t span = longest;
  if (a.left >= 0) {
    const uint64_t window = (uint64_t)a.left + a.sinks + (a.right >= 0 ? (uint64_t)a.right + 1 : longest);
    span = window < span ? window : span;
  }
  // The more rows a tile has, the less often keys are read; but the GPU needs a workgroup for most of
  // its CUs. us by tiles of 128, 64, 32 and 16 rows: bf16 8 x 1024 of 3 + 1 x 256, window 512: 42, 56, 67, -;
  // 4 x 1024 40, 31, 46, 72; 1 x 2048 -, 28.5, 24.9, 49; 16 x 128 -, 15.8, 13.4, 20.7; causal 3 x 1024 of 16 + 4 x 128
  // 45, 50, 75, -; 1 x 1024 33, 22, 27, 42; 1 x 2048 57, 44, 73, -; fp32 4 x 1024 -, 101, 126, 191; 1 x 2048 -, 100, 65, 127.
  if (pairs > kFewRows * busy) {
    const bool uneven = a.right >= 0 && span > longest / 2;  // causal: the first rows have few keys, the last all
    if (a.type != EG2_TYPE_F32 && groups(128) >= (uneven ? 320 : 144)) return Plan{128, 1};
    if (groups(64) >= 144) return Plan{64, 1};
    if (groups(32) >= 144) return Plan{32, 1};
  }
  // The keys split over one round of workgroups: two to a CU where a row of keys takes 128 bytes, one
  // beyond (24 caches at 192 workgroups 28 us, at 480 39). Each at least 64 keys (1 x 8192 x 256: 13.8 us; 256 keys 17, 512 23),
  // and none below 512, where the join costs more (300 keys: split 8.8 us, whole 7.3; 1000: 10.8, 14.9). Tiles
  // of 32 and 64 rows are not split: their sums make the join too long (300 rows over 3000: 34 us, whole
  // 36; 500 over 1000: 32, 20).
  const uint64_t row = (a.d <= 64 ? 64u : a.d <= 128 ? 128u : 256u) * (a.type == EG2_TYPE_F32 ? 4u : 2u);
  uint64_t splits = (row <= 128 ? 2 * kCus : kCus) / groups(kFewRows);
  if (splits > span / 64) splits = span / 64;
  if (splits > kMostSplits) splits = kMostSplits;
  // Sequences without queries have workgroups as well, which end at once: at most 2^22 more of them.
  const uint64_t most = (1u << 22) / ((uint64_t)a.batch * a.kv_heads);
  if (splits > most) splits = most;
  if (span < 512) splits = 1;
  return Plan{kFewRows, splits ? (unsigned)splits : 1u};
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
  const float c = scale > 0.0f ? scale : 0x1p-149f;  // 0: every finite score below 2^-21, and a hidden key still at -inf
  const unsigned group = a.heads / a.kv_heads, n = (unsigned)((uint64_t)a.rows * group / pl.rows) + a.batch;
  auto whole = [&](auto qb, auto wm, auto wk, auto bn) {
    constexpr int QB = decltype(qb)::value, WM = decltype(wm)::value, WK = decltype(wk)::value, BN = decltype(bn)::value;
    constexpr int PARTS = k32 || 16 * QB * WM > 64 ? 1 : 2;
    window_attention_kernel<T, DP, QB, WM, WK, BN, 2, PARTS><<<n * a.kv_heads, 64 * WM * WK, 0, st>>>(a, n, 1, nullptr, nullptr, c);
    return hipGetLastError();
  };
  switch (pl.rows) {
    case 128:
      if constexpr (!k32) return whole(Const<DP <= 128 ? 2 : 1>{}, Const<DP <= 128 ? 4 : 8>{}, Const<1>{}, Const<DP <= 128 ? 64 : 32>{});
      return hipErrorInvalidValue;
    case 64:
      return whole(Const<1>{}, Const<4>{}, Const<(RB > 512) ? 1 : 2>{}, Const<(RB > 256) ? 32 : 64>{});
    case 32:
      return whole(Const<1>{}, Const<2>{}, Const<(RB > 128) ? 2 : 4>{}, Const<(RB > 512) ? 16 : (RB > 256) ? 32 : 64>{});
    default:
      break;
  }
  constexpr int BN = k32 ? 16 : 32, WK = 4, NBUF = BN * RB <= 8192 ? 2 : 1;  // at most 128 KB of LDS
  float* sums = static_cast<float*>(a.workspace);
  float2* ml = reinterpret_cast<float2*>(sums + (uint64_t)pl.splits * a.rows * a.heads * a.d);
  window_attention_kernel<T, DP, 1, 1, WK, BN, NBUF, k32 ? 1 : 2><<<n * a.kv_heads * pl.splits, 64 * WK, 0, st>>>(a, n, pl.splits, sums, ml, c);
  if (pl.splits > 1)
    window_join_kernel<T, DP><<<a.rows * a.heads, 256, 0, st>>>(a, pl.splits, sums, ml);
  return hipGetLastError();
}

}  // namespace

uint64_t window_attention_workspace(const Args& a) {
  const Plan pl = plan(a);
  return join_bytes(a, pl.splits);
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
