// The kernels of eg2_hip_linear and eg2_hip_linear_gated, for one activation
// type each (kernels_linear_*.hip).
//
//   y = act(x W^T + b) + r            y = act(x Wg^T + bg) * (x Wu^T + bu)
//
// Products run on the matrix units with 32-bit sums: v_mfma_f32_16x16x32 of the
// 16-bit types, v_mfma_f32_16x16x4_f32 of fp32. The weights are the first operand, so
// that a lane holds consecutive columns of one row of y: bias, residual and y move
// in 16 bytes. Q8_0 weights with 16-bit activations: a block's 32 whole numbers of
// 8 bits are exact in the type and are one MFMA's depth; its scale is one fma
// per output and block. With fp32 activations the other weights are decoded to fp32, exactly.
#pragma once

#include <hip/hip_runtime.h>

#include "block_device.hpp"
#include "eg2_block.hpp"

namespace eg2 {
namespace block {

template <class W>
constexpr bool kIsQ8 = __is_same(W, Q8);

// Loads at any alignment of the values (one instruction: global loads need none).
template <class V>
__device__ __forceinline__ V load_any(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}

// 16 bytes of T from the W values [k, k + kPer16) of a row, zeros from `end` on.
template <class T, class W>
__device__ __forceinline__ uintx4 load_chunk(const W* row, unsigned k, unsigned end) {
  constexpr int N = kPer16<T>;
  union {
    uintx4 all;
    T v[N];
  } r;
  if (k + N <= end) {
    if constexpr (__is_same(T, W)) return load_any<uintx4>(row + k);
    struct Raw {
      W v[N];
    };
    const Raw w = load_any<Raw>(row + k);
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[e] = (T)to_float(w.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[e] = k + e < end ? (T)to_float(row[k + e]) : (T)0.0f;
  }
  return r.all;
}

// The output of a lane: COLS consecutive columns of one row, from their sums.
template <class T, bool GATED, int COLS>
__device__ __forceinline__ void finish(const Linear& p, unsigned row, unsigned col, const float (&a)[COLS],
                                       const float (&b)[COLS]) {
  static_assert(COLS % 4 == 0, "");
  if (row >= p.n || col >= p.m) return;
  T* y = static_cast<T*>(p.y) + row * p.ldy + col;
  const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr + col : nullptr;
  struct alignas(sizeof(T) * 4) Four {
    T v[4];
  };
  auto on = [](const void* q) { return q == nullptr || reinterpret_cast<uintptr_t>(q) % sizeof(Four) == 0; };
  const bool whole = col + COLS <= p.m && on(y) && on(r);
#pragma unroll
  for (int c = 0; c < COLS; c += 4) {
    Four res, out;
    if (r && whole) res = *reinterpret_cast<const Four*>(r + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned at = min(col + c + e, p.m - 1);
      float z = a[c + e];
      if (p.bias[0]) z = z + p.bias[0][at];
      z = activate(z, p.act);
      if constexpr (GATED) {
        float u = b[c + e];
        if (p.bias[1]) u = u + p.bias[1][at];
        z = z * u;
      } else if (r) {
        if (!whole) res.v[e] = r[at - col];
        z = z + to_float(res.v[e]);
      }
      out.v[e] = (T)z;
      if (!whole && col + c + e < p.m) y[c + e] = out.v[e];
    }
    if (whole) *reinterpret_cast<Four*>(y + c) = out;
  }
}

// ------------------------------------------------------------------ tiles
//
// BM rows of x times BN rows of the weights (of a gated pair BN / 2 of each
// matrix) per workgroup of four waves, 2 x 2, each 16 x 16 blocks over its
// quarter. Slices of 128 bytes of every row go through two LDS buffers, the next
// on its way while one is multiplied. The 16-byte chunks of a row are
// swizzled so that the 16 rows of a fragment read lie on distinct banks.
constexpr int kRowBytes = 128, kChunks = kRowBytes / 16;

// A wave's block j of JBG, lane i: which of its 16 JBG weight rows it feeds, so
// that a lane's outputs of the blocks are consecutive columns.
template <int JBG>
__device__ __forceinline__ int weight_row(int j, int i) {
  return 4 * JBG * (i >> 2) + 4 * j + (i & 3);
}
template <int JBG>
__device__ __forceinline__ int weight_key(int row) {
  return (row & 3) | ((row / (4 * JBG)) & 1) << 2;
}

// One Q8_0 item: 16 values of a row and the scale of their block.
struct Q8Item {
  uint32_t q[4];
  uint32_t d;
};

template <class T, class W, bool GATED, bool DMA, int BM, int BN>
__global__ void __launch_bounds__(256) linear_tile_kernel(Linear p) {
  constexpr int G = GATED ? 2 : 1, COLS = BN / G;  // columns of y
  constexpr int IB = BM / 32, JB = BN / 32, JBG = JB / G;
  constexpr int N = kPer16<T>, BK = kChunks * N;  // values per chunk and slice
  constexpr bool kScaled = kIsQ8<W> && !__is_same(T, float);
  constexpr bool kDmaW = DMA && __is_same(T, W);
  constexpr int kBlocks = BK / 32;  // Q8_0 blocks of a slice
  struct Lds {
    alignas(16) unsigned char x[2][BM * kRowBytes];
    alignas(16) unsigned char w[2][BN * kRowBytes];
    alignas(16) float d[2][kScaled ? kBlocks * BN : 4];
  };
  __shared__ Lds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15, wm = wave >> 1, wn = wave & 1;

  // Workgroups go round the 8 XCDs; each XCD takes a run of tiles, eight rows
  // of tiles down before the next column, so that its L2 serves both operands.
  const unsigned down = (p.n + BM - 1) / BM, across = (p.m + COLS - 1) / COLS, tiles = down * across;
  const unsigned xcd = blockIdx.x & 7, share = tiles / 8, more = tiles % 8;
  const unsigned at = xcd * share + min(xcd, more) + (blockIdx.x >> 3);
  const unsigned band = at / (8 * across), in_band = at - band * 8 * across, high = min(8u, down - 8 * band);
  const unsigned row0 = (8 * band + in_band % high) * BM, col0 = in_band / high * COLS;

  auto weight_base = [&](int rr) -> const unsigned char* {  // the row of the weights that is row rr of the tile
    const int z = GATED && rr >= COLS;
    const size_t row = min(col0 + rr - z * COLS, p.m - 1);
    const unsigned char* w = static_cast<const unsigned char*>(p.w[z]);
    if constexpr (kIsQ8<W>)
      return w + row * (p.ldw / 32) * kBlockBytes;
    else
      return w + row * p.ldw * sizeof(W);
  };
  const T* xrows = static_cast<const T*>(p.x);

  // A slice on its way through registers.
  constexpr int kXItems = BM * kChunks / 256;
  constexpr int kWItems = kIsQ8<W> ? (BN * BK / 16 + 255) / 256 : BN * kChunks / 256;
  uintx4 xv[kXItems], wv[kIsQ8<W> ? 1 : kWItems];
  Q8Item qv[kIsQ8<W> ? kWItems : 1];
  auto load = [&](unsigned k0) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < kXItems; ++i) {
        const int item = tid + 256 * i, rr = item / kChunks, c = item % kChunks;
        xv[i] = load_chunk<T, T>(xrows + min(row0 + rr, p.n - 1) * p.ldx, k0 + N * c, p.k);
      }
    }
    if constexpr (kIsQ8<W>) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + 256 * i, rr = item / (BK / 16), part = item % (BK / 16);
        const unsigned k = k0 + 16 * part;
        qv[i] = Q8Item{};
        if (rr < BN && k < p.k) {
          const unsigned char* b = weight_base(rr) + (size_t)(k / 32) * kBlockBytes;
          qv[i].d = load_any<uint16_t>(b);
          const uintx4 q = load_any<uintx4>(b + 2 + k % 32);
#pragma unroll
          for (int e = 0; e < 4; ++e) qv[i].q[e] = q[e];
        }
      }
    } else if constexpr (!kDmaW) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + 256 * i, rr = item / kChunks, c = item % kChunks;
        wv[i] = load_chunk<T, W>(reinterpret_cast<const W*>(weight_base(rr)), k0 + N * c, p.k);
      }
    }
  };
  auto put = [&](int buf) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < kXItems; ++i) {
        const int item = tid + 256 * i, rr = item / kChunks, c = item % kChunks;
        *reinterpret_cast<uintx4*>(lds.x[buf] + rr * kRowBytes + 16 * (c ^ (rr & 7))) = xv[i];
      }
    }
    if constexpr (kIsQ8<W>) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + 256 * i, rr = item / (BK / 16), part = item % (BK / 16);
        if (rr >= BN) continue;
        const float d = fp16_bits_to_fp32(qv[i].d);
        if constexpr (kScaled)
          if (part % 2 == 0) lds.d[buf][part / 2 * BN + rr] = d;
#pragma unroll
        for (int c = 0; c < 16 / N; ++c) {
          union {
            uintx4 all;
            T v[N];
          } o;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int at = N * c + e;
            const float q = (float)(int8_t)(qv[i].q[at / 4] >> (8 * (at % 4)));
            o.v[e] = (T)(kScaled ? q : d * q);
          }
          *reinterpret_cast<uintx4*>(lds.w[buf] + rr * kRowBytes +
                                     16 * ((16 / N * part + c) ^ weight_key<JBG>(rr))) = o.all;
        }
      }
    } else if constexpr (!kDmaW) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + 256 * i, rr = item / kChunks, c = item % kChunks;
        *reinterpret_cast<uintx4*>(lds.w[buf] + rr * kRowBytes + 16 * (c ^ weight_key<JBG>(rr))) = wv[i];
      }
    }
  };
  // The same straight to LDS: a wave's load fills 1 KB, 8 rows, lane l the chunk
  // l % 8 of row l / 8; the swizzle is in which chunk it reads. Chunks past k are zeroed.
  constexpr int kXDma = DMA ? BM / 32 : 0, kWDma = kDmaW ? BN / 32 : 0;  // per wave
  uint32_t xoff[DMA ? kXDma : 1], woff[kDmaW ? kWDma : 1];
  int xc = 0, wc[kDmaW ? kWDma : 1];
  const unsigned char* wbase[kDmaW ? kWDma : 1];
  const T* xbase = xrows + row0 * p.ldx;
  if constexpr (DMA) {
    xc = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < kXDma; ++i) {
      const unsigned rr = 8 * (kXDma * wave + i) + (lane >> 3);
      xoff[i] = (uint32_t)((min(row0 + rr, p.n - 1) - row0) * p.ldx * sizeof(T)) + 16 * xc;
    }
  }
  if constexpr (kDmaW) {
#pragma unroll
    for (int i = 0; i < kWDma; ++i) {
      const int first = 8 * (kWDma * wave + i), rr = first + (lane >> 3);
      wc[i] = (lane & 7) ^ weight_key<JBG>(rr);
      wbase[i] = weight_base(first);  // uniform
      woff[i] = (uint32_t)(weight_base(rr) - wbase[i]) + 16 * wc[i];
    }
  }
  auto lds_at = [](const void* q) {
    return __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)static_cast<const unsigned char*>(q));
  };
  auto dma = [&](int buf, unsigned k0) {
    const bool full = k0 + BK <= p.k;
    const uintx4 zero = {};
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < kXDma; ++i) {
        unsigned char* to = lds.x[buf] + 1024 * (kXDma * wave + i);
        if (full || k0 + N * xc < p.k)
          dma16(xbase + k0, xoff[i], lds_at(to));
        else
          *reinterpret_cast<uintx4*>(to + 16 * lane) = zero;
      }
    }
    if constexpr (kDmaW) {
#pragma unroll
      for (int i = 0; i < kWDma; ++i) {
        unsigned char* to = lds.w[buf] + 1024 * (kWDma * wave + i);
        if (full || k0 + N * wc[i] < p.k)
          dma16(wbase[i] + k0 * sizeof(T), woff[i], lds_at(to));
        else
          *reinterpret_cast<uintx4*>(to + 16 * lane) = zero;
      }
    }
  };

  floatx4 acc[IB][JB];
#pragma unroll
  for (int i = 0; i < IB; ++i)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  // The first tile row of the wave's block j, and the block's place in its group.
  auto group_row = [&](int j) { return (j / JBG) * COLS + wn * (16 * JBG); };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uintx4 a[JB], b[IB];
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        const int row = group_row(j) + weight_row<JBG>(j % JBG, r);
        a[j] = *reinterpret_cast<const uintx4*>(lds.w[buf] + row * kRowBytes + 16 * ((4 * kk + g) ^ weight_key<JBG>(row)));
      }
#pragma unroll
      for (int i = 0; i < IB; ++i) {
        const int row = 16 * (IB * wm + i) + r;
        b[i] = *reinterpret_cast<const uintx4*>(lds.x[buf] + row * kRowBytes + 16 * ((4 * kk + g) ^ (row & 7)));
      }
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        floatx4 d;
        if constexpr (kScaled)  // of the lane's four columns
          d = *reinterpret_cast<const floatx4*>(lds.d[buf] + kk * BN + group_row(j) + weight_row<JBG>(j % JBG, 4 * g));
#pragma unroll
        for (int i = 0; i < IB; ++i) {
          if constexpr (kScaled) {
            const floatx4 dot = mfma16<T>(a[j], b[i], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] = __builtin_fmaf(dot[v], d[v], acc[i][j][v]);
          } else {
            acc[i][j] = mfma16<T>(a[j], b[i], acc[i][j]);
          }
        }
      }
    }
  };

  const unsigned slices = (p.k + BK - 1) / BK;
  dma(0, 0);
  load(0);
  put(0);
  for (unsigned s = 0; s < slices; ++s) {
    // The slice is in its buffer, and the other buffer has been read.
    if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (s + 1 < slices) {
      dma((s + 1) & 1, (s + 1) * BK);
      load((s + 1) * BK);
    }
    multiply(s & 1);
    if (s + 1 < slices) put((s + 1) & 1);
  }
#pragma unroll
  for (int i = 0; i < IB; ++i) {
    float a[4 * JBG], b[4 * JBG];
#pragma unroll
    for (int j = 0; j < JBG; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        a[4 * j + v] = acc[i][j][v];
        b[4 * j + v] = acc[i][JB - JBG + j][v];
      }
    finish<T, GATED, 4 * JBG>(p, row0 + 16 * (IB * wm + i) + r, col0 + wn * (16 * JBG) + 4 * JBG * g, a, b);
  }
}

// ------------------------------------------------------------------ few rows
//
// 16 NB rows of x times 16 rows of the weights (of a gated pair of each
// matrix) per workgroup of eight waves, which take every eighth step of k
// and add their sums through LDS: the weights come straight from memory in
// the order of the operand, and every workgroup's chain is an eighth of k.
constexpr int kFewWaves = 8;

template <class T, class W>
struct FewWeights {  // a step of a row: 32 values (fp32: two chunks of 16)
  static constexpr int kChunk = __is_same(T, float) ? 2 : 1;
  uintx4 v[kChunk];
  __device__ __forceinline__ void load(const unsigned char* row, unsigned k, unsigned g, unsigned end) {
#pragma unroll
    for (int c = 0; c < kChunk; ++c)
      v[c] = load_chunk<T, W>(reinterpret_cast<const W*>(row), k + kPer16<T> * (4 * c + g), end);
  }
  __device__ __forceinline__ uintx4 get(int c) const { return v[c]; }
};
template <class T>
struct FewWeights<T, Q8> {
  uint32_t q[2];
  uint32_t d;
  __device__ __forceinline__ void load(const unsigned char* row, unsigned k, unsigned g, unsigned end) {
    q[0] = q[1] = d = 0;
    if (k >= end) return;
    const unsigned char* b = row + (size_t)(k / 32) * kBlockBytes;
    d = load_any<uint16_t>(b);
    if constexpr (__is_same(T, float)) {  // values 4 g .. and 16 + 4 g ..
      q[0] = load_any<uint32_t>(b + 2 + 4 * g);
      q[1] = load_any<uint32_t>(b + 18 + 4 * g);
    } else {
      const uint2 v = load_any<uint2>(b + 2 + 8 * g);
      q[0] = v.x;
      q[1] = v.y;
    }
  }
  __device__ __forceinline__ uintx4 get(int c) const {
    constexpr int N = kPer16<T>;
    union {
      uintx4 all;
      T v[N];
    } o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float f = (float)(int8_t)(q[N == 4 ? c : e / 4] >> (8 * (e % 4)));
      o.v[e] = (T)(N == 4 ? fp16_bits_to_fp32(d) * f : f);
    }
    return o.all;
  }
};

template <class T, class W, bool GATED, int NB>
__global__ void __launch_bounds__(64 * kFewWaves) linear_few_kernel(Linear p) {
  constexpr int G = GATED ? 2 : 1, kChunk = __is_same(T, float) ? 2 : 1;
  constexpr bool kScaled = kIsQ8<W> && !__is_same(T, float);
  constexpr int kDepth = NB * G >= 4 ? 2 : 4;  // steps on their way
  __shared__ floatx4 part[kFewWaves][G][NB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const unsigned across = (p.m + 15) / 16;
  const unsigned row0 = blockIdx.x / across * 16 * NB, col0 = blockIdx.x % across * 16;
  const unsigned char* wrow[G];
#pragma unroll
  for (int z = 0; z < G; ++z) {
    const size_t row = min(col0 + r, p.m - 1);
    wrow[z] = static_cast<const unsigned char*>(p.w[z]);
    if constexpr (kIsQ8<W>)
      wrow[z] += row * (p.ldw / 32) * kBlockBytes;
    else
      wrow[z] += row * p.ldw * sizeof(W);
  }
  const T* xrow[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) xrow[i] = static_cast<const T*>(p.x) + min(row0 + 16 * i + r, p.n - 1) * p.ldx;

  floatx4 acc[G][NB];
#pragma unroll
  for (int z = 0; z < G; ++z)
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[z][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  const unsigned steps = (p.k + 31) / 32;
  FewWeights<T, W> w[kDepth][G];
  uintx4 x[kDepth][NB][kChunk];
  auto load = [&](int slot, unsigned step) {
    if (step >= steps) return;  // uniform
    const unsigned k = 32 * step;
#pragma unroll
    for (int z = 0; z < G; ++z) w[slot][z].load(wrow[z], k, g, p.k);
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int c = 0; c < kChunk; ++c) x[slot][i][c] = load_chunk<T, T>(xrow[i], k + kPer16<T> * (4 * c + g), p.k);
  };
#pragma unroll
  for (int s = 0; s < kDepth; ++s) load(s, wave + kFewWaves * s);
  for (unsigned step = wave; step < steps; step += kFewWaves * kDepth) {
#pragma unroll
    for (int s = 0; s < kDepth; ++s) {
      if (step + kFewWaves * s >= steps) break;  // uniform
#pragma unroll
      for (int z = 0; z < G; ++z) {
        floatx4 d;
        if constexpr (kScaled) {  // of the lane's four columns 4 g .., from the lanes that loaded them
#pragma unroll
          for (int v = 0; v < 4; ++v) d[v] = fp16_bits_to_fp32(__shfl((int)w[s][z].d, 4 * g + v, 64));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          if constexpr (kScaled) {
            const floatx4 dot = mfma16<T>(w[s][z].get(0), x[s][i][0], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[z][i][v] = __builtin_fmaf(dot[v], d[v], acc[z][i][v]);
          } else {
#pragma unroll
            for (int c = 0; c < kChunk; ++c) acc[z][i] = mfma16<T>(w[s][z].get(c), x[s][i][c], acc[z][i]);
          }
        }
      }
      load(s, step + kFewWaves * (s + kDepth));
    }
  }
#pragma unroll
  for (int z = 0; z < G; ++z)
#pragma unroll
    for (int i = 0; i < NB; ++i) part[wave][z][i][lane] = acc[z][i];
  __syncthreads();
  if (wave >= NB) return;
  float sum[2][4];
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    floatx4 s = part[0][z < G ? z : 0][wave][lane];
#pragma unroll
    for (int u = 1; u < kFewWaves; ++u) s = s + part[u][z < G ? z : 0][wave][lane];
#pragma unroll
    for (int v = 0; v < 4; ++v) sum[z][v] = s[v];
  }
  finish<T, GATED, 4>(p, row0 + 16 * wave + r, col0 + 4 * g, sum[0], sum[1]);
}

// ------------------------------------------------------------------ launches

inline bool on16(const void* p, uint64_t ld, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0;
}

template <class T, class W, bool GATED>
hipError_t launch_linear_form(const Linear& p, hipStream_t st) {
  constexpr unsigned kCus = 256;
  auto count = [](unsigned n, unsigned by) { return (n + by - 1) / by; };
  // n m <= 2^32: at most 2^24 + 2^21 workgroups of any form.
  constexpr unsigned kSmallCols = GATED ? 32 : 64, kLargeCols = GATED ? 64 : 128;
  if (p.n <= 64 || count(p.n, 64) * count(p.m, kSmallCols) < kCus / 2) {
    const unsigned nb = p.n <= 16 ? 1 : p.n <= 32 ? 2 : 4;
    const unsigned groups = count(p.n, 16 * nb) * count(p.m, 16);
    if (nb == 1)
      linear_few_kernel<T, W, GATED, 1><<<groups, 64 * kFewWaves, 0, st>>>(p);
    else if (nb == 2)
      linear_few_kernel<T, W, GATED, 2><<<groups, 64 * kFewWaves, 0, st>>>(p);
    else
      linear_few_kernel<T, W, GATED, 4><<<groups, 64 * kFewWaves, 0, st>>>(p);
    return hipGetLastError();
  }
  // Straight to LDS where rows lie on 16 bytes, hold whole chunks, and a tile's rows within 2 GiB.
  bool dma = on16(p.x, p.ldx, sizeof(T)) && p.k % kPer16<T> == 0 && p.ldx < 1u << 20;
  if constexpr (__is_same(T, W)) {
    dma = dma && p.ldw < 1u << 20;
    for (int z = 0; z < (GATED ? 2 : 1); ++z) dma = dma && on16(p.w[z], p.ldw, sizeof(T));
  }
  const bool large = count(p.n, 128) * count(p.m, kLargeCols) >= kCus;
  const unsigned tiles = large ? count(p.n, 128) * count(p.m, kLargeCols) : count(p.n, 64) * count(p.m, kSmallCols);
  if (large) {
    if (dma)
      linear_tile_kernel<T, W, GATED, true, 128, 128><<<tiles, 256, 0, st>>>(p);
    else
      linear_tile_kernel<T, W, GATED, false, 128, 128><<<tiles, 256, 0, st>>>(p);
  } else {
    if (dma)
      linear_tile_kernel<T, W, GATED, true, 64, 64><<<tiles, 256, 0, st>>>(p);
    else
      linear_tile_kernel<T, W, GATED, false, 64, 64><<<tiles, 256, 0, st>>>(p);
  }
  return hipGetLastError();
}

// Every weight type of activations T (the record's types have been checked).
template <class T>
hipError_t launch_linear_type(const Linear& p, unsigned weight_type, bool gated, hipStream_t st) {
  auto go = [&](auto w) {
    using W = decltype(w);
    return gated ? launch_linear_form<T, W, true>(p, st) : launch_linear_form<T, W, false>(p, st);
  };
  if (weight_type == EG2_TYPE_Q8_0) return go(Q8{});
  if constexpr (__is_same(T, float)) {
    if (weight_type == EG2_TYPE_F16) return go(_Float16{});
    if (weight_type == EG2_TYPE_BF16) return go(__bf16{});
  }
  return go(T{});
}

}  // namespace block
}  // namespace eg2
