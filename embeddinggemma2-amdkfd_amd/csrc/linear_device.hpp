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
template <class T, class W>
struct OtherThanQ8 {
  typedef W type;
};
template <class T>
struct OtherThanQ8<T, Q8> {
  typedef T type;
};

// Loads and stores at any alignment of the values (one instruction: the global ones need none).
template <class V>
__device__ __forceinline__ V load_any(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <class V>
__device__ __forceinline__ void store_any(void* p, const V& v) {
  __builtin_memcpy(p, &v, sizeof(V));
}

// The W values [k, k + kPer16<T>) of a row as they lie, zeros from `end` on, and as 16
// bytes of T. (Converted where they are used, not where they are loaded, which would wait for them.)
template <class T, class W>
struct Chunk {
  static constexpr int N = kPer16<T>;
  struct Raw {
    W v[N];
  };
  Raw raw;
  __device__ __forceinline__ void load(const W* row, unsigned k) { raw = load_any<Raw>(row + k); }
  __device__ __forceinline__ void load(const W* row, unsigned k, unsigned end) {
    if (k + N <= end) {
      load(row, k);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) raw.v[e] = row[min(k + e, end - 1)];  // all on their way at once
#pragma unroll
      for (int e = 0; e < N; ++e) raw.v[e] = k + e < end ? raw.v[e] : (W)0.0f;
    }
  }
  __device__ __forceinline__ uintx4 get() const {
    if constexpr (__is_same(T, W)) {
      return __builtin_bit_cast(uintx4, raw);
    } else {
      union {
        uintx4 all;
        T v[N];
      } r;
#pragma unroll
      for (int e = 0; e < N; ++e) r.v[e] = (T)to_float(raw.v[e]);
      return r.all;
    }
  }
};

// The biases of COLS columns from `col` on (the last one past the end; 0 where there is none).
template <int COLS>
struct Biases {
  float v[COLS];
  __device__ __forceinline__ Biases(const float* bias, unsigned col, unsigned m) {
#pragma unroll
    for (int e = 0; e < COLS; ++e) v[e] = bias ? bias[min(col + e, m - 1)] : 0.0f;
  }
};

// The output of a lane: COLS consecutive columns of one row, from their sums.
template <class T, bool GATED, unsigned ACT, int COLS>
__device__ __forceinline__ void finish(const Linear& p, unsigned row, unsigned col, const float (&a)[COLS],
                                       const float (&b)[COLS], const Biases<COLS>& a_bias, const Biases<COLS>& b_bias) {
  if (row >= p.n || col >= p.m) return;
  constexpr int N = COLS % kPer16<T> == 0 ? kPer16<T> : 4;  // values of a store
  static_assert(COLS % 4 == 0, "");
  struct Some {
    T v[N];
  };
  T* y = static_cast<T*>(p.y) + row * p.ldy + col;
  const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr + col : nullptr;
  float z[COLS];
#pragma unroll
  for (int e = 0; e < COLS; ++e) {
    z[e] = activate<ACT>(a[e] + a_bias.v[e]);
    if constexpr (GATED) z[e] = z[e] * (b[e] + b_bias.v[e]);
  }
  if (col + COLS <= p.m) {
#pragma unroll
    for (int c = 0; c < COLS; c += N) {
      if constexpr (!GATED)
        if (r) {
          const Some s = load_any<Some>(r + c);
#pragma unroll
          for (int e = 0; e < N; ++e) z[c + e] = z[c + e] + to_float(s.v[e]);
        }
      Some out;
#pragma unroll
      for (int e = 0; e < N; ++e) out.v[e] = (T)z[c + e];
      store_any(y + c, out);
    }
  } else {
    if constexpr (!GATED)
      if (r) {  // all on their way at once
        T v[COLS];
#pragma unroll
        for (int e = 0; e < COLS; ++e) v[e] = r[min((unsigned)e, p.m - 1 - col)];
#pragma unroll
        for (int e = 0; e < COLS; ++e) z[e] = z[e] + to_float(v[e]);
      }
#pragma unroll
    for (int e = 0; e < COLS; ++e)
      if (col + e < p.m) y[e] = (T)z[e];
  }
}

// A piece of a Q8_0 block on its way: N values from value `at` (a multiple of N) on,
// N / 4 + 1 aligned words from byte `at` of the block, rounded down to 4, on. The
// block lies on 2 bytes: `odd` is at 2 mod 4. Then the values are the words but the
// first, else they start 2 bytes in; the first word also holds the scale if at is 0.
// (Loads that are not on 4 bytes take several times as long: 64 cycles each in the
// few-row form.) The first word may begin 2 bytes before the block, the last
// end 2 behind it; with `edge` (a matrix's first or last row, or rows that overlap) no byte
// outside the block is read.
template <int N>
struct Q8Piece {
  uint32_t w[N / 4 + 1];
  bool odd;
  __device__ __forceinline__ void load(const unsigned char* block, unsigned at, bool edge) {
    odd = (reinterpret_cast<uintptr_t>(block) & 2) != 0;
    const unsigned char* from = block + at - (odd ? 2 : 0);
    if (!edge) {
#pragma unroll
      for (int i = 0; i <= N / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(from)[i];
    } else {  // the half word at one end alone
      const uint32_t half = *reinterpret_cast<const uint16_t*>(block + at + (odd ? 0 : N));
      const uint32_t* words = reinterpret_cast<const uint32_t*>(from) + (odd ? 1 : 0);
      uint32_t v[N / 4];
#pragma unroll
      for (int i = 0; i < N / 4; ++i) v[i] = words[i];
#pragma unroll
      for (int i = 0; i <= N / 4; ++i) w[i] = odd ? (i == 0 ? half << 16 : v[i == 0 ? 0 : i - 1]) : (i == N / 4 ? half : v[i == N / 4 ? 0 : i]);
    }
  }
  __device__ __forceinline__ float scale() const { return fp16_bits_to_fp32(odd ? w[0] >> 16 : w[0] & 0xffffu); }
  __device__ __forceinline__ float value(int e) const {
    const uint32_t four = odd ? w[e / 4 + 1] : __builtin_amdgcn_alignbyte(w[e / 4 + 1], w[e / 4], 2);
    return (float)(int8_t)(four >> (8 * (e % 4)));
  }
};

// ------------------------------------------------------------------ tiles
//
// BM rows of x times BN rows of the weights (of a gated pair BN / 2 of each
// matrix) per workgroup of WM x WN waves, each 16 x 16 blocks over its part, or
// of WK times as many, each share over every WK-th slice of k, added at the
// end. Slices of 128 bytes of every row go through NBUF LDS buffers, all but one
// on their way while one is multiplied. The 16-byte chunks of a row are swizzled
// so that no read waits for LDS's banks (counted: 0 conflicts). Rows on 4 bytes go
// straight to LDS (DMA), others and what has to be decoded through registers.
//
// Bound: large products by the matrix units. 4096 x 2048 x 8192 bf16 with bias
// and GELU takes 123 to 127 us, 1080 to 1120 TFLOP/s, of which 55 % of the cycles the matrix units work
// (a product of 8192^3 by the installed library, no epilogue: 1244 TFLOP/s; its own
// of this size, no epilogue: 103 us). Products that leave most CUs one or two tiles, by how fast a
// CU takes slices from L2 (22 to 26 bytes a cycle): 2048 x 768 x 1152 gated bf16 14 us.
// Deeper buffers (3, 4 slices of 128 or 256 rows) and tiles of 128 x 192 where those
// would save a round of workgroups measured within 3 % of these.
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

template <class T, class W, bool GATED, bool DMA, int BM, int BN, int WM, int WN, int WK, int NBUF>
__global__ void __launch_bounds__(64 * WM * WN * WK) linear_tile_kernel(Linear p) {
  constexpr int G = GATED ? 2 : 1, COLS = BN / G;  // columns of y
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;  // of a share of k
  constexpr int IB = BM / 16 / WM, JB = BN / 16 / WN, JBG = JB / G;
  constexpr int N = kPer16<T>, BK = kChunks * N;  // values per chunk and slice
  constexpr bool kScaled = kIsQ8<W> && !__is_same(T, float);
  constexpr bool kDmaW = DMA && __is_same(T, W);
  constexpr int kBlocks = BK / 32;  // Q8_0 blocks of a slice
  static_assert(NBUF == 2 || kDmaW, "registers hold one slice");
  struct Lds {
    alignas(16) unsigned char x[NBUF][BM * kRowBytes];
    alignas(16) unsigned char w[NBUF][BN * kRowBytes];
    alignas(16) float d[kScaled ? 2 : 1][kScaled ? kBlocks * BN : 4];
  };
  __shared__ union {
    Lds share[WK];
    floatx4 part[WK > 1 ? WK - 1 : 1][WK > 1 ? WAVES * IB * JB : 1][64];
  } all;
  const int wk = WK > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS) : 0;
  const int tid = WK > 1 ? threadIdx.x % THREADS : threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15, wm = wave / WN, wn = wave % WN;
  Lds& lds = all.share[wk];

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
  constexpr int kXItems = BM * kChunks / THREADS;
  constexpr int kWItems = kIsQ8<W> ? (BN * BK / 16 + THREADS - 1) / THREADS : BN * kChunks / THREADS;
  typedef Chunk<T, typename OtherThanQ8<T, W>::type> WChunk;
  Chunk<T, T> xv[DMA ? 1 : kXItems];
  WChunk wv[kIsQ8<W> || kDmaW ? 1 : kWItems];
  Q8Piece<16> qv[kIsQ8<W> ? kWItems : 1];
  uint32_t qd[kIsQ8<W> && !kScaled ? kWItems : 1];
  const bool edge = col0 == 0 || col0 + COLS >= p.m || p.ldw < p.k;
  auto load = [&](unsigned k0) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < kXItems; ++i) {
        const int item = tid + THREADS * i, rr = item / kChunks, c = item % kChunks;
        xv[i].load(xrows + min(row0 + rr, p.n - 1) * p.ldx, k0 + N * c, p.k);
      }
    }
    if constexpr (kIsQ8<W>) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + THREADS * i, rr = item / (BK / 16), part = item % (BK / 16);
        const unsigned k = k0 + 16 * part;
        qv[i] = Q8Piece<16>{};
        if constexpr (!kScaled) qd[i] = 0;
        if (rr < BN && k < p.k) {
          const unsigned char* b = weight_base(rr) + (size_t)(k / 32) * kBlockBytes;
          qv[i].load(b, k % 32, edge);
          if constexpr (!kScaled) qd[i] = *reinterpret_cast<const uint16_t*>(b);
        }
      }
    } else if constexpr (!kDmaW) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + THREADS * i, rr = item / kChunks, c = item % kChunks;
        wv[i].load(reinterpret_cast<const W*>(weight_base(rr)), k0 + N * c, p.k);
      }
    }
  };
  auto put = [&](int buf) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < kXItems; ++i) {
        const int item = tid + THREADS * i, rr = item / kChunks, c = item % kChunks;
        *reinterpret_cast<uintx4*>(lds.x[buf] + rr * kRowBytes + 16 * (c ^ (rr & 7))) = xv[i].get();
      }
    }
    if constexpr (kIsQ8<W>) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + THREADS * i, rr = item / (BK / 16), part = item % (BK / 16);
        if (rr >= BN) continue;
        float d = 1.0f;
        if constexpr (kScaled) {
          if (part % 2 == 0) lds.d[buf][part / 2 * BN + rr] = qv[i].scale();
        } else {
          d = fp16_bits_to_fp32(qd[i]);
        }
#pragma unroll
        for (int c = 0; c < 16 / N; ++c) {
          union {
            uintx4 all;
            T v[N];
          } o;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float q = qv[i].value(N * c + e);
            o.v[e] = (T)(kScaled ? q : d * q);
          }
          *reinterpret_cast<uintx4*>(lds.w[buf] + rr * kRowBytes +
                                     16 * ((16 / N * part + c) ^ weight_key<JBG>(rr))) = o.all;
        }
      }
    } else if constexpr (!kDmaW) {
#pragma unroll
      for (int i = 0; i < kWItems; ++i) {
        const int item = tid + THREADS * i, rr = item / kChunks, c = item % kChunks;
        *reinterpret_cast<uintx4*>(lds.w[buf] + rr * kRowBytes + 16 * (c ^ weight_key<JBG>(rr))) = wv[i].get();
      }
    }
  };
  // The same straight to LDS: a wave's load fills 1 KB, 8 rows, lane l the chunk
  // l % 8 of row l / 8; the swizzle is in which chunk it reads. In the last slice
  // chunks that pass k go through registers, zeros from k on.
  constexpr int kXDma = DMA ? BM / 8 / WAVES : 0, kWDma = kDmaW ? BN / 8 / WAVES : 0;  // per wave
  uint32_t xoff[DMA ? kXDma : 1], woff[kDmaW ? kWDma : 1];
  const unsigned char *xbase = nullptr, *wbase[G] = {};
  if constexpr (DMA) {
    xbase = reinterpret_cast<const unsigned char*>(xrows + row0 * p.ldx);
#pragma unroll
    for (int i = 0; i < kXDma; ++i) {
      const unsigned rr = 8 * (kXDma * wave + i) + (lane >> 3);
      xoff[i] = (uint32_t)((min(row0 + rr, p.n - 1) - row0) * p.ldx * sizeof(T)) + 16 * ((lane & 7) ^ (lane >> 3));
    }
  }
  if constexpr (kDmaW) {
#pragma unroll
    for (int z = 0; z < G; ++z) wbase[z] = weight_base(z * COLS);
#pragma unroll
    for (int i = 0; i < kWDma; ++i) {
      const int rr = 8 * (kWDma * wave + i) + (lane >> 3);
      woff[i] = (uint32_t)(weight_base(rr) - weight_base(GATED && rr >= COLS ? COLS : 0)) + 16 * ((lane & 7) ^ weight_key<JBG>(rr));
    }
  }
  auto lds_address = [](const void* q) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)static_cast<const unsigned char*>(q);
  };
  const uint32_t lds_x = lds_address(lds.x[0]), lds_w = lds_address(lds.w[0]);
  auto dma = [&](int buf, unsigned k0) {
    const uint32_t to_x = lds_x + buf * BM * kRowBytes + 1024 * kXDma * wave, to_w = lds_w + buf * BN * kRowBytes + 1024 * kWDma * wave;
    if (k0 + BK <= p.k) {  // uniform; straight-line code
      if constexpr (DMA) {
#pragma unroll
        for (int i = 0; i < kXDma; ++i) dma16(xbase + k0 * sizeof(T), xoff[i], to_x + 1024 * i);
      }
      if constexpr (kDmaW) {
#pragma unroll
        for (int i = 0; i < kWDma; ++i)
          dma16(wbase[GATED && 8 * (kWDma * wave + i) >= COLS] + k0 * sizeof(T), woff[i], to_w + 1024 * i);
      }
      return;
    }
    // Chunk c of a row as far as it lies before k: straight to LDS if it does as a whole.
    auto whole = [&](unsigned chunk) { return k0 + N * chunk + N <= p.k; };
    auto part = [&](const unsigned char* base, uint32_t off, unsigned chunk) {
      Chunk<T, T> c;
      c.load(reinterpret_cast<const T*>(base + off - 16 * chunk), k0 + N * chunk, p.k);
      return c;
    };
    const unsigned xchunk = (lane & 7) ^ (lane >> 3);
    auto wchunk = [&](int i) { return (lane & 7) ^ weight_key<JBG>(8 * (kWDma * wave + i) + (lane >> 3)); };
    auto wfrom = [&](int i) { return wbase[GATED && 8 * (kWDma * wave + i) >= COLS]; };
    Chunk<T, T> xs[DMA ? kXDma : 1], ws[kDmaW ? kWDma : 1];
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < kXDma; ++i) {
        if (whole(xchunk))
          dma16(xbase + k0 * sizeof(T), xoff[i], to_x + 1024 * i);
        else
          xs[i] = part(xbase, xoff[i], xchunk);
      }
    }
    if constexpr (kDmaW) {
#pragma unroll
      for (int i = 0; i < kWDma; ++i) {
        if (whole(wchunk(i)))
          dma16(wfrom(i) + k0 * sizeof(T), woff[i], to_w + 1024 * i);
        else
          ws[i] = part(wfrom(i), woff[i], wchunk(i));
      }
    }
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < kXDma; ++i)
        if (!whole(xchunk)) *reinterpret_cast<uintx4*>(lds.x[buf] + 1024 * (kXDma * wave + i) + 16 * lane) = xs[i].get();
    }
    if constexpr (kDmaW) {
#pragma unroll
      for (int i = 0; i < kWDma; ++i)
        if (!whole(wchunk(i))) *reinterpret_cast<uintx4*>(lds.w[buf] + 1024 * (kWDma * wave + i) + 16 * lane) = ws[i].get();
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
        if constexpr (kScaled) __builtin_amdgcn_sched_barrier(0);  // the dots of a block of columns at a time
      }
    }
  };

  // A share takes every WK-th slice.
  const unsigned slices = (p.k + BK - 1) / BK, turns = (slices + WK - 1) / WK;
#pragma unroll
  for (int i = 0; i < NBUF - 1; ++i)
    if (wk + i * WK < slices) dma(i, (wk + i * WK) * BK);
  load(wk * BK);
  put(0);
  int buf = 0;
  for (unsigned turn = 0; turn < turns; ++turn) {
    const unsigned s = wk + turn * WK;
    // The slice is in its buffer (those behind it may be on their way: a slice is
    // kXDma + kWDma loads of a wave, or drained), and the buffer before it has been read.
    if constexpr (DMA) {
      if (NBUF > 2 && s + (NBUF - 2) * WK < slices)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 2) * (kXDma + kWDma)) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
    if (s + (NBUF - 1) * WK < slices) dma(buf == 0 ? NBUF - 1 : buf - 1, (s + (NBUF - 1) * WK) * BK);
    if (s + WK < slices) load((s + WK) * BK);
    if (s < slices) multiply(buf);
    if (s + WK < slices) put(buf ^ 1);  // of two
    buf = buf + 1 < NBUF ? buf + 1 : 0;
  }
  if constexpr (WK > 1) {
    __syncthreads();
    if (wk > 0) {
#pragma unroll
      for (int i = 0; i < IB; ++i)
#pragma unroll
        for (int j = 0; j < JB; ++j) all.part[wk - 1][(wave * IB + i) * JB + j][lane] = acc[i][j];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int i = 0; i < IB; ++i)
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int w = 1; w < WK; ++w) acc[i][j] = acc[i][j] + all.part[w - 1][(wave * IB + i) * JB + j][lane];
  }
  const unsigned col = col0 + wn * (16 * JBG) + 4 * JBG * g;
  const Biases<4 * JBG> a_bias(p.bias[0], col, p.m), b_bias(GATED ? p.bias[1] : nullptr, col, p.m);
  with_activation(p.act, [&](auto act) {
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
      finish<T, GATED, decltype(act)::value>(p, row0 + 16 * (IB * wm + i) + r, col, a, b, a_bias, b_bias);
    }
  });
}

// ------------------------------------------------------------------ few rows
//
// 16 NB rows of x times 16 rows of the weights (of a gated pair of each
// matrix) per workgroup of eight waves, which take an eighth of k's steps each
// and add their sums through LDS: the weights come straight from memory in
// the order of the operand, and every workgroup's chain is an eighth of k.
//
// Bound: the weights' bytes once there are some (1 x 4096 x 8192 bf16: 13.5 us, 5.0
// TB/s; 4 x 2048 x 8192 gated Q8_0: 15 us, 2.4 TB/s, where unpacking the blocks counts as well:
// 40 VALU instructions a step), below that the launch and one chain of loads (1 x 768 x 768:
// 3.7 us).
constexpr int kFewWaves = 8;

template <class T, class W, bool EDGE>
struct FewWeights {  // a step of a row: 32 values (fp32: two chunks of 16)
  static constexpr int kChunk = __is_same(T, float) ? 2 : 1;
  Chunk<T, W> v[kChunk];
  __device__ __forceinline__ void load(const unsigned char* row, unsigned k, unsigned g) {
#pragma unroll
    for (int c = 0; c < kChunk; ++c) v[c].load(reinterpret_cast<const W*>(row), k + kPer16<T> * (4 * c + g));
  }
  __device__ __forceinline__ void load(const unsigned char* row, unsigned k, unsigned g, unsigned end) {
#pragma unroll
    for (int c = 0; c < kChunk; ++c) v[c].load(reinterpret_cast<const W*>(row), k + kPer16<T> * (4 * c + g), end);
  }
  __device__ __forceinline__ float scale() const { return 1.0f; }
  __device__ __forceinline__ uintx4 get(int c, float) const { return v[c].get(); }
};
template <class T, bool EDGE>
struct FewWeights<T, Q8, EDGE> {
  static constexpr int N = kPer16<T>;
  Q8Piece<N> q[N == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const unsigned char* row, unsigned k, unsigned g) {
#pragma unroll
    for (int c = 0; c < (N == 4 ? 2 : 1); ++c) q[c].load(row + (size_t)(k / 32) * kBlockBytes, 16 * c + N * g, EDGE);
  }
  __device__ __forceinline__ void load(const unsigned char*, unsigned, unsigned, unsigned) {}  // k is a multiple of 32
  // The block's scale, which the first lane of its four loaded.
  __device__ __forceinline__ float scale() const { return __shfl(q[0].scale(), threadIdx.x & 15, 64); }
  __device__ __forceinline__ uintx4 get(int c, float d) const {
    union {
      uintx4 all;
      T v[N];
    } o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float f = q[c].value(e);
      o.v[e] = (T)(N == 4 ? d * f : f);
    }
    return o.all;
  }
};

template <class T, class W, bool GATED, int NB>
__global__ void __launch_bounds__(64 * kFewWaves) linear_few_kernel(Linear p) {
  constexpr int G = GATED ? 2 : 1, kChunk = __is_same(T, float) ? 2 : 1;
  constexpr bool kScaled = kIsQ8<W> && !__is_same(T, float);
  // Steps on their way: of a pair two, so that its registers leave room for as many
  // waves as one matrix has with four (4 x 2048 x 8192 Q8_0: 16.7 us, 18.9 with four).
  constexpr int kDepth = NB * G >= 4 || GATED ? 2 : 4;
  constexpr int kSlots = GATED && NB == 1 ? 3 : kDepth;  // all the steps of a wave that has no more, at once (1 x 768 x 1152 pairs 8 % less)
  // A wave takes a run of steps, or every eighth: runs keep a row's memory together (1 x 4096 x 4096 fp32
  // 13.9 us, 16.2 by eighths; 1 x 4096 x 8192 bf16 13.5, 14.2), while Q8_0 blocks share their cache lines with the
  // next steps, which eighths fetch at the same time (4 x 2048 x 8192 gated 16.9, 17.1 by runs; 1 x 4096 x 4096 12.1, 12.2).
  constexpr bool kRuns = !kIsQ8<W> && !GATED;
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
  auto run = [&](auto edge) {
    constexpr bool EDGE = decltype(edge)::value != 0;
    FewWeights<T, W, EDGE> w[kSlots][G];
    Chunk<T, T> x[kSlots][NB][kChunk];
    auto multiply = [&](int slot) {
#pragma unroll
      for (int z = 0; z < G; ++z) {
        const float d = w[slot][z].scale();  // of column r
        uintx4 a[kChunk];
#pragma unroll
        for (int c = 0; c < kChunk; ++c) a[c] = w[slot][z].get(c, d);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          if constexpr (kScaled) {  // rows 4 g .. of column r
            const floatx4 dot = mfma16<T>(x[slot][i][0].get(), a[0], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[z][i][v] = __builtin_fmaf(dot[v], d, acc[z][i][v]);
          } else {  // columns 4 g .. of row r
#pragma unroll
            for (int c = 0; c < kChunk; ++c) acc[z][i] = mfma16<T>(a[c], x[slot][i][c].get(), acc[z][i]);
          }
        }
      }
    };
    // The wave's whole steps. The loop's loads stand in no branch (past the last
    // step it is loaded again), so that a step waits for its own alone.
    const unsigned steps = p.k / 32, begin = kRuns ? steps * wave / kFewWaves : wave;
    const unsigned mine = kRuns ? steps * (wave + 1) / kFewWaves - begin : steps > begin ? (steps - begin + kFewWaves - 1) / kFewWaves : 0;
    auto load = [&](int slot, unsigned n) {
      const unsigned k = 32 * (begin + (kRuns ? 1 : kFewWaves) * min(n, mine - 1));
#pragma unroll
      for (int z = 0; z < G; ++z) w[slot][z].load(wrow[z], k, g);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int c = 0; c < kChunk; ++c) x[slot][i][c].load(xrow[i], k + kPer16<T> * (4 * c + g));
    };
    if (mine > kSlots) {
#pragma unroll
      for (int s = 0; s < kDepth; ++s) load(s, s);
      unsigned n = 0;
      for (; n + kDepth < mine; n += kDepth) {
#pragma unroll
        for (int s = 0; s < kDepth; ++s) {
          multiply(s);
          load(s, n + kDepth + s);
        }
      }
#pragma unroll
      for (int s = 0; s < kDepth; ++s)
        if (n + s < mine) multiply(s);
    } else {
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (s < (int)mine) load(s, s);
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (s < (int)mine) multiply(s);
    }
    // The values past the last whole step.
    if (p.k % 32 != 0 && wave == (int)(kRuns ? 0 : steps % kFewWaves)) {
#pragma unroll
      for (int z = 0; z < G; ++z) w[0][z].load(wrow[z], 32 * steps, g, p.k);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int c = 0; c < kChunk; ++c) x[0][i][c].load(xrow[i], 32 * steps + kPer16<T> * (4 * c + g), p.k);
      multiply(0);
    }
  };
  if (kIsQ8<W> && (col0 == 0 || col0 + 16 >= p.m || p.ldw < p.k))
    run(Const<1>{});
  else
    run(Const<0>{});
#pragma unroll
  for (int z = 0; z < G; ++z)
#pragma unroll
    for (int i = 0; i < NB; ++i) part[wave][z][i][lane] = acc[z][i];
  __syncthreads();
  if (wave >= NB) return;
  float sum[2][4];
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < kFewWaves; ++u) {
      const floatx4* from = part[u][z < G ? z : 0][wave];
      if constexpr (kScaled) {  // row r of column 4 g + v: lane 16 (r / 4) + column, element r % 4
#pragma unroll
        for (int v = 0; v < 4; ++v)
          s[v] = s[v] + reinterpret_cast<const float*>(from)[4 * (16 * (r >> 2) + 4 * g + v) + (r & 3)];
      } else {
        s = s + from[lane];
      }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) sum[z][v] = s[v];
  }
  const unsigned col = col0 + 4 * g;
  const Biases<4> a_bias(p.bias[0], col, p.m), b_bias(GATED ? p.bias[1] : nullptr, col, p.m);
  with_activation(p.act, [&](auto act) {
    finish<T, GATED, decltype(act)::value>(p, row0 + 16 * wave + r, col, sum[0], sum[1], a_bias, b_bias);
  });
}

// ------------------------------------------------------------------ launches

inline bool on4(const void* p, uint64_t ld, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld * size % 4 == 0 && ld < 1u << 21;
}

template <class T, class W, bool GATED>
hipError_t launch_linear_form(const Linear& p, hipStream_t st) {
  constexpr unsigned kCus = 256;
  constexpr bool k32 = __is_same(T, float);
  auto count = [](unsigned n, unsigned by) { return (n + by - 1) / by; };
  // n m <= 2^32: at most 2^22 workgroups of any form.
  auto few = [&](auto blocks) {
    constexpr int NB = decltype(blocks)::value;
    linear_few_kernel<T, W, GATED, NB><<<count(p.n, 16 * NB) * count(p.m, 16), 64 * kFewWaves, 0, st>>>(p);
    return hipGetLastError();
  };
  // Few rows, or so few blocks of 16 x 16 that they are one round of the GPU's
  // workgroups (two to a CU). Then more row blocks to a workgroup instead of more
  // rounds; fp32 goes on so where 16-bit types are better off with tiles. us by 1, 2 and 4 blocks and by
  // tiles: 45 x 768 x 1280 fp32 Q8_0 6.6, 8.4, 10.6, 20; 64 x 768 x 768 fp32 5.9, 7.6, 10.9, 17;
  // 300 x 768 x 768 fp32 15.8, 13.4, 12.1, 20.6; 32 x 2048 x 2048 bf16 6.8, 8.6, 9.6, 9.3;
  // 100 x 768 x 768 bf16 5.6, 5.2, 6.6, 6.6; 256 x 768 x 2304 bf16 16, 13.9, 14.1, 6.8.
  const uint64_t down16 = count(p.n, 16), across16 = count(p.m, 16);
  if (p.n <= 16 || down16 * across16 <= 2 * kCus) return few(Const<1>{});
  if (p.n <= 32 || (k32 && (down16 + 1) / 2 * across16 <= 2 * kCus)) return few(Const<2>{});
  if (k32 && (down16 + 3) / 4 * across16 <= 2 * kCus) return few(Const<4>{});
  constexpr unsigned kSmallCols = GATED ? 32 : 64, kLargeCols = GATED ? 64 : 128;
  // Straight to LDS where rows lie on 4 bytes (333 x 1152 x 768 f16: 7.5 us; 1151, whose rows do
  // not: 12.7), and a tile's within 2^31 bytes of each other.
  bool dma = on4(p.x, p.ldx, sizeof(T));
  if constexpr (__is_same(T, W))
    for (int z = 0; z < (GATED ? 2 : 1); ++z) dma = dma && on4(p.w[z], p.ldw, sizeof(T));
  constexpr bool kSame = __is_same(T, W);
  auto tiles = [&](auto size, auto wm, auto wn, auto wk, auto nbuf) {
    constexpr int B = decltype(size)::value, WM = decltype(wm)::value, WN = decltype(wn)::value, WK = decltype(wk)::value;
    constexpr int NBUF = kSame ? decltype(nbuf)::value : 2;
    const unsigned groups = count(p.n, B) * count(p.m, B / (GATED ? 2 : 1));
    if (dma)
      linear_tile_kernel<T, W, GATED, true, B, B, WM, WN, WK, NBUF><<<groups, 64 * WM * WN * WK, 0, st>>>(p);
    else
      linear_tile_kernel<T, W, GATED, false, B, B, WM, WN, WK, 2><<<groups, 64 * WM * WN * WK, 0, st>>>(p);
    return hipGetLastError();
  };
  // The largest tile of which there is one for every CU: it reads its operands least often. us by
  // tiles of 64, 128 and 256: 4096 x 2048 x 8192 bf16 250, 151, 128; 4096^3 223, 136, 120; gated 4096 x 2048 x 4096
  // 213, 137, 118; 2048 x 768 x 2304 f16 22, 18, 28; 1000 x 1150 x 2001 20, 30, 55; fp32 4096 x 2048 x 2048
  // 289, 252 (2048 x 768 x 1152, too few: 49, 58). 16-bit activations on Q8_0 stay with 64, whose scales
  // leave it registers (2048 x 768 x 2304 32, 50; 4096 x 2048 x 4096 169, 229).
  if constexpr (kSame && !k32)
    if (count(p.n, 256) * count(p.m, 2 * kLargeCols) >= kCus)
      return tiles(Const<256>{}, Const<2>{}, Const<4>{}, Const<1>{}, Const<2>{});
  if constexpr (!kIsQ8<W> || k32)
    if (count(p.n, 128) * count(p.m, kLargeCols) >= kCus)
      return tiles(Const<128>{}, Const<2>{}, Const<2>{}, Const<1>{}, Const<2>{});
  // Fewer tiles than CUs: four shares of k to a workgroup. us of 1, 2 and 4 shares: 512 x 768 x 768 bf16 7.3, 6.7, 6.9;
  // 128 x 2048 x 2048 12.9, 13.8, 11.9; 64 x 4096 x 4096 22, 24, 20; 300 x 768 x 1152 f16 Q8_0 13.6, 10.4, 9.1; with more
  // tiles one (1000 x 1150 x 2001 20.2, 19.6, 24.5), or two of fp32 (2048 x 768 x 1152 50, 47, 51).
  if (count(p.n, 64) * count(p.m, kSmallCols) < kCus)
    return tiles(Const<64>{}, Const<2>{}, Const<2>{}, Const<4>{}, Const<2>{});
  return tiles(Const<64>{}, Const<2>{}, Const<2>{}, Const<k32 ? 2 : 1>{}, Const<k32 ? 2 : 4>{});
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
