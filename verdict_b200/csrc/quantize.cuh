// Casts to 8-bit floating point (e4m3) with an fp32 scale per block.
//
// Activations: for each row and block of 128 columns, with v = x or
// v = act(gate) * x,
//   a = max(max |v|, 1e-30),  scale = a / 448,  q = e4m3(v * (448 / a)).
// A block that holds inf or NaN gets that as its scale, so that the whole
// block stands for non-finite values and the product's row shows it.
//
// Bound by memory: one read of x (and gate), one write of a byte per element.
// 16 lanes hold a block (8 elements each, one 16-byte load for 16-bit types),
// so its maximum is four shuffles; each thread takes kQuantUnroll blocks,
// whose loads are all issued before the first is used.  Two blocks a thread
// and six CTAs on an SM (40 registers) beat four and three (145 -> 90 us).
// Gated 8192 x 12288 fp16 with SiLU: 92 us, 5.5 TB/s, 0.84 of the measured
// copy rate; ungated fp32 8192 x 5120: 34 us, 6.3 TB/s.
#pragma once

#include "gemm.cuh"
#include "row_io.cuh"

namespace vd {

struct QuantizeParams {
  const void* x;
  const void* gate;
  int64_t ld_x, ld_gate, ld_q, ld_scale;
  uint32_t blocks, col_blocks;   // rows * col_blocks, ceil(cols / 128)
  FastDiv per_row;               // by col_blocks
  int cols, act;
  uint8_t* q;
  float* scale;
};

constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 2;

// What multiplies x: the gate's activation, SiLU apart from the others so that
// the common kernels stay short (fetching instructions was a fifth of their time).
enum QuantGate : int { kGateNone, kGateSilu, kGateAny };

template <int GATE>
__device__ __forceinline__ float gate_act(float g, int act) {
  if (GATE == kGateSilu) {  // one exp2 and one reciprocal; the reciprocal of inf is 0
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * r;
  }
  return apply_act(g, act);
}

// WHOLE: rows of x, gate and q that 8 elements divide and that are aligned for
// vector access.
template <class T, int GATE, bool WHOLE>
__global__ void __launch_bounds__(kQuantThreads, WHOLE && sizeof(T) == 2 ? 6 : 1) quantize_rows_kernel(QuantizeParams p) {
  const int lane16 = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (kQuantUnroll * kQuantThreads / 16) + (threadIdx.x >> 4);
  // A lane's eight columns of a block: neighbours, or 16 apart so that the
  // lanes' single accesses are contiguous.
  const int lane_col = WHOLE ? lane16 * 8 : lane16;
  constexpr int GAP = WHOLE ? 1 : 16;
  using Chunk = typename std::conditional<WHOLE, Chunk8<T>, T[8]>::type;
  Chunk xr[kQuantUnroll], gr[kQuantUnroll];
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    const uint32_t id = first + u * (kQuantThreads / 16);
    const uint32_t row = p.per_row(id);
    const int col = static_cast<int>(id - row * p.col_blocks) * kF8Block + lane_col;
    const int n = id < p.blocks ? p.cols - col : 0;
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x + col;
    const T* g = GATE != kGateNone ? static_cast<const T*>(p.gate) + row * p.ld_gate + col : nullptr;
    if constexpr (WHOLE) {
      xr[u].zero();
      if (GATE != kGateNone) gr[u].zero();
      if (n > 0) {
        xr[u].load(x);
        if (GATE != kGateNone) gr[u].load(g);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xr[u][j] = j * GAP < n ? x[j * GAP] : Elem<T>::from(0.0f);
        if (GATE != kGateNone) gr[u][j] = j * GAP < n ? g[j * GAP] : Elem<T>::from(0.0f);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    const uint32_t id = first + u * (kQuantThreads / 16);
    const uint32_t row = p.per_row(id);
    const uint32_t kb = id - row * p.col_blocks;
    const int col = static_cast<int>(kb) * kF8Block + lane_col;
    float v[8], g[8];
    if constexpr (WHOLE) {
      xr[u].get(v);
      if (GATE != kGateNone) gr[u].get(g);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = Elem<T>::to(xr[u][j]);
        if (GATE != kGateNone) g[j] = Elem<T>::to(gr[u][j]);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (GATE != kGateNone) v[j] *= gate_act<GATE>(g[j], p.act);
      m = max(m, magnitude_bits(v[j]));
    }
    const F8Scale s = f8_scale(max16(m));
    if (id < p.blocks) {
      if (lane16 == 0) p.scale[row * p.ld_scale + kb] = s.scale;
      uint8_t* q = p.q + row * p.ld_q + col;
      const uint2 w = f8_pack8(v, s.inv);
      if constexpr (WHOLE) {
        if (col < p.cols) *reinterpret_cast<uint2*>(q) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j * GAP < p.cols - col) q[j * GAP] = static_cast<uint8_t>((j < 4 ? w.x : w.y) >> ((j & 3) * 8));
      }
    }
  }
}

// Weights, once at load: a block is 128 rows x 128 columns, one CTA each.
template <class T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const T* __restrict__ w, int64_t ld_w, int rows, int cols,
                                                              uint8_t* __restrict__ q, int64_t ld_q,
                                                              float* __restrict__ scale, int64_t ld_scale) {
  __shared__ uint32_t warp_max[8];
  const int col = blockIdx.x * kF8Block + (threadIdx.x & 15) * 8;
  const int row0 = blockIdx.y * kF8Block + (threadIdx.x >> 4);
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + i * 16;
    Chunk8<T> c;
    c.zero();
    if (row < rows && col < cols) c.load_part(w + row * ld_w + col, cols - col);
    c.get(v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, magnitude_bits(v[i][j]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, warp_max[i]);
  const F8Scale s = f8_scale(m);
  if (threadIdx.x == 0) scale[blockIdx.y * ld_scale + blockIdx.x] = s.scale;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + i * 16;
    if (row < rows && col < cols) f8_store(q + row * ld_q + col, f8_pack8(v[i], s.inv), cols - col);
  }
}

}  // namespace vd
