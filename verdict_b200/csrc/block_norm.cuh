// The step between two blocks of a decoder: the norm after a block, its gate,
// the scaled residual add and the norm before the next block, in one pass.
//   u  = y * rsqrt(mean(y^2) + eps) * post_gain      (or u = y without a gain)
//   h' = residual_scale * h + block_scale * gate * u
//   z  = h' * rsqrt(mean(h'^2) + eps) * pre_gain     (as 16 bits, fp32, or
//        e4m3 with a scale per 128 columns: the next product's operand)
// Statistics, h' and z stay in fp32 until each is stored once; z is formed
// from h' before h' is rounded to the residual's type.
//
// Bound by memory: y and h are read once, h' and z written once.  One CTA per
// row; a thread keeps NV chunks of four columns in registers through both
// norms, so nothing is read twice.  Four columns make every access of a warp
// contiguous, the gains' (fp32, read by every row) among them: eight kept the
// L1 busy 74 % of the time.
// 16384 x 4096, y bf16, residual fp32, 8-bit z: 134 us, 5.5 TB/s, 0.84 of the
// measured copy rate; what is left is the two reductions' latency at four CTAs
// on an SM (five at 48 registers were no faster).
#pragma once

#include "row_io.cuh"

namespace vd {

enum NormOut : int { kNormOutNone = 0, kNormOutF16, kNormOutBF16, kNormOutF32, kNormOutF8 };

struct BlockNormParams {
  const void* y;         // null: no block output (u = 0)
  const void* h;         // null: no residual
  const float* post;     // null: no norm after the block
  const void* gate;      // null: 1
  int gate_f32;          // gate in fp32, else in y's type
  int64_t gate_row, gate_col;  // element strides; 0 broadcasts
  const float* pre;      // gains of z; null: no z
  void* h_out;           // null: h' is not stored
  void* z;
  float* z_scale;
  int64_t ld_y, ld_h, ld_h_out, ld_z, ld_scale;
  int cols;
  int out;               // NormOut
  float residual_scale, block_scale, eps, gain_add;
};

// Sum over the CTA; every thread gets it.  `slots`: one float per warp, used
// by one reduction only.
__device__ __forceinline__ float cta_sum(float x, float* slots) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = x;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  float s = (threadIdx.x & 31) < warps ? slots[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <bool FULL, class T>
__device__ __forceinline__ void columns4(const T* p, int n, float (&v)[4]) {
  Chunk4<T> c;
  if (FULL) c.load(p);
  else c.load_gap(p, n);
  c.get(v);
}

// FULL: every thread has NV whole, aligned chunks (cols = 4 NV blockDim.x);
// otherwise element by element, a thread's four 32 columns apart.
template <class TY, class TH, int NV, bool FULL>
__global__ void block_norm_kernel(BlockNormParams p) {
  __shared__ float slots[2][32];
  const int64_t row = blockIdx.x;
  const int step = blockDim.x * 4;
  const int col0 = FULL ? threadIdx.x * 4 : (threadIdx.x >> 5) * 128 + (threadIdx.x & 31);
  constexpr int GAP = FULL ? 1 : kGap;
  Chunk4<TY> yr[NV];
  Chunk4<TH> hr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) yr[i].zero(), hr[i].zero();
  if (p.y) {
    const TY* y = static_cast<const TY*>(p.y) + row * p.ld_y + col0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (FULL) yr[i].load(y + i * step);
      else yr[i].load_gap(y + i * step, p.cols - col0 - i * step);
    }
  }
  if (p.h) {
    const TH* h = static_cast<const TH*>(p.h) + row * p.ld_h + col0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (FULL) hr[i].load(h + i * step);
      else hr[i].load_gap(h + i * step, p.cols - col0 - i * step);
    }
  }
  const float inv_cols = 1.0f / static_cast<float>(p.cols);
  float u[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) yr[i].get(u[i]);
  if (p.post) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = fmaf(u[i][j], u[i][j], ss);
    const float rstd = rsqrtf(cta_sum(ss, slots[0]) * inv_cols + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float g[4];
      columns4<FULL>(p.post + col0 + i * step, p.cols - col0 - i * step, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) u[i][j] = u[i][j] * rstd * (g[j] + p.gain_add);
    }
  }
  float row_gate = p.block_scale;
  if (p.gate) {
    if (p.gate_col == 0) {
      row_gate *= p.gate_f32 ? static_cast<const float*>(p.gate)[row * p.gate_row]
                             : Elem<TY>::to(static_cast<const TY*>(p.gate)[row * p.gate_row]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t at = row * p.gate_row + col0 + i * step;
        const int n = p.cols - col0 - i * step;
        float g[4];
        if (p.gate_f32) columns4<FULL>(static_cast<const float*>(p.gate) + at, n, g);
        else columns4<FULL>(static_cast<const TY*>(p.gate) + at, n, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[i][j] *= g[j];
      }
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float h[4];
    hr[i].get(h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[i][j] = p.residual_scale * h[j] + row_gate * u[i][j];
      ss = fmaf(u[i][j], u[i][j], ss);
    }
  }
  if (p.h_out) {
    TH* o = static_cast<TH*>(p.h_out) + row * p.ld_h_out + col0;
#pragma unroll
    for (int i = 0; i < NV; ++i) store4<FULL>(o + i * step, u[i], p.cols - col0 - i * step);
  }
  if (p.out == kNormOutNone) return;
  const float rstd = rsqrtf(cta_sum(ss, slots[1]) * inv_cols + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float g[4];
    columns4<FULL>(p.pre + col0 + i * step, p.cols - col0 - i * step, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) u[i][j] = u[i][j] * rstd * (g[j] + p.gain_add);
  }
  const int64_t at = row * p.ld_z + col0;
  if (p.out == kNormOutF8) {
    // A warp holds NV 128-column blocks; lane i forms the scales of block i
    // (two divisions a warp, not two a block).
    const int lane = threadIdx.x & 31;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (FULL || col0 + i * step + j * GAP < p.cols) m = max(m, magnitude_bits(u[i][j]));
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == i) mine = m;
    }
    const F8Scale s = f8_scale(mine);
    const int block0 = col0 / kF8Block;  // the warp's first
    if (lane < NV && (block0 + lane * (step / kF8Block)) * kF8Block < p.cols)
      p.z_scale[row * p.ld_scale + block0 + lane * (step / kF8Block)] = s.scale;
    uint8_t* o = static_cast<uint8_t*>(p.z) + at;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t q = f8_pack4(u[i], __shfl_sync(0xffffffffu, s.inv, i));
      const int n = p.cols - col0 - i * step;
      if (FULL) {
        *reinterpret_cast<uint32_t*>(o + i * step) = q;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j * GAP < n) o[i * step + j * GAP] = static_cast<uint8_t>(q >> (8 * j));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int n = p.cols - col0 - i * step;
    if (p.out == kNormOutF16) store4<FULL>(static_cast<__half*>(p.z) + at + i * step, u[i], n);
    else if (p.out == kNormOutBF16) store4<FULL>(static_cast<__nv_bfloat16*>(p.z) + at + i * step, u[i], n);
    else store4<FULL>(static_cast<float*>(p.z) + at + i * step, u[i], n);
  }
}

}  // namespace vd
