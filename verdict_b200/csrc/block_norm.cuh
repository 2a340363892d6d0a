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
// row; a thread keeps NV chunks of eight columns in registers through both
// norms, so nothing is read twice.
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
  bool z_aligned;
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

__device__ __forceinline__ void gains8(const float* g, int n, bool aligned, float add, float (&v)[8]) {
  Chunk8<float> c;
  if (aligned && n >= 8) c.load(g);
  else c.load_part(g, n);
  c.get(v);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += add;
}

template <class TY, class TH, int NV, bool ALIGNED>
__global__ void block_norm_kernel(BlockNormParams p) {
  __shared__ float slots[2][32];
  const int64_t row = blockIdx.x;
  const int threads = blockDim.x;
  Chunk8<TY> yr[NV];
  Chunk8<TH> hr[NV];
  const TY* y = p.y ? static_cast<const TY*>(p.y) + row * p.ld_y : nullptr;
  const TH* h = p.h ? static_cast<const TH*>(p.h) + row * p.ld_h : nullptr;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (threadIdx.x + i * threads) * 8;
    const int n = p.cols - col;
    yr[i].zero();
    hr[i].zero();
    if (ALIGNED && n >= 8) {
      if (y) yr[i].load(y + col);
      if (h) hr[i].load(h + col);
    } else if (n > 0) {
      if (y) yr[i].load_part(y + col, n);
      if (h) hr[i].load_part(h + col, n);
    }
  }
  const float inv_cols = 1.0f / static_cast<float>(p.cols);
  float post_rstd = 1.0f;
  if (p.post) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
      yr[i].get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
    }
    post_rstd = rsqrtf(cta_sum(ss, slots[0]) * inv_cols + p.eps);
  }
  float hv[NV][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (threadIdx.x + i * threads) * 8;
    const int n = p.cols - col;
    float u[8];
    yr[i].get(u);
    hr[i].get(hv[i]);
    if (n > 0) {
      if (p.post) {
        float g[8];
        gains8(p.post + col, n, ALIGNED, p.gain_add, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = u[j] * post_rstd * g[j];
      }
      if (p.gate) {
        if (p.gate_col == 0) {
          const float g = p.gate_f32 ? static_cast<const float*>(p.gate)[row * p.gate_row]
                                     : Elem<TY>::to(static_cast<const TY*>(p.gate)[row * p.gate_row]);
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] *= g;
        } else {
          float g[8];
          if (p.gate_f32) {
            gains8(static_cast<const float*>(p.gate) + row * p.gate_row + col, n, ALIGNED, 0.0f, g);
          } else {
            Chunk8<TY> c;
            const TY* gp = static_cast<const TY*>(p.gate) + row * p.gate_row + col;
            if (ALIGNED && n >= 8) c.load(gp);
            else c.load_part(gp, n);
            c.get(g);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] *= g[j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) hv[i][j] = p.residual_scale * hv[i][j] + p.block_scale * u[j];
    if (n > 0 && p.h_out) {
      TH* o = static_cast<TH*>(p.h_out) + row * p.ld_h_out + col;
      if (ALIGNED && n >= 8) store8(o, hv[i]);
      else store8_part(o, hv[i], n);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(hv[i][j], hv[i][j], ss);
  }
  if (p.out == kNormOutNone) return;
  const float rstd = rsqrtf(cta_sum(ss, slots[1]) * inv_cols + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (threadIdx.x + i * threads) * 8;
    const int n = p.cols - col;
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = 0.0f;
    if (n > 0) {
      float g[8];
      gains8(p.pre + col, n, ALIGNED, p.gain_add, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = hv[i][j] * rstd * g[j];
    }
    if (p.out == kNormOutF8) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, magnitude_bits(z[j]));
      const F8Scale s = f8_scale(max16(m));  // 16 threads share a 128-column block
      if (n > 0) {
        if ((threadIdx.x & 15) == 0) p.z_scale[row * p.ld_scale + col / kF8Block] = s.scale;
        f8_store(static_cast<uint8_t*>(p.z) + row * p.ld_z + col, f8_pack8(z, s.inv), n, p.z_aligned);
      }
    } else if (n > 0) {
      const bool whole = p.z_aligned && n >= 8;
      const int64_t at = row * p.ld_z + col;
      if (p.out == kNormOutF16) {
        __half* o = static_cast<__half*>(p.z) + at;
        if (whole) store8(o, z);
        else store8_part(o, z, n);
      } else if (p.out == kNormOutBF16) {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.z) + at;
        if (whole) store8(o, z);
        else store8_part(o, z, n);
      } else {
        float* o = static_cast<float*>(p.z) + at;
        if (whole) store8(o, z);
        else store8_part(o, z, n);
      }
    }
  }
}

}  // namespace vd
