// Rotary positions for query and key heads.
//   angle = position * f_i,  (a, b) -> m * (a cos - b sin, b cos + a sin)
// for the pairs (i, i + rotary_dim / 2) ("half") or (2i, 2i + 1)
// ("interleaved") of the first rotary_dim columns of each head; the others are
// copied.  `inverse` negates the angle.
//
// A frequency comes as turns per position in 64-bit fixed point, f_i / 2 pi *
// 2^64.  position * turns modulo 2^64 is then the exact fraction of a turn of
// any 64-bit position (whole turns drop out of the product by themselves), so
// the angle does not lose precision far into a long context and no table
// bounds the positions.
//
// Bound by memory: q and k are read and written once.  A CTA takes
// kRotaryTokens tokens: it forms their cosines and sines once, in shared
// memory, and every head of those tokens reads them there.
#pragma once

#include "row_io.cuh"

namespace vd {

struct RotaryHeads {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;  // element strides
  int heads;
};

struct RotaryParams {
  RotaryHeads q, k;
  const void* positions;  // null: first_position + token
  int positions64;
  int64_t first_position, tokens;
  const uint64_t* turns;  // [rotary_dim / 2]
  int head_dim, rotary_dim, interleaved;
  float factor, sin_sign;
};

constexpr int kRotaryTokens = 4;
constexpr int kRotaryThreads = 256;

__device__ __forceinline__ float2 rotary_cos_sin(int64_t pos, uint64_t turns) {
  // The top 32 bits of the fraction as a signed number: (-1/2, 1/2] turn.
  const uint64_t frac = static_cast<uint64_t>(pos) * turns;
  const int32_t t = static_cast<int32_t>(frac >> 32);
  float s, c;
  sincospif(static_cast<float>(t) * 4.656612873077393e-10f /* 2^-31: half turns */, &s, &c);
  return make_float2(c, s);
}

// VEC: rows of eight elements at a time (every stride, both dims and the
// halves are multiples of eight, pointers 16-byte aligned); else a pair or an
// element at a time.
template <class T, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(RotaryParams p) {
  extern __shared__ float2 cs[];  // [kRotaryTokens][rotary_dim / 2]
  const int half = p.rotary_dim >> 1;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kRotaryTokens;
  const int nt = static_cast<int>(min(static_cast<int64_t>(kRotaryTokens), p.tokens - t0));
  for (int i = threadIdx.x; i < nt * half; i += kRotaryThreads) {
    const int t = i / half;
    const int64_t at = t0 + t;
    const int64_t pos = !p.positions     ? p.first_position + at
                        : p.positions64 ? static_cast<const int64_t*>(p.positions)[at]
                                        : static_cast<int64_t>(static_cast<const int32_t*>(p.positions)[at]);
    float2 v = rotary_cos_sin(pos, p.turns[i - t * half]);
    v.x *= p.factor;
    v.y *= p.factor * p.sin_sign;
    cs[i] = v;
  }
  __syncthreads();
  constexpr int W = VEC ? 8 : 1;
  // Work units of a head: rotated ones first, then the columns that pass through.
  const int rot_units = (VEC && p.interleaved) ? p.rotary_dim / 8 : half / W;
  const int copy_units = (p.head_dim - p.rotary_dim) / W;
  const int units = rot_units + copy_units;
  const int heads = p.q.heads + p.k.heads;
  const uint32_t per_token = static_cast<uint32_t>(heads) * units;
  for (uint32_t w = threadIdx.x; w < nt * per_token; w += kRotaryThreads) {
    const uint32_t t = w / per_token;
    uint32_t rest = w - t * per_token;
    uint32_t head = rest / units;
    const int u = static_cast<int>(rest - head * units);
    const bool is_q = head < static_cast<uint32_t>(p.q.heads);
    const RotaryHeads& r = is_q ? p.q : p.k;
    if (!is_q) head -= p.q.heads;
    const T* in = static_cast<const T*>(r.in) + (t0 + t) * r.in_token + head * r.in_head;
    T* out = static_cast<T*>(r.out) + (t0 + t) * r.out_token + head * r.out_head;
    const float2* c = cs + t * half;
    if (u >= rot_units) {
      const int at = p.rotary_dim + (u - rot_units) * W;
      if (in + at == out + at) continue;
      if constexpr (VEC) {
        Chunk8<T> x;
        x.load(in + at);
        x.store(out + at);
      } else {
        out[at] = in[at];
      }
    } else if (!p.interleaved) {
      const int at = u * W;
      if constexpr (VEC) {
        Chunk8<T> xa, xb;
        xa.load(in + at);
        xb.load(in + at + half);
        float a[8], b[8];
        xa.get(a);
        xb.get(b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = c[at + j];
          const float x = a[j] * f.x - b[j] * f.y;
          b[j] = b[j] * f.x + a[j] * f.y;
          a[j] = x;
        }
        store8(out + at, a);
        store8(out + at + half, b);
      } else {
        const float2 f = c[at];
        const float a = Elem<T>::to(in[at]), b = Elem<T>::to(in[at + half]);
        out[at] = Elem<T>::from(a * f.x - b * f.y);
        out[at + half] = Elem<T>::from(b * f.x + a * f.y);
      }
    } else {
      if constexpr (VEC) {
        Chunk8<T> x;
        x.load(in + u * 8);
        float v[8];
        x.get(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = c[u * 4 + j];
          const float a = v[2 * j], b = v[2 * j + 1];
          v[2 * j] = a * f.x - b * f.y;
          v[2 * j + 1] = b * f.x + a * f.y;
        }
        store8(out + u * 8, v);
      } else {
        const float2 f = c[u];
        const float a = Elem<T>::to(in[2 * u]), b = Elem<T>::to(in[2 * u + 1]);
        out[2 * u] = Elem<T>::from(a * f.x - b * f.y);
        out[2 * u + 1] = Elem<T>::from(b * f.x + a * f.y);
      }
    }
  }
}

}  // namespace vd
