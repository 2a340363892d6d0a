// Rotary positions for query and key heads.
//   angle = position * f_i,  (a, b) -> m * (a cos - b sin, b cos + a sin)
// for the pairs (i, i + rotary_dim / 2) ("half") or (2i, 2i + 1)
// ("interleaved") of the first rotary_dim columns of each head; the others are
// copied.  `inverse` negates the angle.
//
// A frequency comes as turns per position in 64-bit fixed point, f_i / 2 pi *
// 2^64.  position * turns modulo 2^64 is then the fraction of a turn of any
// 64-bit position (whole turns drop out of the product by themselves), with no
// table that bounds the positions.  The product adds no error; the frequency's
// own, at most 2^-62 of a turn (host, in more than a double's 53 bits), grows
// with the position: below the fp32 cosines' up to position 2^37, a thousandth
// of a turn at 2^52.
//
// Bound by memory: q and k are read and written once.  A CTA takes
// kRotaryTokens tokens: it forms their cosines and sines once, in shared
// memory, and every head of those tokens reads them there.  One unit in flight
// a thread left loads exposed (79 us below), four cost occupancy (71).
// 16384 tokens of 16 + 4 heads of 256, 64 columns rotated, fp16: 65 us, 5.2
// TB/s, 0.79 of the measured copy rate; 12288 of 32 + 8 heads of 128, fp32: 82
// us, 6.1 TB/s.
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
  // Work units of a head: rotated ones first, then the columns that pass through.
  int rot_units, units;
  FastDiv per_token, per_head;  // by heads * units, by units
};

constexpr int kRotaryTokens = 4;
constexpr int kRotaryThreads = 256;
constexpr int kRotaryUnroll = 2;  // units whose loads a thread has in flight

// The fraction of a turn as a quarter and a signed rest of at most an eighth,
// both exact in integers: rounding the rest to fp32 then costs 2^-28 of a turn
// at most and a part in 2^24 of a small one (the whole fraction: 2^-26).
__device__ __forceinline__ float2 rotary_cos_sin(int64_t pos, uint64_t turns) {
  const uint64_t frac = static_cast<uint64_t>(pos) * turns;
  const uint64_t moved = frac + (uint64_t(1) << 61);  // quarter boundaries now between the eighths around them
  const int64_t rest = static_cast<int64_t>(moved << 2 >> 2) - (int64_t(1) << 61);
  float s, c;
  sincospif(static_cast<float>(rest) * 0x1p-63f /* half turns */, &s, &c);
  const uint32_t quarter = static_cast<uint32_t>(moved >> 62);
  if (quarter & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  if (quarter & 2) c = -c, s = -s;
  return make_float2(c, s);
}

// VEC: rows of eight elements at a time (every stride, both dims and the
// halves are multiples of eight, pointers 16-byte aligned); else a pair or an
// element at a time.
template <class T, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads, sizeof(T) == 2 ? 5 : 1) rotary_kernel(RotaryParams p) {
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
  const uint32_t heads = p.q.heads + p.k.heads;
  const uint32_t per_token = heads * p.units, total = nt * per_token;
  using Chunk = typename std::conditional<VEC, Chunk8<T>, T>::type;
  for (uint32_t w0 = threadIdx.x; w0 < total; w0 += kRotaryThreads * kRotaryUnroll) {
    const T* in[kRotaryUnroll];
    T* out[kRotaryUnroll];
    int unit[kRotaryUnroll], first[kRotaryUnroll];
    Chunk a[kRotaryUnroll], b[kRotaryUnroll];
#pragma unroll
    for (int i = 0; i < kRotaryUnroll; ++i) {
      const uint32_t w = w0 + i * kRotaryThreads;
      if (w >= total) break;
      const uint32_t t = p.per_token(w), rest = w - t * per_token;
      uint32_t head = p.per_head(rest);
      const int u = static_cast<int>(rest - head * p.units);
      const bool is_q = head < static_cast<uint32_t>(p.q.heads);
      const RotaryHeads& r = is_q ? p.q : p.k;
      if (!is_q) head -= p.q.heads;
      const bool rot = u < p.rot_units;
      const bool pairs = p.interleaved && !VEC && rot;  // the unit is the neighbours 2u and 2u + 1
      const int at = rot ? (pairs ? 2 * u : u * W) : p.rotary_dim + (u - p.rot_units) * W;
      in[i] = static_cast<const T*>(r.in) + (t0 + t) * r.in_token + head * r.in_head + at;
      out[i] = static_cast<T*>(r.out) + (t0 + t) * r.out_token + head * r.out_head + at;
      unit[i] = u;
      first[i] = static_cast<int>(t) * half;  // of the token's cosines and sines
      const int other = pairs ? 1 : half;     // from a to b
      const bool two = rot && (pairs || !p.interleaved);
      if constexpr (VEC) {
        a[i].load(in[i]);
        if (two) b[i].load(in[i] + other);
      } else {
        a[i] = *in[i];
        if (two) b[i] = in[i][other];
      }
    }
#pragma unroll
    for (int i = 0; i < kRotaryUnroll; ++i) {
      if (w0 + i * kRotaryThreads >= total) break;
      const float2* c = cs + first[i];
      if (unit[i] >= p.rot_units) {
        if (in[i] == out[i]) continue;
        if constexpr (VEC) a[i].store(out[i]);
        else *out[i] = a[i];
      } else if constexpr (!VEC) {
        const float2 f = c[unit[i]];
        const float x = Elem<T>::to(a[i]), y = Elem<T>::to(b[i]);
        out[i][0] = Elem<T>::from(x * f.x - y * f.y);
        out[i][p.interleaved ? 1 : half] = Elem<T>::from(y * f.x + x * f.y);
      } else if (p.interleaved) {
        float v[8];
        a[i].get(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = c[unit[i] * 4 + j];
          const float x = v[2 * j], y = v[2 * j + 1];
          v[2 * j] = x * f.x - y * f.y;
          v[2 * j + 1] = y * f.x + x * f.y;
        }
        store8(out[i], v);
      } else {
        float x[8], y[8];
        a[i].get(x);
        b[i].get(y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = c[unit[i] * 8 + j];
          const float r = x[j] * f.x - y[j] * f.y;
          y[j] = y[j] * f.x + x[j] * f.y;
          x[j] = r;
        }
        store8(out[i], x);
        store8(out[i] + half, y);
      }
    }
  }
}

}  // namespace vd
