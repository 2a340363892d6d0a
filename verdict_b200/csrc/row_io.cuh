// Row access for the bandwidth-bound operators: eight consecutive elements of
// a 16-bit or fp32 row at a time, held as loaded until they are used (so that
// a thread's loads are all in flight before the first conversion), and the
// same eight element by element where a row is not 16-byte aligned or ends
// inside the eight.  Plain loads: an output may be its input's own buffer.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace vd {

template <>
struct Elem<float> {
  __device__ __forceinline__ static float from(float x) { return x; }
  __device__ __forceinline__ static float to(float x) { return x; }
};

// Division of numbers below 2^31 by one fixed on the host: ceil(2^(31 + l) / d)
// with l = ceil(log2 d) gives exact quotients.
struct FastDiv {
  uint32_t mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t d) {
    if (d <= 1) return;
    uint32_t l = 0;
    while ((uint64_t(1) << l) < d) ++l;
    mul = static_cast<uint32_t>(((uint64_t(1) << (31 + l)) + d - 1) / d);
    shift = l - 1;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return mul == 0 ? n : __umulhi(n, mul) >> shift; }
};

template <class T>
struct Chunk8 {
  uint4 r;
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void load_part(const T* p, int n) {
    uint32_t w[4] = {0, 0, 0, 0};
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) w[j >> 1] |= static_cast<uint32_t>(s[j]) << ((j & 1) * 16);
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = Elem<T>::unpack2(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
};

template <>
struct Chunk8<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void load_part(const float* p, int n) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.0f;
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
};

// Rows that vector accesses do not fit: a warp takes 128 columns, a lane
// every 32nd of them.
constexpr int kGap = 32;

// Four elements: 8 bytes of a 16-bit type, 16 of fp32.  A warp's access is
// contiguous in either, which eight fp32 elements a thread are not (two
// accesses of every other 16 bytes: twice the shared L1 wavefronts).
template <class T>
struct Chunk4 {
  typename std::conditional<sizeof(T) == 4, float4, uint2>::type r;
  __device__ __forceinline__ void zero() {
    if constexpr (sizeof(T) == 4) r = make_float4(0.f, 0.f, 0.f, 0.f);
    else r = make_uint2(0, 0);
  }
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const decltype(r)*>(p); }
  // Elements kGap apart (a warp's accesses contiguous), those below n.
  __device__ __forceinline__ void load_gap(const T* p, int n) {
    constexpr int G = kGap;
    if constexpr (sizeof(T) == 4) {
      r = make_float4(n > 0 ? p[0] : 0.f, n > G ? p[G] : 0.f, n > 2 * G ? p[2 * G] : 0.f, n > 3 * G ? p[3 * G] : 0.f);
    } else {
      const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
      r.x = (n > 0 ? s[0] : 0u) | ((n > G ? s[G] : 0u) << 16);
      r.y = (n > 2 * G ? s[2 * G] : 0u) | ((n > 3 * G ? s[3 * G] : 0u) << 16);
    }
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    if constexpr (sizeof(T) == 4) {
      v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
    } else {
      const float2 a = Elem<T>::unpack2(r.x), b = Elem<T>::unpack2(r.y);
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
  }
};

template <bool WHOLE, class T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4], int n) {
  if constexpr (WHOLE) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(Elem<T>::pack2(v[0], v[1]), Elem<T>::pack2(v[2], v[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j * kGap < n) p[j * kGap] = Elem<T>::from(v[j]);
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(Elem<T>::pack2(v[0], v[1]), Elem<T>::pack2(v[2], v[3]),
                                              Elem<T>::pack2(v[4], v[5]), Elem<T>::pack2(v[6], v[7]));
  }
}

// |x| as ordered bits: the maximum over these is the largest magnitude, with
// inf above every finite value and NaN above inf (a float maximum drops NaN).
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The e4m3 format's largest value, and the smallest magnitude a block's scale
// is formed from: an all-zero block keeps a normal fp32 scale.
constexpr float kF8Max = 448.0f;
constexpr float kF8AmaxFloor = 1e-30f;
constexpr int kF8Block = 128;

struct F8Scale {
  float scale, inv;
};

// Both divisions are correctly rounded: the scale is part of the result, and
// a value that lies between two e4m3 numbers must not move with the build.
__device__ __forceinline__ F8Scale f8_scale(uint32_t amax_bits) {
  float a = __uint_as_float(amax_bits);
  if (a < kF8AmaxFloor) a = kF8AmaxFloor;  // false for NaN
  return {__fdiv_rn(a, kF8Max), __fdiv_rn(kF8Max, a)};
}

// Values to e4m3, round to nearest even, saturating (NaN stays NaN).
__device__ __forceinline__ uint32_t f8_pack2(float a, float b, float inv) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t f8_pack4(const float (&v)[4], float inv) {
  return f8_pack2(v[0], v[1], inv) | (f8_pack2(v[2], v[3], inv) << 16);
}
__device__ __forceinline__ uint2 f8_pack8(const float (&v)[8], float inv) {
  return make_uint2(f8_pack2(v[0], v[1], inv) | (f8_pack2(v[2], v[3], inv) << 16),
                    f8_pack2(v[4], v[5], inv) | (f8_pack2(v[6], v[7], inv) << 16));
}

__device__ __forceinline__ void f8_store(uint8_t* p, uint2 q, int n) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) p[j] = static_cast<uint8_t>((j < 4 ? q.x : q.y) >> ((j & 3) * 8));
}

// Largest of 16 neighbouring lanes (the 16 chunks of a 128-column block).
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

}  // namespace vd
