// Log probabilities over a whole vocabulary: for each row of logits x and a
// temperature, with z = (x - max x) / temperature and S = sum exp(z),
//   logp(id) = z[id] - log S,  lse = max x / temperature + log S,
//   entropy  = log S - sum(exp(z) z) / S,
// and the `top` largest logits with their ids (equal ones: lowest id first).
//
// Masked entries are -inf: no probability, never listed.  A row that holds
// nothing else has logp and lse -inf, entropy 0 and no alternatives (id -1,
// -inf).  A row with NaN or +inf has no distribution: NaN, ids -1.
//
// Bound by memory: each logit is read once.  Each thread keeps a running
// maximum with the sums of exp(z) and exp(z) z scaled to it; threads, warps
// and the CTAs of a row are joined at the end, in a fixed order.  The
// alternatives come out of the same pass: the first batch of logits gives a
// lower bound on the k-th largest (the k-th largest of 64 groups' maxima), and
// only entries at or above it go to a candidate buffer in shared memory, a few
// hundred of a vocabulary.  A row whose entries keep rising can overflow the
// buffer; it is then read again for a bound found by radix selection, at most
// eight more times.
//
// Few rows: a cluster of up to eight CTAs shares a row and joins through
// distributed shared memory.
#pragma once

#include "gemm2.cuh"
#include "row_io.cuh"

namespace vd {

struct LogprobParams {
  const void* logits;
  int64_t ld;
  int64_t rows;
  int vocab;
  const int64_t* targets;  // [rows, n_targets]; null: none
  int n_targets, top;
  float inv_temperature;
  float* logprobs;      // [rows, n_targets]
  float* entropy;       // [rows]
  float* lse;           // [rows]
  int32_t* top_ids;     // [rows, top]
  float* top_logprobs;  // [rows, top]
  int splits;           // CTAs of a row: the cluster's size
};

constexpr int kLpThreads = 512;
constexpr int kLpUnroll = 4;        // 16-byte loads in flight per thread
constexpr int kLpGroups = kLpThreads / 8;
constexpr int kLpMaxTop = kLpGroups;
constexpr int kLpCap = 1024;        // candidates
constexpr int kLpMaxSplits = 8;
// In units of log2: exponents below this are 0 in fp32.
constexpr float kLpFloor = -1000.0f;

// Keys order by logit, then lowest id first; 0 is below every entry's key.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t id) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
  const uint32_t ordered = b ^ (static_cast<int32_t>(b) < 0 ? 0xffffffffu : 0x80000000u);
  return (static_cast<uint64_t>(ordered) << 32) | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ float lp_key_value(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o ^ (static_cast<int32_t>(o) < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t lp_key_id(uint64_t key) { return ~static_cast<uint32_t>(key); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Running maximum m with s = sum 2^t and u = sum 2^t t, t = (x - m) c.
struct LpStats {
  float m, s, u;
};

__device__ __forceinline__ LpStats lp_rescale(LpStats a, float m, float c) {
  // a.m = -inf: nothing summed (s = u = 0, or NaN, which stays).  NaN logits
  // are not maxima, and +inf - +inf is NaN: both reach s.
  const float d = a.m == -INFINITY ? kLpFloor : max_nan((a.m - m) * c, kLpFloor);
  const float f = exp2_approx(d);
  return {m, a.s * f, f * (a.u + a.s * d)};
}
__device__ __forceinline__ LpStats lp_join(LpStats a, LpStats b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.u + b.u};
  a = lp_rescale(a, m, c);
  b = lp_rescale(b, m, c);
  return {m, a.s + b.s, a.u + b.u};
}
__device__ __forceinline__ LpStats lp_join_lanes(LpStats a, float c, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) {
    LpStats b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.u = __shfl_xor_sync(0xffffffffu, a.u, o);
    a = lp_join(a, b, c);
  }
  return a;
}

template <class T>
struct LpBatch {
  static constexpr int VEC = 16 / sizeof(T);
  uint4 r[kLpUnroll];

  // Slots of 16 bytes counted from the row's start rounded down to 16 bytes;
  // slot v holds elements v * VEC - skew ..  Edge slots are filled with -inf
  // outside the row.
  __device__ __forceinline__ void load(const T* row, int vocab, int skew, int slot, int end) {
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      const int v = slot + k * kLpThreads;
      const int at = v * VEC - skew;
      if (v < end && at >= 0 && at + VEC <= vocab) {
        r[k] = __ldg(reinterpret_cast<const uint4*>(row + at));
      } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) {
            w[j] = v < end && at + j >= 0 && at + j < vocab ? __float_as_uint(row[at + j]) : 0xff800000u;
          } else {
            const unsigned short* s = reinterpret_cast<const unsigned short*>(row);
            const uint32_t none = Elem<T>::kUmmaFormat == 1 ? 0xff80u : 0xfc00u;  // -inf
            const int e = at + 2 * j;
            const uint32_t lo = v < end && e >= 0 && e < vocab ? s[e] : none;
            const uint32_t hi = v < end && e + 1 >= 0 && e + 1 < vocab ? s[e + 1] : none;
            w[j] = lo | (hi << 16);
          }
        }
        r[k] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  __device__ __forceinline__ void get(int k, float (&x)[VEC]) const {
    const uint32_t w[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        x[j] = __uint_as_float(w[j]);
      } else {
        const float2 f = Elem<T>::unpack2(w[j]);
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    }
  }
};

struct LpShared {
  uint64_t cand[kLpCap];
  uint64_t kept[kLpCap];
  uint64_t best[kLpMaxTop];  // this CTA's alternatives, largest first
  uint64_t group[kLpGroups];
  uint64_t bound;
  int count, kept_count;
  int hist[256];
  int above;
  LpStats warp[kLpThreads / 32];
  LpStats total;
};

// The k-th largest of the 64 groups' largest keys (a group is eight threads):
// at least k entries reach it.  0 where fewer groups have an entry.
__device__ __forceinline__ uint64_t lp_group_bound(LpShared& sh, uint64_t best, int k) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
    best = b > best ? b : best;
  }
  if ((threadIdx.x & 7) == 0) sh.group[threadIdx.x >> 3] = best;
  if (threadIdx.x == 0) sh.bound = 0;
  __syncthreads();
  if (threadIdx.x < kLpGroups) {
    const uint64_t mine = sh.group[threadIdx.x];
    int larger = 0;
    for (int i = 0; i < kLpGroups; ++i) larger += sh.group[i] > mine;
    if (larger == k - 1 && mine != 0) sh.bound = mine;  // keys are distinct
  }
  __syncthreads();
  return sh.bound;
}

// The k largest of n <= kLpCap keys in sh.cand, into sh.best (0 past the last).
__device__ __forceinline__ void lp_select(LpShared& sh, int n, int k) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < n; i += kLpThreads) best = sh.cand[i] > best ? sh.cand[i] : best;
  if (threadIdx.x == 0) sh.kept_count = 0;
  const uint64_t bound = lp_group_bound(sh, best, k);
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const uint64_t key = sh.cand[i];
    if (key != 0 && key >= bound) sh.kept[atomicAdd(&sh.kept_count, 1)] = key;
  }
  if (threadIdx.x < kLpMaxTop) sh.best[threadIdx.x] = 0;
  __syncthreads();
  const int kept = sh.kept_count;
  for (int i = threadIdx.x; i < kept; i += kLpThreads) {
    const uint64_t key = sh.kept[i];
    int larger = 0;
    for (int j = 0; j < kept; ++j) larger += sh.kept[j] > key;
    if (larger < k) sh.best[larger] = key;
  }
  __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(LogprobParams p) {
  using Batch = LpBatch<T>;
  constexpr int VEC = Batch::VEC;
  extern __shared__ __align__(16) uint8_t lp_smem[];
  LpShared& sh = *reinterpret_cast<LpShared*>(lp_smem);
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / p.splits;
  const int part = static_cast<int>(blockIdx.x - row * p.splits);
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int slots = (p.vocab + skew + VEC - 1) / VEC;
  const int per = (slots + p.splits - 1) / p.splits;
  const int begin = min(part * per, slots), end = min(begin + per, slots);
  const float c = p.inv_temperature * 1.4426950408889634f;
  const int k = p.top;

  LpStats st{-INFINITY, 0.0f, 0.0f};
  uint64_t bound = 0;
  float bound_x = -INFINITY;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  // Entries at or above the bound; -inf (and NaN) are never listed.
  auto collect = [&](const Batch& b, int slot) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float v[VEC];
      b.get(u, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (v[j] >= bound_x && v[j] > -INFINITY) {
          const uint64_t key = lp_key(v[j], static_cast<uint32_t>((slot + u * kLpThreads) * VEC - skew + j));
          if (key >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kLpCap) sh.cand[at] = key;
          }
        }
      }
    }
  };
  for (int base = begin; base < end; base += kLpThreads * kLpUnroll) {
    Batch b;
    b.load(x, p.vocab, skew, base + tid, end);
    float bm = -INFINITY;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float v[VEC];
      b.get(u, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) bm = fmaxf(bm, v[j]);
    }
    if (bm > st.m) st = lp_rescale(st, bm, c);
    const float m = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float v[VEC];
      b.get(u, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float t = max_nan((v[j] - m) * c, kLpFloor);
        const float e = exp2_approx(t);
        st.s += e;
        st.u = fmaf(e, t, st.u);
      }
    }
    if (k > 0) {
      if (base == begin) {
        uint64_t best = 0;
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) {
          float v[VEC];
          b.get(u, v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const uint64_t key = lp_key(v[j], static_cast<uint32_t>((base + tid + u * kLpThreads) * VEC - skew + j));
            if (v[j] > -INFINITY && key > best) best = key;
          }
        }
        bound = lp_group_bound(sh, best, k);
        if (bound) bound_x = lp_key_value(bound);
      }
      if (bm >= bound_x) collect(b, base + tid);
    }
  }

  st = lp_join_lanes(st, c, 32);
  if ((tid & 31) == 0) sh.warp[tid >> 5] = st;
  __syncthreads();
  if (tid < 32) {
    st = tid < kLpThreads / 32 ? sh.warp[tid] : LpStats{-INFINITY, 0.0f, 0.0f};
    st = lp_join_lanes(st, c, 32);
    if (tid == 0) sh.total = st;
  }

  if (k > 0) {
    __syncthreads();
    if (sh.count > kLpCap) {
      // Radix selection of a bound that k to kLpCap entries reach: the keys'
      // bytes from the top, one pass each.
      uint64_t prefix = 0;
      int above = 0;  // entries above the prefix's range
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kLpThreads) sh.hist[i] = 0;
        __syncthreads();
        for (int base = begin; base < end; base += kLpThreads * kLpUnroll) {
          Batch b;
          b.load(x, p.vocab, skew, base + tid, end);
#pragma unroll 1
          for (int u = 0; u < kLpUnroll; ++u) {
            float v[VEC];
            b.get(u, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const uint64_t key = lp_key(v[j], static_cast<uint32_t>((base + tid + u * kLpThreads) * VEC - skew + j));
              const bool in = shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8));
              if (v[j] > -INFINITY && in) atomicAdd(&sh.hist[(key >> shift) & 255], 1);
            }
          }
        }
        __syncthreads();
        if (tid == 0) {
          int sum = above, bin = 255;
          while (bin > 0 && sum + sh.hist[bin] < k) sum += sh.hist[bin--];
          sh.above = sum;
          sh.count = sum + sh.hist[bin];
          sh.bound = prefix | (static_cast<uint64_t>(bin) << shift);
        }
        __syncthreads();
        above = sh.above;
        prefix = sh.bound;
        const int reach = sh.count;
        __syncthreads();
        if (reach <= kLpCap) break;
      }
      bound = prefix;
      bound_x = lp_key_value(bound);
      if (!(bound_x >= -INFINITY)) bound_x = -INFINITY;  // a prefix can fall outside the numbers
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int base = begin; base < end; base += kLpThreads * kLpUnroll) {
        Batch b;
        b.load(x, p.vocab, skew, base + tid, end);
        collect(b, base + tid);
      }
      __syncthreads();
    }
    lp_select(sh, sh.count, k);
  }
  __syncthreads();

  if (p.splits > 1) {
    cluster_sync_all();  // every CTA's total and alternatives are in place
    if (part == 0) {
      if (tid == 0) {
        LpStats t = sh.total;
        for (int r = 1; r < p.splits; ++r) {
          const uint32_t at = mapa_shared(smem_u32(&sh.total), r);
          LpStats o;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(at));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.s) : "r"(at + 4));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.u) : "r"(at + 8));
          t = lp_join(t, o, c);
        }
        sh.total = t;
      }
      if (k > 0) {
        for (int i = tid; i < p.splits * k; i += kLpThreads) {
          const int r = i / k;
          const uint32_t at = mapa_shared(smem_u32(&sh.best[i - r * k]), r);
          uint64_t key;
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(at));
          sh.cand[i] = key;
        }
        __syncthreads();
        lp_select(sh, p.splits * k, k);
      }
      __syncthreads();
    }
    cluster_sync_all();  // no CTA leaves while its shared memory is read
    if (part != 0) return;
  }

  const LpStats t = sh.total;
  const bool empty = t.m == -INFINITY && t.s == 0.0f;
  const float log_s = logf(t.s);  // NaN rows: s is NaN
  const float lse = empty ? -INFINITY : t.m * p.inv_temperature + log_s;
  if (tid == 0) {
    if (p.lse) p.lse[row] = t.s != t.s ? NAN : lse;
    if (p.entropy) p.entropy[row] = empty ? 0.0f : log_s - 0.6931471805599453f * (t.u / t.s);
  }
  auto logp = [&](float v) {
    if (t.s != t.s) return __int_as_float(0x7fffffff);
    if (empty || v == -INFINITY) return -INFINITY;
    return (v - t.m) * p.inv_temperature - log_s;
  };
  for (int i = tid; i < p.n_targets; i += kLpThreads) {
    const int64_t id = p.targets[row * p.n_targets + i];
    float r = 0.0f;  // a negative id: no token
    if (id >= p.vocab) r = __int_as_float(0x7fffffff);
    else if (id >= 0) r = logp(Elem<T>::to(x[id]));
    p.logprobs[row * p.n_targets + i] = r;
  }
  for (int i = tid; i < k; i += kLpThreads) {
    const uint64_t key = t.s != t.s ? 0 : sh.best[i];
    p.top_ids[row * k + i] = key ? static_cast<int32_t>(lp_key_id(key)) : -1;
    p.top_logprobs[row * k + i] = t.s != t.s ? __int_as_float(0x7fffffff) : key ? logp(lp_key_value(key)) : -INFINITY;
  }
}

}  // namespace vd
