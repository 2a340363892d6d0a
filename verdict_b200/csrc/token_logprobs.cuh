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
// Few rows: a cluster of up to eight CTAs shares a row; each pushes its sums
// and candidates to the first through distributed shared memory.
//
// Accuracy: sums are fp32 and the exponentials ex2.approx (1.4e-7 off at most,
// 5e-8 low on average), of arguments rounded once more by the factor log2(e) /
// temperature.  All of it stays below the rounding of fp32 outputs of this size:
// 1.1e-7 relative on a large batch, where exp of an fp32 difference gives 5e-8
// with more instructions an entry, which are what the batch is bound by.
//
// 1024 x 256000 bf16, 8 alternatives: 136 us, 3.9 TB/s, 0.59 of the measured
// copy rate.  The logits alone are 80 us; the rest is arithmetic (issue slots
// 61 %, special-function unit 49 %: an exp2 an entry) and the 1.7 waves that
// 1024 rows make of 592 resident CTAs.  Four loads a thread and four CTAs on an
// SM beat two and five or six (165, 183 us) and eight and three (158).  One row
// of 152064: 12 us, latency.
#pragma once

#include <type_traits>

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

constexpr int kLpThreads = 256;
constexpr int kLpCtasPerSm = 4;
constexpr int kLpUnroll = 4;        // 16-byte loads in flight per thread
constexpr int kLpGroups = 64;
constexpr int kLpGroupSize = kLpThreads / kLpGroups;
constexpr int kLpMaxTop = kLpGroups;
constexpr int kLpCap = 1024;        // candidates
constexpr int kLpMaxSplits = 8;
constexpr int kLpInbox = 128;       // candidates a CTA sends on
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

// 16 bytes of a row: slot v, counted from the row's start rounded down to 16
// bytes, holds entries v * VEC - skew and on; -inf outside the row.
template <class T>
__device__ __forceinline__ uint4 lp_load(const T* row, int vocab, int skew, int v, int end) {
  constexpr int VEC = 16 / sizeof(T);
  const int at = v * VEC - skew;
  if (v < end && at >= 0 && at + VEC <= vocab) return __ldg(reinterpret_cast<const uint4*>(row + at));
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
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T>
__device__ __forceinline__ void lp_unpack(uint4 r, float (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
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

template <class T>
struct LpBatch {
  static constexpr int VEC = 16 / sizeof(T);
  uint4 r[kLpUnroll];

  __device__ __forceinline__ void load(const T* row, int vocab, int skew, int base, int end) {
    const int slot = base + static_cast<int>(threadIdx.x);
    // Inside the row and the CTA's part of it: no checks per load.
    if (base > 0 && base + kLpThreads * kLpUnroll < end) {
      const uint4* p = reinterpret_cast<const uint4*>(row + (static_cast<int64_t>(slot) * VEC - skew));
#pragma unroll
      for (int k = 0; k < kLpUnroll; ++k) r[k] = __ldg(p + k * kLpThreads);
      return;
    }
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) r[k] = lp_load(row, vocab, skew, slot + k * kLpThreads, end);
  }
  // The largest entry of load u (NaN is passed over), two 16-bit entries at a time.
  __device__ __forceinline__ float largest(int u) const {
    if constexpr (sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(&r[u]);
      return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
    } else {
      using T2 = typename std::conditional<Elem<T>::kUmmaFormat == 1, __nv_bfloat162, __half2>::type;
      const T2* v = reinterpret_cast<const T2*>(&r[u]);
      const T2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
      const float2 f = Elem<T>::unpack2(*reinterpret_cast<const uint32_t*>(&m));
      return fmaxf(f.x, f.y);
    }
  }
  // Bit u * VEC + j for each entry of at least `low` (which is above -inf).
  __device__ __forceinline__ uint32_t reaching(const float (&top)[kLpUnroll], float low) const {
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      if (top[u] >= low) {
        float v[VEC];
        lp_unpack<T>(r[u], v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) bits |= v[j] >= low ? 1u << (u * VEC + j) : 0u;
      }
    }
    return bits;
  }
};

struct LpShared {
  uint64_t cand[kLpCap];
  uint64_t kept[kLpCap];
  uint64_t best[kLpMaxTop];  // this CTA's alternatives, largest first
  uint64_t group[kLpGroups];
  uint64_t bound[2];
  int count, kept_count;
  int hist[256];
  int above;
  LpStats warp[kLpThreads / 32];
  LpStats total;
  float target_x[kLpThreads];  // each thread its own
  int target_is[kLpThreads];
  // What the cluster's CTAs send to its first.
  LpStats part[kLpMaxSplits];
  int part_count[kLpMaxSplits];
  uint64_t inbox[kLpMaxSplits * kLpInbox];
};

// The k-th largest of the 64 groups' largest keys (a group is kLpGroupSize threads):
// at least k entries reach it.  0 where fewer groups have an entry.  `word`: a
// thread may still read the call before's result when another begins this call,
// so calls with no barrier of the caller's between them take the two words in turn.
__device__ __forceinline__ uint64_t lp_group_bound(LpShared& sh, uint64_t best, int k, int word) {
#pragma unroll
  for (int o = kLpGroupSize / 2; o > 0; o >>= 1) {
    const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
    best = b > best ? b : best;
  }
  const int group = threadIdx.x / kLpGroupSize, in_group = threadIdx.x % kLpGroupSize;
  if (in_group == 0) sh.group[group] = best;
  if (threadIdx.x == 0) sh.bound[word] = 0;
  __syncthreads();
  // A group's threads count the keys above its own.
  const uint64_t mine = sh.group[group];
  int larger = 0;
#pragma unroll
  for (int i = 0; i < kLpGroups; i += kLpGroupSize) larger += sh.group[i + in_group] > mine;
#pragma unroll
  for (int o = kLpGroupSize / 2; o > 0; o >>= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
  if (larger == k - 1 && mine != 0) sh.bound[word] = mine;  // keys are distinct
  __syncthreads();
  return sh.bound[word];
}

// The k largest of get(0) .. get(n - 1), n <= kLpCap, into sh.best (0 past the last).
template <class Get>
__device__ __forceinline__ void lp_select(LpShared& sh, int n, int k, Get&& get) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < n; i += kLpThreads) best = get(i) > best ? get(i) : best;
  if (threadIdx.x == 0) sh.kept_count = 0;
  const uint64_t bound = lp_group_bound(sh, best, k, 0);
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const uint64_t key = get(i);
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
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) token_logprobs_kernel(LogprobParams p) {
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
  int batches = 0;
  uint64_t bound = 0;
  float bound_x = -3.402823466e38f;  // every entry but -inf
  if (tid == 0) sh.count = 0;
  // The targets' logits, on their way while the row is read (more than
  // kLpThreads of them: the others at the end).
  auto fetch_target = [&](int i) {
    const int64_t id = p.targets[row * p.n_targets + i];
    const int is = id < 0 ? -1 : id >= p.vocab;  // -1: no token, 1: past the vocabulary
    sh.target_is[tid] = is;
    if (is == 0) sh.target_x[tid] = Elem<T>::to(x[id]);
  };
  if (part == 0 && tid < p.n_targets) fetch_target(tid);
  __syncthreads();
  // Says that this CTA runs: its shared memory may be written once all have.
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  auto id_of = [&](int slot, int bit) { return (slot + bit / VEC * kLpThreads) * VEC - skew + bit % VEC; };
  // Entries at or above the bound go to the buffer.
  auto collect = [&](const Batch& b, const float (&top)[kLpUnroll], int slot) {
    uint32_t bits = b.reaching(top, bound_x);
#pragma unroll 1
    while (bits) {
      const int id = id_of(slot, __ffs(bits) - 1);
      bits &= bits - 1;
      const uint64_t key = lp_key(Elem<T>::to(x[id]), static_cast<uint32_t>(id));
      if (key >= bound) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kLpCap) sh.cand[at] = key;
      }
    }
  };
  for (int base = begin; base < end; base += kLpThreads * kLpUnroll) {
    Batch b;
    b.load(x, p.vocab, skew, base, end);
    float top[kLpUnroll];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) top[u] = b.largest(u);
    static_assert(kLpUnroll == 4, "");
    const float bm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    if (bm > st.m) st = lp_rescale(st, bm, c);
    const float m = st.m == -INFINITY ? 0.0f : st.m;
    // Two running pairs (even and odd entries), joined at the batch's end.
    float2 sum = make_float2(st.s, 0.0f), mom = make_float2(st.u, 0.0f);
    const float2 neg_m = make_float2(-m, -m), cc = make_float2(c, c);
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float v[VEC];
      lp_unpack<T>(b.r[u], v);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        float2 t = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), neg_m), cc);
        t.x = max_nan(t.x, kLpFloor);
        t.y = max_nan(t.y, kLpFloor);
        const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
        sum = __fadd2_rn(sum, e);
        mom = __ffma2_rn(e, t, mom);
      }
    }
    st.s = sum.x + sum.y;
    st.u = mom.x + mom.y;
    if (k > 0) {
      if (base == begin) {
        // The thread's largest entry, the first of equal ones.
        uint64_t best = 0;
        if (bm > -INFINITY) best = lp_key(bm, static_cast<uint32_t>(id_of(base + tid, __ffs(b.reaching(top, bm)) - 1)));
        bound = lp_group_bound(sh, best, k, 0);
        if (bound) bound_x = lp_key_value(bound);
      }
      if (bm >= bound_x) collect(b, top, base + tid);
      // After 2, 4, 8 .. batches the bound rises with the maxima so far (their
      // ids are not kept: the key of any entry with that value will do), so
      // that each doubling of what has been read adds about k candidates.  Not
      // where less than half as much is left.
      if (++batches > 1 && (batches & (batches - 1)) == 0 &&
          ((end - base) / (kLpThreads * kLpUnroll) - 1) * 2 >= batches) {
        const uint64_t higher = lp_group_bound(sh, st.m > -INFINITY ? lp_key(st.m, 0xffffffffu - tid) : 0, k,
                                               (31 - __clz(batches)) & 1);
        if (higher != 0 && (higher | 0xffffffffu) > (bound | 0xffffffffu)) {
          bound = higher & ~0xffffffffull;
          bound_x = lp_key_value(bound);
        }
      }
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
#pragma unroll 1
          for (int u = 0; u < kLpUnroll; ++u) {
            const int slot = base + tid + u * kLpThreads;
            float v[VEC];
            lp_unpack<T>(lp_load(x, p.vocab, skew, slot, end), v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const uint64_t key = lp_key(v[j], static_cast<uint32_t>(slot * VEC - skew + j));
              if (v[j] > -INFINITY && (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8))))
                atomicAdd(&sh.hist[(key >> shift) & 255], 1);
            }
          }
        }
        __syncthreads();
        if (tid == 0) {
          int sum = above, bin = 255;
          while (bin > 0 && sum + sh.hist[bin] < k) sum += sh.hist[bin--];
          sh.above = sum;
          sh.count = sum + sh.hist[bin];
          sh.bound[0] = prefix | (static_cast<uint64_t>(bin) << shift);
        }
        __syncthreads();
        above = sh.above;
        prefix = sh.bound[0];
        const int reach = sh.count;
        __syncthreads();
        if (reach <= kLpCap) break;
      }
      bound = prefix;
      bound_x = lp_key_value(bound);
      if (!(bound_x >= -3.402823466e38f)) bound_x = -3.402823466e38f;  // a prefix can lie below every number
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int base = begin; base < end; base += kLpThreads * kLpUnroll) {
        Batch b;
        b.load(x, p.vocab, skew, base, end);
        float top[kLpUnroll];
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) top[u] = b.largest(u);
        collect(b, top, base + tid);
      }
      __syncthreads();
    }
  }
  int found = sh.count;
  if (p.splits == 1) {
    if (k > 0) lp_select(sh, found, k, [&](int i) { return sh.cand[i]; });
    __syncthreads();
  } else {
    // More candidates than the inbox holds: the k largest of them.
    const uint64_t* send = sh.cand;
    if (k > 0 && found > kLpInbox) {
      lp_select(sh, found, k, [&](int i) { return sh.cand[i]; });
      send = sh.best;
      found = k;
    }
    __syncwarp();  // the aligned barrier wants whole warps, and the loops and branches above split them
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA runs
    if (k > 0)
      for (int i = tid; i < found; i += kLpThreads)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&sh.inbox[part * kLpInbox + i]), 0)),
                     "l"(send[i])
                     : "memory");
    if (tid == 0) {
      const uint32_t at = mapa_shared(smem_u32(&sh.part[part]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(st.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(st.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(st.u) : "memory");
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&sh.part_count[part]), 0)),
                   "r"(k > 0 ? found : 0)
                   : "memory");
    }
    __syncwarp();
    cluster_sync_all();  // all has arrived
    if (part != 0) return;
    if (tid < 32) {
      LpStats t = tid < p.splits ? sh.part[tid] : LpStats{-INFINITY, 0.0f, 0.0f};
      t = lp_join_lanes(t, c, kLpMaxSplits);
      if (tid == 0) sh.total = t;
    }
    if (k > 0)
      lp_select(sh, p.splits * kLpInbox, k, [&](int i) -> uint64_t {
        return i % kLpInbox < sh.part_count[i / kLpInbox] ? sh.inbox[i] : 0;
      });
    __syncthreads();
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
    if (i >= kLpThreads) fetch_target(i);
    const int is = sh.target_is[tid];
    p.logprobs[row * p.n_targets + i] = is < 0 ? 0.0f : is ? __int_as_float(0x7fffffff) : logp(sh.target_x[tid]);
  }
  for (int i = tid; i < k; i += kLpThreads) {
    const uint64_t key = t.s != t.s ? 0 : sh.best[i];
    p.top_ids[row * k + i] = key ? static_cast<int32_t>(lp_key_id(key)) : -1;
    p.top_logprobs[row * k + i] = t.s != t.s ? __int_as_float(0x7fffffff) : key ? logp(lp_key_value(key)) : -INFINITY;
  }
}

}  // namespace vd
