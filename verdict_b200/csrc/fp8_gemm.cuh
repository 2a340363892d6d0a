// Matrix product in 8-bit floating point (e4m3) with a scale per block of 128:
//   out[m, n] = sum_b sa[m, b] * sw[n / 128, b] * (sum_{k in block b} a[m, k] w[n, k]) + bias[n]
// a [M, K] with scales per row and 128 columns, w [N, K] with scales per 128 x
// 128 block (nn.Linear layout), products and sums in fp32.
//
// The scales change every 128 columns of K, so the tensor core's accumulator
// holds one k-block only: for each of them tcgen05 MMAs (kind::f8f6f4, four
// steps of K = 32) write a fresh TMEM accumulator, and the drain warps add it,
// times its scale, to fp32 sums that stay in registers over the whole of K.
// Several TMEM accumulators keep the MMAs ahead of the drain.
//
// Scales and bias are read by plain loads: these kernels are set up while the
// ones before them still write, and the read-only path is for memory that no one
// writes while a kernel lives.
//
// Two kernels: fp8_gemm_pair_kernel (CTA pairs, 256 x 256 tiles) for many
// rows, fp8_gemm_rows_kernel (below) for few.
#pragma once

#include "gemm2.cuh"
#include "row_io.cuh"

namespace vd {

struct F8Shape {
  int M, N, K;
  const float* sa;  // [M, ceil(K / 128)], row stride ld_sa
  const float* sw;  // [ceil(N / 128), ceil(K / 128)], row stride ld_sw
  int64_t ld_sa, ld_sw;
  const float* bias;
  void* out;        // row-major, stride ld_out
  int64_t ld_out;
  int out_aligned;  // rows of out start on 16 bytes
  int splits;       // CTAs along K: the cluster's size
  int stages;       // of the shared-memory ring (fp8_gemm_rows_kernel)
  // Failure-path tests: the limit of every barrier wait, and the k-blocks after
  // which each CTA stops loading (-1: never), so that its other warps wait for a
  // stage that nothing will fill.
  uint64_t wait_ns = VD_WAIT_TIMEOUT_NS;
  int stall_after = -1;
};

// mbar_wait with the clock read only after a run of polls: reading the global
// timer takes longer than the k-block that most waits here are for.
__device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code,
                                        uint64_t limit_ns) {
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
      if (*abort_flag) return false;
    }
    const uint64_t t = globaltimer();
    if (t0 == 0) {
      t0 = t;
    } else if (t - t0 > limit_ns) {
      *abort_flag = 1;
      record_error(err, code);
      return false;
    }
  }
}

// After a wait ran out: the last phase that a ring's barriers were armed for,
// slots before `at` in the pass with parity `phase`, the others in the one
// before (true at once where that never was).  Lets the copies and MMAs that
// are under way land before the CTA gives up its memory.
__device__ __forceinline__ void f8_settle(uint64_t* bars, int n, int at, uint32_t phase) {
  for (int i = 0; i < n; ++i) mbar_wait_own(&bars[i], i < at ? phase : phase ^ 1, VD_WAIT_TIMEOUT_NS / 8);
}

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 inputs, fp32 accumulate.
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// e4m3 x e4m3 -> fp32, both operands K-major: the format codes are 0.
__host__ __device__ constexpr uint32_t umma_idesc_f8(int m, int n) { return umma_idesc_f16kind(m, n, 0); }

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

// N = 16, 32 or 64 consecutive columns of this thread's TMEM lane.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 16 || N == 32 || N == 64, "");
  if constexpr (N == 32) {
    tmem_ld32(taddr, r);
  } else if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr));
  }
}

// ---------------------------------------------------------------------------
// Few rows: the weights are read once and everything else is small, so this
// side is bound by memory and, for the shortest calls, by latency.
//
// A tile is 128 weight rows (the 128-row side of the MMA) by BN tokens; a CTA
// owns one tile over its share of K.  Where the tiles do not fill the GPU, a
// cluster of CTAs splits K: each CTA pushes its sums to the CTA that owns a
// token's column through distributed shared memory, and that one adds them in
// rank order, so the result does not depend on who came first.
//
// A drain thread owns a weight row.  The scales a[token] * w of 8 or 16
// k-blocks at a time lie in shared memory and are read four tokens at once.
//
// bf16, device time: 1 x 6144 x 4096 6.5 us (floor 3.8: the weights' 25 MB),
// 16 x 24576 x 4096 20.5 us (4.9 TB/s), 37 x 4096 x 12288 16.2 us (floor 7.8;
// while it streams 5.5 TB/s, the rest is the first loads' latency and the join).
// ---------------------------------------------------------------------------
template <int BN>
struct F8RowsConfig {
  static constexpr int BM = 128;
  static constexpr int BK = 128;
  // Ring depth: with two CTAs on an SM, and for one that has it to itself.
  static constexpr int SHARED_STAGES = BN == 128 ? 0 : BN == 64 ? 3 : 4;
  static constexpr int STAGES = BN == 128 ? 4 : BN == 64 ? 6 : 8;
  static constexpr int W_BYTES = BM * BK;
  static constexpr int A_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = W_BYTES + A_BYTES;
  static constexpr int BUFS = 4;  // TMEM accumulators
  static constexpr int TMEM_COLS = BUFS * BN;
  static constexpr int DRAIN_WARPS = BN >= 64 ? 8 : 4;
  static constexpr int COLS = BN / (DRAIN_WARPS / 4);  // columns of a drain warp
  static constexpr int SCALE_KB = BN >= 64 ? 8 : 16;   // k-blocks of scales staged at a time
  static constexpr int SCALE_BYTES = 2 * SCALE_KB * BN * 4;
  static constexpr int MAX_SPLITS = BN >= 32 ? 8 : BN / 4;  // shares of at least four columns
  static constexpr int SUM_BYTES = BN * BM * 4;  // what the cluster's CTAs send here
  // Up to 64 tokens two CTAs may share an SM: one's latencies hide under the other.
  static constexpr int CTAS_PER_SM = SHARED_STAGES > 0 ? 2 : 1;
  static constexpr int smem_bytes(int stages, int splits) {
    return 1024 + stages * STAGE_BYTES + 512 + SCALE_BYTES + (splits > 1 ? SUM_BYTES : 0);
  }
  static constexpr int THREADS = 64 + 32 * DRAIN_WARPS;
};

template <int BN, class O>
__global__ void __launch_bounds__(F8RowsConfig<BN>::THREADS, F8RowsConfig<BN>::CTAS_PER_SM)
    fp8_gemm_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, F8Shape s,
                         int* err) {
  using Cfg = F8RowsConfig<BN>;
  constexpr int BM = Cfg::BM, BK = Cfg::BK, BUFS = Cfg::BUFS, COLS = Cfg::COLS;
  constexpr int DRAIN = 32 * Cfg::DRAIN_WARPS;
  const int stages = s.stages;
  constexpr uint32_t IDESC = umma_idesc_f8(BM, BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sA = smem + stages * Cfg::W_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * Cfg::STAGE_BYTES);
  float* sScale = reinterpret_cast<float*>(smem + stages * Cfg::STAGE_BYTES + 512);
  float* sSum = reinterpret_cast<float*>(smem + stages * Cfg::STAGE_BYTES + 512 + Cfg::SCALE_BYTES);  // splits > 1
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint64_t* acc_empty = acc_full + BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int kblocks = (s.K + BK - 1) / BK;
  const int tile = static_cast<int>(blockIdx.x) / s.splits;
  const int part = static_cast<int>(blockIdx.x) - tile * s.splits;
  const int n0 = tile * BM;
  const int m0 = static_cast<int>(blockIdx.y) * BN;
  const int kb0 = static_cast<int>(static_cast<int64_t>(kblocks) * part / s.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(kblocks) * (part + 1) / s.splits);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmA);
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], Cfg::DRAIN_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  // Says that this CTA runs: its shared memory may be written once all have.
  if (s.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The set-up above ran under the tail of the kernel before this one; global
  // memory is touched only when that one is done.
  pdl_trigger_next();
  pdl_wait_prior();

  float acc[COLS];
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb - kb0 == s.stall_after) break;
        ok = f8_wait(&empty[stage], phase ^ 1, abort_flag, err, kErrTimeoutEmpty, s.wait_ns);
        if (!ok) break;
        mbar_arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
        tma_load_2d(sW + stage * Cfg::W_BYTES, &tmW, &full[stage], kb * BK, n0);
        tma_load_2d(sA + stage * Cfg::A_BYTES, &tmA, &full[stage], kb * BK, m0);
        if (++stage == stages) stage = 0, phase ^= 1;
      }
      // Every load has landed and been consumed before the CTA may exit.
      const int at = stage;
      const uint32_t at_phase = phase;
      for (int i = 0; i < stages && ok; ++i) {
        ok = f8_wait(&empty[stage], phase ^ 1, abort_flag, err, kErrTimeoutEmpty, s.wait_ns);
        if (++stage == stages) stage = 0, phase ^= 1;
      }
      if (!ok) f8_settle(full, stages, at, at_phase);
    }
    __syncwarp();
  } else if (warp == 1) {
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    const uint64_t w_desc0 = sw128_kmajor_desc(smem_u32(sW)), a_desc0 = sw128_kmajor_desc(smem_u32(sA));
    for (int kb = kb0; kb < kb1; ++kb) {
      bool ok = f8_wait(&acc_empty[buf], buf_phase ^ 1, abort_flag, err, kErrTimeoutAccEmpty, s.wait_ns) &&
                f8_wait(&full[stage], phase, abort_flag, err, kErrTimeoutFull, s.wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        f8_settle(acc_full, BUFS, buf, buf_phase);
        f8_settle(empty, stages, stage, phase);
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        // Descriptors hold addresses in units of 16 bytes; 32 bytes per step of K.
        const uint64_t w_desc = w_desc0 + stage * (Cfg::W_BYTES >> 4);
        const uint64_t a_desc = a_desc0 + stage * (Cfg::A_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f8(tmem_base + buf * BN, w_desc + 2 * k, a_desc + 2 * k, IDESC, k != 0);
        umma_commit(&acc_full[buf]);
        umma_commit(&empty[stage]);
      }
      __syncwarp();
      if (++stage == stages) stage = 0, phase ^= 1;
      if (++buf == BUFS) buf = 0, buf_phase ^= 1;
    }
  } else {
    // Drain: TMEM lane quarter warp % 4, columns [COLS * part, ...).
    const int quarter = warp & 3;
    const int col0 = ((warp - 2) >> 2) * COLS;
    const int t = threadIdx.x - 64;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + col0;
    const float* sw = s.sw + static_cast<int64_t>(n0 / kF8Block) * s.ld_sw;
    constexpr int PER = Cfg::SCALE_KB * BN / DRAIN;  // scales of a chunk per thread
    float next[PER];
    auto fetch = [&](int base) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = i * DRAIN + t;
        const int tok = m0 + e / Cfg::SCALE_KB, kb = base + e % Cfg::SCALE_KB;
        next[i] = tok < s.M && kb < kb1 ? s.sa[tok * s.ld_sa + kb] * sw[kb] : 0.0f;
      }
    };
    auto put = [&](int chunk) {
      float* to = sScale + (chunk & 1) * (Cfg::SCALE_KB * BN);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = i * DRAIN + t;
        to[e % Cfg::SCALE_KB * BN + e / Cfg::SCALE_KB] = next[i];
      }
    };
    fetch(kb0);
#pragma unroll
    for (int j = 0; j < COLS; ++j) acc[j] = 0.0f;
    put(0);
    int buf = 0, chunk = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int base = kb0; base < kb1; base += Cfg::SCALE_KB, ++chunk) {
      // The chunk is in place; the other buffer's chunk has been used up.  A warp
      // whose wait ran out keeps coming here: the others may still be at work, and
      // this barrier counts on all of them.
      asm volatile("bar.sync 1, %0;" ::"n"(DRAIN) : "memory");
      const int stop = min(base + Cfg::SCALE_KB, kb1);
      if (stop < kb1) fetch(stop);
      const float* scales = sScale + (chunk & 1) * (Cfg::SCALE_KB * BN) + col0;
      for (int kb = base; kb < stop && ok; ++kb, scales += BN) {
        ok = __all_sync(0xffffffffu, f8_wait(&acc_full[buf], buf_phase, abort_flag, err, kErrTimeoutAccFull, s.wait_ns));
        if (!ok) break;
        tc_fence_after();
        uint32_t r[COLS];
        tmem_ld<COLS>(taddr + buf * BN, r);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
#pragma unroll
        for (int j = 0; j < COLS; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(scales + j);
          acc[j] = fmaf(__uint_as_float(r[j]), f.x, acc[j]);
          acc[j + 1] = fmaf(__uint_as_float(r[j + 1]), f.y, acc[j + 1]);
          acc[j + 2] = fmaf(__uint_as_float(r[j + 2]), f.z, acc[j + 2]);
          acc[j + 3] = fmaf(__uint_as_float(r[j + 3]), f.w, acc[j + 3]);
        }
        if (++buf == BUFS) buf = 0, buf_phase ^= 1;
      }
      if (stop < kb1) put(chunk + 1);
    }
  }

  const int row = (warp & 3) * 32 + lane;  // of a drain thread
  const int n = n0 + row;
  O* out = static_cast<O*>(s.out);
  if (s.splits == 1) {
    if (warp >= 2 && n < s.N) {
      const int col0 = ((warp - 2) >> 2) * COLS;
      const float bias = s.bias ? s.bias[n] : 0.0f;
      O* o = out + static_cast<int64_t>(m0 + col0) * s.ld_out + n;
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (m0 + col0 + j < s.M) o[j * s.ld_out] = Elem<O>::from(acc[j] + bias);
    }
  } else {
    // Four columns at a time: column j goes to CTA j / share, there to
    // [rank][(j % share) / 4][row][4].
    const int share = BN / s.splits;
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA runs
    if (warp >= 2) {
      const int col0 = ((warp - 2) >> 2) * COLS;
      const uint32_t mine = smem_u32(sSum) + (part * share * BM + row * 4) * 4;
#pragma unroll
      for (int j = 0; j < COLS; j += 4) {
        const int to = (col0 + j) / share, at = (col0 + j) - to * share;
        if (m0 + col0 + j < s.M)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_shared(mine + at * (BM * 4), to)),
                       "f"(acc[j]), "f"(acc[j + 1]), "f"(acc[j + 2]), "f"(acc[j + 3])
                       : "memory");
      }
    }
    __syncwarp();
    cluster_sync_all();  // the sums have arrived
    if (warp >= 2 && n < s.N) {
      const float bias = s.bias ? s.bias[n] : 0.0f;
      const int first = part * share;
      const int count = min(share, s.M - m0 - first);
      const float4* sums = reinterpret_cast<const float4*>(sSum) + row;
      for (int j = ((warp - 2) >> 2) * 4; j < count; j += Cfg::DRAIN_WARPS) {
        float v[4] = {bias, bias, bias, bias};
#pragma unroll 4
        for (int r = 0; r < s.splits; ++r) {
          const float4 x = sums[(r * share + j) * (BM / 4)];
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        }
        O* o = out + static_cast<int64_t>(m0 + first + j) * s.ld_out + n;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i < count) o[i * s.ld_out] = Elem<O>::from(v[i]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// CTA pairs (cta_group::2): 256 x 256 tiles for shapes with enough of them.
//
// A pair stages 2 x 32 KB per k-block for 256 x 256 x 128 products, a third
// less shared-memory traffic per product than 128 x 256 tiles on one CTA.  The
// MMAs of a k-block write one of two 256-column TMEM accumulators; eight drain
// warps per CTA (two per TMEM lane quarter, 128 columns each) add it to their
// registers while the next k-block's MMAs fill the other.  The grid is
// persistent, one pair per two SMs; outputs leave through shared memory and
// TMA stores while the next tile's MMAs run.
//
// 8192 x 24576 x 4096 bf16: 890-910 us, 1.83 PFLOP/s back to back, under the
// power cap (1000 W, 1515 MHz); 760 us, 2.17 PFLOP/s, in short bursts.  515 x
// 6144 x 4096: 24 us.  A k-block takes about 890 cycles, 512 of them MMAs: two
// accumulators are all that TMEM holds at this width, and the way from a
// finished accumulator to its reuse (two 64-column loads with the first half's
// FMAs between them, 325 cycles, then the hand-back to the leader and the MMAs'
// own 750 cycles of latency) is longer than one k-block.  Tried, slower: 16
// drain warps of 64 columns (1030 cycles), 32-column loads in two buffers
// (950), scales four k-blocks ahead (920), MMAs of N = 128 with four
// accumulators (1120: A is read twice), 192-column tiles whose 96 columns a
// warp loads at once and hands back before any FMA (1057 us).
// ---------------------------------------------------------------------------
struct F8PairConfig {
  static constexpr int BM = 128;  // rows per CTA
  static constexpr int BN = 256;
  static constexpr int BK = 128;
  static constexpr int STAGES = 6;
  static constexpr int A_BYTES = BM * BK;
  static constexpr int B_BYTES = BN / 2 * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int DRAIN_WARPS = 8;
  static constexpr int OUT_BYTES = 4096;  // per drain warp: 32 rows of 128 bytes
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + DRAIN_WARPS * OUT_BYTES + 1024;
  static constexpr int THREADS = 128 + 32 * DRAIN_WARPS;
  // Registers: the launch's 168 a thread are redistributed, 40 to the control
  // warpgroup and 232 to the two of the drain.
  static constexpr int LAUNCH_REGS = 168, CONTROL_REGS = 40, DRAIN_REGS = 232;
  static_assert(128 * CONTROL_REGS + 256 * DRAIN_REGS <= THREADS * LAUNCH_REGS, "register split");
  static constexpr int GROUP_M = 8;  // pair tiles (256 rows) per raster group
};

__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on an mbarrier of either CTA with the default semantics.  What it
// tells the leader is that this warp's TMEM loads are complete, which
// tcgen05.wait::ld and the tcgen05 fences order; no memory access is handed
// over.  (mbarrier.arrive.release.cluster is a memory barrier on top, which
// waited for the scale loads in flight: 600 cycles a k-block.)
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

template <class O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8PairConfig::THREADS, 1)
    fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmC, F8Shape s, int* err) {
  using Cfg = F8PairConfig;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BK = Cfg::BK, STAGES = Cfg::STAGES;
  constexpr uint32_t IDESC = umma_idesc_f8(2 * BM, BN);
  constexpr int CHUNK = 128 / sizeof(O);  // columns of a 128-byte output row in shared memory
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint8_t* sOut = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + Cfg::DRAIN_WARPS * Cfg::OUT_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);   // the leader's arm; both CTAs' bytes complete it
      mbar_init(&empty[i], 1);  // the leader's commit, multicast to both CTAs
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * Cfg::DRAIN_WARPS);  // both CTAs' drain warps (the leader's copy is used)
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger_next();  // as in the other kernel
  pdl_wait_prior();

  const int num_m = (s.M + 2 * BM - 1) / (2 * BM);
  const int num_n = (s.N + BN - 1) / BN;
  const int tiles = num_m * num_n;
  const int kblocks = (s.K + BK - 1) / BK;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::CONTROL_REGS));
    if (warp == 0) {
      if (lane == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        tma_prefetch_desc(&tmC);
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true, stalled = false;
        for (int tile = pair; tile < tiles && ok && !stalled; tile += pairs) {
          int m, n;
          tile_coords(tile, num_m, num_n, Cfg::GROUP_M, m, n);
          const int ya = m * 2 * BM + static_cast<int>(rank) * BM;
          const int yb = n * BN + static_cast<int>(rank) * (BN / 2);
          for (int kb = 0; kb < kblocks; ++kb) {
            if (issued++ == s.stall_after) {
              stalled = true;
              break;
            }
            if (!f8_wait(&empty[stage], phase ^ 1, abort_flag, err, kErrTimeoutEmpty, s.wait_ns)) {
              ok = false;
              break;
            }
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::STAGE_BYTES);
            const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
            tma_load_2d_pair(sA + stage * Cfg::A_BYTES, &tmA, bar, kb * BK, ya);
            tma_load_2d_pair(sB + stage * Cfg::B_BYTES, &tmB, bar, kb * BK, yb);
            if (++stage == STAGES) stage = 0, phase ^= 1;
          }
        }
        // Every stage this CTA filled has been consumed before the CTA may exit.
        const int at = stage;
        const uint32_t at_phase = phase;
        for (int i = 0; i < STAGES && ok; ++i) {
          ok = f8_wait(&empty[stage], phase ^ 1, abort_flag, err, kErrTimeoutEmpty, s.wait_ns);
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
        // The leader's barriers count both CTAs' loads; the other CTA meets it
        // at the cluster barrier below.
        if (!ok && leader) f8_settle(full, STAGES, at, at_phase);
      }
    } else if (warp == 1) {
      // The whole warp waits and one elected lane issues, so that addresses and
      // descriptors stay in uniform registers: with a k-block's MMAs over in 512
      // cycles, what the issuing thread does between them counts.
      if (leader) {
        int stage = 0, buf = 0;
        uint32_t phase = 0, buf_phase = 0;
        const uint64_t a_desc0 = sw128_kmajor_desc(smem_u32(sA)), b_desc0 = sw128_kmajor_desc(smem_u32(sB));
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
          for (int kb = 0; kb < kblocks; ++kb) {
            ok = f8_wait(&full[stage], phase, abort_flag, err, kErrTimeoutFull, s.wait_ns) &&
                 f8_wait(&acc_empty[buf], buf_phase ^ 1, abort_flag, err, kErrTimeoutAccEmpty, s.wait_ns);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
              f8_settle(acc_full, 2, buf, buf_phase);
              f8_settle(empty, STAGES, stage, phase);
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              // Descriptors hold addresses in units of 16 bytes; 32 bytes per step of K.
              const uint64_t a_desc = a_desc0 + stage * (Cfg::A_BYTES >> 4);
              const uint64_t b_desc = b_desc0 + stage * (Cfg::B_BYTES >> 4);
              const uint32_t d = tmem_base + buf * BN;
              umma_f8_pair(d, a_desc, b_desc, IDESC, 0);
              umma_f8_pair(d, a_desc + 2, b_desc + 2, IDESC, 1);
              umma_f8_pair(d, a_desc + 4, b_desc + 4, IDESC, 1);
              umma_f8_pair(d, a_desc + 6, b_desc + 6, IDESC, 1);
              umma_commit_pair(&acc_full[buf], 0x3);
              umma_commit_pair(&empty[stage], 0x3);
            }
            __syncwarp();
            if (++stage == STAGES) stage = 0, phase ^= 1;
            if (++buf == 2) buf = 0, buf_phase ^= 1;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::DRAIN_REGS));
    // Drain warp: TMEM lane quarter warp % 4, columns [128 half, +128), one
    // weight block: thread = output row, one scale per k-block.
    const int quarter = warp & 3;
    const int half = (warp - 4) >> 2;
    uint8_t* stage_out = sOut + (warp - 4) * Cfg::OUT_BYTES;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
    const uint32_t release0 = mapa_shared(smem_u32(&acc_empty[0]), 0);
    const uint32_t release1 = mapa_shared(smem_u32(&acc_empty[1]), 0);
    const int wblocks = (s.N + kF8Block - 1) / kF8Block;
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      int m, n;
      tile_coords(tile, num_m, num_n, Cfg::GROUP_M, m, n);
      const int row0 = m * 2 * BM + static_cast<int>(rank) * BM + quarter * 32;
      const int row = row0 + lane;
      const int col0 = n * BN + half * 128;
      // Rows and blocks past the end: any scale, their products are zero.
      const float* sa = s.sa + min(row, s.M - 1) * s.ld_sa;
      const float* sw = s.sw + min(col0 / kF8Block, wblocks - 1) * s.ld_sw;
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.0f, 0.0f);
      // Scales are loaded two k-blocks ahead.
      float a1 = sa[0], w1 = sw[0];
      float a2 = kblocks > 1 ? sa[1] : 0.0f, w2 = kblocks > 1 ? sw[1] : 0.0f;
      for (int kb = 0; kb < kblocks; ++kb) {
        const float f = a1 * w1;
        a1 = a2, w1 = w2;
        if (kb + 2 < kblocks) a2 = sa[kb + 2], w2 = sw[kb + 2];
        ok = __all_sync(0xffffffffu, f8_wait(&acc_full[buf], buf_phase, abort_flag, err, kErrTimeoutAccFull, s.wait_ns));
        if (!ok) break;
        tc_fence_after();
        const float2 ff = make_float2(f, f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t r[64];
          tmem_ld<64>(taddr + buf * BN + c * 64, r);
          tmem_wait_ld();
          if (c == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_remote(buf ? release1 : release0);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j)
            acc[c * 32 + j] = __ffma2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), ff,
                                         acc[c * 32 + j]);
        }
        if (++buf == 2) buf = 0, buf_phase ^= 1;
      }
      if (!ok) break;
      if (s.bias) {
        if (col0 + 128 <= s.N && (reinterpret_cast<uintptr_t>(s.bias) & 15) == 0) {
          const float4* b = reinterpret_cast<const float4*>(s.bias + col0);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float4 v = b[j];
            acc[2 * j] = __fadd2_rn(acc[2 * j], make_float2(v.x, v.y));
            acc[2 * j + 1] = __fadd2_rn(acc[2 * j + 1], make_float2(v.z, v.w));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            const int col = col0 + 2 * j;
            if (col < s.N) acc[j].x += s.bias[col];
            if (col + 1 < s.N) acc[j].y += s.bias[col + 1];
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 128 / CHUNK; ++c) {
        const int x = col0 + c * CHUNK;
        if (x >= s.N || row0 >= s.M) break;
        if (lane == 0) bulk_wait_read<0>();  // the store before has read the buffer
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          uint4 w;
          const float2* v = acc + c * (CHUNK / 2) + q * (CHUNK / 16);
          if constexpr (sizeof(O) == 4) {
            w = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                           __float_as_uint(v[1].y));
          } else {
            w = make_uint4(Elem<O>::pack2(v[0].x, v[0].y), Elem<O>::pack2(v[1].x, v[1].y),
                           Elem<O>::pack2(v[2].x, v[2].y), Elem<O>::pack2(v[3].x, v[3].y));
          }
          *reinterpret_cast<uint4*>(stage_out + lane * 128 + ((q ^ (lane & 7)) << 4)) = w;
        }
        // A TMA store writes whole 16-byte units, past the last column of out as
        // well: only where a unit does not cross it.
        if (s.out_aligned && (x + CHUNK <= s.N || s.N % (16 / static_cast<int>(sizeof(O))) == 0)) {
          fence_proxy_async_smem_gemm();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmC, stage_out, x, row0);
            bulk_commit();
          }
          continue;
        }
        // What TMA cannot store: row by row, lanes along columns.
        __syncwarp();
        constexpr int EL = 4 / sizeof(O);  // outputs in a lane's four bytes
        const int left = s.N - x - lane * EL, rows = min(32, s.M - row0);
        O* o = static_cast<O*>(s.out) + row0 * s.ld_out + x + lane * EL;
#pragma unroll 4
        for (int r = 0; r < rows; ++r, o += s.ld_out) {
          const uint32_t v =
              *reinterpret_cast<const uint32_t*>(stage_out + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
          const O* e = reinterpret_cast<const O*>(&v);
#pragma unroll
          for (int k = 0; k < EL; ++k)
            if (k < left) o[k] = e[k];
        }
        __syncwarp();
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its peer may still read or signal its shared memory
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace vd
