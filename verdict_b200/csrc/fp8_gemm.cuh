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
// One-CTA kernel (this file's first): a tile is 128 rows of P by BN rows of Q.
//   SWAP = false: P = a (a thread of the drain owns a token; its scale is one
//     number per k-block), Q = w.
//   SWAP = true: P = w, Q = a, for few tokens: the 128-row side of the MMA is
//     filled with weight rows, and a tile needs no more than 32 or 64 tokens.
// Where the tiles do not fill the GPU, a cluster of CTAs splits K and joins its
// sums through distributed shared memory, in rank order.
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
};

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

template <int BN>
struct F8Config {
  static constexpr int BM = 128;
  static constexpr int BK = 128;
  static constexpr int STAGES = BN == 128 ? 6 : 8;
  static constexpr int P_BYTES = BM * BK;
  static constexpr int Q_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES;
  static constexpr int BUFS = 4;  // TMEM accumulators
  static constexpr int TMEM_COLS = BUFS * BN;
  static constexpr int SCALE_KB = 16;  // k-blocks of token scales staged at a time (SWAP)
  static constexpr int SCALE_BYTES = 2 * SCALE_KB * BN * 4;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 1024 + SCALE_BYTES;
  static constexpr int THREADS = 192;
};

__device__ __forceinline__ void drain_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <class O>
__device__ __forceinline__ void f8_out(O* out, float v, int n, const float* bias) {
  *out = Elem<O>::from(bias ? v + __ldg(bias + n) : v);
}

template <bool SWAP, int BN, class O>
__global__ void __launch_bounds__(F8Config<BN>::THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, F8Shape s,
                    int* err) {
  using Cfg = F8Config<BN>;
  constexpr int STAGES = Cfg::STAGES, BUFS = Cfg::BUFS;
  constexpr uint32_t IDESC = umma_idesc_f8(Cfg::BM, BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sP = smem;
  uint8_t* sQ = smem + STAGES * Cfg::P_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + BUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sScale = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE_BYTES + 1024);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
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
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int kblocks = (s.K + Cfg::BK - 1) / Cfg::BK;
  const int part = static_cast<int>(blockIdx.x) % s.splits;
  const int p0 = static_cast<int>(blockIdx.x) / s.splits * Cfg::BM;
  const int q0 = static_cast<int>(blockIdx.y) * BN;
  const int kb0 = static_cast<int>(static_cast<int64_t>(kblocks) * part / s.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(kblocks) * (part + 1) / s.splits);

  float acc[BN];
  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmP);
      tma_prefetch_desc(&tmQ);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, err, kErrTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
        tma_load_2d(sP + stage * Cfg::P_BYTES, &tmP, &full[stage], kb * Cfg::BK, p0);
        tma_load_2d(sQ + stage * Cfg::Q_BYTES, &tmQ, &full[stage], kb * Cfg::BK, q0);
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
      // Every load has landed and been consumed before the CTA may exit.
      for (int i = 0; i < STAGES; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, err, kErrTimeoutEmpty)) break;
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&acc_empty[buf], buf_phase ^ 1, abort_flag, err, kErrTimeoutAccEmpty)) break;
        if (!mbar_wait(&full[stage], phase, abort_flag, err, kErrTimeoutFull)) break;
        tc_fence_after();
        const uint32_t p_addr = smem_u32(sP + stage * Cfg::P_BYTES);
        const uint32_t q_addr = smem_u32(sQ + stage * Cfg::Q_BYTES);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f8(tmem_base + buf * BN, sw128_kmajor_desc(p_addr + k * 32), sw128_kmajor_desc(q_addr + k * 32), IDESC,
                  k != 0);
        umma_commit(&empty[stage]);
        umma_commit(&acc_full[buf]);
        if (++stage == STAGES) stage = 0, phase ^= 1;
        if (++buf == BUFS) buf = 0, buf_phase ^= 1;
      }
    }
  } else {
    // Drain: thread (lane quarter warp % 4, lane) owns row p of the tile.
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int t = threadIdx.x - 64;
    const int p = p0 + row;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
    for (int j = 0; j < BN; ++j) acc[j] = 0.0f;
    int buf = 0;
    uint32_t buf_phase = 0;
    // SWAP: one weight-block scale for the whole tile, a scale per column
    // (token), staged SCALE_KB k-blocks at a time.  Otherwise: one scale per
    // thread (token) and one for the tile (BN = 128: one weight block).
    const float* sw = s.sw + static_cast<int64_t>((SWAP ? p0 : q0) / kF8Block) * s.ld_sw;
    const float* sa = !SWAP && p < s.M ? s.sa + p * s.ld_sa : nullptr;
    bool ok = true;
    for (int base = kb0; base < kb1 && ok; base += Cfg::SCALE_KB) {
      const int stop = min(base + Cfg::SCALE_KB, kb1);
      float* scales = sScale + ((base - kb0) / Cfg::SCALE_KB & 1) * (Cfg::SCALE_KB * BN);
      if constexpr (SWAP) {
        // Column-major by k-block; two buffers: the barrier below also tells
        // that every warp is done with the buffer before last.
        for (int i = t; i < Cfg::SCALE_KB * BN; i += 128) {
          const int tok = i / Cfg::SCALE_KB, kb = base + i % Cfg::SCALE_KB;
          scales[i % Cfg::SCALE_KB * BN + tok] =
              q0 + tok < s.M && kb < stop ? __ldg(s.sa + (q0 + tok) * s.ld_sa + kb) : 0.0f;
        }
        drain_barrier();
      }
      for (int kb = base; kb < stop; ++kb) {
        const float w = __ldg(sw + kb);
        const float f = SWAP ? w : w * (sa ? __ldg(sa + kb) : 0.0f);
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], buf_phase, abort_flag, err, kErrTimeoutAccFull));
        if (!ok) break;
        tc_fence_after();
        uint32_t r[2][32];
        tmem_ld32(taddr + buf * BN, r[0]);
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          tmem_wait_ld();
          if (c + 1 < BN / 32) {
            tmem_ld32(taddr + buf * BN + (c + 1) * 32, r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float d = __uint_as_float(r[c & 1][j]);
            const float g = SWAP ? f * scales[(kb - base) * BN + c * 32 + j] : f;
            acc[c * 32 + j] = fmaf(d, g, acc[c * 32 + j]);
          }
        }
        if (++buf == BUFS) buf = 0, buf_phase ^= 1;
      }
    }
    if (s.splits > 1) {
      // All MMAs of this CTA are done (its last accumulator was read), so the
      // stages are free: [column][row], one 128-byte line per warp access.
      float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int j = 0; j < BN; ++j) sums[j * Cfg::BM + row] = acc[j];
    }
  }
  if (s.splits > 1) {
    __syncthreads();
    cluster_sync_all();
    if (warp >= 2) {
      const int quarter = warp & 3;
      const int row = quarter * 32 + lane;
      const int p = p0 + row;
      const int j0 = BN * part / s.splits, j1 = BN * (part + 1) / s.splits;
      const uint32_t local = smem_u32(smem);
      O* out = static_cast<O*>(s.out);
      for (int j = j0; j < j1; ++j) {
        float v = 0.0f;
        for (int r = 0; r < s.splits; ++r) {
          float x;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(x)
                       : "r"(mapa_shared(local + (j * Cfg::BM + row) * 4, r)));
          v += x;
        }
        const int m = SWAP ? q0 + j : p, n = SWAP ? p : q0 + j;
        if (m < s.M && n < s.N) f8_out(out + m * s.ld_out + n, v, n, s.bias);
      }
    }
    cluster_sync_all();  // no CTA leaves while its sums are read
  } else if (warp >= 2) {
    const int p = p0 + (warp & 3) * 32 + lane;
    O* out = static_cast<O*>(s.out);
    if constexpr (SWAP) {
#pragma unroll
      for (int j = 0; j < BN; ++j)
        if (q0 + j < s.M && p < s.N) f8_out(out + (q0 + j) * s.ld_out + p, acc[j], p, s.bias);
    } else if (p < s.M) {
      O* o = out + p * s.ld_out + q0;
#pragma unroll
      for (int j = 0; j < BN; j += 8) {
        if (q0 + j >= s.N) break;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[j + i] + (s.bias && q0 + j + i < s.N ? __ldg(s.bias + q0 + j + i) : 0.0f);
        if (s.out_aligned && q0 + j + 8 <= s.N) store8(o + j, v);
        else store8_part(o + j, v, s.N - q0 - j);
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

}  // namespace vd
