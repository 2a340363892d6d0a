// C entry points of the 8-bit decoder operators (include/vdexec_kernels.h):
// argument checks, the choice of a kernel variant and the launch on the
// caller's stream.  Nothing here allocates or waits.

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <limits>
#include <string>
#include <type_traits>

#include "vdexec_kernels.h"

#include "block_norm.cuh"
#include "fp8_gemm.cuh"
#include "host.hpp"
#include "overlap.hpp"
#include "quantize.cuh"
#include "rotary.cuh"
#include "token_logprobs.cuh"

namespace vd {
namespace {

constexpr int64_t kMaxInt = 0x7fffffff;

void need(bool ok, const char* what) {
  if (!ok) fail(VD_EINVAL, what);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int elem_bytes(int dtype) { return dtype == VDK_FP32 ? 4 : 2; }

// What a kernel dereferences has to lie on its element's boundary.
template <class T>
void need_aligned(const T* p, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % alignof(T)) fail(VD_EINVAL, std::string(what) + " is not aligned to its type");
}
void need_aligned(const void* p, int dtype, const char* what) {
  const int bytes = dtype == VDK_FP8 ? 1 : elem_bytes(dtype);
  if (reinterpret_cast<uintptr_t>(p) % bytes) fail(VD_EINVAL, std::string(what) + " is not aligned to its type");
}

// Matrix [rows, cols] of `dtype` with row stride ld.
ByteRows matrix(const void* p, int64_t rows, int64_t cols, int64_t ld, int dtype) {
  const int64_t bytes = dtype == VDK_FP8 ? 1 : elem_bytes(dtype);
  return {p, cols * bytes, rows, ld * bytes};
}

// What one thread writes no other may read or write: an output lies apart from
// everything else, or (where the kernel reads an element in the thread that
// writes it) it is the same rows.
void need_apart(const ByteRows& out, const ByteRows& other, const char* what, bool or_same = false) {
  if (overlap(out, other) && !(or_same && same_rows(out, other))) fail(VD_EINVAL, std::string(what) + " overlap");
}

// Rows of `dtype` that all start on a 16-byte boundary.
bool rows16(const void* p, int64_t ld, int dtype) { return aligned16(p) && ld * elem_bytes(dtype) % 16 == 0; }

template <class F>
void by_type(int dtype, F&& f) {
  switch (dtype) {
    case VDK_FP16: f(__half()); break;
    case VDK_BF16: f(__nv_bfloat16()); break;
    case VDK_FP32: f(float()); break;
    default: fail(VD_EINVAL, "dtype must be VDK_FP16, VDK_BF16 or VDK_FP32");
  }
}

int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64) fail(VD_EINVAL, "device index out of range");
  if (!sms[dev]) {  // the same value whichever thread stores it
    int n = 0;
    cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
    sms[dev] = n;
  }
  return sms[dev];
}

void launched() { cuda_check(cudaGetLastError(), "kernel launch"); }

// cluster = 0: the kernel's own cluster size.  programmatic: the kernel may be
// set up while the one before it in the stream still runs (it waits for that
// one itself).
template <class K, class... Args>
void launch(K kernel, dim3 grid, int threads, size_t smem, int cluster, bool programmatic, cudaStream_t stream,
            const Args&... args) {
  if (cluster == 1 && !programmatic) {
    kernel<<<grid, threads, smem, stream>>>(args...);
    return launched();
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  unsigned n = 0;
  if (cluster > 0) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (programmatic) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), "kernel launch");
}

// Row-major [rows, cols] bytes with row stride ld, boxes of box_rows x 128
// with the 128-byte swizzle; columns and rows past the end read as zero.
CUtensorMap f8_map(const void* ptr, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(VD_ECUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")");
  return m;
}

// Clusters of `splits` CTAs of fp8_gemm_rows_kernel that the device holds at
// once, one CTA on an SM (what the occupancy call assumes of kernels that use
// tensor memory; two were seen to run); asked once per device and kernel.
template <int BN, class O>
int f8_rows_clusters(int splits) {
  using Cfg = F8RowsConfig<BN>;
  static std::atomic<int> known[64][4];
  int dev = 0;
  cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64) fail(VD_EINVAL, "device index out of range");
  std::atomic<int>& slot = known[dev][splits == 1 ? 0 : splits == 2 ? 1 : splits == 4 ? 2 : 3];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    auto kernel = fp8_gemm_rows_kernel<BN, O>;
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Cfg::smem_bytes(Cfg::STAGES, Cfg::MAX_SPLITS)),
               "shared memory size");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(splits * 1024);
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::smem_bytes(Cfg::STAGES, splits);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cuda_check(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg), "cluster occupancy");
    slot.store(n = std::max(n, 1), std::memory_order_relaxed);
  }
  return n;
}

struct F8RowsPlan {
  int splits, stages;
  int steps;  // k-blocks that the last CTA to finish goes through, one after another
};

template <int BN, class O>
F8RowsPlan plan_f8_rows(const F8Shape& s) {
  using Cfg = F8RowsConfig<BN>;
  const int kblocks = (s.K + 127) / 128;
  const int tiles = ((s.N + 127) / 128) * ((s.M + BN - 1) / BN);
  // The most CTAs per tile that still run at once, each with at least four
  // k-blocks: a second wave costs more than the split gains.
  F8RowsPlan p{Cfg::MAX_SPLITS, 0, 0};
  int room = f8_rows_clusters<BN, O>(p.splits);
  while (p.splits > 1 && (kblocks / p.splits < 4 || tiles > Cfg::CTAS_PER_SM * room))
    room = f8_rows_clusters<BN, O>(p.splits /= 2);
  p.stages = Cfg::CTAS_PER_SM == 1 || tiles <= room ? Cfg::STAGES : Cfg::SHARED_STAGES;
  p.steps = (tiles + room - 1) / room * ((kblocks + p.splits - 1) / p.splits);
  return p;
}

template <int BN, class O>
void launch_f8_rows(const void* a, int64_t ld_a, const void* w, int64_t ld_w, F8Shape s, const F8RowsPlan& plan,
                    int* status, cudaStream_t stream) {
  using Cfg = F8RowsConfig<BN>;
  s.splits = plan.splits;
  s.stages = plan.stages;
  const int n_tiles = (s.N + 127) / 128, m_tiles = (s.M + BN - 1) / BN;
  launch(fp8_gemm_rows_kernel<BN, O>, dim3(n_tiles * s.splits, m_tiles), Cfg::THREADS,
         Cfg::smem_bytes(s.stages, s.splits), s.splits, true, stream, f8_map(w, s.N, s.K, ld_w, 128),
         f8_map(a, s.M, s.K, ld_a, BN), s, status);
}

// Which kernel a product runs on.
struct F8Choice {
  int bn;           // tokens a tile of fp8_gemm_rows_kernel; 0: CTA pairs
  F8RowsPlan rows;  // of the former
};

template <class O>
F8Choice choose_f8(const F8Shape& s) {
  if (s.M <= 16) return {16, plan_f8_rows<16, O>(s)};
  if (s.M <= 32) return {32, plan_f8_rows<32, O>(s)};
  if (s.M <= 64) return {64, plan_f8_rows<64, O>(s)};
  // A pair goes through a k-block of a 256 x 256 tile in 0.53 us, a CTA of
  // the other kernel through one of a 128 x 128 tile in 0.6, but it can split
  // K, for about four k-blocks' time (bf16, us, pairs / rows: 128 x 6144 x
  // 4096 19.4 / 14.8, 100 x 4096 x 12288 46.8 / 19.0, 200 x 4096 x 4096 19.1
  // / 14.8; 256 x 6144 x 4096 19.5 / 21.2, 100 x 24576 x 4096 36.0 / 41.1).
  const int pairs = sm_count() / 2;
  const int pair_tiles = ((s.M + 255) / 256) * ((s.N + 255) / 256);
  const int pair_steps = (pair_tiles + pairs - 1) / pairs * ((s.K + 127) / 128);
  const F8RowsPlan plan = plan_f8_rows<128, O>(s);
  const bool rows = plan.steps * 1.1 + 4 < pair_steps && (s.M + 127) / 128 <= 65535;
  return {rows ? 128 : 0, plan};
}

// Row-major outputs [rows, cols] with row stride ld, boxes of 32 rows x 128
// bytes with the 128-byte swizzle; stores past the end are dropped, columns in
// units of 16 bytes.
CUtensorMap out_map(const void* ptr, int64_t rows, int64_t cols, int64_t ld, int dtype) {
  CUtensorMap m;
  const int es = elem_bytes(dtype);
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * es};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / es), 32};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType t = dtype == VDK_FP32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : dtype == VDK_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = encode_fn()(&m, t, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(VD_ECUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")");
  return m;
}

template <class O>
void launch_f8_pair(const void* a, int64_t ld_a, const void* w, int64_t ld_w, const F8Shape& s, int dtype, int* status,
                    cudaStream_t stream) {
  using Cfg = F8PairConfig;
  auto kernel = fp8_gemm_pair_kernel<O>;
  cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES),
             "shared memory size");
  cudaFuncAttributes attr;
  cuda_check(cudaFuncGetAttributes(&attr, kernel), "kernel attributes");
  if (attr.numRegs != Cfg::LAUNCH_REGS) fail(VD_ECUDA, "fp8_gemm_pair_kernel was built with another register count");
  const int tiles = ((s.M + 255) / 256) * ((s.N + 255) / 256);
  const int grid = 2 * std::min(tiles, sm_count() / 2);
  launch(kernel, dim3(grid), Cfg::THREADS, Cfg::SMEM_BYTES, 0, true, stream, f8_map(a, s.M, s.K, ld_a, 128),
         f8_map(w, s.N, s.K, ld_w, 128), s.out_aligned ? out_map(s.out, s.M, s.N, s.ld_out, dtype) : CUtensorMap{}, s,
         status);
}

}  // namespace
}  // namespace vd

using namespace vd;

extern "C" VD_API int vdk_quantize_fp8(const void* x, int64_t ld_x, const void* gate, int64_t ld_gate, int act,
                                       int64_t rows, int64_t cols, int dtype, void* q, int64_t ld_q, float* scale,
                                       int64_t ld_scale, void* stream, char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need(rows >= 0 && cols >= 1 && cols <= kMaxInt - 128, "need rows >= 0 and 1 <= cols < 2^31 - 128");
    need(act >= VDK_ACT_NONE && act <= VDK_ACT_SILU, "unknown activation");
    need(gate || act == VDK_ACT_NONE, "an activation needs a gate");
    const int64_t col_blocks = (cols + 127) / 128;
    need(rows <= kMaxInt / col_blocks, "rows * ceil(cols / 128) must be below 2^31");
    need(ld_x >= cols && ld_q >= cols && ld_scale >= col_blocks && (!gate || ld_gate >= cols),
         "a row stride is smaller than its row");
    if (rows == 0) return;
    need(x && q && scale, "null buffer");
    need_aligned(x, dtype, "x");
    need_aligned(gate, dtype, "gate");
    need_aligned(scale, "scale");
    const ByteRows mx = matrix(x, rows, cols, ld_x, dtype), mg = matrix(gate, rows, cols, ld_gate, dtype),
                   mq = matrix(q, rows, cols, ld_q, VDK_FP8), ms = matrix(scale, rows, col_blocks, ld_scale, VDK_FP32);
    need_apart(mq, mx, "q and x");
    need_apart(mq, mg, "q and gate");
    need_apart(ms, mx, "scale and x");
    need_apart(ms, mg, "scale and gate");
    need_apart(mq, ms, "q and scale");
    QuantizeParams p{};
    p.x = x, p.gate = gate;
    p.ld_x = ld_x, p.ld_gate = ld_gate, p.ld_q = ld_q, p.ld_scale = ld_scale;
    p.blocks = static_cast<uint32_t>(rows * col_blocks);
    p.col_blocks = static_cast<uint32_t>(col_blocks);
    p.per_row = FastDiv(static_cast<uint32_t>(col_blocks));
    p.cols = static_cast<int>(cols);
    p.act = act;
    p.q = static_cast<uint8_t*>(q);
    p.scale = scale;
    const unsigned per = kQuantUnroll * kQuantThreads / 16;
    const unsigned grid = (p.blocks + per - 1) / per;
    const bool whole = cols % 8 == 0 && rows16(x, ld_x, dtype) && (!gate || rows16(gate, ld_gate, dtype)) &&
                       (reinterpret_cast<uintptr_t>(q) & 7) == 0 && ld_q % 8 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    by_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      auto run = [&](auto whole_kernel, auto kernel) {
        if (whole) whole_kernel<<<grid, kQuantThreads, 0, s>>>(p);
        else kernel<<<grid, kQuantThreads, 0, s>>>(p);
      };
      if (!gate) run(quantize_rows_kernel<T, kGateNone, true>, quantize_rows_kernel<T, kGateNone, false>);
      else if (act == VDK_ACT_SILU)
        run(quantize_rows_kernel<T, kGateSilu, true>, quantize_rows_kernel<T, kGateSilu, false>);
      else run(quantize_rows_kernel<T, kGateAny, true>, quantize_rows_kernel<T, kGateAny, false>);
    });
    launched();
  });
}

extern "C" VD_API int vdk_quantize_fp8_weight(const void* w, int64_t ld_w, int64_t rows, int64_t cols, int dtype,
                                              void* q, int64_t ld_q, float* scale, int64_t ld_scale, void* stream,
                                              char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need(rows >= 1 && rows <= 65535ll * 128 && cols >= 1 && cols <= kMaxInt - 128,
         "need 1 <= rows <= 8388480 and 1 <= cols < 2^31 - 128");
    need(ld_w >= cols && ld_q >= cols && ld_scale >= (cols + 127) / 128, "a row stride is smaller than its row");
    need(w && q && scale, "null buffer");
    need_aligned(w, dtype, "w");
    need_aligned(scale, "scale");
    const ByteRows mw = matrix(w, rows, cols, ld_w, dtype), mq = matrix(q, rows, cols, ld_q, VDK_FP8),
                   ms = matrix(scale, (rows + 127) / 128, (cols + 127) / 128, ld_scale, VDK_FP32);
    need_apart(mq, mw, "q and w");
    need_apart(ms, mw, "scale and w");
    need_apart(mq, ms, "q and scale");
    const dim3 grid(static_cast<unsigned>((cols + 127) / 128), static_cast<unsigned>((rows + 127) / 128));
    by_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      quantize_weight_kernel<T><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(w), ld_w, static_cast<int>(rows), static_cast<int>(cols), static_cast<uint8_t*>(q), ld_q,
          scale, ld_scale);
    });
    launched();
  });
}

static void need_f8_shape(int64_t M, int64_t N, int64_t K, int out_dtype) {
  need(M >= 0 && N >= 1 && K >= 1, "need M >= 0, N >= 1 and K >= 1");
  need(M <= (int64_t(1) << 30) && N <= 65535ll * 32 && K <= (int64_t(1) << 30), "a dimension is too large");
  need(out_dtype >= VDK_FP16 && out_dtype <= VDK_FP32, "out_dtype must be VDK_FP16, VDK_BF16 or VDK_FP32");
}

extern "C" VD_API int vdk_fp8_linear_plan(int64_t M, int64_t N, int64_t K, int out_dtype, int* tile_rows, int* splits,
                                          int* stages, char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need_f8_shape(M, N, K, out_dtype);
    need(M >= 1 && tile_rows && splits && stages, "need rows and somewhere to put the answer");
    F8Shape s{};
    s.M = static_cast<int>(M), s.N = static_cast<int>(N), s.K = static_cast<int>(K);
    by_type(out_dtype, [&](auto tag) {
      const F8Choice c = choose_f8<decltype(tag)>(s);
      *tile_rows = c.bn;
      *splits = c.bn ? c.rows.splits : 1;
      *stages = c.bn ? c.rows.stages : F8PairConfig::STAGES;
    });
  });
}

static int fp8_linear(const void* a, int64_t ld_a, const float* a_scale, int64_t ld_a_scale, const void* w, int64_t ld_w,
                      const float* w_scale, int64_t ld_w_scale, int64_t M, int64_t N, int64_t K, const float* bias,
                      void* out, int64_t ld_out, int out_dtype, int* status, uint64_t wait_ns, int stall_after,
                      void* stream, char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need_f8_shape(M, N, K, out_dtype);
    const int64_t kb = (K + 127) / 128;
    need(ld_a >= K && ld_w >= K && ld_out >= N && ld_a_scale >= kb && ld_w_scale >= kb,
         "a row stride is smaller than its row");
    if (M == 0) return;
    need(a && w && a_scale && w_scale && out, "null buffer");
    need(aligned16(a) && ld_a % 16 == 0 && aligned16(w) && ld_w % 16 == 0,
         "rows of a and w must start on 16-byte boundaries");
    need_aligned(a_scale, "a_scale");
    need_aligned(w_scale, "w_scale");
    need_aligned(bias, "bias");
    need_aligned(out, out_dtype, "out");
    need_aligned(status, "status");
    const ByteRows mo = matrix(out, M, N, ld_out, out_dtype);
    need_apart(mo, matrix(a, M, K, ld_a, VDK_FP8), "out and a");
    need_apart(mo, matrix(w, N, K, ld_w, VDK_FP8), "out and w");
    need_apart(mo, matrix(a_scale, M, kb, ld_a_scale, VDK_FP32), "out and a_scale");
    need_apart(mo, matrix(w_scale, (N + 127) / 128, kb, ld_w_scale, VDK_FP32), "out and w_scale");
    need_apart(mo, ByteRows(bias, 4 * N), "out and bias");
    need_apart(mo, ByteRows(status, 4), "out and status");
    F8Shape s{};
    s.M = static_cast<int>(M), s.N = static_cast<int>(N), s.K = static_cast<int>(K);
    s.sa = a_scale, s.sw = w_scale;
    s.ld_sa = ld_a_scale, s.ld_sw = ld_w_scale;
    s.bias = bias;
    s.out = out;
    s.ld_out = ld_out;
    s.out_aligned = rows16(out, ld_out, out_dtype);
    s.wait_ns = wait_ns;
    s.stall_after = stall_after;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    by_type(out_dtype, [&](auto tag) {
      using O = decltype(tag);
      const F8Choice c = choose_f8<O>(s);
      switch (c.bn) {
        case 16: return launch_f8_rows<16, O>(a, ld_a, w, ld_w, s, c.rows, status, st);
        case 32: return launch_f8_rows<32, O>(a, ld_a, w, ld_w, s, c.rows, status, st);
        case 64: return launch_f8_rows<64, O>(a, ld_a, w, ld_w, s, c.rows, status, st);
        case 128: return launch_f8_rows<128, O>(a, ld_a, w, ld_w, s, c.rows, status, st);
        default: return launch_f8_pair<O>(a, ld_a, w, ld_w, s, out_dtype, status, st);
      }
    });
  });
}

extern "C" VD_API int vdk_fp8_linear(const void* a, int64_t ld_a, const float* a_scale, int64_t ld_a_scale,
                                     const void* w, int64_t ld_w, const float* w_scale, int64_t ld_w_scale, int64_t M,
                                     int64_t N, int64_t K, const float* bias, void* out, int64_t ld_out, int out_dtype,
                                     int* status, void* stream, char* err, size_t errlen) {
  return fp8_linear(a, ld_a, a_scale, ld_a_scale, w, ld_w, w_scale, ld_w_scale, M, N, K, bias, out, ld_out, out_dtype,
                    status, VD_WAIT_TIMEOUT_NS, -1, stream, err, errlen);
}

extern "C" VD_API int vdk_fp8_linear_stalled(const void* a, int64_t ld_a, const float* a_scale, int64_t ld_a_scale,
                                             const void* w, int64_t ld_w, const float* w_scale, int64_t ld_w_scale,
                                             int64_t M, int64_t N, int64_t K, const float* bias, void* out,
                                             int64_t ld_out, int out_dtype, int* status, int64_t wait_limit_us,
                                             int stall_after, void* stream, char* err, size_t errlen) {
  const int rc = guarded_call(err, errlen, [&] {
    need(wait_limit_us >= 1 && wait_limit_us <= 2000000 && stall_after >= -1,
         "need 1 <= wait_limit_us <= 2e6 and stall_after >= -1");
  });
  if (rc != VD_OK) return rc;
  return fp8_linear(a, ld_a, a_scale, ld_a_scale, w, ld_w, w_scale, ld_w_scale, M, N, K, bias, out, ld_out, out_dtype,
                    status, static_cast<uint64_t>(wait_limit_us) * 1000, stall_after, stream, err, errlen);
}

extern "C" VD_API int vdk_block_norm(const void* y, int64_t ld_y, int y_dtype, const void* h, int64_t ld_h, int h_dtype,
                                     const float* post_gain, const void* gate, int gate_dtype, int64_t gate_row_stride,
                                     int64_t gate_col_stride, float residual_scale, float block_scale,
                                     const float* pre_gain, float eps, int plus_one, int64_t rows, int64_t cols,
                                     void* h_out, int64_t ld_h_out, void* z, int64_t ld_z, int z_dtype, float* z_scale,
                                     int64_t ld_z_scale, void* stream, char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need(rows >= 0 && rows <= kMaxInt && cols >= 1 && cols <= VDK_NORM_MAX_COLS,
         "need 0 <= rows < 2^31 and 1 <= cols <= VDK_NORM_MAX_COLS");
    need(y_dtype >= VDK_FP16 && y_dtype <= VDK_FP32, "y_dtype must be VDK_FP16, VDK_BF16 or VDK_FP32");
    need(h_dtype == VDK_FP32 || h_dtype == y_dtype, "h_dtype must be VDK_FP32 or y's type");
    need(!gate || gate_dtype == VDK_FP32 || gate_dtype == y_dtype, "gate_dtype must be VDK_FP32 or y's type");
    need(!gate || ((gate_col_stride == 0 || gate_col_stride == 1) && gate_row_stride >= 0),
         "gate strides: 0 or 1 between columns, not negative between rows");
    need(y || (!post_gain && !gate), "post_gain and gate need y");
    need(std::isfinite(residual_scale) && std::isfinite(block_scale) && eps >= 0.0f && std::isfinite(eps),
         "scales must be finite and eps finite and not negative");
    need(!z == !pre_gain, "z and pre_gain come together");
    need(!z || (z_dtype >= VDK_FP16 && z_dtype <= VDK_FP8), "z_dtype must be VDK_FP16, VDK_BF16, VDK_FP32 or VDK_FP8");
    const int64_t kb = (cols + 127) / 128;
    need((!y || ld_y >= cols) && (!h || ld_h >= cols) && (!h_out || ld_h_out >= cols) && (!z || ld_z >= cols),
         "a row stride is smaller than its row");
    if (rows == 0) return;
    need(y || h, "need a block output or a residual");
    need(h_out || z, "nothing to write");
    need(!z || z_dtype != VDK_FP8 || (z_scale && ld_z_scale >= kb), "8-bit z needs z_scale with a row per token");
    need_aligned(y, y_dtype, "y");
    need_aligned(h, h_dtype, "h");
    need_aligned(gate, gate_dtype, "gate");
    need_aligned(post_gain, "post_gain");
    need_aligned(pre_gain, "pre_gain");
    need_aligned(h_out, h_dtype, "h_out");
    need_aligned(z, z_dtype, "z");
    need_aligned(z_scale, "z_scale");
    // y, h and a gate with a value per element are read by the thread that
    // writes the same element: an output may be one of them.
    const ByteRows my = matrix(y, rows, cols, ld_y, y_dtype), mh = matrix(h, rows, cols, ld_h, h_dtype),
                   mg = matrix(gate, rows, gate_col_stride ? cols : 1, gate_row_stride, gate_dtype),
                   mo = matrix(h_out, rows, cols, ld_h_out, h_dtype), mz = matrix(z, rows, cols, ld_z, z_dtype),
                   ms = matrix(z && z_dtype == VDK_FP8 ? z_scale : nullptr, rows, kb, ld_z_scale, VDK_FP32);
    for (const ByteRows* o : {&mo, &mz, &ms}) {
      if (!o->p) continue;
      need_apart(*o, my, "an output and y", o != &ms);
      need_apart(*o, mh, "an output and h", o != &ms);
      need_apart(*o, mg, "an output and gate", o != &ms && gate_col_stride);
      need_apart(*o, ByteRows(post_gain, 4 * cols), "an output and post_gain");
      need_apart(*o, ByteRows(pre_gain, 4 * cols), "an output and pre_gain");
    }
    need_apart(mo, mz, "h_out and z");
    need_apart(mo, ms, "h_out and z_scale");
    need_apart(mz, ms, "z and z_scale");
    BlockNormParams p{};
    p.y = y, p.h = h, p.post = post_gain, p.gate = gate;
    p.gate_f32 = gate_dtype == VDK_FP32;
    p.gate_row = gate_row_stride, p.gate_col = gate_col_stride;
    p.pre = pre_gain, p.h_out = h_out, p.z = z, p.z_scale = z_scale;
    p.ld_y = ld_y, p.ld_h = ld_h, p.ld_h_out = ld_h_out, p.ld_z = ld_z, p.ld_scale = ld_z_scale;
    p.cols = static_cast<int>(cols);
    p.out = !z ? kNormOutNone
               : z_dtype == VDK_FP16 ? kNormOutF16
               : z_dtype == VDK_BF16 ? kNormOutBF16
               : z_dtype == VDK_FP32 ? kNormOutF32
                                     : kNormOutF8;
    p.residual_scale = residual_scale, p.block_scale = block_scale, p.eps = eps;
    p.gain_add = plus_one ? 1.0f : 0.0f;
    // Four columns a thread and step; few steps for short rows (latency), up to
    // eight for long ones (at most 512 threads).
    const int chunks = static_cast<int>((cols + 3) / 4);
    const int nv = chunks <= 256 ? 1 : chunks <= 512 ? 2 : chunks <= 1280 ? 4 : 8;
    const int threads = ((chunks + nv - 1) / nv + 31) / 32 * 32;
    const bool full =
        cols == 4ll * nv * threads && (!y || rows16(y, ld_y, y_dtype)) && (!h || rows16(h, ld_h, h_dtype)) &&
        (!h_out || rows16(h_out, ld_h_out, h_dtype)) && aligned16(post_gain) && aligned16(pre_gain) &&
        (!gate || gate_col_stride == 0 || rows16(gate, gate_row_stride, gate_dtype)) &&
        (!z || (z_dtype == VDK_FP8 ? (reinterpret_cast<uintptr_t>(z) & 3) == 0 && ld_z % 4 == 0 : rows16(z, ld_z, z_dtype)));
    const unsigned grid = static_cast<unsigned>(rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    by_type(y_dtype, [&](auto ty) {
      using TY = decltype(ty);
      auto run = [&](auto th) {
        using TH = decltype(th);
        auto go = [&](auto k) { k<<<grid, threads, 0, s>>>(p); };
        if (!full) {
          if (nv == 1) go(block_norm_kernel<TY, TH, 1, false>);
          else if (nv == 2) go(block_norm_kernel<TY, TH, 2, false>);
          else if (nv == 4) go(block_norm_kernel<TY, TH, 4, false>);
          else go(block_norm_kernel<TY, TH, 8, false>);
        } else {
          if (nv == 1) go(block_norm_kernel<TY, TH, 1, true>);
          else if (nv == 2) go(block_norm_kernel<TY, TH, 2, true>);
          else if (nv == 4) go(block_norm_kernel<TY, TH, 4, true>);
          else go(block_norm_kernel<TY, TH, 8, true>);
        }
      };
      if (h_dtype == VDK_FP32) run(float());
      else run(TY());
    });
    launched();
  });
}

extern "C" VD_API int vdk_rotary_turns(double theta, int rotary_dim, int scaling, const double* args,
                                       const double* divisors, uint64_t* turns, float* factor, char* err,
                                       size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= VDK_ROTARY_MAX_DIM,
         "rotary_dim must be even, from 2 to VDK_ROTARY_MAX_DIM");
    need(std::isfinite(theta) && theta > 0.0, "theta must be positive");
    need(scaling >= VDK_ROPE_NONE && scaling <= VDK_ROPE_DIVISORS, "unknown scaling");
    need(turns && factor, "null buffer");
    need(scaling == VDK_ROPE_NONE || args, "the scaling needs its arguments");
    need(scaling != VDK_ROPE_DIVISORS || divisors, "the scaling needs one divisor per pair");
    // A turn in 64 bits wants more than a double's 53 at every step up to it:
    // the position multiplies what is lost here.
    using real = long double;
#ifndef __CUDA_ARCH__
    static_assert(std::numeric_limits<real>::digits >= 64, "the turns need 64 bits");
#endif
    const real two_pi = 6.283185307179586476925286766559005768L;
    const int half = rotary_dim / 2;
    const double d = rotary_dim;
    double m = 1.0;
    real base = theta;
    const double f = scaling != VDK_ROPE_NONE ? args[0] : 1.0;
    if (scaling != VDK_ROPE_NONE && scaling != VDK_ROPE_DIVISORS)
      need(std::isfinite(f) && f >= 1.0, "the scaling factor must be at least 1");
    double lo = 0.0, hi = 0.0;
    if (scaling == VDK_ROPE_NTK) {
      need(rotary_dim > 2, "this scaling needs rotary_dim > 2");
      base = theta * std::pow(static_cast<real>(f), static_cast<real>(d) / (d - 2.0));
    } else if (scaling == VDK_ROPE_YARN) {
      const double orig = args[1], fast = args[2], slow = args[3];
      need(orig > 0.0 && fast > slow && slow > 0.0, "need original_max_position > 0 and beta_fast > beta_slow > 0");
      need(theta != 1.0, "this scaling needs theta != 1");
      auto dim = [&](double turns_over) {
        return d * std::log(orig / (turns_over * static_cast<double>(two_pi))) / (2.0 * std::log(theta));
      };
      lo = std::max(std::floor(dim(fast)), 0.0);
      hi = std::min(std::ceil(dim(slow)), d - 1.0);
      m = args[4] > 0.0 ? args[4] : 0.1 * std::log(f) + 1.0;
    } else if (scaling == VDK_ROPE_LLAMA3) {
      need(args[1] > 0.0 && args[3] > args[2], "need original_max_position > 0 and high_freq_factor > low_freq_factor");
    } else if (scaling == VDK_ROPE_DIVISORS) {
      m = args[0];
      need(std::isfinite(m) && m > 0.0, "the factor on the rotated values must be positive");
    }
    const real zero = 0, one = 1;
    for (int i = 0; i < half; ++i) {
      real r = std::pow(base, static_cast<real>(-2 * i) / rotary_dim);  // radians per position
      if (scaling == VDK_ROPE_LINEAR) {
        r /= f;
      } else if (scaling == VDK_ROPE_YARN) {
        const real ramp = std::min(std::max((i - static_cast<real>(lo)) / std::max(hi - lo, 0.001), zero), one);
        r = r / f * ramp + r * (one - ramp);
      } else if (scaling == VDK_ROPE_LLAMA3) {
        const real t = std::min(std::max((args[1] * r / two_pi - args[2]) / (args[3] - args[2]), zero), one);
        r = (one - t) * r / f + t * r;
      } else if (scaling == VDK_ROPE_DIVISORS) {
        need(std::isfinite(divisors[i]) && divisors[i] > 0.0, "divisors must be positive");
        r /= divisors[i];
      }
      const real t = r / two_pi;
      const real scaled = std::round(std::ldexp(t - std::floor(t), 64));
      turns[i] = scaled < std::ldexp(one, 64) ? static_cast<uint64_t>(scaled) : 0;  // rounded up to a whole turn
    }
    *factor = static_cast<float>(m);
  });
}

extern "C" VD_API int vdk_rotary(const vdk_rotary_heads* q, const vdk_rotary_heads* k, int64_t tokens, int head_dim,
                                 int rotary_dim, int dtype, int interleaved, int inverse, const void* positions,
                                 int positions_bits, int64_t first_position, const uint64_t* turns, float factor,
                                 void* stream, char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need(tokens >= 0 && tokens <= (int64_t(1) << 32), "need 0 <= tokens <= 2^32");
    need(head_dim >= 2 && head_dim <= 65536 && rotary_dim >= 2 && rotary_dim <= head_dim && rotary_dim % 2 == 0 &&
             rotary_dim <= VDK_ROTARY_MAX_DIM,
         "rotary_dim must be even, from 2 to head_dim and to VDK_ROTARY_MAX_DIM");
    need(!positions || positions_bits == 32 || positions_bits == 64, "positions are 32- or 64-bit");
    need(q || k, "need queries or keys");
    need(std::isfinite(factor), "factor must be finite");
    RotaryParams p{};
    const int es = elem_bytes(dtype);
    bool vec = rotary_dim % 8 == 0 && (head_dim - rotary_dim) % 8 == 0 && (interleaved || rotary_dim % 16 == 0);
    int64_t heads = 0;
    auto fill = [&](const vdk_rotary_heads* v, RotaryHeads& r) {
      if (!v) return;
      need(v->heads >= 1 && v->heads <= 65536, "heads must be from 1 to 65536");
      need(tokens == 0 || (v->in && v->out), "null buffer");
      need_aligned(v->in, dtype, "heads");
      need_aligned(v->out, dtype, "output heads");
      need(v->in_token >= 0 && v->in_head >= 0 && v->out_token >= 0 && v->out_head >= 0, "negative stride");
      // Output rows of head_dim lie apart: heads within a token, or tokens within a head.
      const int64_t hs = v->out_head, ts = v->out_token;
      need((v->heads == 1 || hs >= head_dim) && (tokens <= 1 || ts >= head_dim) &&
               (v->heads == 1 || tokens <= 1 || ts / v->heads >= hs || hs / tokens >= ts),
           "output heads overlap");
      r = {v->in, v->out, v->in_token, v->in_head, v->out_token, v->out_head, v->heads};
      for (const int64_t st : {v->in_token, v->in_head, v->out_token, v->out_head}) vec = vec && st * es % 16 == 0;
      vec = vec && aligned16(v->in) && aligned16(v->out);
      heads += v->heads;
    };
    fill(q, p.q);
    fill(k, p.k);
    need(heads * head_dim <= (int64_t(1) << 28), "too many heads");
    if (tokens == 0) return;
    need(turns != nullptr, "null buffer");
    need_aligned(turns, "turns");
    need(reinterpret_cast<uintptr_t>(positions) % (positions_bits == 64 ? 8 : 4) == 0,
         "positions are not aligned to their type");
    const int64_t row = static_cast<int64_t>(head_dim) * es;
    const auto rows_in = [&](const vdk_rotary_heads* v) {
      return v ? ByteRows(v->in, row, tokens, v->in_token * es, v->heads, v->in_head * es) : ByteRows();
    };
    const auto rows_out = [&](const vdk_rotary_heads* v) {
      return v ? ByteRows(v->out, row, tokens, v->out_token * es, v->heads, v->out_head * es) : ByteRows();
    };
    const ByteRows q_in = rows_in(q), k_in = rows_in(k), q_out = rows_out(q), k_out = rows_out(k);
    need_apart(q_out, q_in, "queries and their output", true);
    need_apart(k_out, k_in, "keys and their output", true);
    need_apart(q_out, k_in, "keys and the queries' output");
    need_apart(k_out, q_in, "queries and the keys' output");
    need_apart(q_out, k_out, "the outputs");
    for (const ByteRows* o : {&q_out, &k_out}) {
      need_apart(*o, ByteRows(positions, tokens * (positions_bits / 8)), "an output and positions");
      need_apart(*o, ByteRows(turns, rotary_dim / 2 * 8), "an output and turns");
    }
    p.positions = positions;
    p.positions64 = positions_bits == 64;
    p.first_position = first_position;
    p.tokens = tokens;
    p.turns = turns;
    p.head_dim = head_dim, p.rotary_dim = rotary_dim, p.interleaved = interleaved != 0;
    p.factor = factor;
    p.sin_sign = inverse ? -1.0f : 1.0f;
    const int width = vec ? 8 : 1;
    p.rot_units = vec && interleaved ? rotary_dim / 8 : rotary_dim / 2 / width;
    p.units = p.rot_units + (head_dim - rotary_dim) / width;
    p.per_token = FastDiv(static_cast<uint32_t>(heads * p.units));
    p.per_head = FastDiv(static_cast<uint32_t>(p.units));
    const unsigned grid = static_cast<unsigned>((tokens + kRotaryTokens - 1) / kRotaryTokens);
    const size_t smem = kRotaryTokens * (rotary_dim / 2) * sizeof(float2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    by_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      if (vec) rotary_kernel<T, true><<<grid, kRotaryThreads, smem, s>>>(p);
      else rotary_kernel<T, false><<<grid, kRotaryThreads, smem, s>>>(p);
    });
    launched();
  });
}

extern "C" VD_API int vdk_token_logprobs(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int dtype,
                                         float temperature, const int64_t* targets, int64_t n_targets, int top,
                                         float* logprobs, float* entropy, float* lse, int32_t* top_ids,
                                         float* top_logprobs, void* stream, char* err, size_t errlen) {
  return guarded_call(err, errlen, [&] {
    need(rows >= 0 && rows <= kMaxInt / 8 && vocab >= 1 && vocab <= kMaxInt - 65536,
         "need 0 <= rows < 2^28 and 1 <= vocab < 2^31 - 65536");
    need(ld >= vocab, "a row stride is smaller than its row");
    need(std::isfinite(temperature) && temperature > 0.0f &&
             std::isfinite(static_cast<float>(1.4426950408889634 / temperature)),
         "temperature must be positive (at least 4.3e-39)");
    need(top >= 0 && top <= VDK_LOGPROBS_MAX_TOP, "top must be from 0 to VDK_LOGPROBS_MAX_TOP");
    need(n_targets >= 0 && n_targets <= kMaxInt, "n_targets must not be negative");
    if (rows == 0) return;
    need(logits != nullptr, "null buffer");
    need(n_targets == 0 || (targets && logprobs), "targets need their ids and an output");
    need(top == 0 || (top_ids && top_logprobs), "alternatives need their outputs");
    need_aligned(logits, dtype, "logits");
    need_aligned(targets, "targets");
    need_aligned(logprobs, "logprobs");
    need_aligned(entropy, "entropy");
    need_aligned(lse, "lse");
    need_aligned(top_ids, "top_ids");
    need_aligned(top_logprobs, "top_logprobs");
    const ByteRows outs[] = {ByteRows(n_targets ? logprobs : nullptr, rows * n_targets * 4), ByteRows(entropy, rows * 4),
                             ByteRows(lse, rows * 4), ByteRows(top ? top_ids : nullptr, rows * top * 4),
                             ByteRows(top ? top_logprobs : nullptr, rows * top * 4)};
    for (int i = 0; i < 5; ++i) {
      need_apart(outs[i], matrix(logits, rows, vocab, ld, dtype), "an output and logits");
      need_apart(outs[i], ByteRows(n_targets ? targets : nullptr, rows * n_targets * 8), "an output and targets");
      for (int j = 0; j < i; ++j) need_apart(outs[i], outs[j], "two outputs");
    }
    static_assert(VDK_LOGPROBS_MAX_TOP == kLpMaxTop, "");
    LogprobParams p{};
    p.logits = logits;
    p.ld = ld, p.rows = rows;
    p.vocab = static_cast<int>(vocab);
    p.targets = targets;
    p.n_targets = static_cast<int>(n_targets);
    p.top = top;
    p.inv_temperature = 1.0f / temperature;
    p.logprobs = logprobs, p.entropy = entropy, p.lse = lse, p.top_ids = top_ids, p.top_logprobs = top_logprobs;
    // CTAs share a row while all of them still run at once and each keeps a
    // batch of loads (kLpThreads * kLpUnroll * 16 bytes): joining them costs more
    // than idle SMs do (1024 x 256000 bf16: 134 us with one CTA a row, 159 with
    // two, 203 with four; 512 x 50369: 39 with two).
    p.splits = 1;
    const int64_t bytes = vocab * elem_bytes(dtype);
    while (p.splits < kLpMaxSplits && rows * p.splits * 2 <= kLpCtasPerSm * sm_count() &&
           bytes / (p.splits * 2) >= 16384)
      p.splits *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    by_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      launch(token_logprobs_kernel<T>, dim3(static_cast<unsigned>(rows * p.splits)), kLpThreads, sizeof(LpShared),
             p.splits, false, s, p);
    });
  });
}
