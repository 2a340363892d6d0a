/*
 * vdexec kernel-level entry points: the individual sm_100a kernels of the
 * decision forward on caller-owned DEVICE buffers, for composing other
 * forwards and for testing each kernel against a reference implementation.
 *
 * These have no single counterpart in the reference (which runs cuBLAS / SDPA
 * through torch, executor/torch_exec.py:205-261); each entry names the torch op
 * it replaces.  Calls are synchronous on `stream` (a cudaStream_t, or NULL for
 * the legacy default stream) unless said otherwise, and return 0 or a negative VD_E* code from
 * vdexec.h with a message in err.
 */
#ifndef VDEXEC_KERNELS_H_
#define VDEXEC_KERNELS_H_

#include <stddef.h>
#include <stdint.h>

#include "vdexec.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Epilogues of vdk_gemm. */
#define VDK_EPI_STORE 0     /* out = act(A W^T + bias), 16-bit                                     */
#define VDK_EPI_RESIDUAL 1  /* out_f32 += A W^T + bias                                              */
#define VDK_EPI_GATED 2     /* out[:, j] = act(g_j) * u_j, 16-bit; W rows interleaved in 128-row blocks */
#define VDK_EPI_QKROPE 3    /* per-head q/k RMSNorm + rotary embedding (see vdk_gemm_qkrope)   */

/* 16-bit element types of A, W, qkv and 16-bit outputs. */
#define VDK_FP16 0
#define VDK_BF16 1
/* Further types of the 8-bit decoder operators below. */
#define VDK_FP32 2
#define VDK_FP8 3 /* e4m3 (4 exponent bits, 3 mantissa bits, no infinities), with fp32 scales beside it */

/* Activations. */
#define VDK_ACT_NONE 0
#define VDK_ACT_GELU_ERF 1
#define VDK_ACT_GELU_TANH 2
#define VDK_ACT_RELU 3
#define VDK_ACT_SILU 4

/*
 * tcgen05 GEMM: A [M, K] row-major, W [N, K] row-major (nn.Linear weight
 * layout), both of the 16-bit type `dtype`, fp32 accumulation; replaces
 * torch.nn.functional.linear.  N % 128 == 0 (N % 256 == 0 for
 * VDK_EPI_GATED), K % 64 == 0.
 * out: dtype [M, ld_out] (store, gated) or fp32 [M, ld_out] (residual).
 */
VD_API int vdk_gemm(const void* A, const void* W, int64_t M, int64_t N, int64_t K, int dtype, int epi, int act,
                    const float* bias, void* out, int64_t ld_out, void* stream, char* err, size_t errlen);

/*
 * QKV projection with the attention-input epilogue: columns [0, q_cols) are
 * query heads and [q_cols, q_cols + k_cols) key heads of size head_dim (128 or
 * 256); each gets the optional bias, the optional per-head RMSNorm with gains
 * q_norm / k_norm (NULL: none; plus_one: gain = 1 + w) and the rotary embedding
 * at positions[m] with base theta; the remaining columns (values) are stored as
 * they are.  Replaces q_norm(q_proj(x)) / k_norm(k_proj(x)) + apply_rotary_pos_emb.
 */
VD_API int vdk_gemm_qkrope(const void* A, const void* W, int64_t M, int64_t N, int64_t K, int dtype, const float* bias,
                           const float* q_norm, const float* k_norm, int q_cols, int k_cols, int head_dim,
                           int plus_one, float eps, const int32_t* positions, double theta, int max_pos, void* out,
                           int64_t ld_out, void* stream, char* err, size_t errlen);

/*
 * Varlen attention over packed rows.  qkv [T, ld_qkv] (16-bit dtype) holds query head h
 * at column q_col0 + h*head_dim and K/V head g at k_col0 / v_col0 + g*head_dim
 * (g = h / (heads / kv_heads)); cu_seqlens_host [nseq + 1] (host) delimits the
 * sequences; out [T, ld_out] (dtype) at column h*head_dim.  causal = 1 for
 * decoders.  Replaces F.scaled_dot_product_attention (is_causal) per sequence.
 */
VD_API int vdk_attention(const void* qkv, int64_t ld_qkv, int64_t q_col0, int64_t k_col0, int64_t v_col0, int heads,
                         int kv_heads, int head_dim, int dtype, int causal, const int32_t* cu_seqlens_host,
                         int64_t nseq, void* out, int64_t ld_out, void* stream, char* err, size_t errlen);

/*
 * The same attention on the 5th-generation tensor cores (tcgen05 MMAs with
 * TMEM accumulators, TMA-fed), causal with head_dim 128 or 256 or
 * bidirectional with head_dim 64, one query head per CTA, 128-row query tiles
 * and 64-key tiles; the kernel the engine uses for decoders with those head
 * sizes and for the marker-head encoders.  Same arguments and result as
 * vdk_attention; strides and column offsets multiples of 8.
 */
VD_API int vdk_attention_tc(const void* qkv, int64_t ld_qkv, int64_t q_col0, int64_t k_col0, int64_t v_col0,
                            int heads, int kv_heads, int head_dim, int dtype, int causal,
                            const int32_t* cu_seqlens_host, int64_t nseq, void* out, int64_t ld_out, void* stream,
                            char* err, size_t errlen);

/*
 * vdk_attention with no allocation of its own.  It has no counterpart in the
 * reference; it exists for callers that must not call cudaMalloc: a host
 * process whose GPU memory is entirely owned by another allocator (a serving
 * framework's caching pool that reserves the HBM budget up front), or a
 * latency-critical path where cudaMalloc/cudaFree would block on the device.
 *
 * Same arguments and results as vdk_attention.  The per-call work table (one
 * entry per 64-row query tile) lives in a fixed device array of 16384 entries
 * (512 KiB) that every GPU loading this library keeps until the process
 * exits; a batch needing more tiles (sum over sequences of ceil(len / 64)) is
 * rejected with VD_EINVAL before anything is launched.
 * The first call on a device looks up that array's device address (with the
 * device current) and keeps it; make that first call before any stream
 * capture.  All calls in a process share the one array per GPU and it keeps
 * the last call's contents; calls that overlapped on the GPU would race on it,
 * so each call holds a process-wide lock until its kernel has finished.  Every
 * entry a call reads is written by that same call, so nothing needs clearing.
 */
VD_API int vdk_attention_noalloc(const void* qkv, int64_t ld_qkv, int64_t q_col0, int64_t k_col0, int64_t v_col0,
                                 int heads, int kv_heads, int head_dim, int dtype, int causal,
                                 const int32_t* cu_seqlens_host, int64_t nseq, void* out, int64_t ld_out,
                                 void* stream, char* err, size_t errlen);

/*
 * The 8-bit decoder operators: what a decoder layer on 8-bit weights consists
 * of besides attention, and its readout over the whole vocabulary.  They have
 * no counterpart in the reference.  Unlike the entries above they only
 * enqueue work on `stream` and return: no allocation, no wait, usable under
 * stream capture.  Buffers belong to the current device and must stay valid
 * until the work has run.  Arguments are checked before anything is launched
 * (VD_EINVAL); zero rows are no work and no error.  Strides count elements.
 * Outputs share no memory with each other or with inputs, save where an entry
 * says that one may be the same rows as an input.
 */

/*
 * Activations to e4m3 with a scale per row and 128 columns: with v = x, or
 * v = act(gate) * x where gate is given, and a = max(max |v|, 1e-30) of the
 * block,  scale = a / 448,  q = e4m3(v * (448 / a)), rounded to nearest even.
 * A block with inf or NaN has that as its scale.  x, gate [rows, cols] of
 * `dtype` (VDK_FP16 / BF16 / FP32); q [rows, cols] bytes; scale
 * [rows, ceil(cols / 128)].
 */
VD_API int vdk_quantize_fp8(const void* x, int64_t ld_x, const void* gate, int64_t ld_gate, int act, int64_t rows,
                            int64_t cols, int dtype, void* q, int64_t ld_q, float* scale, int64_t ld_scale,
                            void* stream, char* err, size_t errlen);

/* The same for weights [rows, cols], a scale per 128 x 128 block: scale [ceil(rows / 128), ceil(cols / 128)]. */
VD_API int vdk_quantize_fp8_weight(const void* w, int64_t ld_w, int64_t rows, int64_t cols, int dtype, void* q,
                                   int64_t ld_q, float* scale, int64_t ld_scale, void* stream, char* err,
                                   size_t errlen);

/*
 * out[m, n] = sum_b a_scale[m, b] w_scale[n / 128, b] (sum_{k in b} a[m, k] w[n, k]) + bias[n]
 * over blocks b of 128 columns, e4m3 operands, fp32 sums; a [M, K] and w
 * [N, K] as the casts above lay them out, rows starting on 16-byte boundaries;
 * any M, N and K.  out [M, N] of out_dtype (VDK_FP16 / BF16 / FP32); bias fp32
 * or NULL.  status: a device int or NULL; a pipeline wait that runs out (2 s)
 * ends the kernel and stores its code there if it holds 0.
 */
VD_API int vdk_fp8_linear(const void* a, int64_t ld_a, const float* a_scale, int64_t ld_a_scale, const void* w,
                          int64_t ld_w, const float* w_scale, int64_t ld_w_scale, int64_t M, int64_t N, int64_t K,
                          const float* bias, void* out, int64_t ld_out, int out_dtype, int* status, void* stream,
                          char* err, size_t errlen);

/*
 * How vdk_fp8_linear runs a product on the current device: tokens in a tile (0:
 * CTA pairs on tiles of 256 x 256), CTAs that share K, and stages of the
 * shared-memory ring.  Nothing is launched.
 */
VD_API int vdk_fp8_linear_plan(int64_t M, int64_t N, int64_t K, int out_dtype, int* tile_rows, int* splits, int* stages,
                               char* err, size_t errlen);

/*
 * Failure-path tests only: vdk_fp8_linear with a limit of its own on every pipeline
 * wait, and with each CTA's loads stopping after stall_after blocks of 128
 * columns (-1: never).  Where they stop early, a wait runs out: the kernel
 * ends, status has the wait's code and out is not to be used.
 */
VD_API int vdk_fp8_linear_stalled(const void* a, int64_t ld_a, const float* a_scale, int64_t ld_a_scale, const void* w,
                                  int64_t ld_w, const float* w_scale, int64_t ld_w_scale, int64_t M, int64_t N,
                                  int64_t K, const float* bias, void* out, int64_t ld_out, int out_dtype, int* status,
                                  int64_t wait_limit_us, int stall_after, void* stream, char* err, size_t errlen);

/*
 * The step between two blocks of a decoder, one pass:
 *   u = rmsnorm(y) * post_gain, or y without post_gain;
 *   h_out = residual_scale * h + block_scale * gate * u;
 *   z = rmsnorm(h_out) * pre_gain.
 * rmsnorm(x) = x / sqrt(mean(x^2) + eps); plus_one: gains are 1 + gain.
 * y (VDK_FP16 / BF16 / FP32, or NULL: u = 0), h (fp32 or y's type, or NULL:
 * 0), gate (fp32 or y's type, or NULL: 1) with strides that may be 0 to
 * broadcast (columns: 0 or 1); h_out has h's type (NULL: not stored); h_out or
 * z may be the rows of h, y or a gate with a value per element.  z is VDK_FP16,
 * BF16, FP32 or FP8; FP8 comes with z_scale [rows, ceil(cols / 128)] as
 * vdk_quantize_fp8 gives it; z and pre_gain NULL: no second norm.  z is formed
 * in fp32 from h_out before that is rounded.
 */
#define VDK_NORM_MAX_COLS 16384
VD_API int vdk_block_norm(const void* y, int64_t ld_y, int y_dtype, const void* h, int64_t ld_h, int h_dtype,
                          const float* post_gain, const void* gate, int gate_dtype, int64_t gate_row_stride,
                          int64_t gate_col_stride, float residual_scale, float block_scale, const float* pre_gain,
                          float eps, int plus_one, int64_t rows, int64_t cols, void* h_out, int64_t ld_h_out, void* z,
                          int64_t ld_z, int z_dtype, float* z_scale, int64_t ld_z_scale, void* stream, char* err,
                          size_t errlen);

/*
 * Rotary frequencies for vdk_rotary: turns per position of each pair in 64-bit
 * fixed point (frequency / 2 pi * 2^64, whole turns dropped, within 4 units for
 * frequencies of up to one radian) and the factor on the rotated values.  Host
 * only.  Pair i turns theta^(-2 i / rotary_dim)
 * radians per position, then by `scaling`:
 *   VDK_ROPE_LINEAR   args {factor}: divided by factor
 *   VDK_ROPE_NTK      args {factor}: theta * factor^(d / (d - 2)) as the base
 *   VDK_ROPE_YARN     args {factor, original_max_position, beta_fast,
 *                     beta_slow, factor on values (0: 0.1 ln(factor) + 1)}:
 *                     pairs that turn more than beta_fast times in the
 *                     original context keep their frequency, those below
 *                     beta_slow are divided by factor, a ramp between
 *   VDK_ROPE_LLAMA3   args {factor, original_max_position, low_freq_factor,
 *                     high_freq_factor}: the same by wavelength
 *   VDK_ROPE_DIVISORS args {factor on values}: pair i divided by divisors[i]
 */
#define VDK_ROPE_NONE 0
#define VDK_ROPE_LINEAR 1
#define VDK_ROPE_NTK 2
#define VDK_ROPE_YARN 3
#define VDK_ROPE_LLAMA3 4
#define VDK_ROPE_DIVISORS 5
#define VDK_ROTARY_MAX_DIM 1024
VD_API int vdk_rotary_turns(double theta, int rotary_dim, int scaling, const double* args, const double* divisors,
                            uint64_t* turns, float* factor, char* err, size_t errlen);

/* Heads of vdk_rotary: [tokens, heads, head_dim] with unit stride in a head; out may be in's rows. */
typedef struct vdk_rotary_heads {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;
  int32_t heads;
} vdk_rotary_heads;

/*
 * Rotary positions on query and key heads (either may be NULL): the pairs
 * (i, i + rotary_dim / 2), or (2i, 2i + 1) with interleaved, of the first
 * rotary_dim columns of each head turn by positions[token] * turns[i]
 * (inverse: back); the other columns are copied.  positions: device int32 or
 * int64, any value, or NULL: first_position + token; what turns[i] is off by is
 * multiplied by the position (2^-62 of a turn each: below fp32's rounding of
 * the cosines up to position 2^37).  turns: device.
 */
VD_API int vdk_rotary(const vdk_rotary_heads* q, const vdk_rotary_heads* k, int64_t tokens, int head_dim,
                      int rotary_dim, int dtype, int interleaved, int inverse, const void* positions,
                      int positions_bits, int64_t first_position, const uint64_t* turns, float factor, void* stream,
                      char* err, size_t errlen);

/*
 * Log probabilities over the whole vocabulary at a temperature: per row of
 * logits [rows, vocab] (VDK_FP16 / BF16 / FP32, row stride ld)
 *   logprobs [rows, n_targets] of targets (a negative id: 0; one past the
 *     vocabulary: NaN), entropy [rows] and lse [rows] (either may be NULL),
 *   top_ids, top_logprobs [rows, top]: the largest logits, equal ones by id.
 * -inf logits are masked: no probability, not listed (id -1, -inf past the
 * last).  A row with nothing else: logprobs and lse -inf, entropy 0.  A row
 * with NaN or +inf: NaN, ids -1.
 */
#define VDK_LOGPROBS_MAX_TOP 64
VD_API int vdk_token_logprobs(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int dtype,
                              float temperature, const int64_t* targets, int64_t n_targets, int top, float* logprobs,
                              float* entropy, float* lse, int32_t* top_ids, float* top_logprobs, void* stream,
                              char* err, size_t errlen);

#ifdef __cplusplus
}
#endif

#endif /* VDEXEC_KERNELS_H_ */
