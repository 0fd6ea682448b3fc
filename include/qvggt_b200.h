/*
 * qvggt_b200 -- C ABI of the B200 (sm_100a) kernels for QVGGT's quantised
 * transformer hot path.
 *
 * Every entry point takes raw device pointers, sizes and a CUDA stream
 * (cudaStream_t passed as void*; NULL = legacy default stream) and returns
 * QVGGT_OK or an error code; qvggt_last_error() gives the message of the last
 * failure on the calling thread.  Kernels are launched asynchronously on the
 * stream; nothing here synchronises.  Tensors are dense row-major unless a
 * stride argument says otherwise.  fp16 means IEEE binary16.
 *
 * Reference citations are paths inside the QVGGT repository
 * (E/ = qvggt/runtime/awq_inference_engine/csrc/).
 */
#ifndef QVGGT_B200_H
#define QVGGT_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QVGGT_OK 0
#define QVGGT_ERR_INVALID 1      /* bad shape or argument */
#define QVGGT_ERR_UNSUPPORTED 2  /* configuration the kernels do not implement */
#define QVGGT_ERR_CUDA 3         /* CUDA runtime / launch error */
#define QVGGT_ERR_TIMEOUT 4      /* a bounded device-side wait gave up */
#define QVGGT_ERR_ALIGN 5        /* pointer or stride not 16-byte aligned */

#define QVGGT_DTYPE_F16 0
#define QVGGT_DTYPE_BF16 1

/* Library version (major*10000 + minor*100 + patch). */
int qvggt_version(void);

/* Message of the last error returned on this thread ("" if none). */
const char* qvggt_last_error(void);

/* Device status word of the current device: 0, or the code of the first
 * bounded device-side wait that gave up since the last clear.  Synchronises
 * the current device.  clear != 0 resets the word to 0 afterwards. */
int qvggt_device_status(uint32_t* status_out, int clear);

/* Budget of every bounded device-side wait (default 2 s). */
int qvggt_set_wait_timeout_ns(uint64_t ns);

/* Number of kernels this library launched on this process (all devices). */
uint64_t qvggt_launch_count(void);

/* ---------------------------------------------------------------- W4A16 */

/* out[M, N] = in_feats[M, K] . deq(qweight)^T (+ bias), fp16 in / fp16 out,
 * fp32 accumulation (tcgen05, TMEM).  qweight int16 [N/4, K] in the AWQ
 * interleaved layout of pack_intweight(interleave=4, kstride=64);
 * scales / scaled_zeros fp16 [gpad, N], gpad >= K / group_size.
 * Requirements: N % 128 == 0, K % group_size == 0, group_size % 64 == 0.
 * bias may be NULL; with a bias the result is half(half(acc) + bias), the same
 * two roundings as the reference's GEMM followed by `out + self.bias`.
 * Replaces gemm_forward_cuda_new (E/quantization_new/gemm/gemm_cuda.cu:1125-1235,
 * bound at E/pybind.cpp:21) and the bias add of WQLinear.forward
 * (qvggt/runtime/awq/qmodule.py:361-367). */
int qvggt_w4a16_gemm(const void* in_feats, const void* qweight, const void* scales, const void* scaled_zeros,
                     const void* bias, void* out, int64_t M, int64_t N, int64_t K, int64_t gpad,
                     int32_t group_size, void* stream);

/* qvggt_w4a16_gemm with bf16 in_feats, scales, scaled_zeros, bias and out
 * (same qweight).  Dequantisation w = q * s + sz in one bf16x2 fma, bf16
 * operands on the tensor cores, fp32 accumulation, out = bf16(acc) (with a
 * bias: bf16(bf16(acc) + bias)).  Replaces the bf16 instantiation of
 * gemm_forward_cuda_new (E/quantization_new/gemm/gemm_cuda.cu:1146 dispatches
 * nv_bfloat16 through the same kernels; dequantize.cuh:53-90). */
int qvggt_w4a16_gemm_bf16(const void* in_feats, const void* qweight, const void* scales, const void* scaled_zeros,
                          const void* bias, void* out, int64_t M, int64_t N, int64_t K, int64_t gpad,
                          int32_t group_size, void* stream);

/* Same GEMM with a fused epilogue for the VGGT block:
 *   act == 1: out = gelu_erf(half(half(acc) + bias))          (fc1 -> GELU)
 *   resid != NULL: resid[M, ldr] += half(half(half(acc)+bias) * gamma)
 *                  (out must equal resid; LayerScale residual of proj / fc2)
 * New entry point (the reference runs these as separate PyTorch ops after
 * WQLinear.forward, qmodule.py:333-369). */
int qvggt_w4a16_linear_ex(const void* in_feats, int64_t lda, const void* qweight, const void* scales,
                          const void* scaled_zeros, const void* bias, void* out, int64_t ldo, int64_t M, int64_t N,
                          int64_t K, int64_t gpad, int32_t group_size, int32_t act, const void* resid,
                          int64_t ldr, const void* gamma, void* stream);

/* The qkv projection of a VGGT block with the q/k/v split, the optional per-head
 * LayerNorm (qk_norm != 0; qn_w/qn_b/kn_w/kn_b fp16 [64]) and the 2-D RoPE
 * fused into the W4A16 GEMM epilogue: y = half(half(in . deq(W)^T) + bias)
 * over N = 3*dim columns [q | k | v]; q -> q_out [M, dim] and [k | v] ->
 * kv_out [M, 2*dim], with q and k rotated exactly as qvggt_qkv_rope2d does
 * (same position rule and fp16 rounding points).  weight_kind 0 = W4A16
 * (qweight/scales/scaled_zeros/gpad/group_size), 1 = dense fp16 [N, K] in
 * `qweight` (scales ignored).  New entry point (the reference model runs the
 * split and RoPE in PyTorch after WQLinear.forward). */
int qvggt_qkv_rope_linear(const void* in_feats, int32_t weight_kind, const void* qweight, const void* scales,
                          const void* scaled_zeros, int64_t gpad, int32_t group_size, const void* bias, void* q_out,
                          void* kv_out, int64_t M, int64_t K, int32_t dim, int64_t token_offset,
                          int32_t tokens_per_frame, int32_t patch_start, int32_t grid_w, const void* cos_tab,
                          const void* sin_tab, int32_t max_pos, int32_t qk_norm, const void* qn_w, const void* qn_b,
                          const void* kn_w, const void* kn_b, float eps, void* stream);

/* Dense fp16 linear with the same fused epilogues (weight fp16 [N, K]); used
 * for the unquantised DINOv2 patch-embed blocks.  No reference counterpart
 * (the reference runs these layers in PyTorch). */
int qvggt_f16_linear_ex(const void* in_feats, int64_t lda, const void* weight, const void* bias, void* out,
                        int64_t ldo, int64_t M, int64_t N, int64_t K, int32_t act, const void* resid, int64_t ldr,
                        const void* gamma, void* stream);

/* Small-M linear (1 <= M <= 256 rows; N % 128 == 0, K % 64 == 0): the same
 * result and epilogues as qvggt_w4a16_linear_ex (weight_kind 0: AWQ int4
 * qweight/scales/scaled_zeros/gpad/group_size) or qvggt_f16_linear_ex
 * (weight_kind 1: fp16 weight [N, K] in `weight`, scales ignored), or
 * qvggt_w4a16_gemm_bf16 (weight_kind 2: AWQ int4 with bf16 activations,
 * scales, bias and output; act = 0 and resid = NULL only), computed
 * with the rows as the tensor-core N dimension and K split across the CTAs
 * of a thread-block cluster (partials summed on chip in a fixed order; no
 * workspace).  Replaces the small-M path of gemm_forward_cuda_new,
 * gemm_w4a16_T1 with its split-K semaphore
 * (E/quantization_new/gemm/gemm_cuda.cu:312-751, 1154-1205). */
int qvggt_small_linear(int32_t weight_kind, const void* in_feats, int64_t lda, const void* weight, const void* scales,
                       const void* scaled_zeros, int64_t gpad, int32_t group_size, const void* bias, void* out,
                       int64_t ldo, int64_t M, int64_t N, int64_t K, int32_t act, const void* resid, int64_t ldr,
                       const void* gamma, void* stream);

/* Launch plan qvggt_small_linear uses for (M, N, K) on the current device:
 * info[0] padded rows (MMA N), info[1] CTAs per cluster (K splits),
 * info[2] 64-wide k-blocks per CTA, info[3] CTAs, info[4] clusters of that
 * size the device holds at once.  Part of the same small-M replacement
 * (E/quantization_new/gemm/gemm_cuda.cu:1154-1205 picks its tiles by M). */
int qvggt_small_linear_plan(int32_t weight_kind, int64_t M, int64_t N, int64_t K, int32_t* info);

/* out[m, N] = in_feats[m, K] . deq(qweight)^T (+ bias) for 1 <= m <= 16.
 * Any group_size that is a multiple of 32 and divides K.
 * Replaces gemv_forward_cuda_new (E/quantization_new/gemv/gemv_cuda.cu:197-281,
 * bound at E/pybind.cpp:22; reference: m <= 7, group_size 128 only). */
int qvggt_w4a16_gemv(const void* in_feats, const void* qweight, const void* scales, const void* scaled_zeros,
                     const void* bias, void* out, int64_t m, int64_t N, int64_t K, int64_t gpad,
                     int32_t group_size, void* stream);

/* qvggt_w4a16_gemv with bf16 in_feats, scales, scaled_zeros, bias and out:
 * bf16 dequantisation as qvggt_w4a16_gemm_bf16, products summed in fp32,
 * out = bf16(sum) (+ bias).  Replaces the bf16 instantiation of
 * gemv_forward_cuda_new (E/quantization_new/gemv/gemv_cuda.cu:210-217, 59,
 * 130-133: the reference sums in bf16). */
int qvggt_w4a16_gemv_bf16(const void* in_feats, const void* qweight, const void* scales, const void* scaled_zeros,
                          const void* bias, void* out, int64_t m, int64_t N, int64_t K, int64_t gpad,
                          int32_t group_size, void* stream);

/* ----------------------------------------------------------------- W8A8 */

/* out[M, N] fp16 = half(float(acc) * (wscales[n] * ascales[m]))                (bias == NULL)
 *              or half(fma(float(acc) * wscales[n], ascales[m], bias[n]))      (bias != NULL)
 * acc = sum_k in[m, k] * w[n, k] in int32 (tcgen05 kind::i8, TMEM).
 * in int8 [M, K], w int8 [N, K], wscales fp16 [N], ascales fp16 [M].
 * Requirements: N % 128 == 0, K % 128 == 0.
 * Replaces w8a8_gemm_forward_cuda and w8a8_gemm_fuse_bias_forward_cuda
 * (E/w8a8/w8a8_gemm_cuda.cu:881-922 and :564-607, E/pybind.cpp:27-28). */
int qvggt_w8a8_gemm(const int8_t* in, const int8_t* w, const void* wscales, const void* ascales, const void* bias,
                    void* out, int64_t M, int64_t N, int64_t K, void* stream);

/* The W8A8 GEMM of a VGGT block with the LayerScale residual fused:
 * resid[M, N] += half(half(y) * gamma), y as in qvggt_w8a8_gemm (bias may be
 * NULL).  New entry point (the reference has no caller of its W8A8 GEMM). */
int qvggt_w8a8_gemm_residual(const int8_t* in, const int8_t* w, const void* wscales, const void* ascales,
                             const void* bias, const void* gamma, void* resid, int64_t M, int64_t N, int64_t K,
                             void* stream);

/* Raw int32 accumulators acc[M, N] of the same GEMM (for bit-exact checks).
 * No reference counterpart (the reference never exposes its accumulators). */
int qvggt_i8_gemm_i32(const int8_t* in, const int8_t* w, int32_t* acc, int64_t M, int64_t N, int64_t K,
                      void* stream);

/* Per-token dynamic int8 quantisation: scale[t] = half(amax_t / 127),
 * out = rni_sat(x * (127 / amax_t)).  in fp16 [tokens, hidden].
 * Replaces invoke_quant (E/w8a8/quantization.cu:81-96, E/pybind.cpp:29). */
int qvggt_invoke_quant(int8_t* out, const void* in, void* scale, int64_t tokens, int64_t hidden, void* stream);

/* LayerNorm (var = E[x^2] - E[x]^2) + int8 quantisation.
 * per_token != 0: out = rni_sat(ln * 127 / amax), scale_io[t] = half(amax/127)
 *   (amax over fp16-rounded ln, floor half(1e-6)); beta used.
 * per_token == 0: out = rni_sat(half(ln) * scale_io[0]) with scale_io a
 *   per-tensor fp16 input; beta ignored (the reference passes none).
 * Replaces rms_norm_general (E/w8a8/layernorm.cu:155-191, E/pybind.cpp:30-32). */
int qvggt_layernorm_quant(int8_t* out, const void* in, const void* gamma, const void* beta, void* scale_io,
                          int64_t tokens, int64_t hidden, float eps, int32_t per_token, void* stream);

/* tmp = gelu_tanh(in) in fp16 arithmetic; scale[t] = half(amax_t / 127) with
 * the reference's |t| rule (t > 1e-4 ? t : -t); out = rni_sat(half(127/amax) * tmp).
 * Replaces gelu_and_quant (E/w8a8/act.cu:77-90, E/pybind.cpp:36). */
int qvggt_gelu_quant(int8_t* out, const void* in, void* scale, void* tmp, int64_t tokens, int64_t d, void* stream);

/* ---------------------------------------------------------------- norms */

/* out = LayerNorm(in) * gamma + beta, fp16 in/out, fp32 statistics
 * (two-pass mean / variance).  rows of `hidden` (multiple of 256, <= 8192).
 * New entry point: the VGGT pre-norm (nn.LayerNorm, run by PyTorch in the
 * reference model). */
int qvggt_layernorm(const void* in, const void* gamma, const void* beta, void* out, int64_t tokens, int64_t hidden,
                    float eps, void* stream);

/* ----------------------------------------------------------------- RoPE */

/* Reference rotate-half RoPE with explicit per-(b, s) angles:
 * in [s, b, h, d] with element strides in_strides[4], freqs fp32 [b, s, d2],
 * out [s, b, h, d] with element strides out_strides[4]; dims >= d2 copied.
 * Replaces fused_rope_with_pos_forward_func (E/rope_new/fused_rope_with_pos.cu:122-164,
 * E/pybind.cpp:26); the caller allocates `out` with the strides it wants. */
int qvggt_rope_with_pos(const void* in, const float* freqs, void* out, int64_t s, int64_t b, int64_t h, int64_t d,
                        int64_t d2, const int64_t* in_strides, const int64_t* out_strides, void* stream);

/* VGGT 2-D RoPE fused with the q/k/v split of the qkv projection output.
 * qkv fp16 [T, 3*H*64] (token-major, [q | k | v], head-major inside each);
 * q_out [T, H*64] (roped), kv_out [T, 2*H*64] ([k roped | v]).
 * Token t's position: p = (t + token_offset) % tokens_per_frame; p < patch_start
 * -> (0, 0) else ((p-patch_start)/grid_w + 1, (p-patch_start)%grid_w + 1).
 * cos_tab / sin_tab fp16 [max_pos, 32] (the per-half tables of the model).
 * qk_norm != 0 applies LayerNorm over each head's 64 dims to q and k first
 * (weights qn_w/qn_b/kn_w/kn_b fp16 [64]).  New entry point. */
int qvggt_qkv_rope2d(const void* qkv, void* q_out, void* kv_out, int64_t T, int32_t heads, int64_t token_offset,
                     int32_t tokens_per_frame, int32_t patch_start, int32_t grid_w, const void* cos_tab,
                     const void* sin_tab, int32_t max_pos, int32_t qk_norm, const void* qn_w, const void* qn_b,
                     const void* kn_w, const void* kn_b, float eps, void* stream);

/* ------------------------------------------------------------ attention */

/* Flash attention, head_dim 64, non-causal, softmax(q k^T / 8) v, tcgen05.
 * Token-major layouts: q [batches*Lq rows, q_stride] with head h at column
 * h*64; k / v rows of kv_stride elements, head h at k_col0 + h*64 and
 * v_col0 + h*64; out [batches*Lq, o_stride], head h at column h*64.
 * Batch b covers q rows [b*Lq, (b+1)*Lq) and kv rows [b*Lkv, (b+1)*Lkv).
 * Strides are in elements and must be multiples of 8.
 * New entry point (the reference model runs PyTorch SDPA). */
int qvggt_attention(const void* q, int64_t q_stride, const void* kv, int64_t kv_stride, int64_t k_col0,
                    int64_t v_col0, void* out, int64_t o_stride, int64_t batches, int64_t Lq, int64_t Lkv,
                    int32_t heads, void* stream);

/* qvggt_attention over a chosen subset of each batch's keys, in pieces that
 * merge exactly (the frame-sharded global block of the aggregator: a rank
 * attends to its own K/V rows while the all-gather of the other ranks' rows is
 * in flight, then to those rows, and the two results are merged).
 *
 * Keys: rows [seg0_start, seg0_start + seg0_len) and
 * [seg1_start, seg1_start + seg1_len) of each batch's Lkv rows (seg1_len may
 * be 0; seg0_len > 0).
 * splits: 1..4 CTAs share each (batch, head, 256-query block), each over a
 * consecutive part of the keys; their results are merged on the device by the
 * last of them to finish (no CTA waits for another).  splits > 1 needs
 * `scratch` of qvggt_attention_scratch_bytes() bytes (16-byte aligned); its
 * first bytes are cleared on `stream` before the launch, so calls on one
 * stream may share it, calls that may overlap on the GPU may not.
 * lse (fp32 [batches][heads][Lq]) holds ln(sum_k exp(q.k / 8)) of each row:
 *   lse_mode 0: not used;  1: written;  2: `out` and `lse` hold the result of
 *   an earlier call over other keys of the same rows, which is merged with
 *   this call's; both are overwritten with the merged result.
 * qvggt_attention_plan() gives the split count the library would choose for a
 * shape on the current device (fewest waves of CTAs over its SMs) and the
 * scratch it needs.
 * New entry points (the reference model runs PyTorch SDPA). */
int qvggt_attention_ex(const void* q, int64_t q_stride, const void* kv, int64_t kv_stride, int64_t k_col0,
                       int64_t v_col0, void* out, int64_t o_stride, int64_t batches, int64_t Lq, int64_t Lkv,
                       int64_t seg0_start, int64_t seg0_len, int64_t seg1_start, int64_t seg1_len, int32_t heads,
                       int32_t splits, int32_t lse_mode, float* lse, void* scratch, int64_t scratch_bytes,
                       void* stream);
int qvggt_attention_plan(int64_t batches, int64_t Lq, int64_t keys, int32_t heads, int32_t* splits,
                         int64_t* scratch_bytes);
int qvggt_attention_scratch_bytes(int64_t batches, int64_t Lq, int32_t heads, int32_t splits,
                                  int64_t* scratch_bytes);

/* qvggt_attention_ex over all keys (lse_mode 0) with `splits` (1..4) split-KV
 * CTAs, for callers that cannot allocate device memory: it allocates nothing.
 * Its scratch is a fixed 64 MiB array in the library's device memory, present
 * on every GPU that loads the library until the process exits; a shape whose
 * scratch (qvggt_attention_scratch_bytes) exceeds 64 MiB is rejected with
 * QVGGT_ERR_UNSUPPORTED.  The first call on a device looks up the array's
 * device address (cudaGetSymbolAddress, with that device current); make that
 * first call before any stream capture.  All calls on a device share the array
 * and leave their data in it; each call clears the counters it needs on
 * `stream` before its kernel, so calls in order on one stream are safe, and
 * calls whose kernels may run at the same time on the GPU (other streams,
 * other host threads) race.  Same arguments and results as qvggt_attention_ex.
 * No counterpart in the reference. */
int qvggt_attention_split_static(const void* q, int64_t q_stride, const void* kv, int64_t kv_stride,
                                 int64_t k_col0, int64_t v_col0, void* out, int64_t o_stride, int64_t batches,
                                 int64_t Lq, int64_t Lkv, int32_t heads, int32_t splits, void* stream);

/* Attention over short sequences with head_dim 128 (the camera-head trunk:
 * 16 heads x 128 over the S <= 256 camera tokens of each batch),
 * softmax(q k^T / sqrt(128)) v on CUDA cores in fp32.  Same token-major
 * layout as qvggt_attention with heads at column h*128 and Lq = Lkv = L.
 * New entry point (the reference model runs PyTorch SDPA in its camera head,
 * loader.py:338-344 quantises the trunk's linears around it). */
int qvggt_attention_small(const void* q, int64_t q_stride, const void* kv, int64_t kv_stride, int64_t k_col0,
                          int64_t v_col0, void* out, int64_t o_stride, int64_t batches, int64_t L, int32_t heads,
                          void* stream);

/* --------------------------------------------------- streaming K/V cache
 * These calls take their arguments in a structure of 64-bit fields (sizes,
 * strides in elements, device pointers).  Sizes that have to fit 32 bits are
 * checked. */

/* Rotary positions with 1..4 axes (time, height, width, ...), q and k in one
 * launch.  x [T, heads, head_dim] with element strides (tok, head) and unit
 * stride inside a head; fp16 or bf16 (dtype); out may be the input itself.
 * Axis a owns sections[a] consecutive pairs of the R/2 = sum(sections) pairs,
 * and pair j turns by positions[axis_j][t] * inv_freq[j]:
 *   y[lo] = x[lo] cos - x[hi] sin,  y[hi] = x[hi] cos + x[lo] sin.
 * layout 0 (axial): each axis' pairs are the two halves of its own 2 *
 *   sections[a] dims; 1 (split): pair j is dims (j, j + R/2); 2 (interleaved):
 *   dims (2j, 2j + 1).  Dims >= R are copied.  inverse != 0 turns back (the
 * gradient).  positions int32 [n_axes, T] with row stride pos_stride, inv_freq
 * fp32 [R/2].  head_dim <= 256.  k_heads may be 0.  New entry point. */
typedef struct {
  const void* q;
  int64_t q_tok, q_head;
  void* q_out;
  int64_t qo_tok, qo_head, q_heads;
  const void* k;
  int64_t k_tok, k_head;
  void* k_out;
  int64_t ko_tok, ko_head, k_heads;
  int64_t T, head_dim;
  const int32_t* positions;
  int64_t pos_stride;
  const float* inv_freq;
  int64_t sections[4], n_axes, layout, inverse, dtype;
} qvggt_rope_axes_args;
int qvggt_rope_axes(const qvggt_rope_axes_args* args, void* stream);

/* Block tables and slot maps of a paged cache, from request lengths.  Request
 * b goes from cached_lens[b] to target_lens[b] tokens (more: blocks are taken
 * from the free ring; fewer, 0 to end it: its surplus blocks go back).
 * free_ring [num_blocks] holds the free blocks at positions [free_range[0],
 * free_range[1]) modulo num_blocks: blocks are taken at the first, in request
 * order, and given back at the second.
 * Written: block_tables [requests, max_blocks] and free_ring in place (entries
 * past a request's length are stale); lens_out; free_range_out; cu_new and
 * cu_blocks [requests + 1], the running sums of new tokens and of blocks that
 * get new tokens; slots [max_new], block * block_size + offset of each new
 * token in request order, then -1; status[0].
 * status: 0 done; otherwise nothing is changed, no token gets a slot and
 * lens_out = cached_lens: 1 too few free blocks, 2 a table row too short, 3 a
 * negative length, 4 more than max_new tokens, 5 free_range is not 0 <= first <=
 * second <= first + num_blocks or more blocks come back than it leaves room for
 * (lengths that do not fit the pool).  Block ids are handed on as they stand;
 * one outside the cache sets the device status word (0x201) and gives its
 * tokens the slot -1.  One launch, no host
 * synchronisation; the same inputs give the same result again.  At most 8192
 * requests; block_size a power of two.  New entry point. */
typedef struct {
  const int32_t *cached_lens, *target_lens;
  int64_t requests;
  int32_t* block_tables;
  int64_t max_blocks;
  int32_t* free_ring;
  int64_t num_blocks;
  const int64_t* free_range;
  int64_t block_size, max_new;
  int32_t *slots, *cu_new, *cu_blocks, *lens_out;
  int64_t* free_range_out;
  int32_t* status;
} qvggt_block_plan_args;
int qvggt_block_plan(const qvggt_block_plan_args* args, void* stream);

/* The 8-bit cache: k_cache / v_cache int8 [num_blocks][kv_heads][block_size]
 * [head_dim] (block_stride codes between blocks, 16-byte aligned), k_scale /
 * v_scale fp32 [num_blocks][kv_heads], all positive; an element is code *
 * scale.  block_size 32, 64 or 128, head_dim 64 or 128. */
typedef struct {
  int8_t *k_cache, *v_cache;
  int64_t block_stride;
  float *k_scale, *v_scale;
  int64_t num_blocks, kv_heads, block_size, head_dim;
} qvggt_kv_cache;

/* Writes new K and V rows into the 8-bit cache.
 * k, v [tokens, kv_heads, head_dim] (element strides of token and head, unit
 * stride inside, rows 16-byte aligned), fp16 or bf16, requests packed one
 * after another as cu_new says; cu_new and cu_blocks as qvggt_block_plan
 * writes them, cached_lens the lengths before.  max_units: an upper bound of
 * cu_blocks[requests] (tokens / block_size + 2 * requests always is one).
 * Per (block, head): s = max(s_old if the block holds earlier tokens, amax /
 * 127, 2^-60), code = rint(x / s) within +-127 (computed as x * (1 / s));
 * earlier codes c of the block become rint(c * s_old / s).  Only finite values
 * count in amax; infinities are stored as the largest code, NaN as 0.  A block
 * id or length outside its range sets the device status word (0x201 / 0x202)
 * and skips the block; so does a max_units that is too small (0x202, the blocks
 * past it are not written).  New entry point. */
typedef struct {
  qvggt_kv_cache cache;
  const void* k;
  int64_t k_tok, k_head;
  const void* v;
  int64_t v_tok, v_head, tokens, dtype;
  const int32_t* block_tables;
  int64_t max_blocks;
  const int32_t *cached_lens, *cu_new, *cu_blocks;
  int64_t requests, max_units;
} qvggt_kv_append_args;
int qvggt_kv_append(const qvggt_kv_append_args* args, void* stream);

/* Reads cache rows back: out [n][out_stride] fp16 or bf16, row i = [K of all
 * heads | V of all heads] of slots[i] (the layout qvggt_attention reads as
 * kv); a negative slot gives zeros.  New entry point. */
typedef struct {
  qvggt_kv_cache cache;
  const int32_t* slots;
  int64_t n;
  void* out;
  int64_t out_stride, dtype;
} qvggt_kv_gather_args;
int qvggt_kv_gather(const qvggt_kv_gather_args* args, void* stream);

/* Attention over the 8-bit cache: softmax(scale q k^T + mask) v for ragged
 * requests whose query rows are packed one after another.
 * q, out [Tq, q_heads, head_dim], fp16 or bf16, element strides of token and
 * head, rows 16-byte aligned; query head h reads key head h / (q_heads /
 * kv_heads).  Request b's queries are rows [cu_q[b], cu_q[b + 1]) (at most
 * max_q of them) and its keys the first kv_lens[b] tokens of table row b;
 * max_kv is about the largest length (it sets how the work is laid out; any
 * length up to the table's is served).
 * Mask: query i of ql sits at position p = kv_len - ql + i.  causal_chunk 0:
 * it sees every key; c > 0: keys j < (p / c + 1) * c (1: causal; the tokens of
 * a frame: its own and all earlier frames), none when p < 0.  A row that sees
 * no key gives 0; rows outside cu_q are left as they are.  lse (fp32
 * [q_heads][Tq], may be NULL): ln sum_j exp(scale q.k_j), -inf for a row
 * without a key.
 * scale: above 1e-30, at most 1e30.  Sums, maxima and products are held in fp32;
 * the weights are rounded to fp16 for the product with V, and with many rows one
 * in eight of them comes from a polynomial (relative error up to 7.5e-5, a sixth of
 * that rounding's).  The V scales of one request's blocks may lie 2^80 apart.
 * scratch: qvggt_cached_attention_scratch() bytes (0 for some shapes), 16-byte
 * aligned; its contents need no preparation and are free after the call, and
 * calls that may overlap on the GPU may not share it.  A block id or length
 * outside its range sets the device status word (0x201: the block's keys are
 * skipped, 0x202: the request is skipped, its rows of out and lse are left as
 * they are).  New entry points. */
typedef struct {
  qvggt_kv_cache cache;
  const void* q;
  int64_t q_tok, q_head;
  void* out;
  int64_t o_tok, o_head;
  float* lse;
  int64_t Tq, q_heads, dtype;
  const int32_t* block_tables;
  int64_t max_blocks;
  const int32_t *cu_q, *kv_lens;
  int64_t requests, max_q, max_kv, causal_chunk;
  double scale;
  void* scratch;
  int64_t scratch_bytes;
} qvggt_cached_attention_args;
int qvggt_cached_attention(const qvggt_cached_attention_args* args, void* stream);
int qvggt_cached_attention_scratch(int64_t Tq, int32_t q_heads, int32_t kv_heads, int32_t requests, int32_t max_q,
                                   int64_t max_kv, int32_t head_dim, int64_t* bytes);

/* What a cached key has gathered: for the keys of each request, out = old +
 * sum of exp(scale q_i . k_j - lse_i) over the queries i that see key j and the
 * query heads that read its head, where old is decay * weights for tokens before
 * fresh_from[b] (of all tokens, if it is NULL) and 0 for the others, whose places
 * may hold anything.
 * weights, out fp32 [num_blocks][kv_heads][block_size], the cache's order, and
 * may be the same; places that hold no key of a request are left as they are.
 * lse fp32 [q_heads][Tq] as the attention over the same keys gives it (a row then
 * hands out 1 in all; over the keys before they were rounded to codes, e^d times
 * more or less at most, d being what the rounding may change a score by); a row
 * whose lse is not finite (no key, or NaN) counts for nothing.  q, cu_q, kv_lens,
 * block_tables, max_q, max_kv, causal_chunk, scale as in qvggt_cached_attention;
 * requests have their own blocks.  decay: 0 to 1.  Sums are held in fp32 and
 * taken in one order, so they repeat bit for bit.  A block id or length outside
 * its range sets the device status word (0x201: the block is skipped, 0x202: the
 * request is).  New entry point. */
typedef struct {
  const int8_t* k_cache;
  int64_t block_stride;
  const float* k_scale;
  int64_t num_blocks, kv_heads, block_size, head_dim;
  const void* q;
  int64_t q_tok, q_head, Tq, q_heads, dtype;
  const float* lse;
  const int32_t* block_tables;
  int64_t max_blocks;
  const int32_t *cu_q, *kv_lens, *fresh_from;
  int64_t requests, max_q, max_kv, causal_chunk;
  const float* weights;
  float* out;
  double scale, decay;
} qvggt_key_weights_args;
int qvggt_key_weights(const qvggt_key_weights_args* args, void* stream);

/* Which tokens stay when request b goes from lens[b] to keep[b] tokens, for
 * every layer and kv head apart: the first `sink` and the last `recent` (as
 * far as keep[b] goes, the first ones before the last), then those of largest
 * weight; of equal ones the lower position.  NaN counts as the lowest weight,
 * infinities as the largest finite ones.  A token that stays although it stands
 * at keep[b] or later moves into the place of one that goes: dst
 * [layers][requests][kv_heads][max_moves] holds the places below keep[b] that
 * fall free and src the tokens that move, both ascending, then -1; counts
 * [layers][requests][kv_heads] how many.  keep[b] >= lens[b]: none.
 * weights fp32 [layers][num_blocks][kv_heads][block_size], 16-byte aligned.
 * max_moves: at least the largest min(keep[b], lens[b] - keep[b]); moves past it
 * are dropped and the status word says so (0x202).  max_len: about the longest
 * length (0: what the tables hold); it sets how the work is laid out.  A length
 * outside its range gives no moves, a block outside the cache lowest weights;
 * the status word says so (0x202, 0x201).  At most 2^30 tokens a request.
 * New entry point. */
typedef struct {
  const float* weights;
  int64_t layers, num_blocks, kv_heads, block_size;
  const int32_t* block_tables;
  int64_t max_blocks;
  const int32_t *lens, *keep;
  int64_t requests, sink, recent, max_moves, max_len;
  int32_t *src, *dst, *counts;
} qvggt_evict_plan_args;
int qvggt_evict_plan(const qvggt_evict_plan_args* args, void* stream);

/* Carries out the moves of qvggt_evict_plan in the cache: codes, scales and, if
 * not NULL, weights [layers][num_blocks][kv_heads][block_size] of token src[i]
 * enter the place of token dst[i].
 * cache: the tensors of the first layer; layer_stride codes between layers
 * (16-byte aligned), the scales [layers][num_blocks][kv_heads].  Per (layer,
 * head) and block that receives rows of magnitude amax: s = max(s_old, amax /
 * 127, 2^-60), incoming values x become rint(x * (1 / s)), and if s grew all
 * other codes c of the block rint(c * (s_old * (1 / s))).  Blocks that receive
 * nothing are left as they are, and so is what stands at keep[b] or later, but
 * for the rest of the block that keep[b] falls into.  Requests have their own
 * blocks.  Places outside [0, keep[b]) in dst, or before keep[b] in src, and block
 * ids outside the cache are skipped and reported (0x202, 0x201).  New entry point. */
typedef struct {
  qvggt_kv_cache cache;
  int64_t layers, layer_stride;
  float* weights;
  const int32_t* block_tables;
  int64_t max_blocks;
  const int32_t* keep;
  int64_t requests;
  const int32_t *src, *dst, *counts;
  int64_t max_moves;
} qvggt_kv_evict_args;
int qvggt_kv_evict(const qvggt_kv_evict_args* args, void* stream);

/* Attention over whole sequences packed one after another: softmax(scale q k^T +
 * mask) v within each.
 * q, out [T, q_heads, head_dim], k, v [T, kv_heads, head_dim], fp16 or bf16,
 * element strides of token and head (positive multiples of 8 where there is more
 * than one), unit stride inside, 16-byte aligned, out apart from k and v;
 * head_dim 64 or 128; query head h reads key head h / (q_heads / kv_heads), at
 * most 128 query heads to a key head.  Sequence b is rows [cu[b], cu[b + 1]), at
 * most max_len of them.
 * Mask: causal_chunk 0: every token sees its whole sequence; c > 0: token i sees
 * tokens j < (i / c + 1) * c (1: causal; the tokens of a frame: its own and all
 * earlier frames).  What a token does not see adds nothing to it, NaN and
 * infinities and the largest finite values among it.  Rows outside cu are left as
 * they are.  lse (fp32 [q_heads][T], may be NULL): ln sum_j exp(scale q.k_j).
 * scale: above 1e-30, at most 1e30.  Sums, maxima and products are held in fp32:
 * a row that sees a score of NaN or, scaled and times log2 e, above 2^27 (fp16) or
 * 2^31 (bf16) is NaN, and its largest should not be under the negatives of these.
 * The weights are rounded to the inputs' type for the product with V, and one
 * under 2^-125 of the row's largest counts as 0.  The product is divided by the
 * sum of the weights last, which are up to 2^8 each: bf16 values near fp32's
 * largest, seen with such weights, can overflow it.
 * scratch: qvggt_prompt_attention_scratch() bytes (0 for some shapes), 16-byte
 * aligned; calls that may overlap on the GPU may not share it.  A sequence
 * outside [0, T) or longer than max_len is skipped and sets the device status
 * word (0x202).  New entry points. */
typedef struct {
  const void* q;
  int64_t q_tok, q_head;
  const void* k;
  int64_t k_tok, k_head;
  const void* v;
  int64_t v_tok, v_head;
  void* out;
  int64_t o_tok, o_head;
  float* lse;
  int64_t T, q_heads, kv_heads, head_dim, dtype;
  const int32_t* cu;
  int64_t sequences, max_len, causal_chunk;
  double scale;
  void* scratch;
  int64_t scratch_bytes;
} qvggt_prompt_attention_args;
int qvggt_prompt_attention(const qvggt_prompt_attention_args* args, void* stream);
int qvggt_prompt_attention_scratch(int64_t T, int32_t q_heads, int32_t kv_heads, int32_t sequences, int64_t max_len,
                                   int32_t head_dim, int64_t* bytes);

/* ---------------------------------------------------------- patch embed */

/* images fp16 [S, 3, H, W] (pixels in [0, 1]) -> patches fp16
 * [S*(H/patch)*(W/patch), k_pad]: column c*patch^2 + ky*patch + kx holds
 * half(half(x - mean[c]) / std[c]), columns >= 3*patch^2 are zero.  Turns the
 * patch-embed convolution of the DINOv2 front into a GEMM.  No reference
 * counterpart (the model runs the convolution in PyTorch). */
int qvggt_patchify(const void* images, void* out, int64_t S, int32_t H, int32_t W, int32_t patch, int32_t k_pad,
                   const float* mean3, const float* std3, void* stream);

/* out [S, P, C]: rows p < n_special of frame f copy specials[set][p] (set = 1
 * for every frame whose global index f + frame_offset > 0 when two_sets != 0,
 * else 0); rows p >= n_special copy src row
 * f*src_rows_per_frame + src_row_offset + (p - n_special).  If pos != NULL,
 * pos[p] (fp16 [P, C]) is added (one fp16 rounding).  Builds the DINOv2 token
 * sequence (cls / registers / patches + position embedding) and the aggregator
 * sequence (camera / registers / patch tokens).  No reference counterpart. */
int qvggt_assemble_tokens(const void* src, int64_t src_rows_per_frame, int64_t src_row_offset, const void* specials,
                          int32_t n_special, int32_t two_sets, const void* pos, void* out, int64_t S, int32_t P,
                          int32_t C, int64_t frame_offset, void* stream);

/* Kernel configuration of every large-M GEMM entry point (W4A16, dense fp16,
 * int8): 0 = chosen per shape (default: the configuration with the fewest
 * estimated cycles, waves of tiles over the SMs x time per tile), 1 = CTA
 * pairs with 256 x 256 tiles, 2 = one SM per 128 x 256 tile, 3 = one SM per
 * 128 x 128 tile.  A forced configuration a shape cannot use falls back to
 * the automatic choice.  Process-wide; for tuning and tests.  The
 * QVGGT_GEMM_CONFIG environment variable sets the initial value.  No
 * reference counterpart (the reference picks its GEMM by M alone,
 * gemm_cuda.cu:1154-1232). */
int qvggt_set_gemm_config(int32_t cfg);

/* ------------------------------------------------------- post-processing */

/* Camera matrices from VGGT's pose encoding "absT_quaR_FoV": pose_enc fp32
 * [n, 9] = (t, quaternion x y z w, fov_h, fov_w) -> extrinsics fp32 [n, 3, 4] =
 * [R | t] and, when `intrinsics` is not NULL, intrinsics fp32 [n, 3, 3]
 * (fx = (w/2) / tan(fov_w/2), fy = (h/2) / tan(fov_h/2), fields of view
 * clamped to [1e-6, pi - 1e-6], focal lengths to [1, 1e6], principal point
 * (w/2, h/2)).  Replaces qvggt/common/pose_enc.py:7-65
 * (pose_encoding_to_extri_intri) and rotation.py:4-25 (quat_to_mat). */
int qvggt_pose_encoding_to_extri_intri(const float* pose_enc, int64_t n, int32_t image_h, int32_t image_w,
                                        float* extrinsics, float* intrinsics, void* stream);

/* World points from depth maps: depth fp32 [S, H, W] (16-byte aligned),
 * extrinsics fp32 [S, 3, 4], intrinsics fp32 [S, 3, 3] -> world_points fp32
 * [S, H, W, 3] (16-byte aligned) = R^T (cam - t) with cam = ((u - cu) d / fu,
 * (v - cv) d / fv, d), fu and fv floored at 1e-6; every pixel is converted
 * (no mask), as in the reference.  Replaces qvggt/common/geometry.py:43-96
 * (unproject_depth_map_to_point_map, computed there in numpy on the host). */
int qvggt_unproject_depth(const float* depth, int64_t S, int32_t H, int32_t W, const float* extrinsics,
                          const float* intrinsics, float* world_points, void* stream);

/* ------------------------------------------------------------- self-test */

/* Runs one kernel whose bounded wait waits on an mbarrier nothing arrives on;
 * it must give up after the wait budget and report QVGGT_ERR_TIMEOUT through
 * the status word (which this call clears).  Synchronises.  For tests of the
 * failure path; faults nothing. */
int qvggt_selftest_wait_timeout(uint64_t timeout_ns, uint32_t* status_out);

#ifdef __cplusplus
}
#endif

#endif /* QVGGT_B200_H */
