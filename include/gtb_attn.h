/* B200 (sm_100a) scaled-dot-product-attention engine: raw-pointer C ABI.
 *
 * Every entry point takes device pointers, sizes and element strides, and a CUDA stream
 * (cudaStream_t passed as void*; NULL = the legacy default stream). No entry point takes a
 * framework type. All return 0 on success and -1 on failure with a thread-local message in
 * gtb_last_error(), the convention of the reference's gt_last_error (csrc/gt_core.cpp:7-23).
 * Tensors must live on the current CUDA device. There is no CPU path: host pointers are an error.
 *
 * The reference-shaped handle ABI (gt_tensor *, gguf_train.h) is declared in gguf_train_attn.h and
 * is implemented on top of these functions.
 */
#ifndef GTB_ATTN_H
#define GTB_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GTB_API __attribute__((visibility("default")))

/* A strided 4-D view of device memory. data points at element [0,0,0,0]; strides count elements
 * (a stride of 0 broadcasts a size-1 dimension). dtype is a gt_dtype code (gguf_train.h:22-36):
 * 0 = f32, 1 = f16, 2 = bf16, 3 = f64, 9 = bool (masks only). */
typedef struct gtb_tensor4 {
    void *data;
    int64_t shape[4];
    int64_t stride[4];
    int32_t dtype;
} gtb_tensor4;

/* Attention forward.
 * Replaces the body of gt_flash_attention (reference csrc/gt_ops_nn.cpp:2423-2525, declared
 * csrc/gguf_train.h:311) for CUDA tensors.
 *   q (B,H,L,D), k (B,Hkv,S,D), v (B,Hkv,S,Dv); H % Hkv == 0 (query head h reads kv head
 *   h / (H/Hkv)); out (B,H,L,Dv) in q's dtype.
 *   mask: NULL or (B|1,H|1,L|1,S|1), bool (0 = may not attend) or float (added to the scores).
 *   scale <= 0 means 1/sqrt(D). is_causal masks s > l (top-left aligned).
 *   lse: NULL or a (B,H,L) contiguous buffer that receives the natural-log sum of exp(scores)
 *   per row (-inf for a row with no allowed key, whose output is 0): float64 for f64 inputs,
 *   float32 otherwise.
 * Kernel choice: bf16/f16 with D == Dv in {64,128}, unit inner stride, and no mask or a bool / f32 /
 * f16 / bf16 mask, runs the tcgen05/TMA kernel; everything else runs the SIMT kernel (f32/f64
 * accumulate as the input). With a mask, a pre-pass classifies each 128-row x 128-key block of it
 * (every key allowed with nothing added / none allowed / mixed) into a small table from the
 * stream-ordered allocator, and only mixed blocks read the mask entry by entry.
 * For L <= 8192 the tcgen05 kernel runs persistent CTAs that claim work from a 4-byte counter taken
 * from the stream-ordered allocator and zeroed on the stream. */
GTB_API int gtb_sdpa_fwd(const gtb_tensor4 *q, const gtb_tensor4 *k, const gtb_tensor4 *v,
                         const gtb_tensor4 *mask, float scale, int is_causal,
                         gtb_tensor4 *out, void *lse, void *stream);

/* Prefill attention with rotary position embedding fused in: out = attention(rope(q), rope(k), v) and
 * k_rot = rope(k), the rotation that of gtb_rope (backward = 0) with q's positions pos_q (>= L entries)
 * and k's positions pos_k (>= S entries). New export; replaces gt_rope on q and on k (reference
 * csrc/gt_ops_nn.cpp:2409-2421) followed by gt_flash_attention (csrc/gt_ops_nn.cpp:2423-2525).
 *   q (B,H,L,D), k (B,Hkv,S,D) contiguous f32/f16/bf16; v, mask, scale, is_causal, out and lse as in
 *   gtb_sdpa_fwd; k_rot: a contiguous buffer of k's shape and dtype that receives rope(k) (the rotated
 *   keys a caller keeps as its K cache).
 * k is rotated once in HBM (every query tile reads every key tile). q is rotated into a stream-ordered
 * scratch copy first, or, with q_in_kernel != 0 where the tcgen05 kernel runs with no mask and
 * n_dims % 16 == 0, inside the kernel: each Q tile in shared memory once it has landed, from a
 * (cos, sin) table of the L query positions (gtb_last_path "tcgen05+rope"; no q copy, but slower on
 * B200: the next item's Q lands only when the previous item's score products are issued, so the
 * rotation is not hidden). Either way the results equal gtb_rope on q and k followed by gtb_sdpa_fwd
 * bit for bit. */
GTB_API int gtb_sdpa_fwd_rope(const gtb_tensor4 *q, const gtb_tensor4 *k, const gtb_tensor4 *v,
                              const gtb_tensor4 *mask, float scale, int is_causal, const int32_t *pos_q,
                              int64_t n_pos_q, const int32_t *pos_k, int64_t n_pos_k, int n_dims, int mode,
                              float freq_base, float freq_scale, int q_in_kernel, gtb_tensor4 *k_rot,
                              gtb_tensor4 *out, void *lse, void *stream);

/* The forward for q, k, v and out in HOST memory (contiguous, row-major; pinned for the copies to
 * overlap, pageable works with serialised copies), no mask. New export for callers whose tensors live
 * on the host, as the reference's do (gt_flash_attention, csrc/gt_ops_nn.cpp:2423-2525, reads and
 * writes host tensors). The work is cut into `pieces` (<= 0: 8) pieces — whole sequences, or one
 * sequence's kv heads in groups when the batch is smaller than that — and on the calling thread's
 * device piece i's q, k, v are copied in on one internal stream while piece i-1 is attended on
 * `stream` and piece i-2's output is copied out on another; two device slots from the stream-ordered
 * allocator are reused in turn. Asynchronous like the other calls: `out` is complete once `stream`
 * has passed the call. Results are bit for bit those of gtb_sdpa_fwd on the same values. */
GTB_API int gtb_sdpa_fwd_host(const gtb_tensor4 *q, const gtb_tensor4 *k, const gtb_tensor4 *v, float scale,
                              int is_causal, gtb_tensor4 *out, int pieces, void *stream);

/* Attention backward: dq, dk, dv from dout, the forward inputs, the forward output and its lse.
 * Replaces FlashAttentionFn.backward (reference gguf_train/_functions.py:1934-1965), which
 * recomputes the probabilities with a chain of separate ops. dk/dv are summed over the query
 * heads of each kv head, as that function does (:1958-1962). Scratch (rowsum(dout*out) per row;
 * on the tcgen05 path with D = 128 also f32 dq sums, B*H*Lpad*128*4 bytes, Lpad = L rounded up to
 * 128) is taken from the stream-ordered allocator. With D = 128 dq is summed with f32 reductions
 * in global memory, so its bits may differ from run to run in the last place; the environment
 * variable GTB_BWD_SPLIT_DQ=1 (read once per process) selects a separate, deterministic dq kernel,
 * which then runs on an internal per-device stream forked from and joined back into `stream`
 * within the call, so the call's work stays ordered on `stream` (and under stream capture, in the
 * captured graph). */
GTB_API int gtb_sdpa_bwd(const gtb_tensor4 *dout, const gtb_tensor4 *q, const gtb_tensor4 *k,
                         const gtb_tensor4 *v, const gtb_tensor4 *mask, const gtb_tensor4 *out,
                         const void *lse, float scale, int is_causal,
                         gtb_tensor4 *dq, gtb_tensor4 *dk, gtb_tensor4 *dv, void *stream);

/* Options of gtb_sdpa_fwd_ex / gtb_sdpa_bwd_ex (NULL = all zero).
 *   flags: GTB_BWD_DETERMINISTIC (backward): dq from the separate dq kernel, the same bits on every
 *     run (what the environment variable GTB_BWD_SPLIT_DQ=1 selects for every call); needed where a
 *     recomputed backward must repeat exactly, as under activation checkpointing (reference
 *     gguf_train/utils/checkpoint.py:159-222) or torch.use_deterministic_algorithms.
 *   dropout_p in [0, 1): dropout on the attention probabilities, as the reference's
 *     F.scaled_dot_product_attention(dropout_p > 0) (gguf_train/nn/functional.py:750-767): each
 *     probability is dropped with probability dropout_p and the kept ones scaled by 1/(1 - dropout_p);
 *     the softmax normaliser and the lse are those of the undropped probabilities.
 *   dropout_seed: the keep / drop decision of element (b, h, l, s) is a pure function of the seed and
 *     the indices (a counter-based hash, no generator state), so the backward given the forward's
 *     seed reproduces the forward's mask exactly, on any kernel. */
typedef struct gtb_sdpa_opts {
    int32_t flags;
    float dropout_p;
    uint64_t dropout_seed;
} gtb_sdpa_opts;
#define GTB_BWD_DETERMINISTIC 1

/* gtb_sdpa_fwd with options (dropout). Replaces the same reference function as gtb_sdpa_fwd, and the
 * dropout branch of F.scaled_dot_product_attention (gguf_train/nn/functional.py:750-767). */
GTB_API int gtb_sdpa_fwd_ex(const gtb_tensor4 *q, const gtb_tensor4 *k, const gtb_tensor4 *v,
                            const gtb_tensor4 *mask, float scale, int is_causal,
                            gtb_tensor4 *out, void *lse, const gtb_sdpa_opts *opts, void *stream);

/* gtb_sdpa_bwd with options (determinism, dropout: pass the forward's dropout_p and seed).
 * Replaces the same reference function as gtb_sdpa_bwd. */
GTB_API int gtb_sdpa_bwd_ex(const gtb_tensor4 *dout, const gtb_tensor4 *q, const gtb_tensor4 *k,
                            const gtb_tensor4 *v, const gtb_tensor4 *mask, const gtb_tensor4 *out,
                            const void *lse, float scale, int is_causal,
                            gtb_tensor4 *dq, gtb_tensor4 *dk, gtb_tensor4 *dv, const gtb_sdpa_opts *opts,
                            void *stream);

/* Attention weights (probabilities) of a forward that has run, from its lse: the need_weights=True
 * output of MultiheadAttention (reference gguf_train/nn/modules/transformer.py:153-166, which forms
 * them with matmul + softmax). P[b,h,l,s] = exp(scale * q.k + mask - lse[b,h,l]), 0 where masked or
 * (causal) s > l; with opts->dropout_p > 0 and the forward's seed, times keep / (1 - p) with the
 * forward's decisions (the weights the output was formed with). q, k, mask, scale, is_causal as in
 * gtb_sdpa_fwd; lse as gtb_sdpa_fwd wrote it. out: contiguous in q's dtype, (B, 1, L, S) with
 * average != 0 (mean over the H heads) or (B, H, L, S). Any head size up to 256. */
GTB_API int gtb_attn_weights(const gtb_tensor4 *q, const gtb_tensor4 *k, const gtb_tensor4 *mask, const void *lse,
                             float scale, int is_causal, int average, const gtb_sdpa_opts *opts, gtb_tensor4 *out,
                             void *stream);

/* Linear layer on the tensor cores: c (M, N) = a (M, K) b (N, K)^T (+ bias (N)), i.e. F.linear(a, b, bias)
 * for row-major a and b. Replaces gt_linear (reference csrc/gt_ops_nn.cpp:256-335, a ggml_mul_mat graph)
 * for 16-bit operands: dtype bf16 or f16 for a, b, bias (nullable) and c; f32 accumulation.
 * lda, ldb, ldc: elements between consecutive rows, multiples of 8 (16-byte rows); pointers 16-byte
 * aligned; K > 0. MultiheadAttention's projections and their backward products use it. */
GTB_API int gtb_linear(const void *a, const void *b, const void *bias, void *c, int64_t M, int64_t N, int64_t K,
                       int64_t lda, int64_t ldb, int64_t ldc, int dtype, void *stream);

/* Q8_0 quantisation of n_rows rows of row_len values (row_len % 32 == 0) into GGUF Q8_0 blocks
 * (fp16 scale + 32 int8, 34 bytes per 32 values), bit-exact with ggml's reference quantiser.
 * Replaces gt_quantize(t, GT_Q_BASE + 8) (reference csrc/gt_ops_extra.cpp:2002, which goes
 * through a host float buffer in gt_tensor_to_dtype, csrc/gt_core.cpp:792-840).
 * x: contiguous f32/f16/bf16 (x_dtype); out: n_rows * row_len / 32 * 34 bytes. */
GTB_API int gtb_q8_0_quantize(const void *x, int x_dtype, int64_t n_rows, int64_t row_len,
                              void *out, void *stream);

/* KV-cache append on the device (new export; the reference appends by quantising on the host through
 * gt_tensor_to_dtype, csrc/gt_core.cpp:792-840, and concatenating). x: contiguous (B, Hkv, n_new, D)
 * f32/f16/bf16, D % 32 == 0; row t of (b, hk) is quantised exactly as gtb_q8_0_quantize does into
 * row pos[b] + t of cache (B, Hkv, Smax, D/32*34 bytes, the layout gtb_decode_q8_0 reads). pos:
 * device int32 (B), the sequences' current lengths (gtb_decode_q8_0's seq_lens); with advance != 0 a
 * second kernel then adds n_new to every pos[b]. A destination row outside [0, Smax) is skipped and
 * sets the device status word to 60 (read with gtb_device_status). */
GTB_API int gtb_q8_0_append(const void *x, int x_dtype, int64_t B, int64_t Hkv, int64_t n_new, int64_t D,
                            void *cache, int64_t Smax, int32_t *pos, int advance, void *stream);

/* The same with each new row first rotated (RoPE, as gtb_rope with backward = 0) for its cache
 * position pos[b] + t, in f32 before quantising: the rotated keys land in the cache without an
 * intermediate rounding. Replaces gt_rope (csrc/gt_ops_nn.cpp:2409) followed by the quantising append. */
GTB_API int gtb_q8_0_append_rope(const void *x, int x_dtype, int64_t B, int64_t Hkv, int64_t n_new, int64_t D,
                                 void *cache, int64_t Smax, int32_t *pos, int advance, int n_dims, int mode,
                                 float freq_base, float freq_scale, void *stream);

/* Rotary position embedding on the device. Replaces gt_rope / gt_rope_backward (reference
 * csrc/gt_ops_nn.cpp:2409-2421, ggml_rope_ext with ext_factor 0, attn_factor 1): x, out (B, H, S, D)
 * contiguous f32/f16/bf16 (computed in f32, stored in x's type), pos device int32 with n_pos >= S
 * entries (one per sequence element, shared by batch and heads), n_dims even in [2, D], mode 0
 * (pairs 2i, 2i+1) or 2 (NeoX: pairs i, i + n_dims/2), angle of pair i = freq_scale * p *
 * freq_base^(-2i/n_dims) accumulated as ggml's rope cache does; backward != 0 rotates by -angle.
 * Error texts are the reference's. */
GTB_API int gtb_rope(const void *x, int dtype, int64_t B, int64_t H, int64_t S, int64_t D, const int32_t *pos,
                     int64_t n_pos, int n_dims, int mode, float freq_base, float freq_scale, int backward, void *out,
                     void *stream);

/* Q8_0 -> f32/f16/bf16 (out_dtype), x = q * d. Replaces gt_dequantize (csrc/gt_ops_extra.cpp:2006). */
GTB_API int gtb_q8_0_dequantize(const void *blocks, int64_t n_rows, int64_t row_len,
                                void *out, int out_dtype, void *stream);

/* One decode step against a Q8_0 KV cache.
 * Replaces the reference's route for this step: k.dequantize(), v.dequantize(), then
 * F.scaled_dot_product_attention(q, k, v) with q (B,H,1,D) (gguf_train/_tensor.py:1188-1196,
 * csrc/gt_ops_nn.cpp:2423-2525), which has no fused path.
 *   q: (B,H,D) contiguous, q_dtype f16/bf16/f32; k_q8, v_q8: (B,Hkv,Smax,D) as rows of D/32
 *   Q8_0 blocks; seq_lens: int32 (B), sequence b attends its first seq_lens[b] rows (clamped to
 *   [0, Smax]); out: (B,H,D) in q_dtype. D % 32 == 0 and D <= 256.
 * Split-KV: each (b, kv head) is cut into chunks of up to GTB_DECODE_CHUNK rows that run in
 * parallel; a second kernel merges the partial results. The partials, and a small work area
 * (item counter, per-sequence item prefix and item list of the tensor-core kernels), live in scratch taken
 * from the stream-ordered allocator. With D = 128, an f16 q, H/Hkv in {1,2,4,8}, an even Smax
 * and 16-byte aligned q/k/v the step runs on the tensor cores; otherwise on CUDA cores. */
#define GTB_DECODE_CHUNK 2048
GTB_API int gtb_decode_q8_0(const void *q, int q_dtype, const void *k_q8, const void *v_q8,
                            const int32_t *seq_lens, int64_t B, int64_t H, int64_t Hkv, int64_t Smax,
                            int64_t D, float scale, void *out, void *stream);

/* The same decode step as gtb_decode_q8_0, for callers that cannot let the library allocate device
 * memory: a serving runtime whose own allocator owns the GPU, or a loop that must never reach
 * cudaMalloc/cudaFree (they synchronise the device) or grow a memory pool mid-run. It allocates
 * nothing: the split-KV partial results go to a fixed device array of
 * GTB_DECODE_NOALLOC_SCRATCH_BYTES that every GPU loading this library holds until the process
 * exits. A call needs a work area of 8*(B+2) + 8*B*Hkv*ceil(Smax/GTB_DECODE_CHUNK) bytes rounded up
 * to 256, plus B*Hkv*ceil(Smax/GTB_DECODE_CHUNK)*(H/Hkv)*(D+2)*4 bytes of partials when Smax spans
 * more than one chunk; calls needing more than the array holds, or with B, Smax above 2^31 - 1, H
 * above 65535 or D above 256, are rejected with an error before any kernel runs (config 5a, B=64
 * Hkv=8 H=32 D=128 Smax=32768, needs 17.1 MB).
 * The first call on a device sets up the array's device address (call it once before any stream
 * capture). Calls share the array: calls whose kernels overlap on the GPU race. Its kernels report
 * a bounded wait that ran out through gtb_device_status(), like every other kernel.
 * No counterpart in the reference: it is an addition of this engine. */
#define GTB_DECODE_NOALLOC_SCRATCH_BYTES (40u << 20)
GTB_API int gtb_decode_q8_0_noalloc(const void *q, int q_dtype, const void *k_q8, const void *v_q8,
                                    const int32_t *seq_lens, int64_t B, int64_t H, int64_t Hkv,
                                    int64_t Smax, int64_t D, float scale, void *out, void *stream);

/* Log-sum-exp merge of a partial attention result into an accumulator (the combine step of the
 * long-context K/V ring: a causal attention over a sequence sharded across GPUs):
 *   o_acc: groups x rows x D float32, lse_acc: groups x rows float32 (contiguous; start at 0 / -inf),
 *   o_part: element g*part_gstride + r*D + d of part_dtype (f32/f16/bf16), lse_part: g*lse_gstride + r
 *   (natural-log sums as gtb_sdpa_fwd writes them). Rows with lse -inf contribute nothing.
 * No counterpart in the reference, which has no multi-device path. */
GTB_API int gtb_attn_merge(float *o_acc, float *lse_acc, const void *o_part, const float *lse_part,
                           int part_dtype, int64_t groups, int64_t rows, int64_t D, int64_t part_gstride,
                           int64_t lse_gstride, void *stream);

/* Rotary position embedding with several position axes (time, height, width of images and video), of
 * one tensor or of q and k in one launch. New export; gtb_rope takes one position per token.
 *   x (B,H,S,D), out of x's shape and dtype; k, k_out (B,Hkv,S,D) or both NULL; f32/f16/bf16, any
 *   strides with a unit innermost one; out may be x (in place) when both have the same strides.
 *   pos: device int32, axis a's position of token (b, s) at pos[a * pos_axis + b * pos_batch + s]
 *   (pos_batch 0: shared by the batch).
 *   sections[n_axes] (1 to 4 axes): pairs of dimensions per axis, P = their sum, 2 P <= D <= 256.
 *   Axis of pair i: blocks (the first sections[0] pairs axis 0, ...), or with GTB_ROPE_INTERLEAVED
 *   a = i mod n_axes if i < n_axes * sections[a], else 0 (which has to give every axis its sections).
 *   Frequency of pair i: freq_scale * freq_base^(-i / P); with GTB_ROPE_PER_AXIS the j-th pair of axis a
 *   has freq_scale * freq_base^(-j / sections[a]).
 *   mode 0 (pairs 2i, 2i+1) or 2 (pairs i, i + P); dims >= 2 P pass through; backward != 0 rotates by
 *   -angle (the gradient).
 * Angles are turns in 64-bit fixed point: position x frequency modulo one turn is right to 2^-31 of a turn at any int32
 * position (frequencies up to 1 radian a position) and then rounded to f32 (2^-26 of a turn at most), so long positions
 * lose nothing against short ones; gtb_rope instead follows ggml's f32 accumulation, and the two differ by that rounding
 * where they can express the same rotation. */
#define GTB_ROPE_INTERLEAVED 1
#define GTB_ROPE_PER_AXIS 2
GTB_API int gtb_rope_axes(const gtb_tensor4 *x, gtb_tensor4 *out, const gtb_tensor4 *k, gtb_tensor4 *k_out,
                          const int32_t *pos, int64_t pos_axis, int64_t pos_batch, const int32_t *sections, int n_axes,
                          int mode, int flags, float freq_base, float freq_scale, int backward, void *stream);

/* A KV cache held in 8 bits with one scale for each block of `block` tokens and kv head:
 * value = code * scale. New exports; the reference's only 8-bit cache is Q8_0 (a scale per 32 values).
 *   k, v: (B,Hkv,Smax,D) contiguous codes, 16-byte aligned: int8 (GTB_KV8_INT8, largest code 127) or OCP
 *   e4m3 (GTB_KV8_E4M3, 448). k_scale, v_scale: (B,Hkv,ceil(Smax/block)) f32. lens: device int32 (B), rows
 *   held of each sequence (values outside [0, Smax] are read as the nearest end). block 16, 32, 64 or
 *   128; D a multiple of 16, at most 256; B * Hkv at most 2^31 - 1, Smax below 2^30.
 * Rows at and past lens[b], and scales of blocks that hold none of the rows before it, may hold anything
 * (NaN included): no call lets them into a result. */
typedef struct gtb_kv8 {
    void *k, *v;
    float *k_scale, *v_scale;
    int32_t *lens;
    int64_t B, Hkv, Smax, D;
    int32_t block;
    int32_t format;
} gtb_kv8;
#define GTB_KV8_INT8 0
#define GTB_KV8_E4M3 1

/* Append rows: k, v (B,Hkv,n,D) f32/f16/bf16 (one dtype, any strides with a unit innermost one); the first
 * counts[b] of them (device int32, clamped to [0, n]; NULL: n) go to rows lens[b] .. of sequence b.
 * Per touched block: scale' = max(scale, amax * (1/M)), amax the largest finite |value| of the block's
 * new rows, M the largest code and 1/M its f32 reciprocal, `scale` only if the block held rows; where that grew the rows held are
 * requantised, code' = Q((code * scale) / scale'); new codes are Q(x / scale'). Every step is one
 * correctly rounded f32 operation; Q rounds to nearest even and saturates; NaN becomes code 0 and a
 * zero scale gives zero codes. With advance != 0 a second kernel sets lens[b] = min(lens[b] + counts[b],
 * Smax). Rows that would land past Smax are dropped and leave status 61 (gtb_device_status). */
GTB_API int gtb_kv8_append(const gtb_kv8 *cache, const gtb_tensor4 *k, const gtb_tensor4 *v, const int32_t *counts,
                           int advance, void *stream);

/* Rows start[b] .. start[b] + n - 1 of every head as values: k_out, v_out (B,Hkv,n,D) contiguous
 * f32/f16/bf16, code * scale rounded once. lens is not consulted (stored rows come back as they are);
 * rows outside [0, Smax) give 0. start: device int32 (B) or NULL (0). */
GTB_API int gtb_kv8_read(const gtb_kv8 *cache, const int32_t *start, gtb_tensor4 *k_out, gtb_tensor4 *v_out, void *stream);

/* Attention of q (B,H,Lq,D), H % Hkv == 0, over the cache: the queries are the last counts[b] (device int32,
 * clamped to [0, Lq]; NULL: Lq) of the lens[b] tokens cached, query i < counts[b] attending rows
 * s <= lens[b] - counts[b] + i. A query at or past counts[b], or with no row to attend, gives 0 and lse -inf.
 *   q f32/f16/bf16, any strides with a unit innermost one; out (B,H,Lq,D) in q's dtype, contiguous, 16-byte
 *   aligned; lse NULL or (B,H,Lq) f32; scale <= 0 means 1/sqrt(D).
 *   score_out NULL, or (B,Hkv,Smax) f32 that receives score_in (same shape, may be score_out itself) + the
 *   attention weight each row s < lens[b] got, summed over the kv head's query heads and all queries; other
 *   entries are not written. The sums run in a fixed order: the same bits on every run.
 * A weight is 2^(score - log-sum-exp) of f32 numbers: off by about |score| 2^-22 of itself (scores in powers of 2).
 * A v_scale below 2^-80 (a largest value below 1.1e-22) counts as 2^-80, and the v_scales of a head's blocks that hold
 * other values than zeros may lie up to 2^120 apart.
 * Scratch comes from the stream-ordered allocator: up to 1 GB for the scores (or, where query rows
 * are many, the f16 queries) that score_out is made from, up to 2 GB (or what one sequence takes: 2 bytes a code of its
 * capacity) for f16 copies of K and V where query rows are many, and some MB. */
GTB_API int gtb_kv8_attention(const gtb_tensor4 *q, const gtb_kv8 *cache, float scale, const int32_t *counts,
                              const float *score_in, float *score_out, gtb_tensor4 *out, float *lse, void *stream);

/* Eviction by accumulated attention weight, from src into dst (same B, Hkv, D, format; dst.Smax >= budget; the two
 * share no memory): of each (sequence, kv head) with more than `budget` rows the last `recent` and, of the
 * rows before those, the budget - recent of largest score (score (B,Hkv,src.Smax) f32; NaN counts as
 * -inf, ties go to the lowest row) are kept, in their order; a sequence of at most `budget` rows is kept whole. dst's
 * blocks get scale' = amax * (1/M) over their kept rows' values and codes Q((code * scale) / scale'), as an
 * append to an empty cache would; dst.lens = min(lens, budget). kept: (B,Hkv,budget) int32, the source row of
 * each kept row, -1 past the length. score_out: NULL or (B,Hkv,dst.Smax) f32, the kept rows' scores, 0 for
 * rows from there up to dst.Smax. 0 <= recent <= budget, 1 <= budget. */
GTB_API int gtb_kv8_evict(const gtb_kv8 *src, const float *score, int64_t budget, int64_t recent, const gtb_kv8 *dst,
                          float *score_out, int32_t *kept, void *stream);

/* A cache for latent attention: of each token one latent vector of R values, from which every head's keys and values
 * are made, and one rotary key of Dr values that the heads share. New exports; the reference has no such attention.
 *   rows: (B,Smax,R+Dr) contiguous f16 or bf16, 16-byte aligned, a row the latent followed by the rotary key; lens:
 *   device int32 (B), rows held of each sequence (values outside [0, Smax] are read as the nearest end). R a
 *   multiple of 64 from 64 to 512, Dr a multiple of 16 from 16 to 64; Smax below 2^30.
 * Rows at and past lens[b] may hold anything (NaN included): no call lets them into a result. */
typedef struct gtb_latent {
    void *rows;
    int32_t *lens;
    int64_t B, Smax;
    int32_t R, Dr;
    int32_t dtype;
} gtb_latent;

/* Append rows: latent (B,1,n,R) and k_rope (B,1,n,Dr), f32/f16/bf16 (one dtype, any strides with a unit innermost one);
 * the first counts[b] of them (device int32, clamped to [0, n]; NULL: n) go to rows lens[b] .. of sequence b, rounded
 * once to the cache's type. With rope_mode 0 (pairs 2i, 2i+1) or 2 (pairs i, i + Dr/2) the rotary key is first rotated,
 * in f32, for position offset[0] + lens[b] + i (offset: device int32, or NULL: 0; mostly the lens of a prefix, but any number
 * of positions, whether or not a cache holds as many rows: read as it is, below 0 as 0), its pairs' frequencies freq_scale * freq_base^(-2i / Dr) and angles those of gtb_rope_axes; with -1 it is taken as given.
 * With advance != 0 a second kernel sets lens[b] = min(lens[b] + counts[b], Smax). Rows that would land past Smax are
 * dropped and leave status 62 (gtb_device_status). */
GTB_API int gtb_latent_append(const gtb_latent *cache, const gtb_tensor4 *latent, const gtb_tensor4 *k_rope,
                              const int32_t *counts, const int32_t *offset, int rope_mode, float freq_base,
                              float freq_scale, int advance, void *stream);

/* Attention in the absorbed form: q (B,H,Lq,R+Dr) in the cache's dtype, its first R values the query taken through the
 * keys' up-projection, the other Dr the rotated ones. The queries are the last counts[b] (device int32, clamped to
 * [0, Lq]; NULL: Lq) of the lens[b] tokens cached, and query i < counts[b] attends every row of the prefix and rows
 * s <= lens[b] - counts[b] + i of its sequence: score = scale * q . row, out (B,H,Lq,R) = sum of weight * latent
 * (the values' up-projection is the caller's next product). A query at or past counts[b], or with no row to attend,
 * gives 0 and lse -inf.
 *   prefix: NULL, or a cache of one sequence (B = 1, same R, Dr and dtype) whose rows come before every sequence's own.
 *   Where H * Lq is at most 32, as many sequences as fill 64 query rows read them together; beyond that each block of up to 64 query
 *   rows of a sequence does. q 16-byte aligned, any strides that are positive multiples of 8 with a unit innermost one; out
 *   contiguous, 16-byte aligned; lse NULL or (B,H,Lq) f32; scale positive, below 1e38.
 * Scores, maxima, sums and outputs are f32; a weight is rounded to the cache's type (in f16 to 11 bits, or to steps of 2^-24 of
 * its row's largest where those are coarser) before it meets the latents, and out is rounded once.
 * Scratch from the stream-ordered allocator, for f32 parts of rows that several thread blocks worked on, some 4 R + 8 bytes a row: two slots a
 * multiprocessor of an item's rows (up to 64; 38 MB on 148 with R = 512). Where sequences read a prefix together, 64 rows for each
 * multiprocessor and each such group of sequences, and H * Lq rows (to a multiple of 16) for each multiprocessor and sequence. */
GTB_API int gtb_latent_attention(const gtb_tensor4 *q, const gtb_latent *cache, const gtb_latent *prefix, float scale,
                                 const int32_t *counts, gtb_tensor4 *out, float *lse, void *stream);

/* Attention in the expanded form, for prompts and training: q (B,H,L,Dn+Dr), k (B,Hkv,S,Dn), k_rope (B,1,S,Dr) shared by the
 * heads, v (B,Hkv,S,Dn); f16 or bf16 (one dtype), Dn 64 or 128, Dr a multiple of 16 from 16 to 64, H % Hkv == 0;
 *   score = scale * (q[..Dn] . k + q[Dn..] . k_rope), out (B,H,L,Dn); is_causal masks s > l (top-left aligned).
 *   seq_lens: NULL, or device int32 (B) with L = S: tokens from seq_lens[b] (clamped to [0, S]) on are not attended, whatever
 *   they hold; their out is 0, and all their gradients.
 *   lse: NULL or (B,H,L) f32, -inf where nothing is attended (out is 0 there). scale positive, below 1e38.
 * All tensors start on 16 bytes, with a unit innermost stride and others that are positive multiples of 8.
 * Without sequences, without heads, or with neither queries nor keys nothing is done, but the backward refuses keys that there is no
 * head for (their gradients have values); queries without keys, and keys without queries, are refused.
 * The backward takes the forward's out and lse and writes dq, dk, dk_rope (summed over all heads) and dv, in fixed order:
 * the same bits on every run. Its weights are 2^(score - log-sum-exp) of f32 numbers: off by about |score| 2^-22 of themselves
 * (scores in powers of 2). Its scratch, 4 (2 B H L' + B Hkv S Dr) bytes with L' = L to a multiple of 64, comes from the
 * stream-ordered allocator.
 * Scores, maxima, sums and what the products add up to are f32. Rounded to the inputs' type are, once each: a weight before it meets v or
 * grad_out; ds = weight * (grad_out . v - grad_out . out) before it meets q or k (f16 has steps of 2^-24 for both, and ds becomes
 * infinite past 65504); the results. grad_out . out is formed of the rounded out. Gradients of bf16 inputs are off by some 0.0024
 * of their norm (over a handful of keys 0.0036), where rounding the exact ones leaves 0.0017. */
GTB_API int gtb_latent_sdpa_fwd(const gtb_tensor4 *q, const gtb_tensor4 *k, const gtb_tensor4 *k_rope, const gtb_tensor4 *v,
                                const int32_t *seq_lens, float scale, int is_causal, gtb_tensor4 *out, float *lse,
                                void *stream);
GTB_API int gtb_latent_sdpa_bwd(const gtb_tensor4 *grad_out, const gtb_tensor4 *q, const gtb_tensor4 *k,
                                const gtb_tensor4 *k_rope, const gtb_tensor4 *v, const gtb_tensor4 *out, const float *lse,
                                const int32_t *seq_lens, float scale, int is_causal, gtb_tensor4 *dq, gtb_tensor4 *dk,
                                gtb_tensor4 *dk_rope, gtb_tensor4 *dv, void *stream);

/* Kernel family of the calling thread's last gtb_sdpa_fwd / gtb_sdpa_fwd_rope / gtb_sdpa_bwd call:
 * "tcgen05" (tensor cores, TMA), "tcgen05+rope" (the same with q rotated inside the kernel),
 * "f32_tiled" (fp32 with head size 64, register-blocked on the CUDA cores) or "simt" (one warp per
 * row; "" before the first). Lets a caller or a test see which path a call took. */
GTB_API const char *gtb_last_path(void);

/* Thread-local message of the last failure ("" if none). */
GTB_API const char *gtb_last_error(void);
GTB_API void gtb_clear_error(void);

/* Synchronises the current device and returns (then clears) its kernel status words: 0 = fine,
 * otherwise the code a kernel wrote when one of its bounded waits ran out or a check failed (the
 * first nonzero of the main word and of the fixed word of gtb_decode_q8_0_noalloc). Allocates
 * nothing. Replaces nothing in the reference, which runs no device kernels; its errors follow
 * gt_last_error (csrc/gt_core.cpp:7-23). */
GTB_API int gtb_device_status(void);

/* Failure-detection self-test: launches on `stream` a one-warp kernel that waits on an mbarrier
 * nothing ever arrives at, with the same bounded wait every kernel of this library uses but a limit
 * of `limit_cycles` SM cycles (1000 .. 2^31) instead of about a second. The wait gives up, the
 * kernel records status 90 and returns: gtb_device_status() then reports 90 once, and the device
 * stays usable. No counterpart in the reference, which has no device code. */
GTB_API int gtb_selftest_wait_timeout(int64_t limit_cycles, void *stream);

/* Build-time facts: number of sm_100a kernels compiled in, and a version string. */
GTB_API const char *gtb_version(void);

#ifdef __cplusplus
}
#endif

#endif /* GTB_ATTN_H */
