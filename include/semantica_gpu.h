/*
 * semantica_gpu.h -- C ABI of the MI355X (gfx950) EmbeddingGemma-300M Q8_0
 * forward library (libsemantica_gpu.so).
 *
 * Plain C types only: host or device pointers, sizes, int status codes.  No
 * exception or abort crosses this boundary; failures return a negative SG_ERR_*
 * code and sg_last_error() (thread-local) describes the most recent one.
 *
 * Each entry point replaces one seam of the reference Go implementation
 * (headlands-org/go-semantica); the citation is given beside it.  Paths are
 * relative to that source tree.
 */
#ifndef SEMANTICA_GPU_H
#define SEMANTICA_GPU_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SG_ABI_VERSION 2

/* Status codes.  The first four are the error cases of forwardINT8WithDim
 * (internal/runtime/model_int8.go:150-171) and ForwardWithDim
 * (internal/runtime/model.go:661-667). */
#define SG_OK 0
#define SG_ERR_EMPTY (-1)     /* "empty input": a sequence with no tokens        */
#define SG_ERR_TOO_LONG (-2)  /* "sequence too long: %d > %d"                    */
#define SG_ERR_TOKEN (-3)     /* "token ID out of range: %d"                     */
#define SG_ERR_DIM (-4)       /* "target dimension %d out of range (1..%d)"      */
#define SG_ERR_INVALID (-5)   /* bad argument / unsupported shape (kernel seams panic here) */
#define SG_ERR_DEVICE (-6)    /* HIP runtime failure                              */
#define SG_ERR_NOMEM (-7)     /* device or host allocation failed                 */

typedef struct sg_ctx sg_ctx;             /* one GPU: device ordinal + stream + scratch */
typedef struct sg_model sg_model;         /* weights resident in HBM + forward workspace */
typedef struct sg_q8_weight sg_q8_weight; /* one repacked Q8_0 matrix                    */

/* ModelConfig, internal/runtime/model.go:16-31 (fields parseConfig fills,
 * :424-517).  head_dim = embed_dim / num_heads and the attention scale
 * 1/sqrt(head_dim) are derived exactly as parseConfig derives them. */
typedef struct sg_model_config {
  int32_t embed_dim;    /* gemma-embedding.embedding_length  (768)  */
  int32_t num_layers;   /* block_count                        (24)   */
  int32_t num_heads;    /* attention.head_count               (3)    */
  int32_t num_kv_heads; /* attention.head_count_kv            (1)    */
  int32_t interm_dim;   /* feed_forward_length                (1152) */
  int32_t max_seq_len;  /* context_length                     (2048) */
  int32_t vocab_size;   /* len(tokenizer.ggml.tokens)         (262144) */
  float norm_eps;       /* attention.layer_norm_rms_epsilon   (1e-6) */
  float rope_base;      /* rope.freq_base                     (10000) */
} sg_model_config;

/* Host pointers to one layer's GGUF tensors, exactly as stored in the file
 * (loadLayerINT8, internal/runtime/model_int8.go:54-119): Q8_0 matrices are
 * raw 34-byte blocks, row-major [out][in/32]; norms are F32 vectors. */
typedef struct sg_layer_desc {
  const void *attn_q, *attn_k, *attn_v, *attn_output; /* blk.N.attn_{q,k,v,output}.weight */
  const void *ffn_gate, *ffn_up, *ffn_down;           /* blk.N.ffn_{gate,up,down}.weight  */
  const float *attn_norm, *attn_q_norm, *attn_k_norm; /* blk.N.attn_norm / attn_{q,k}_norm */
  const float *post_attention_norm, *ffn_norm, *post_ffw_norm;
} sg_layer_desc;

typedef struct sg_model_desc {
  sg_model_config config;
  const void *token_embd;     /* token_embd.weight, Q8_0 [vocab][embed_dim/32][34 B] */
  const float *output_norm;   /* output_norm.weight [embed_dim] */
  const sg_layer_desc *layers;/* num_layers entries */
} sg_model_desc;

/* ---- context ----------------------------------------------------------- */

/* Opens device `device_ordinal`, creates a default-priority stream.
 * (The reference has no device; this is the handle the Go cgo shim keeps.) */
int sg_init(int device_ordinal, sg_ctx **out);
void sg_shutdown(sg_ctx *ctx);
const char *sg_last_error(void);
int sg_abi_version(void);

/* ---- model seam --------------------------------------------------------- */

/* Replaces LoadModel/loadModel's weight setup (internal/runtime/model.go:233-315,
 * :520-552; model_int8.go:54-140): copies every tensor to HBM once, repacks
 * the Q8_0 matrices for the MFMA GEMM and extracts the fp32 block scales with
 * the IEEE converter (model_int8.go:543-597); the token embedding keeps the
 * halving converter of DequantizeQ8_0Row (gguf/tensor.go:157-240).  Host
 * buffers may be freed after return (unlike the Go zero-copy views). */
int sg_model_load(sg_ctx *ctx, const sg_model_desc *desc, sg_model **out);
void sg_model_free(sg_model *model);

/* ---- GGUF model images ---------------------------------------------------
 * parseConfig (internal/runtime/model.go:424-517) over a GGUF v3 image
 * (gguf/reader.go:98-178): fills *out from the metadata.  Host only; no
 * device call. */
int sg_gguf_read_config(const void *data, size_t size, sg_model_config *out);

/* LoadModelFromBytes (model.go:250-262) for the INT8 path: parses the image,
 * checks the tensors the forward reads (token_embd and the seven layer
 * matrices Q8_0; attn_norm/ffn_norm F32 or Q8_0; q/k norms, post norms and
 * output_norm optional) and calls sg_model_load.  The image may be released
 * after return.  No tokenizer is built: the library takes token IDs. */
int sg_model_load_gguf(sg_ctx *ctx, const void *data, size_t size, sg_model **out);

/* LoadModel (model.go:236-248): the same from a file, memory-mapped for the
 * duration of the call. */
int sg_model_load_gguf_file(sg_ctx *ctx, const char *path, sg_model **out);

/* Batched ForwardWithDim (internal/runtime/model.go:661-667 ->
 * forwardINT8WithDim model_int8.go:148-256) over n_seq packed sequences:
 * tokens[seq_offsets[i] .. seq_offsets[i+1]) is sequence i (CSR offsets,
 * seq_offsets[0] == 0).  out[n_seq][out_dim] receives each sequence's
 * mean-pooled, L2-normalized embedding truncated to out_dim (1..embed_dim).
 * Every sequence is computed exactly as the reference computes it alone
 * (per-sequence activation scales, attention and pooling).  Host buffers;
 * synchronous.  A model serves one call at a time (calls are serialized by a
 * per-model mutex), as the reference serves concurrent callers. */
int sg_forward(sg_model *model, const int32_t *tokens, const int32_t *seq_offsets,
               int32_t n_seq, int32_t out_dim, float *out);

/* Same, with tokens and out in device memory (tokens already resident in
 * HBM); seq_offsets stays on the host.  `stream` (hipStream_t, may be NULL
 * for the context stream) orders the work; the call returns after the
 * result is complete and token IDs have been validated on the device. */
int sg_forward_device(sg_model *model, const int32_t *d_tokens, const int32_t *seq_offsets,
                      int32_t n_seq, int32_t out_dim, float *d_out, void *stream);

/* Layer tap for parity work (no counterpart in the reference API; it mirrors
 * the CPU oracle's stop-layer tap): runs the embedding and the first
 * n_layers layers (0..num_layers) of the batched forward and copies the
 * residual stream h [T][embed_dim] (before the final norm) into d_hidden.
 * Same argument checks and synchronization as sg_forward_device. */
int sg_forward_hidden(sg_model *model, const int32_t *d_tokens, const int32_t *seq_offsets,
                      int32_t n_seq, int32_t n_layers, float *d_hidden, void *stream);

/* Per-layer trace of the batched forward, for parity checks: runs the first
 * n_layers layers (1..num_layers) as sg_forward_hidden does and writes, for
 * each layer l, rows l*T .. l*T + T - 1 (T = seq_offsets[n_seq]) of
 *   d_qkv [n_layers][T][q_dim + 2*kv_dim]: the Q|K|V GEMM output, before
 *         QK-norm and RoPE (runAttentionINT8, model_int8.go:357-372),
 *   d_att [n_layers][T][q_dim]: the attention output before it is quantized
 *         (model_int8.go:481-507),
 *   d_h   [n_layers][T][embed_dim]: the residual stream after the layer
 *         (model_int8.go:232).
 * Any of the three may be NULL.  No counterpart in the reference, which keeps
 * these values internal to forwardINT8WithDim (model_int8.go:148-256). */
int sg_forward_trace(sg_model *model, const int32_t *d_tokens, const int32_t *seq_offsets, int32_t n_seq,
                     int32_t n_layers, float *d_qkv, float *d_att, float *d_h, void *stream);

/* ---- measurement hook ---------------------------------------------------
 * No counterpart in the reference (its benchmark only times whole Embed
 * calls, cmd/benchmark/main.go:553-715).  While enabled, sg_forward*
 * brackets every kernel launch with HIP events on the launch stream and
 * accumulates, per kernel class, the event-measured time, the launch count
 * and the algorithmic work of those launches (int8 ops for the GEMM, flops
 * for attention's two products, bytes read+written at the reference dtypes
 * for the bandwidth kernels).  sg_profile_read synchronizes and returns the
 * totals since the last enable. */
enum {
  SG_K_GEMM = 0,      /* Q8_0 GEMMs (QKV, gate/up; O and down below the fused size) */
  SG_K_ATTENTION = 1, /* fused MQA attention                          */
  SG_K_QUANTIZE = 2,  /* per-sequence int8 quantization               */
  SG_K_NORM = 3,      /* embed+norm, post-norm+residual+norm, QK-norm+RoPE */
  SG_K_GELU = 4,      /* GELUQuick * up                               */
  SG_K_POOL = 5,      /* mean-pool + L2                               */
  SG_K_OTHER = 6,     /* fills                                        */
  SG_K_GEMM_NORM = 7, /* O / down GEMM with the residual post-norm in one launch
                         (work: the GEMM's int8 ops)                   */
  SG_K_CLASSES = 8
};
typedef struct sg_profile {
  double ms[SG_K_CLASSES];        /* summed event time of the class's launches */
  double work[SG_K_CLASSES];      /* ops (GEMM), flops (attention) or bytes    */
  int64_t launches[SG_K_CLASSES];
} sg_profile;
int sg_profile_enable(sg_model *model, int on);
int sg_profile_read(sg_model *model, sg_profile *out);

/* Attention arithmetic of the forward.  SG_ATTN_FAST (the default) runs the
 * score and weight products on fp16 matrix cores as hi/lo splits (within
 * 1e-5 relative of the reference's float32 attention).  SG_ATTN_EXACT runs
 * multiHeadAttentionInternal's float32 operations in its order on the vector
 * ALUs (attention.go:101-363 with dotProductSIMD's eight-lane sums,
 * activation.go:161-213, axpyAccum): with it the whole forward gives the bits
 * of forwardINT8WithDim on the block-serial GEMM path
 * (matmul_inner_loop_fallback.go:16-43, model_int8.go:148-256), several times
 * slower.  Needs max_seq_len <= 2048.  Takes effect from the next forward.
 * No counterpart in the reference (which has one attention): the switch is
 * for callers that need embeddings identical to it, such as parity checks. */
#define SG_ATTN_FAST 0
#define SG_ATTN_EXACT 1
int sg_model_set_attention_mode(sg_model *model, int mode);

/* ---- kernel seam (device pointers, work on `stream`) ---------------------
 * sg_matmul_q8_0_int8 and sg_ffn_gate_up are asynchronous: they return once
 * their work is enqueued on `stream`.  They share the context's operand
 * scratch, so each is ordered on the GPU after the previous one of the same
 * context (an event; no host wait), whatever streams they use.  The other
 * calls (they read host-side seq_offsets, or dump into temporary buffers)
 * return after their work on `stream` has completed. */

/* Repacks one raw Q8_0 matrix [out_dim][in_dim/32][34 B] (host pointer) into
 * the device layout used by the GEMM (the int8 values block-major, one
 * byte per weight, plus the fp32 block scales).  in_dim must be a multiple
 * of 32.
 * (extractQ8_0Scales model_int8.go:543-569 + the weight bytes it views.) */
int sg_q8_weight_create(sg_ctx *ctx, const void *q8, int32_t out_dim, int32_t in_dim,
                        sg_q8_weight **out);
void sg_q8_weight_free(sg_q8_weight *w);

/* QuantizeSymmetricINT8Into (internal/kernels/quantize.go:29-103) applied to
 * each sequence of a packed tensor: x[rows][cols] fp32, rows grouped by the
 * host CSR seq_offsets[n_seq+1].  One scale per sequence (max|x|/127; all-zero
 * input gives scale 1 and zeros).  q_out int8 [rows][cols], scale_out[n_seq]. */
int sg_quantize_act(sg_ctx *ctx, const float *x, int32_t rows, int32_t cols,
                    const int32_t *seq_offsets, int32_t n_seq,
                    int8_t *q_out, float *scale_out, void *stream);

/* MatMulQ8_0INT8 (internal/kernels/quantize.go:346-458):
 * dst[b][n] = (sum_blocks float(P_block) * d[n][block]) * row_scale[b] with
 * P_block the exact int32 dot of a 32-wide block, accumulated block by block
 * with a fused multiply-add.  x int8 [batch][in_dim]; row_scale[batch]
 * (the reference's single input.Scale, repeated per row of a sequence). */
int sg_matmul_q8_0_int8(sg_ctx *ctx, float *dst, const sg_q8_weight *w, const int8_t *x,
                        const float *row_scale, int32_t batch, void *stream);

/* sg_matmul_q8_0_int8 without any device allocation: the same kernels and the
 * same results, with the activation operand relaid in a fixed per-device
 * array of SG_NOALLOC_SCRATCH_BYTES (resolved by sg_init, held until the
 * process ends) instead of a library-grown buffer.  No counterpart in the
 * reference: for callers that cannot allocate (HIP graph capture, serving
 * loops).  Limit: gemm_pad(batch) x in_dim bytes, where gemm_pad rounds up
 * to 256 rows; larger inputs return SG_ERR_INVALID before any launch.  Calls
 * that overlap on one device (e.g. on two streams) race on the array. */
#define SG_NOALLOC_SCRATCH_BYTES (64u << 20)
int sg_matmul_q8_0_int8_noalloc(sg_ctx *ctx, float *dst, const sg_q8_weight *w, const int8_t *x,
                                const float *row_scale, int32_t batch, void *stream);

/* Measurement hook (no counterpart in the reference): the HBM yardstick the
 * bandwidth-bound kernels are set against.  kind 0: c = a + b over n fp32
 * (8 B read, 4 B written per element); kind 1: c = int8 codes of a at a fixed
 * scale (4 B read, 1 B written: the quantizers' I/O; b unused).  One float4
 * per lane, launched `reps` times back to back on `stream` between two HIP
 * events; returns the average time per launch.  n a multiple of 4, device
 * buffers 16-byte aligned.  Synchronizes the stream. */
int sg_hbm_probe(sg_ctx *ctx, int32_t kind, const float *a, const float *b, void *c, int64_t n,
                 int32_t reps, void *stream, float *us_per_launch);

/* Measurement hook (no counterpart in the reference): the issue rate of the
 * Q8_0 GEMM's per-K-block arithmetic with no memory traffic, the compute
 * floor of those kernels.  kind 0: per 32x32 output subtile and K-block one
 * v_mfma_i32_32x32x32_i8 and the block-serial update (16 subtractions + 16
 * v_fmac, as the GEMM kernels issue them); kind 1: the VALU part alone;
 * kind 2: the MFMA alone; kind 3: the attention's v_mfma_f32_16x16x32_f16
 * alone (four independent chains; one instruction per "subtile-block").
 * waves_per_simd (1..8) waves run `iters` steps of two subtiles each on every
 * SIMD.  Returns the SIMD cycles per subtile and K-block (the launch's event
 * time x the shader clock, which the waves' s_memtime / s_memrealtime counts
 * give, / subtile-blocks per SIMD) and that clock in GHz.  Allocates and frees its own small buffers; synchronizes the
 * stream. */
int sg_issue_probe(sg_ctx *ctx, int32_t kind, int32_t waves_per_simd, int32_t iters, void *stream,
                   float *simd_cycles_per_block, float *clock_ghz);

/* Measurement hook for the GEMM kernel alone (no counterpart in the
 * reference): relays x into the operand layout once, then launches the same
 * GEMM kernel sg_matmul_q8_0_int8 uses `reps` times back to back on `stream`
 * between two HIP events and returns the average time per launch.  dst is
 * written as by sg_matmul_q8_0_int8.  Synchronizes the stream. */
int sg_matmul_q8_0_int8_bench(sg_ctx *ctx, float *dst, const sg_q8_weight *w, const int8_t *x,
                              const float *row_scale, int32_t batch, int32_t reps, void *stream,
                              float *us_per_launch);

/* The exact int32 block dot products of the same GEMM, out[batch][out_dim][in_dim/32]
 * (what matmulInnerLoop* converts with VCVTDQ2PS, simd_amd64.s:290). */
int sg_q8_block_sums(sg_ctx *ctx, int32_t *out, const sg_q8_weight *w, const int8_t *x,
                     int32_t batch, void *stream);

/* The FFN's first half as one GEMM (model_int8.go:520-535: MatMulQ8_0INT8 with
 * ffn_gate and with ffn_up, GELUQuickSIMD on the gate output, VecMulF32 by up):
 * dst[b][n] = geluquick(gate[b][n]) * up[b][n], where gate and up are exactly
 * what sg_matmul_q8_0_int8 returns for w_gate and w_up (same shapes, out_dim a
 * multiple of 32); bit-identical to those two calls followed by
 * sg_gelu_quick_mul. */
int sg_ffn_gate_up(sg_ctx *ctx, float *dst, const sg_q8_weight *w_gate, const sg_q8_weight *w_up,
                   const int8_t *x, const float *row_scale, int32_t batch, void *stream);

/* RMSNorm per row (internal/kernels/norm.go:8-36), AVX2 8-lane order.
 * dst may equal src.  n must be a multiple of 8. */
int sg_rmsnorm(sg_ctx *ctx, float *dst, const float *src, const float *weight,
               int32_t rows, int32_t n, float eps, void *stream);

/* Per-head RMSNorm with attn_q_norm / attn_k_norm then RoPE (model_int8.go:371-452;
 * rope_cache.go:15-107) on q[rows][n_heads*head_dim] and k[rows][n_kv*head_dim]
 * (row strides ldq, ldk floats), in place.  Positions restart at 0 for each
 * sequence of the host CSR seq_offsets.  head_dim must be 256. */
int sg_qknorm_rope(sg_ctx *ctx, float *q, int32_t ldq, float *k, int32_t ldk,
                   const float *q_norm, const float *k_norm, int32_t n_heads, int32_t n_kv_heads,
                   int32_t head_dim, float eps, float rope_base, int32_t max_seq_len,
                   const int32_t *seq_offsets, int32_t n_seq, void *stream);

/* MultiHeadAttentionChunked with mask=nil (internal/kernels/attention.go:88-363) per
 * sequence: bidirectional MQA, scale 1/sqrt(head_dim), fastExp softmax.
 * q[rows][ldq] (heads at h*head_dim), k,v[rows][ldkv]; out[rows][n_heads*head_dim].
 * head_dim must be 256 and n_heads/n_kv_heads <= 4. */
int sg_attention(sg_ctx *ctx, float *out, const float *q, int32_t ldq, const float *k,
                 const float *v, int32_t ldkv, int32_t n_heads, int32_t n_kv_heads,
                 int32_t head_dim, const int32_t *seq_offsets, int32_t n_seq, void *stream);

/* sg_attention in the reference's float32 order (MultiHeadAttentionChunked,
 * attention.go:88-363, mask nil; see SG_ATTN_EXACT): bit-identical to it.
 * Same arguments; any n_heads / n_kv_heads ratio, sequences up to 2048 keys,
 * q and k 16-byte aligned with strides multiples of 4. */
int sg_attention_exact(sg_ctx *ctx, float *out, const float *q, int32_t ldq, const float *k,
                       const float *v, int32_t ldkv, int32_t n_heads, int32_t n_kv_heads,
                       int32_t head_dim, const int32_t *seq_offsets, int32_t n_seq, void *stream);

/* GELUQuickSIMD then VecMulF32 (activation.go:47-145, matmul.go:238-259):
 * dst[i] = geluquick(gate[i]) * up[i], for `rows` rows of `cols` (strides ldg, ldu, ldd). */
int sg_gelu_quick_mul(sg_ctx *ctx, float *dst, int32_t ldd, const float *gate, int32_t ldg,
                      const float *up, int32_t ldu, int32_t rows, int32_t cols, void *stream);

/* Token embedding lookup + sqrt(embed_dim) scaling (model_int8.go:166-184, with
 * DequantizeQ8_0Row's halving fp16 converter) for the model's token_embd. */
int sg_embed_tokens(sg_model *model, float *dst, const int32_t *d_tokens, int32_t n_tokens,
                    void *stream);

/* MeanPoolingPartial + l2Normalize (attention.go:423-445, runtime/model.go:808-820)
 * per sequence: x[rows][ldx], out[n_seq][out_dim]. */
int sg_pool_l2(sg_ctx *ctx, float *out, const float *x, int32_t ldx, int32_t out_dim,
               const int32_t *seq_offsets, int32_t n_seq, void *stream);

/* ---- layer operators of sibling models (device pointers, work on `stream`) ----
 * No counterpart in the reference, which runs one architecture with one set of
 * weights: what a layer of another decoder-derived embedder, or a fine-tuned one,
 * needs beside the products above.  All of them take a packed batch whose CSR
 * offsets d_seq_offsets[n_seq + 1] are in device memory (sequence i is rows
 * d_seq_offsets[i] .. d_seq_offsets[i+1] - 1; ascending; empty sequences are
 * allowed), return once their work is enqueued, allocate nothing and wait for
 * nothing, so they may be captured into a HIP graph and called from several
 * threads or on several streams at once.  Rows of no sequence (before the first
 * or behind the last) are left as they were.  The contents of device arrays are
 * not checked; offsets outside 0 .. rows and ids that name nothing are never
 * followed out of the tensors.  With no rows nothing is done, and the rows' tensors
 * may be NULL.  Element types: */
#define SG_F32 0
#define SG_F16 1
#define SG_BF16 2

/* How a score becomes a weight in sg_attention_masked.  i and j: positions of a
 * query and a key in their sequence.  All pointers are device memory. */
typedef struct sg_attn_mask {
  float scale;            /* of q . k; 0: 1/sqrt(head_dim) */
  float softcap;          /* > 0: scores become softcap * tanh(score / softcap); 0: they stay */
  const float *slopes;    /* [n_heads]: slopes[h] * |i - j| is subtracted after the cap (slopes of any sign); NULL: nothing */
  const int32_t *doc_ids; /* [rows]: keys of the query's own document are visible, and none if its id is
                             negative (padding); NULL: the whole sequence is one document */
  const int32_t *prefix;  /* [n_seq]: with causal, a sequence's first prefix[i] keys are visible to all of
                             its queries; NULL: none */
  int32_t causal;         /* keys behind the query are hidden */
  int32_t window;         /* > 0: keys with |i - j| >= window are hidden, prefix or not; 0: none */
} sg_attn_mask;

/* Attention of every sequence with itself: out_i = sum_j softmax_j(score_ij) v_j
 * over the visible keys; zeros for a query that sees none, or none whose score
 * is above -infinity.  Hidden keys do not touch the result, whatever they hold
 * (infinities and NaN included).  What lies before the first sequence or behind the
 * last is not read as a key.  Inside a sequence a hidden key or value that is not finite
 * costs time: queries that see others of the same 32 to 64 keys are computed
 * again one key at a time (400 times as long at 1000 tokens).
 * q [rows][ldq] and out [rows][ldo] hold n_heads heads of head_dim side by side, k
 * [rows][ldk] and v [rows][ldv] n_kv_heads (a divisor of n_heads) of them, all of
 * type dtype; strides in elements.  Sums and softmax statistics are float32.
 * float32 products keep 22 bits of each operand (2^-37 of its row's largest value
 * at worst, of a weight times its value's size 2^-30 of the largest); 16-bit types round
 * the weights to their type (float32 tensors keep them; fp16's to 2^-31 of the
 * largest), and tanh is off by 2^-19 at most.
 * head_dim: a multiple of 8 up to 256; pointers 16-byte aligned, strides whole 16
 * bytes (k's and v's up to 2^22 elements); rows * n_heads up to 2^30 or a little
 * less; out apart from q, k and v (other columns of one tensor, with the same
 * stride, are).
 * mask NULL: scale 1/sqrt(head_dim), nothing hidden. */
int sg_attention_masked(sg_ctx *ctx, void *out, int64_t ldo, const void *q, int64_t ldq, const void *k, int64_t ldk,
                        const void *v, int64_t ldv, int32_t dtype, int32_t n_heads, int32_t n_kv_heads,
                        int32_t head_dim, int32_t rows, const int32_t *d_seq_offsets, int32_t n_seq,
                        const sg_attn_mask *mask, void *stream);

/* What stands between two blocks of a layer, in one pass:
 *   y   = x * rsqrt(mean(x^2) + eps) * w_post      (w_post NULL: y = x)
 *   sum = h + scale * gate * y                     (gate NULL: 1)
 *   xn  = sum * rsqrt(mean(sum^2) + eps) * w_pre   (from sum before it is rounded; xn NULL: not wanted)
 * x, h, sum, xn: [rows][cols] of type dtype with row strides in elements; w_post,
 * w_pre [cols] and gate float32.  d_seq_offsets NULL (n_seq 0): every row, one
 * gate [cols] for all.  Otherwise gate is [n_seq][cols], one for each sequence.
 * cols 1 .. 8192, rows and strides of any whole elements (whole 16 bytes are
 * faster).  The squares are summed in float32, as sg_rmsnorm's are: values past
 * 2^63 overflow them, and those of a row below 2^-75 are zeros, which eps 0 divides by.
 * sum and xn may each be x or h (same pointer and stride); otherwise no output overlaps
 * another tensor (other columns of the same one, with the same stride, do not). */
int sg_block_norm(sg_ctx *ctx, void *xn, int64_t ldxn, void *sum, int64_t lds, const void *x, int64_t ldx,
                  const void *h, int64_t ldh, int32_t dtype, int32_t rows, int32_t cols, const float *w_post,
                  const float *w_pre, float eps, const float *gate, float scale, const int32_t *d_seq_offsets,
                  int32_t n_seq, void *stream);

/* Low-rank adapters of one projection, laid out for the GPU once.  d_a
 * [n_adapters][rank][in_dim] and d_b [n_adapters][out_dim][rank] (device memory,
 * contiguous, type dtype; an adapter of a smaller rank is padded with zeros),
 * d_scales [n_adapters] float32.  rank 1 .. 256, in_dim and out_dim multiples of
 * 8.  The arrays are read on `stream` and may be freed after return, which waits
 * for that.  Freeing the bank waits for the device.  Neither is for a time when a thread
 * captures a graph. */
typedef struct sg_adapter_bank sg_adapter_bank;
int sg_adapter_bank_create(sg_ctx *ctx, const void *d_a, const void *d_b, const float *d_scales, int32_t dtype,
                           int32_t n_adapters, int32_t rank, int32_t in_dim, int32_t out_dim, void *stream,
                           sg_adapter_bank **out);
void sg_adapter_bank_free(sg_adapter_bank *bank);

/* Bytes of workspace that sg_adapters_apply needs for `rows` rows or fewer (so a program
 * that allocates once asks for its largest batch). */
int sg_adapters_work_bytes(const sg_adapter_bank *bank, int32_t rows, size_t *bytes);

/* dst_t = base_t + scale_a * B_a (A_a x_t) for every row t, a = d_adapter_ids[i] of
 * the sequence i that holds it; dst_t = base_t where a names no adapter (-1).
 * base: the shared projection's output (sg_matmul_q8_0_int8's, for one); dst may
 * be base.  x [rows][ldx], base and dst [rows][ldb / ldd] of the bank's type,
 * strides in elements, pointers 16-byte aligned, strides whole 16 bytes.  work:
 * sg_adapters_work_bytes of device memory, 16-byte aligned, in use until the
 * call's work on `stream` is done (one for each stream or graph that runs at the
 * same time; a graph keeps its address, and the bank's).  dst does not overlap x,
 * or base unless it is base (other columns of one tensor, with the same stride, do not
 * overlap); work lies outside them all.  rows * out_dim: up to 2^36 or a little less.
 * The sums are float32 and in the same order every time. */
int sg_adapters_apply(sg_ctx *ctx, void *dst, int64_t ldd, const void *base, int64_t ldb, const sg_adapter_bank *bank,
                      const void *x, int64_t ldx, int32_t rows, const int32_t *d_seq_offsets, int32_t n_seq,
                      const int32_t *d_adapter_ids, void *work, size_t work_bytes, void *stream);

/* ---- kept keys and values ------------------------------------------------
 * For a causal sibling of the built-in model that answers requests behind text it
 * has run before: a document or an instruction is run once, its keys and values are
 * kept, and every request runs only its own tokens.  No counterpart in the reference.
 * The calls are asynchronous on `stream` (NULL: the context's), allocate nothing and may
 * be captured; the order of calls that write slots and calls that read them is the
 * caller's, by streams, as with any memory (a row with an infinity or a NaN, written to a cache
 * of bits 0, counts as written to all 32 slots of its s / 32). */

/* A cache of `slots` tokens' keys and values, n_kv_heads heads of head_dim (a multiple of
 * 8 up to 256; kept as 64, 128 or 256).  dtype: the type of rows in and out, and of
 * queries.  bits 0: kept as they are; bits 8: for each slot and head
 *   scale = max(max|x| / 127, 2^-126) as float32, code = the whole number nearest to
 *   x / scale (halves to even),
 * one scale for its key, one for its value.  A key or value that holds an infinity or a NaN
 * has a NaN for its scale: it reads as NaNs.  Slots that were never written are zeros.
 * Making a cache waits for its clearing, freeing it for the device; neither is for a time when
 * a thread captures a graph. */
typedef struct sg_kv_cache sg_kv_cache;
int sg_kv_cache_create(sg_ctx *ctx, int32_t slots, int32_t n_kv_heads, int32_t head_dim, int32_t dtype, int32_t bits,
                       void *stream, sg_kv_cache **out);
void sg_kv_cache_free(sg_kv_cache *cache);
/* Bytes of device memory that it holds. */
int sg_kv_cache_bytes(const sg_kv_cache *cache, size_t *bytes);

/* Rows of a packed batch into the cache and out of it: row t of sequence i (offsets
 * d_seq_offsets [n_seq+1] in device memory, ascending) is slot d_starts[i] + t -
 * d_seq_offsets[i].  k, v [rows][n_kv_heads * head_dim] of the cache's type with row strides
 * in elements, pointers 16-byte aligned, strides whole 16 bytes; a read's k and v do not
 * overlap (columns of one tensor, with the same stride, do not).  Rows of no sequence are
 * neither written nor read.  A slot outside the cache (every slot of a negative start)
 * is not written, and reads as zeros.  Where two sequences of a write name the same slot, the
 * later one's row is kept.  rows * n_kv_heads: up to 2^30, or somewhat more. */
int sg_kv_cache_write(sg_ctx *ctx, sg_kv_cache *cache, const void *k, int64_t ldk, const void *v, int64_t ldv,
                      int32_t rows, const int32_t *d_seq_offsets, int32_t n_seq, const int32_t *d_starts, void *stream);
int sg_kv_cache_read(sg_ctx *ctx, const sg_kv_cache *cache, void *k, int64_t ldk, void *v, int64_t ldv, int32_t rows,
                     const int32_t *d_seq_offsets, int32_t n_seq, const int32_t *d_starts, void *stream);

/* Which keys a batch's queries see, all arrays in device memory.  Sequence i's own keys are
 * slots starts[i] .. starts[i] + lengths[i] - 1, behind those of its prefix: sequences
 * shared[p] .. shared[p+1] - 1 (shared [n_prefix+1], ascending) share prefix p, slots
 * prefix_starts[p] .. + prefix_lengths[p] - 1; a sequence outside them all has none.
 * A range that does not lie in the cache is empty. */
typedef struct {
  const int32_t *starts;         /* [n_seq]                                             */
  const int32_t *lengths;        /* [n_seq]: own keys, the queries' tokens among them    */
  const int32_t *shared;         /* [n_prefix+1]                                         */
  const int32_t *prefix_starts;  /* [n_prefix]                                           */
  const int32_t *prefix_lengths; /* [n_prefix]                                           */
  int32_t n_prefix;              /* 0: no prefixes, the three above may be NULL           */
  float scale;                   /* of q.k; 0: 1/sqrt(head_dim)                          */
  float softcap;                 /* s = cap * tanh(s / cap); 0: none                     */
  int32_t causal;                /* a query sees no key behind its own place             */
  int32_t window;                /* ... none window places away or farther; 0: any       */
} sg_shared_keys;

/* Bytes of workspace that sg_attention_shared needs for so many rows, sequences and prefixes
 * or fewer of each. */
int sg_attention_shared_work_bytes(const sg_kv_cache *cache, int32_t n_heads, int32_t rows, int32_t n_seq,
                                   int32_t n_prefix, size_t *bytes);

/* Softmax attention of a packed batch's queries over kept keys, a prefix read once for all
 * that share it.  The n queries of a sequence are the last n places of its prefix and
 * own keys together (a query before the first place has none, and sees under causal nothing);
 * a row that sees no key, or only scores of -infinity, is zeros, rows of no sequence stay as
 * they were.  What hidden slots hold does not matter.  An infinity or a NaN in a value that is
 * seen is that dim's result whatever its key's score (a NaN where infinities of both signs are seen; kept
 * as codes it is a NaN in all dims, and none with a score of -infinity, which has no weight).
 * Sums are float32 and up to 2^10 times the number of keys larger than the result: values beyond
 * 2^90 may leave its range, and queries beyond 2^112 over codes, whose scores are formed before the
 * key's scale.  16-bit types round the weights to their type before they multiply values (fp16's to
 * 2^-31 of the largest at worst; over codes, with the value's scale in them, bf16's to bf16 and fp16's
 * within 2^-17); float32 keeps its bits, queries and values behind codes down to 2^-100, weights down to
 * 2^-126.  q, out [rows][n_heads * head_dim] of
 * the cache's type with row strides in elements, pointers 16-byte aligned, strides whole 16
 * bytes, apart from each other (other columns of one tensor are); n_heads is a multiple of the
 * cache's heads, head h reads key head h * n_kv_heads / n_heads.  rows * n_heads up to 2^25.
 * scale and softcap are 0 or lie within 1e-15 .. 1e15 (a scale of either sign).  work:
 * sg_attention_shared_work_bytes of device memory, 16-byte aligned, in use until the call's
 * work on `stream` is done (one for each stream or graph that runs at the same time; a graph
 * keeps its address, and the cache's), apart from q and out.  The same call on the same values
 * gives the same bits. */
int sg_attention_shared(sg_ctx *ctx, void *out, int64_t ldo, const void *q, int64_t ldq, const sg_kv_cache *cache,
                        int32_t n_heads, int32_t rows, const int32_t *d_seq_offsets, int32_t n_seq,
                        const sg_shared_keys *keys, void *work, size_t work_bytes, void *stream);

/* ---- 4-bit weights --------------------------------------------------------
 * A matrix [out_dim][in_dim] of 4-bit codes with a scale, and if need be a zero, for each
 * group of 32, 64 or 128 inputs: w = scale * (code - zero).  d_codes [out_dim][in_dim/2]: byte b
 * of a row holds input 2 b in its lower four bits and 2 b + 1 in its upper; d_scales
 * [out_dim][in_dim/group] of type scale_dtype, d_zeros the same as bytes 0 .. 15 (NULL: 8).
 * Laid out for the GPU once: the arrays (device memory, contiguous) are read on `stream` and
 * may be freed after return, which waits for that.  Making and freeing are not for a time when a
 * thread captures a graph.  No counterpart in the reference, which runs Q8_0 only. */
typedef struct sg_q4_weight sg_q4_weight;
int sg_q4_weight_create(sg_ctx *ctx, const uint8_t *d_codes, const void *d_scales, int32_t scale_dtype,
                        const uint8_t *d_zeros, int32_t out_dim, int32_t in_dim, int32_t group, void *stream,
                        sg_q4_weight **out);
/* The same from GGUF's raw Q4_0 blocks in host memory, row-major [out_dim][in_dim/32][18 B]: an
 * fp16 scale, then 16 bytes, the lower four bits of which are the block's inputs 0 .. 15 and the
 * upper ones 16 .. 31; zero 8.  Synchronous. */
int sg_q4_weight_create_q4_0(sg_ctx *ctx, const void *raw, int32_t out_dim, int32_t in_dim, sg_q4_weight **out);
void sg_q4_weight_free(sg_q4_weight *weight);

/* dst[m][n] = sum over k of w[n][k] x[m][k] for a few rows (16 or 32 of them share one
 * pass over the weights, more take one for every so many: from some 64 rows on a dense product of
 * 16-bit weights is faster, at 512 three to five times).  x [rows][in_dim], dst [rows][out_dim] of
 * type dtype with row strides in elements; x 16-byte aligned, its stride whole 16 bytes; dst does not overlap
 * x (other columns of one tensor, with the same stride, do not).  Weights are not rounded, sums
 * are float32 and in the same order every time; float32 rows keep their bits down to 2^-102 (what
 * lies below 2^-126 is lost of smaller values), and values beyond 2^116 may leave float32's range in a
 * group's sum, which is formed before its scale.  Asynchronous on `stream`, allocates nothing,
 * may be captured. */
int sg_matmul_q4(sg_ctx *ctx, void *dst, int64_t ldd, const sg_q4_weight *weight, const void *x, int64_t ldx,
                 int32_t dtype, int32_t rows, void *stream);

/* ---- tokenizer (internal/tokenizer) -------------------------------------
 * The reference's SentencePiece-style BPE tokenizer on the host: text ->
 * the token IDs sg_forward takes.  Same normalization (NFKC / accents /
 * lowercase), space handling, merge order (highest score, ties to the
 * rightmost pair), byte fallback and special tokens as tokenizer.go. */
typedef struct sg_tokenizer sg_tokenizer;

/* tokenizer.Config (tokenizer.go:46-53) plus the special ids
 * (LoadFromGGUF sets them from metadata, :570-595); -1 = none. */
typedef struct {
  int32_t add_bos, add_eos, lowercase, remove_accents, nfkc;
  int32_t bos_id, eos_id, unk_id, pad_id;
} sg_tokenizer_config;

/* tokenizer.New (tokenizer.go:56-97).  Token i is
 * token_data[token_offsets[i] .. token_offsets[i+1]) (UTF-8, any bytes);
 * token_types may be NULL (all normal).  "vocab and scores length mismatch"
 * cannot occur here (one n for both). */
int sg_tokenizer_create(const char *token_data, const int64_t *token_offsets, const float *scores,
                        const int32_t *token_types, int32_t n, const sg_tokenizer_config *cfg,
                        sg_tokenizer **out);

/* tokenizer.LoadFromGGUF (tokenizer.go:497-598) over a GGUF v3 image / file:
 * tokenizer.ggml.tokens, .scores, .token_type, .add_bos_token,
 * .add_eos_token and the special ids; NFKC on.  Same errors. */
int sg_tokenizer_from_gguf(const void *data, size_t size, sg_tokenizer **out);
int sg_tokenizer_from_gguf_file(const char *path, sg_tokenizer **out);

/* Tokenizer.Encode (tokenizer.go:99-133) of text[0..len): *n_ids receives the
 * number of IDs; the first min(n, cap) are written to ids (ids may be NULL to
 * query the count). */
int sg_tokenizer_encode(const sg_tokenizer *tok, const char *text, size_t len, int32_t *ids, int32_t cap,
                        int32_t *n_ids);

/* Encode of n_texts texts (text i = text_data[text_offsets[i] ..
 * text_offsets[i+1])) into one packed array: id_offsets[n_texts+1] receives
 * CSR offsets (the seq_offsets sg_forward takes); ids (capacity cap) may be
 * NULL to query the total, id_offsets[n_texts]. */
int sg_tokenizer_encode_batch(const sg_tokenizer *tok, const char *text_data, const int64_t *text_offsets,
                              int32_t n_texts, int32_t *ids, int64_t cap, int32_t *id_offsets);

/* Tokenizer.Decode (tokenizer.go:135-159): *len receives the byte length;
 * the first min(len, cap) bytes go to buf (not NUL-terminated). */
int sg_tokenizer_decode(const sg_tokenizer *tok, const int32_t *ids, int32_t n, char *buf, size_t cap,
                        size_t *len);

/* Tokenizer.VocabSize (tokenizer.go:438-440). */
int32_t sg_tokenizer_vocab_size(const sg_tokenizer *tok);

void sg_tokenizer_free(sg_tokenizer *tok);

/* ---- brute-force vector search (search/brute) ----------------------------
 * The reference's quantized brute-force index (search/brute/index.go,
 * builder.go, storage.go) with its vectors in HBM.  Scores are bit-identical
 * to the reference's amd64 AVX2 dot products (quant.go:79-135,
 * index.go:199-214, dot_amd64.s) and the top-k is the reference's streaming
 * selection (index.go:53-147), ties included; only the batching is new: one
 * call searches n_queries queries. */
typedef struct sg_index sg_index;

/* brute.QuantizationMode, search/brute/quant.go:8-15 */
#define SG_BF_FLOAT32 0
#define SG_BF_INT8 1
#define SG_BF_INT16 2

/* brute.NewBuilder(WithDimension(dim), WithQuantization(q)) + AddVector for each
 * (ids[i], vectors[i*dim ..]) + Build (builder.go:40-128): every vector is
 * L2-normalized (builder.go:131-141) and stored in mode q (quant.go:17-41).
 * Host vectors.  Errors as the reference: "brute: no vectors added" (n = 0),
 * "brute: duplicate id %d", "brute: unsupported quantization %d". */
int sg_index_build(sg_ctx *ctx, int32_t dim, int32_t quantization, const int32_t *ids,
                   const float *vectors, int32_t n, sg_index **out);

/* Same with the vectors in device memory (row stride ld floats), e.g. the
 * embeddings sg_forward_device left in HBM; ids stay on the host. */
int sg_index_build_device(sg_ctx *ctx, int32_t dim, int32_t quantization, const int32_t *ids,
                          const float *d_vectors, int64_t ld, int32_t n, void *stream, sg_index **out);

/* Serializer.Deserialize (storage.go:43-45,94-153) of a "BRUT" v1 image. */
int sg_index_deserialize(sg_ctx *ctx, const void *data, size_t size, sg_index **out);

/* Serializer.Serialize (storage.go:31-41,47-91): *size receives the image
 * size; with buf == NULL nothing else is done. */
int sg_index_serialize(sg_index *index, void *buf, size_t cap, size_t *size);

/* Index.Dimension / Count (index.go:149-153) and the storage mode. */
int sg_index_info(const sg_index *index, int32_t *dim, int32_t *count, int32_t *quantization);

/* Index.Vector (index.go:155-172): the dequantized vector stored under id;
 * SG_ERR_INVALID when there is none (the reference returns ok = false). */
int sg_index_vector(sg_index *index, int32_t id, float *out);

/* SearchVector (normalize = 1, index.go:27-41) or SearchNormalized
 * (normalize = 0, index.go:43-51) for n_queries queries [n_queries][dim]
 * (host).  Query q gets n_found[q] = min(top_k, count) results in
 * out_ids/out_dist[q*top_k ...], distance descending, ties by id ascending.
 * top_k <= 0: "brute: topK must be positive".  One call at a time per index
 * (a per-index mutex). */
int sg_index_search(sg_index *index, const float *queries, int32_t n_queries, int32_t top_k,
                    int32_t normalize, int32_t *out_ids, float *out_dist, int32_t *n_found,
                    void *stream);

void sg_index_free(sg_index *index);

#ifdef __cplusplus
}
#endif
#endif /* SEMANTICA_GPU_H */
