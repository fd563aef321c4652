/*
 * libnemo: MI355X (gfx950) Nemotron-3-Embed encoder forward pass behind a
 * plain C ABI. This is the native side of the reference's embedding runtime
 * (src/webgpu/model.ts NemotronWebGPUModel / NemotronExecutionPlan and the
 * EmbeddingRuntime / EmbeddingPlan interfaces of
 * src/webgpu/embedding-engine.ts:7-14). Host bindings (Python ctypes in
 * nemo_amd, the Node-API addon) call exactly these symbols.
 *
 * Conventions: every call returns a nemo_status; on failure
 * nemo_last_error() returns a message for the calling thread (the reference
 * throws an Error with that message). No C++ exception crosses the ABI.
 * Host pointers are copied before a blocking call returns; output buffers
 * are owned by the caller. Pointers documented as "device" are HIP device
 * pointers on the context's device.
 */
#ifndef NEMO_H
#define NEMO_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef int32_t nemo_status;
#define NEMO_OK 0
#define NEMO_ERR_INVALID 1     /* bad argument, shape or format */
#define NEMO_ERR_MISSING 2     /* a tensor the graph needs was never set */
#define NEMO_ERR_DEVICE 3      /* HIP runtime failure */
#define NEMO_ERR_OOM 4         /* device or pinned host allocation failed */
#define NEMO_ERR_UNSUPPORTED 5 /* valid input this build does not execute */

/* GGML tensor type codes, src/gguf/types.ts:17-23. */
#define NEMO_TYPE_F32 0
#define NEMO_TYPE_F16 1
#define NEMO_TYPE_Q4_0 2
#define NEMO_TYPE_Q4_K 12
#define NEMO_TYPE_Q6_K 14
/* Q4_0 in the wgpack "q4_0-tile32-compact" layout: 20-byte records
 * [f16 d][2 zero bytes][16 nibble bytes] ordered tile (32 rows) -> 32-value
 * block -> row (src/prepacked/format.ts:65-99). Not a GGML type code; the
 * tensor is held and returned as NEMO_TYPE_Q4_0. */
#define NEMO_TYPE_Q4_0_TILE32 258

typedef struct nemo_ctx nemo_ctx;
typedef struct nemo_model nemo_model;
typedef struct nemo_plan nemo_plan;
typedef struct nemo_weight nemo_weight;

/* Model shape. The reference hard-codes these (src/webgpu/model.ts:19-28,
 * src/webgpu/ops.ts:126,186,242,258); here they are parameters so one build
 * runs both the reference dims and other shapes of the same architecture. */
typedef struct nemo_dims {
  int32_t hidden;              /* 2048 */
  int32_t q_heads;             /* 24 */
  int32_t kv_heads;            /* 8 */
  int32_t head_dim;            /* 128 (64 also supported) */
  int32_t intermediate;        /* 6144 */
  int32_t layers;              /* 16 */
  int32_t vocab;               /* 131072 */
  int32_t merge_after_layer;   /* 4: MERGE_AFTER_LAYER, model.ts:26; 0..layers,
                                  where == layers merges just before the pool */
  float rms_epsilon;           /* 1e-5: model.ts:27 */
  float rope_theta;            /* 1e6: model.ts:28 */
  int32_t kv_stride_threshold; /* 2048: ops.ts:258 */
  int32_t kv_stride;           /* 3: ops.ts:258 */
  int32_t kv_dense_before_merge; /* 0: the code's rule (ops.ts:258) in every layer, so a request longer
                                    than the threshold samples keys before the merge too; 1: the rule
                                    README.md:26 states: layers before the merge attend every key, and
                                    merged sequences through the threshold use full attention */
} nemo_dims;

/* Fills the reference model's constants (src/webgpu/model.ts:19-28). */
void nemo_dims_reference(nemo_dims* out);

/* Message of the last failing call on this thread ("" if none). */
const char* nemo_last_error(void);

/* Library version string. */
const char* nemo_version(void);

/* Testing hook, no counterpart in the reference: the calling thread's
 * `checks`-th HIP status check from now on (counting every HIP call the
 * library makes and checks on that thread, launches included) fails as if
 * that call had returned an error, so tests can end an enqueue partway with
 * kernels already queued. 0 turns it off. */
void nemo_debug_fail_after(int32_t checks);

/* Open a context on HIP device `device` (replaces requestWebGPUDevice,
 * src/webgpu/device.ts:6-24). */
nemo_status nemo_init(int32_t device, nemo_ctx** out);
nemo_status nemo_shutdown(nemo_ctx* ctx);

/* ---- model (src/webgpu/model.ts:236-329) -------------------------------- */

nemo_status nemo_model_create(nemo_ctx* ctx, const nemo_dims* dims, nemo_model** out);

/* Upload one tensor (replaces createBufferWithData per tensor,
 * src/webgpu/model.ts:264-266,283-286). `dims` are GGUF dims (ne0 first: a
 * matrix of n rows by k columns is {k, n}). Matrices: NEMO_TYPE_Q4_K,
 * NEMO_TYPE_Q6_K or NEMO_TYPE_Q4_0 raw GGUF blocks, or NEMO_TYPE_Q4_0_TILE32
 * records of a .wgpack (k a multiple of 256 for every matrix type); norms:
 * NEMO_TYPE_F32; token_embd.weight:
 * NEMO_TYPE_Q6_K or NEMO_TYPE_F16. Names are the GGUF names; the fused
 * blk.N.attn_qkv.weight / blk.N.ffn_gate_up.weight may be given directly or
 * as their parts (attn_q/attn_k/attn_v, ffn_gate/ffn_up), fused at finalize
 * like combineQ4 (src/webgpu/model.ts:288-304). */
nemo_status nemo_model_set_tensor(nemo_model* model, const char* name, int32_t ggml_type, const int64_t* dims,
                                  int32_t n_dims, const void* bytes, size_t n_bytes);

/* Fill every tensor with seeded synthetic weights generated on the device:
 * matrices N(0, 0.02) quantized to Q4_K (ffn_down to Q6_K), norm weights 1,
 * token_embd.weight N(0, 0.02) as `embedding_type` (F16 or Q6_K). */
nemo_status nemo_model_synthesize(nemo_model* model, uint64_t seed, int32_t embedding_type);

/* Validate and fuse; required before nemo_plan_create. Errors name the
 * missing or malformed tensor (src/webgpu/model.ts:278,291-292,309,315,318). */
nemo_status nemo_model_finalize(nemo_model* model);

/* Copy a tensor back to the host in its GGUF byte layout. With out == NULL
 * only *n_bytes is written. */
nemo_status nemo_model_get_tensor(nemo_model* model, const char* name, int32_t* ggml_type, int64_t* dims4,
                                  void* out, size_t* n_bytes);

nemo_status nemo_model_destroy(nemo_model* model);

/* ---- execution plan (src/webgpu/model.ts:58-234) ------------------------ */

/* createPlan(batch, sequence) (src/webgpu/model.ts:328): activations for
 * `batch` requests of up to `sequence` tokens (batch <= 64). */
nemo_status nemo_plan_create(nemo_model* model, int32_t batch, int32_t sequence, nemo_plan** out);

/* EmbeddingPlan.run (src/webgpu/model.ts:146-176; src/webgpu/embedding-engine.ts:8):
 * ids[batch * sequence] padded after each request's tokens, lengths[batch]
 * with 1 <= lengths[b] <= sequence; writes out[batch * hidden] float32,
 * L2-normalised, in input order. Blocking. n_ids != batch * sequence fails
 * with 'token buffer does not match execution plan' (model.ts:147). */
nemo_status nemo_plan_run(nemo_plan* plan, const uint32_t* ids, size_t n_ids, const uint32_t* lengths,
                          size_t n_lengths, float* out);

/* Same graph with ids and out as device pointers, enqueued on `stream`
 * (hipStream_t; NULL = the plan's own stream); lengths are host values.
 * Returns once enqueued. Work of the plan enqueued earlier on another stream
 * is waited for on the device first (the runs share the plan's buffers). If
 * the enqueue fails partway, the call drains `stream` before it returns the
 * error, and later calls on the plan still order after what was queued. */
nemo_status nemo_plan_run_device(nemo_plan* plan, const uint32_t* d_ids, const uint32_t* lengths, size_t n_lengths,
                                 float* d_out, void* stream);

/* profile() (src/webgpu/model.ts:178-224): milliseconds per stage, summed
 * over layers, in the order of nemo_profile_stage_name. */
nemo_status nemo_plan_profile(nemo_plan* plan, const uint32_t* ids, size_t n_ids, const uint32_t* lengths,
                              size_t n_lengths, float* stage_ms, int32_t n_stages);
int32_t nemo_profile_stage_count(void);
const char* nemo_profile_stage_name(int32_t index);

/* destroy() (src/webgpu/model.ts:141-144). Waits for a call on the plan
 * that another thread is running, then for all work the plan enqueued (on
 * its own stream or a caller's), then frees it. The caller must not start
 * further calls on the plan, nor have any waiting to start: the host
 * bindings count their runs in flight and destroy once the last settles. */
nemo_status nemo_plan_destroy(nemo_plan* plan);

/* The plan's batch, sequence and the model's hidden width (any pointer may
 * be NULL): a binding sizes the embeddings of a run, batch * hidden floats,
 * from the plan itself. No counterpart in the reference, whose plan object
 * carries these fields (src/webgpu/model.ts:58-74). */
nemo_status nemo_plan_shape(nemo_plan* plan, int32_t* batch, int32_t* sequence, int32_t* hidden);

/* Copy one activation buffer of the last run to the host, for stage-wise
 * parity checks (the reference's buffers of src/webgpu/model.ts:80-94 are
 * debuggable the same way through readF16Buffer, src/main.ts:24-34). Names:
 * "x_full", "norm_full", "x_merged", "norm_merged", "qkv", "q", "k",
 * "attention", "delta" (written only by projections without a K split),
 * "ffn" (f16, packed rows of the last layer that wrote them) and
 * "embeddings" (float). With out == NULL only *n_bytes is
 * written (the buffer's capacity). Blocks until the plan's work is done. */
nemo_status nemo_plan_read_buffer(nemo_plan* plan, const char* name, void* out, size_t* n_bytes);

/* ---- kernel level (src/webgpu/quant-matmul.ts:438-563) ------------------- */

/* Upload one quantized matrix of n rows by k columns (k % 256 == 0) from raw
 * GGUF bytes: QuantMatmulKernel.createRun's weight buffer
 * (src/webgpu/quant-matmul.ts:503-509). Types Q4_K, Q6_K, Q4_0 (GGUF blocks) and
 * NEMO_TYPE_Q4_0_TILE32 (the wgpack records; quant-matmul.ts:99-108). */
nemo_status nemo_weight_create(nemo_ctx* ctx, int32_t ggml_type, int32_t n, int32_t k, const void* bytes,
                               size_t n_bytes, nemo_weight** out);
nemo_status nemo_weight_destroy(nemo_weight* weight);

#define NEMO_MATMUL_AUTO 0     /* GEMV for m <= 160, two-pass where it pays, else the fused GEMM */
#define NEMO_MATMUL_GEMM 1     /* MFMA GEMM decoding W inside the kernel (tiles chosen by size) */
#define NEMO_MATMUL_GEMV 2     /* split-K GEMV, m <= 160 */
#define NEMO_MATMUL_TWO_PASS 3 /* W expanded to f16 scratch (n * k halves, held by the weight),
                                  then an f16 MFMA GEMM; bit-identical to NEMO_MATMUL_GEMM */
#define NEMO_MATMUL_GEMM_MID 4 /* the fused GEMM on 64-row tiles with deep prefetch (the plan's choice
                                  for mid-size m); bit-identical to NEMO_MATMUL_GEMM */
#define NEMO_MATMUL_GEMM_SPLIT 5 /* the 64-row tiles with K split into fp32 partials summed in chunk
                                    order (the plan's choice for 17..64 rows); scratch is held by the
                                    weight and grows on demand */

/* Y[m, n] = f16(X[m, k] W[n, k]^T), fp32 accumulate; d_x f16 [m, k] and d_y
 * f16 [m, n] are device pointers (createRun + dispatch,
 * src/webgpu/quant-matmul.ts:503-563). */
nemo_status nemo_weight_matmul(nemo_weight* weight, const uint16_t* d_x, int32_t m, uint16_t* d_y, int32_t algo,
                               void* stream);

/* Bytes of the per-GPU static scratch that nemo_weight_matmul_static uses
 * (64 MiB): split-K partial sums need splits * m * n * 4 bytes, the two-pass
 * expansion n * k * 2 (a 16384 x 2048 or 2048 x 8192 matrix at most). */
#define NEMO_STATIC_SCRATCH_BYTES 67108864

/* No counterpart in the reference. nemo_weight_matmul for callers that
 * cannot allocate device memory (code under HIP graph capture, serving
 * loops, harnesses that forbid hipMalloc): same algorithms, kernels and
 * bits, but any scratch (the GEMV's and the split-K tiles' fp32 partial
 * sums, the two-pass f16 expansion of W) lives in a static array of
 * NEMO_STATIC_SCRATCH_BYTES that the library holds on each GPU until the
 * process ends; the call allocates and frees nothing. A call whose scratch
 * would exceed that size fails with NEMO_ERR_INVALID before launching
 * anything. Every call on one GPU shares the array: calls that overlap on
 * one GPU (concurrent streams, or host threads) race and must be ordered by
 * the caller. Under HIP graph capture: make one eager call of the same
 * shape and algorithm first (the first call of a kernel sets its LDS size
 * attribute); the captured launches record no memset, and replays equal
 * eager calls bit for bit (tests/test_zz_no_alloc.py). */
nemo_status nemo_weight_matmul_static(nemo_weight* weight, const uint16_t* d_x, int32_t m, uint16_t* d_y,
                                      int32_t algo, void* stream);

/* Decode the uploaded matrix to float32 [n, k] (device pointer); bit-exact
 * with dequantizeQ4KBlock / dequantizeQ6KBlock (src/gguf/quantization.ts:19-74). */
nemo_status nemo_weight_dequantize(nemo_weight* weight, float* d_out, void* stream);

/* Decode raw GGUF blocks at a 16-byte aligned device pointer to float32
 * and/or f16 (either output may be NULL): dequantizeQ4KBlock,
 * dequantizeQ6KBlock, dequantizeQ40Block (src/gguf/quantization.ts:19-74).
 * n_values must be a whole number of blocks. */
nemo_status nemo_dequantize(int32_t ggml_type, const void* d_raw, int64_t n_values, float* d_out_f32,
                            uint16_t* d_out_f16, void* stream);

/* Roofline probe, no counterpart in the reference: the floors the HBM-bound
 * kernels are measured against. bytes == 0 launches one empty kernel (the
 * cost of a launch); otherwise one kernel reads `bytes` (a multiple of 16)
 * at the 16-byte aligned device pointer d_src once, with fully coalesced
 * 16-byte loads, `loads_per_thread` (1, 2, 4 or 8) per thread, and does
 * nothing else: the least time a kernel reading those bytes in one launch
 * takes. d_sink is a device buffer of 256 uint32 the kernel may write. */
nemo_status nemo_probe_stream(const void* d_src, size_t bytes, int32_t loads_per_thread, uint32_t* d_sink,
                              void* stream);

/* ---- attention block operators -------------------------------------------
 * The reference has these only inside its encoder pass (src/webgpu/ops.ts:21-56,
 * 168-362), in one form each; here they are operators on device buffers of
 * any layout, for callers that build a layer from nemo_weight_matmul and
 * these. All are enqueued on `stream` (NULL: the default stream) and return;
 * nothing is allocated, so they can be captured into a HIP graph after one
 * eager call of the same kind. Strides count elements and are in [0, 2^23];
 * addresses are multiples of their values' size; rows and heads that are
 * written do not overlap. */

#define NEMO_TYPE_I8 24        /* GGML's code */
#define NEMO_TYPE_BF16 30      /* GGML's code */
#define NEMO_TYPE_F8_E4M3 259  /* 8-bit floats, largest 448; not a GGML type code */

/* Rotary positions. A head's first rotary_dim values are r / 2 pairs, pair i
 * of which is turned by the angle position * f_i and scaled by `magnitude`:
 *   (a, b) -> m (a cos - b sin, a sin + b cos).
 * The head's other values are copied. f_i = theta^(-2i / r), and then by
 * `scaling`: LINEAR f_i / factor; YARN f_i / factor for pairs that turn less
 * than beta_slow times in original_positions, f_i for those that turn more
 * than beta_fast times, a linear ramp over the pair index between (the
 * table of src/webgpu/model.ts:95-106 is YARN with factor 16, 16384, 32, 1,
 * interleaved, magnitude 1); BANDS f_i / factor for wavelengths longer than
 * original_positions / low_band, f_i for those shorter than
 * original_positions / high_band, between them linear in the number of
 * turns. */
#define NEMO_ROPE_INTERLEAVED 0 /* pair i: values 2i and 2i + 1 */
#define NEMO_ROPE_HALF 1        /* pair i: values i and i + r / 2 */
#define NEMO_ROPE_NONE 0
#define NEMO_ROPE_LINEAR 1
#define NEMO_ROPE_YARN 2
#define NEMO_ROPE_BANDS 3

typedef struct nemo_rope nemo_rope;
typedef struct nemo_rope_config {
  int32_t head_dim;           /* 2..1024, even */
  int32_t rotary_dim;         /* 2..head_dim, even; 0: head_dim */
  int32_t layout;             /* NEMO_ROPE_INTERLEAVED or _HALF */
  int32_t scaling;            /* NEMO_ROPE_NONE.._BANDS */
  double theta;               /* > 1 */
  double factor;              /* > 0; LINEAR, YARN, BANDS */
  int32_t original_positions; /* >= 1; YARN, BANDS */
  double beta_fast, beta_slow; /* YARN: beta_fast >= beta_slow > 0 */
  double low_band, high_band;  /* BANDS: high_band > low_band > 0 */
  double magnitude;            /* 0: 1, for YARN 0.1 ln(factor) + 1 (factor > 1) */
} nemo_rope_config;

/* head_dim 128, whole heads, interleaved, theta 1e6, no scaling (its factor
 * 1, 16384 positions, betas 32 and 1, bands 1 and 4), magnitude 0. */
void nemo_rope_config_default(nemo_rope_config* out);

/* The frequencies are computed in 64 bits on the host and held on the
 * context's device. */
nemo_status nemo_rope_create(nemo_ctx* ctx, const nemo_rope_config* config, nemo_rope** out);
/* Waits for the device, then frees it. */
nemo_status nemo_rope_destroy(nemo_rope* rope);

/* `heads` heads of each row: head h of row t starts at x + t x_row + h x_head
 * and goes to y + t y_row + h y_head. y may be x with the same strides (the
 * heads are turned in place); other overlap of an input and an output is not
 * allowed. */
typedef struct nemo_rope_heads {
  const void* x;
  void* y;
  int64_t x_row, x_head, y_row, y_head;
  int32_t heads;
} nemo_rope_heads;

/* Turn the heads of `rows` tokens (at most 2^23), `type` F32, F16 or BF16
 * (arithmetic in 32 bits, one rounding), of q and, unless it is NULL, of k in
 * the same launch. Row t has position base + d_positions[t] (device; NULL: base
 * + t). Angles are position * f_i in 64 bits, reduced there: their error is
 * about 2^-53 of the angle. Negative positions turn back. */
nemo_status nemo_rope_apply(nemo_rope* rope, int32_t type, const nemo_rope_heads* q, const nemo_rope_heads* k,
                            int64_t rows, const int64_t* d_positions, int64_t base, void* stream);

/* Attention with a sliding window and sinks. Request b has query rows
 * q_start[b] .. q_start[b + 1] - 1 of q and out and kv_len[b] key and value rows
 * from kv_start[b] on. Its queries are its last positions: query i of n stands at
 * p = kv_len - n + i, and sees key j when
 *   j <= p + right  and  (j >= p - left  or  j < sinks)
 * (left or right -1: no bound on that side; right 0 is causal). out = softmax(scale q.k) v
 * over the keys it sees, 0 when it sees none. Query head h reads key and
 * value head h / (q_heads / kv_heads). Keys and values that no query of a
 * request sees may hold anything, NaN included; one that some queries see
 * reaches no other query's result. Softmax sums and the output are
 * accumulated in 32 bits; the probabilities are rounded to `type` for the
 * product with v. */
typedef struct nemo_attention_config {
  int32_t q_heads, kv_heads; /* q_heads a multiple of kv_heads, at most 1024 */
  int32_t head_dim;          /* 64 or 128 */
  int32_t type;              /* F16 or BF16 */
  int32_t left, right;       /* >= 0, or -1: unbounded */
  int32_t sinks;             /* >= 0 */
  float scale;               /* > 0, or 0: head_dim^-1/2 */
} nemo_attention_config;

/* Buffers are 16-byte aligned, strides multiples of 8. The index arrays are
 * read on the device when the work runs (a captured graph may be replayed
 * with other lengths); entries outside the buffers are cut to q_rows and
 * kv_rows. Key and value rows are at least head_dim apart; the row strides of
 * a k and v of one row are not used. Rows of `out` that belong to no request are
 * left as they were. `out` and the workspace overlap no other buffer. */
typedef struct nemo_attention_batch {
  int32_t count;             /* requests: 0..2^20, times kv_heads at most 2^22 */
  int64_t q_rows, kv_rows;   /* rows of q and out, times q_heads at most 2^26; of k and v, at most 2^30 */
  int64_t max_kv;            /* the longest kv_len, or more: a hint for the split of the keys over the chip */
  const int32_t* q_start;    /* device [count + 1], ascending */
  const int64_t* kv_start;   /* device [count] */
  const int32_t* kv_len;     /* device [count] */
  const void *q, *k, *v;
  void* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  void* workspace;           /* device, 16-byte aligned; NULL: the keys of a query are not split */
  size_t workspace_bytes;    /* at least nemo_window_attention_workspace's when workspace is given */
} nemo_attention_batch;

/* Bytes of workspace for a batch of these sizes (0: none is used). Its
 * content carries nothing from one call to the next; calls that may overlap,
 * graphs among them, need one each. */
nemo_status nemo_window_attention_workspace(const nemo_attention_config* config, int32_t count, int64_t q_rows,
                                            int64_t max_kv, size_t* bytes);
nemo_status nemo_window_attention(nemo_ctx* ctx, const nemo_attention_config* config,
                                  const nemo_attention_batch* batch, void* stream);

/* Residual addition, RMSNorm and 8-bit output in one pass, for each row:
 *   h = x + delta,  y = h / sqrt(mean(h^2) + epsilon) * weight
 * in 32 bits from the unrounded h; sum = h and y in `type`; and
 *   scales = max |y| / 127 (I8) or / 448 (F8_E4M3), y8 = round(y / scale)
 * of the unrounded y over a whole row or over each `group` columns (scale 0,
 * and y8 0, where y is 0; NaN where y holds a NaN; to even on ties, the
 * quotient as 64 bits give it). Where sum or y is x or delta it has the same
 * row stride; other overlap of an input and an output is not allowed. */
typedef struct nemo_norm_args {
  int32_t type;              /* of x, delta, sum, y: F32, F16 or BF16 */
  int32_t hidden;            /* 1..2^30 */
  int64_t rows;              /* 0..2^23 */
  const void* x;
  const void* delta;         /* NULL: h = x */
  const float* weight;       /* [hidden]; NULL: 1 */
  void* sum;                 /* NULL: not written; may be x or delta */
  void* y;                   /* NULL: not written; may be x or delta */
  void* y8;                  /* NULL: not written */
  float* scales;             /* rows of 1, or of hidden / group; with y8 */
  int64_t x_row, delta_row, sum_row, y_row, y8_row, scales_row;
  int32_t type8;             /* I8 or F8_E4M3, with y8 */
  int32_t group;             /* 0 (a row), 32, 64 or 128, which divides hidden */
  float epsilon;             /* >= 0 */
} nemo_norm_args;

nemo_status nemo_rmsnorm(nemo_ctx* ctx, const nemo_norm_args* args, void* stream);

/* Encoders of the same graph whose layers attend through a window, or whose
 * rotary positions differ from the reference's: before nemo_model_finalize,
 * the model's attention becomes nemo_rope_apply on the query and key heads
 * (positions counted within a request, merged positions after the merge) and
 * nemo_window_attention over each request's own keys, in place of the
 * reference's rotation, key sampling and temperature. Every global_every-th
 * layer (the global_every-th, the 2 global_every-th, ...; 0: none) has no left
 * bound, and no right bound unless right is 0. rope.head_dim is taken from
 * the model. A model without this call computes what the reference does. */
typedef struct nemo_model_attention {
  int32_t left, right, sinks; /* as in nemo_attention_config */
  int32_t global_every;
  nemo_rope_config rope;
} nemo_model_attention;
nemo_status nemo_model_set_attention(nemo_model* model, const nemo_model_attention* attention);

/* The token states of the plan's last run in 8 bits, for indexes of one vector
 * a token: the final RMSNorm of each request's merged rows, unpooled, as
 * nemo_rmsnorm writes it (y8 [rows][hidden], scales [rows] or [rows][hidden /
 * group]), request after request, max(1, ceil(0.64 length)) rows each. `rows`
 * receives their number; more than `capacity`, and a plan that has not run,
 * whose last run failed, or whose model merges after its last layer, are
 * refused. Enqueued on `stream` (NULL: the plan's own) after the run. */
nemo_status nemo_plan_token_states8(nemo_plan* plan, int32_t type8, int32_t group, void* d_y8, float* d_scales,
                                    int64_t capacity, int64_t* rows, void* stream);

/* ---- low-bit operators of an attention block -------------------------------
 * What stands between nemo_rmsnorm's 8-bit rows and the output projection in
 * a block that is served in few bits: products of 8-bit rows, norms of heads
 * before their rotation, a cache of 4-bit floats in pages, and attention over
 * it. The reference has no counterparts. They follow the conventions of the
 * operators above: enqueued on `stream`, nothing allocated, strides in elements
 * and in [0, 2^23]. */

/* RMSNorm of each query and key head, then its rotation, in one pass:
 *   h = x / sqrt(mean over the head of x^2 + epsilon) * weight,  y = h turned
 * by nemo_rope_apply's angles (values that it copies are normed only), in 32
 * bits, the sum of squares too (a head whose largest value is 2^59 or more, or below
 * 2^-55 with an epsilon of 0, is not normed rightly), with one rounding at the
 * end. Head h's weight begins at
 * weight + h weight_head; 0: one weight for all heads. */
typedef struct nemo_head_norm {
  const float* q_weight;       /* [head_dim] each; NULL: 1 */
  const float* k_weight;
  int64_t q_weight_head, k_weight_head;
  float epsilon;               /* >= 0 */
} nemo_head_norm;
nemo_status nemo_rope_norm_apply(nemo_rope* rope, int32_t type, const nemo_rope_heads* q, const nemo_rope_heads* k,
                                 const nemo_head_norm* norm, int64_t rows, const int64_t* d_positions, int64_t base,
                                 void* stream);

/* Products of 8-bit rows, as nemo_rmsnorm writes them with group 0, and 8-bit
 * weights with a scale for each output channel:
 *   y[i][j] = type(x_scale[i] w_scale[j] (sum over k of x[i][k] w[j][k]) + bias[j])
 * The sum is exact (32-bit integers); it is rounded to 32 bits and scaled by
 * x_scale; w_scale's product and the bias's addition round once, in 32 bits. k 0
 * leaves the bias. x and w are 16-byte aligned, their row strides multiples of 16 and at
 * least k (for more than one row); bytes of a row behind k may hold anything.
 * y overlaps no other buffer. */
typedef struct nemo_matmul8_args {
  int32_t type;                /* of y: F32, F16 or BF16 */
  int32_t n, k;                /* 0..2^23 output channels; 0..131071 */
  int64_t m;                   /* 0..2^23 rows */
  const int8_t* x;             /* [m][k] */
  const float* x_scale;        /* [m], x_scale_row apart */
  const int8_t* w;             /* [n][k] */
  const float* w_scale;        /* [n] */
  const float* bias;           /* [n]; NULL: none */
  void* y;                     /* [m][n] */
  int64_t x_row, x_scale_row, w_row, y_row; /* y_row at least n for more than one row */
} nemo_matmul8_args;
nemo_status nemo_matmul8(nemo_ctx* ctx, const nemo_matmul8_args* args, void* stream);

/* A cache of keys and values in 4-bit floats. Each 32 values of a head share a
 * power of two: value = code 2^(byte - 127), the codes E2M1 floats (0, 0.5, 1,
 * 1.5, 2, 3, 4, 6; bit 3 the sign), as CDNA4 converts them to 16 bits in one
 * instruction and without a rounding; byte 255 makes its 32 values NaN.
 *
 * Tokens lie in pages of `page` tokens of one request, P = page, D = head_dim.
 * A page holds its KV heads one after the other, each as
 *   K codes   [P][D / 2]             two codes a byte, the first in the low bits
 *   V codes   [P / 4][16][4][D / 32] 4 tokens' pieces of D / 16 values side by side
 *   K scales  [P / 8][D / 32][8]
 *   V scales  [P / 8][D / 32][8]
 * P (D + D / 16) bytes. Pages may be shared by requests that only read them. */
typedef struct nemo_cache4_config {
  int32_t kv_heads;            /* 1..1024 */
  int32_t head_dim;            /* 64 or 128 */
  int32_t page;                /* 32, 64, 128, 256, 512 or 1024 tokens */
} nemo_cache4_config;

/* Bytes of a page: kv_heads page (head_dim + head_dim / 16). */
nemo_status nemo_cache4_page_bytes(const nemo_cache4_config* config, size_t* bytes);

/* Where the tokens of `count` requests are: token t of request b is token
 * t % page of page table[b table_row + t / page]. The arrays are read on the device when
 * the work runs. Pages outside [0, pages), and tokens past table_row pages,
 * are not there: they are not written, read as zeros, and no query sees them. */
typedef struct nemo_cache4_pages {
  int32_t count;               /* requests: 0..2^20, times kv_heads at most 2^22 */
  int32_t pages;               /* pages that `data` holds */
  void* data;                  /* device, 16-byte aligned */
  const int32_t* table;        /* device [count][table_row] */
  int64_t table_row;           /* pages of a request's row of the table: 0..2^23 */
  const int32_t* kv_len;       /* device [count]: tokens of each request, at most 2^30, those of this call's rows
                                  among them */
} nemo_cache4_pages;

/* Key and value rows of requests' last tokens: rows q_start[b] .. q_start[b + 1]
 * - 1 are request b's; of its n rows, row i is token kv_len - n + i (rows
 * before token 0 have none). Head h of row t starts at k + t k_row + h k_head. */
typedef struct nemo_cache4_rows {
  int32_t type;                /* F32, F16 or BF16 */
  int64_t rows;                /* rows of k and v: 0..2^23 */
  const int32_t* q_start;      /* device [count + 1], ascending; entries are cut to `rows` */
  const int64_t* positions;    /* device [rows]: what the rotation of a row goes by; NULL: its token's number */
  void *k, *v;
  int64_t k_row, k_head, v_row, v_head;
} nemo_cache4_rows;

/* Append rows to a cache: keys are turned by `rope` (NULL: as they are; its
 * head_dim is the cache's), keys and values rounded to 4 bits: the smallest
 * power of two 2^s with max |x| <= 7 2^s, s in [-126, 125], and the nearest
 * code, to an even one on ties, up to 6. Values as they are get the code of the
 * exact value, turned ones that of their rotation in 64 bits (in 32 where a bound on
 * its error shows that to be the same): next to a border between two codes, where
 * the angle's own rounding of about 2^-53 of it decides, the other may be taken. 32
 * values with a NaN or an infinity become NaN. k and v are only read. Rows of a call that share a page write
 * bytes of their own. */
nemo_status nemo_cache4_append(nemo_ctx* ctx, const nemo_cache4_config* config, const nemo_cache4_pages* pages,
                               const nemo_cache4_rows* rows, nemo_rope* rope, void* stream);
/* The other way: the rows' values from the cache, in `type`; `positions` is
 * not used. Rows that belong to no request or token are left as they were. */
nemo_status nemo_cache4_read(nemo_ctx* ctx, const nemo_cache4_config* config, const nemo_cache4_pages* pages,
                             const nemo_cache4_rows* rows, void* stream);

/* nemo_window_attention over a cache in pages: request b's queries are rows
 * q_start[b] .. q_start[b + 1] - 1 of q and out, its keys the kv_len[b] tokens of
 * the cache, and what a query sees goes by nemo_attention_config, whose kv_heads
 * and head_dim are the cache's. Keys and values are read as `type`, exactly in
 * BF16, and in F16 from 2^-14 on and to 65504 (what lies above is an infinity; in
 * v it makes its column of the rows that see it NaN). Softmax sums and outputs are in
 * 32 bits, the probabilities rounded to `type` for the product with v. Keys and values
 * that a query does not see, and other queries, reach its result in no form, NaN
 * neither. Rows of `out` that belong to no request are left as they
 * were. `out` and the workspace overlap no other buffer. */
typedef struct nemo_cache4_queries {
  int64_t q_rows;              /* rows of q and out, times q_heads at most 2^26 */
  int64_t max_kv;              /* the longest kv_len, or more: a hint for the split of the keys over the chip */
  const int32_t* q_start;      /* device [count + 1], ascending; entries are cut to q_rows */
  const void* q;               /* 16-byte aligned, strides multiples of 8, as out */
  void* out;
  int64_t q_row, q_head, out_row, out_head;
  void* workspace;             /* device, 16-byte aligned; NULL: the keys of a query are not split */
  size_t workspace_bytes;      /* at least nemo_cache4_attention_workspace's when workspace is given */
} nemo_cache4_queries;

/* Bytes of workspace for such a call (0: none is used), with the conditions of
 * nemo_window_attention_workspace. */
nemo_status nemo_cache4_attention_workspace(const nemo_attention_config* attention, int32_t count, int64_t q_rows,
                                            int64_t max_kv, size_t* bytes);
nemo_status nemo_cache4_attention(nemo_ctx* ctx, const nemo_cache4_config* config,
                                  const nemo_attention_config* attention, const nemo_cache4_pages* pages,
                                  const nemo_cache4_queries* queries, void* stream);

/* ---- offline requantization (src/gguf/quantization.ts:77-131) ------------ */

/* requantizeMatrixToQ40 (src/gguf/quantization.ts:101-131) on the GPU: the
 * raw GGUF bytes of an n x k matrix of type Q4_K, Q6_K or Q4_0 (host memory,
 * n_src bytes) -> n * k / 32 GGUF Q4_0 blocks of 18 bytes written to `out`
 * (host memory, out_bytes). Bit-exact with the reference's JavaScript, which
 * quantizes each 32 values as quantizeQ40Block (:77-98). Errors as the
 * reference: "K=<k> is not divisible by a K-quant block", "source has <n>
 * bytes; expected <m>". scripts/prepack-model.ts:28-36 calls it per matrix. */
nemo_status nemo_requantize_q40(nemo_ctx* ctx, int32_t src_type, const void* src, size_t n_src, int64_t k, int64_t n,
                                void* out, size_t out_bytes);

#ifdef __cplusplus
}
#endif

#endif /* NEMO_H */
