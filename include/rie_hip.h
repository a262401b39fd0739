/*
 * rie_hip.h — C ABI of the MI355X (gfx950) backend for RIE's per-token forward
 * loop (librie_hip.so).
 *
 * The backend entry points mirror the reference's `trait Backend`
 * (crates/rie-core/src/model/mod.rs:303-320) one for one, so a Rust
 * `impl Backend for HipBackend` over these symbols is a drop-in for the seam
 * that `rie bench`, `rie run` and rie-server already call
 * (crates/rie-cli/src/main.rs:246-262, crates/rie-server/src/lib.rs:602-640,
 * crates/rie-ffi/src/lib.rs:96-129).  Conventions follow rie.h
 * (crates/rie-ffi/include/rie.h:17-73): NULL / negative return on failure with
 * the message written into a caller buffer, no exceptions across the ABI.
 *
 * Thread-safety: one host thread drives a handle at a time (Backend: Send).
 * forward() is synchronous: it returns after the logits are in host memory.
 */
#ifndef RIE_HIP_H
#define RIE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Error codes: one per variant of the reference's Error enum
 * (crates/rie-core/src/error.rs:5-15). */
#define RIE_HIP_OK 0
#define RIE_HIP_ERR_IO (-1)
#define RIE_HIP_ERR_FORMAT (-2)
#define RIE_HIP_ERR_UNSUPPORTED (-3)
#define RIE_HIP_ERR_MISSING (-4)
#define RIE_HIP_ERR_RUNTIME (-5)

/* KV cache formats (KvType, crates/rie-core/src/model/cpu.rs:12-36). */
#define RIE_HIP_KV_F16 0
#define RIE_HIP_KV_Q8_0 1
#define RIE_HIP_KV_TURBO4 2

typedef struct rie_hip_backend rie_hip_backend;

typedef struct rie_hip_config {
    int32_t n_ctx;     /* KV capacity in positions (the caller applies min(n_ctx, ctx_train)) */
    int32_t max_batch; /* tokens per forward (CpuBackend max_batch, clamped to [1, n_ctx]) */
    int32_t kv_type;   /* RIE_HIP_KV_*; falls back to f16 like CpuBackend::with_kv_type */
    int32_t device;    /* HIP device ordinal */
    int32_t use_graph; /* 1: replay the single-token decode step as a HIP graph */
} rie_hip_config;

rie_hip_config rie_hip_default_config(void);

/* Construct a backend from a GGUF image held in host memory (the reference's
 * GgufFile::data(), crates/rie-core/src/gguf.rs:271-276).  Tensor data is copied
 * once to HBM in its native ggml block layout; the image may be released after
 * the call.  Replaces CpuBackend::with_kv_type (model/cpu.rs:100-177) /
 * GpuBackend::new (crates/rie-gpu/src/lib.rs:236-624).  Returns NULL on failure;
 * *err_code (if non-NULL) receives the RIE_HIP_ERR_* class. */
rie_hip_backend *rie_hip_create(const uint8_t *gguf, size_t gguf_len, const rie_hip_config *cfg, int32_t *err_code, char *err,
                                size_t err_len);
void rie_hip_destroy(rie_hip_backend *b);

/* Backend::name (model/mod.rs:305): copies a NUL-terminated name, returns its length. */
size_t rie_hip_name(const rie_hip_backend *b, char *buf, size_t buf_len);
/* Backend::max_batch (model/mod.rs:307) */
size_t rie_hip_max_batch(const rie_hip_backend *b);
/* Backend::n_ctx (model/mod.rs:309) */
size_t rie_hip_n_ctx(const rie_hip_backend *b);
/* Backend::forward (model/mod.rs:310-313; CpuBackend semantics model/cpu.rs:210-409):
 * evaluate tokens[0..n) at positions pos..pos+n; writes the last token's logits
 * (n_vocab floats) or, with all_logits, n·n_vocab floats.  Errors (RUNTIME):
 * empty batch, n > max_batch, pos+n > n_ctx, token id out of range, logits buffer
 * too small (checked before any work is done). */
int32_t rie_hip_forward(rie_hip_backend *b, const uint32_t *tokens, size_t n, size_t pos, int32_t all_logits, float *logits,
                        size_t logits_len, char *err, size_t err_len);
/* Backend::hidden (model/mod.rs:314-319): final normalized hidden rows of the last
 * forward (rows × n_embd), valid until the next call; NULL when none. */
const float *rie_hip_hidden(rie_hip_backend *b, size_t *rows);

/* ---- model facts ---- */
size_t rie_hip_n_vocab(const rie_hip_backend *b);
size_t rie_hip_n_embd(const rie_hip_backend *b);
int32_t rie_hip_kv_type(const rie_hip_backend *b);
size_t rie_hip_kv_bytes(const rie_hip_backend *b);
size_t rie_hip_weight_bytes(const rie_hip_backend *b);

/* ---- engine-side greedy decoding on the device (Engine::bench / eval_next,
 * crates/rie-core/src/engine.rs:384-392, 540-564; sampler.rs:199-209 argmax with
 * first-max tie-break).  No per-token logits readback. ---- */
/* forward(tokens, pos) then argmax of the last logits row; returns 0 and *next. */
int32_t rie_hip_forward_argmax(rie_hip_backend *b, const uint32_t *tokens, size_t n, size_t pos, uint32_t *next, char *err,
                               size_t err_len);
/* forward(tokens, pos), then of every token's logits on the device (no logits readback):
 * logprob[i] = ln p(targets[i]) (NaN for a target that is no token), the entropy in nats,
 * and the n_top (0..64) most likely tokens in order, the lowest id first among equals, with
 * their log probabilities ([n][n_top]); rie_hip_k_token_logprobs has the rules.  For scoring
 * (Engine::perplexity, engine.rs:567-602) and a server's logprobs.  targets with logprob,
 * entropy, and (n_top = 0) top_ids with top_logprobs may be NULL.  Errors: forward's, and
 * RUNTIME for an n_top or a combination of NULLs outside these. */
int32_t rie_hip_forward_logprobs(rie_hip_backend *b, const uint32_t *tokens, size_t n, size_t pos, const uint32_t *targets,
                                 size_t n_top, float *logprob, float *entropy, uint32_t *top_ids, float *top_logprobs, char *err,
                                 size_t err_len);
/* n_gen greedy steps continuing from the token chosen by the previous
 * forward_argmax/generate call, at positions pos, pos+1, ...; out[i] receives the
 * token fed at step i. */
int32_t rie_hip_generate_greedy(rie_hip_backend *b, size_t pos, size_t n_gen, uint32_t *out, char *err, size_t err_len);
/* Engine::bench (engine.rs:540-564): prompt ids (i·7919+13) mod V, warm-up on the
 * first 8, one prompt evaluation in chunks of max_batch, then n_gen greedy steps.
 * Returns prompt and generation throughput in tokens/s. */
int32_t rie_hip_bench(rie_hip_backend *b, size_t n_prompt, size_t n_gen, double *pp_tps, double *tg_tps, char *err, size_t err_len);

/* ---- synthetic GGUF images (`rie bench --synthetic`, crates/rie-core/src/testing.rs:95-383) ---- */
typedef struct rie_hip_synth_spec {
    char arch[32];
    uint32_t n_vocab, n_embd, n_layer, n_head, n_head_kv, head_dim, n_ff, rope_dim, ctx;
    int32_t wtype, embd_type;
    int32_t tied_output, qkv_bias, qk_norm, post_norms, fused;
    uint32_t swa_window, n_expert, n_expert_used, n_ff_exp, n_ff_shexp;
    int32_t chat_template; /* 0 none, 1 chatml, 2 llama3 */
    uint64_t seed;
    /* workload mode: 0 = the reference's random-byte weights (testing.rs:46-91);
     * 1 = N(0, 0.02) values quantized with quantize::q4_0 / Q8_0 (quant/mod.rs:262-298),
     *     unit norms, rope_base below */
    int32_t mode;
    float rope_base;
    int32_t output_type; /* mode 1: type of output.weight (-1 = embd_type) */
    /* mode 1 per-tensor mix: 0 = every matrix wtype; 1 = Q4_K_M: attn_v Q6_K, ffn_down
     * Q6_K in the layers llama.cpp's Q4_K_M gives more bits (i < n/8, i >= 7n/8,
     * (i - n/8) % 3 == 2), wtype elsewhere */
    int32_t mix;
} rie_hip_synth_spec;

/* SyntheticSpec::tiny (testing.rs:127-154) / preset (testing.rs:157-212); 0 or -1. */
int32_t rie_hip_synth_tiny(const char *arch, int32_t wtype, rie_hip_synth_spec *out);
int32_t rie_hip_synth_preset(const char *name, int32_t wtype, rie_hip_synth_spec *out);
/* SyntheticSpec::build (testing.rs:229-383): writes the GGUF image to a buffer
 * owned by the library (release with rie_hip_free); returns its size, 0 on error. */
size_t rie_hip_synth_build(const rie_hip_synth_spec *spec, uint8_t **out, int32_t n_threads);
void rie_hip_free(void *p);
/* The generator's weight quantizers: n values of x to ggml blocks of type ty
 * (Q4_0 and Q8_0 are quantize::q4_0 / quantize::q8_0, quant/mod.rs:262-298;
 * Q4_K and Q6_K, which the reference has no quantizer for, are min/max
 * quantizers of this library).  0, or RIE_HIP_ERR_UNSUPPORTED for other types
 * or n not a multiple of the block size. */
int32_t rie_hip_quantize(int32_t ty, const float *x, size_t n, uint8_t *out);

/* ---- parity hooks (no counterpart in the reference; for tests and debugging) ---- */
/* Keep per-layer copies of intermediate f32 tensors during forward (slow path):
 * what = 0 x after attention, 1 x after FFN, 2 attention output, 3 q after
 * RoPE/scale, 4 k after norm/RoPE, 5 v, 6 FFN gated hidden, 7 MoE router logits,
 * 8 the experts the device routing selected ([n][k] int32 bit patterns, ascending),
 * 9 their combination weights ([n][k]). */
int32_t rie_hip_set_capture(rie_hip_backend *b, int32_t on);
/* on = 1: single-token attention always splits the context into ranges merged
 * across workgroups, also at the short contexts where it otherwise runs one
 * workgroup per query head over the whole cache (so tests can check both kernels
 * on the same positions); on = 0: automatic (the default). */
int32_t rie_hip_set_attention_ranges(rie_hip_backend *b, int32_t on);
int32_t rie_hip_capture(rie_hip_backend *b, size_t layer, int32_t what, float *out, size_t len);
/* Raw KV cache of one layer: which 0 = K, 1 = V; [kv_head][slot][row bytes];
 * Turbo4 scales ([kv_head][slot] f16) go to scales_out. */
int32_t rie_hip_kv_layer(rie_hip_backend *b, size_t layer, int32_t which, uint8_t *out, size_t len, uint8_t *scales_out,
                         size_t scales_len);
size_t rie_hip_kv_row_bytes(const rie_hip_backend *b);
/* Time one eager decode step at pos, reps times, with a HIP event after every
 * launch on the backend's stream; per kernel family: summed ms and launch count.
 * names receives the family names separated by newlines. */
int32_t rie_hip_profile_decode(rie_hip_backend *b, size_t pos, int32_t reps, char *names, size_t names_len, double *ms,
                               int32_t *launches, size_t max_entries, size_t *n_entries);

/* Average duration in microseconds of the single-token gate/up/SwiGLU launch
 * (dense_ffn's gate·x, up·x and silu product, model/cpu.rs:431-467, as one
 * kernel), timed with HIP events on the backend's stream while cycling through
 * every layer's weights reps times; *bytes_per_launch = weight bytes of gate
 * and up + activation read + hidden written.  No counterpart in the reference:
 * it measures the dominant decode kernel for the roofline report. */
int32_t rie_hip_time_ffn_glu(rie_hip_backend *b, int32_t reps, double *avg_us, size_t *bytes_per_launch);

/* ---- kernel entry points on device pointers (stream 0, synchronous) ---- */
/* RMSNorm (w may be NULL: quantize only) + Q8_0 (fmt 1) or Q8_K (fmt 2) quantization
 * of n rows of k values (ops.rs:7-14 with the sum of squares in the order of
 * kernels/avx2.rs:186-203; quant/mod.rs:191-218, kernels/avx2.rs:153-184).  Outputs:
 * Q8_0: qs [n][k], d/s/isum [n][k/32]; Q8_K: qs [n][k], d [n][k/256], bsums [n][k/16]. */
int32_t rie_hip_k_rmsnorm_quant(const float *x, const float *w, float eps, int32_t n, int32_t k, int32_t fmt, float *xn, int8_t *qs,
                                float *d, float *s, int32_t *isum, int16_t *bsums);
/* out[t*rows + r] = W[r] · act[t] for one ggml weight matrix (kernels/mod.rs:136-232).
 * w may end at its last row: the kernels read whole aligned words around each
 * block, up to 4 KiB past the matrix, so these entry points run on a padded copy
 * of w (allocated and freed inside the call). */
int32_t rie_hip_k_gemv(int32_t ty, const uint8_t *w, int32_t rows, int32_t k, const int8_t *qs, const float *d, const float *s,
                       const int32_t *isum, const int16_t *bsums, const float *act_f32, int32_t n_tok, float *out);
/* the int8 MFMA prompt GEMM on the same operands (n_tok > 8) */
int32_t rie_hip_k_gemm(int32_t ty, const uint8_t *w, int32_t rows, int32_t k, const int8_t *qs, const float *d, const float *s,
                       const int32_t *isum, const int16_t *bsums, int32_t n_tok, float *out);
/* MoE routing of n_tok tokens (moe_ffn's routing, model/cpu.rs:487-501): softmax
 * over each token's n_exp router logits (ops.rs:38-49), the k most probable
 * experts with the lower index first on ties (NaN probabilities compare Equal, so
 * a token whose probabilities are NaN takes experts 0..k-1), weights p/Σ_top p
 * (norm_topk), p, or 1 (unit_weights).  sel/wgt [n_tok][k] receive each token's
 * choices in ascending expert order.  1 ≤ k ≤ min(n_exp, 64), n_exp ≤ 512; other
 * sizes return RIE_HIP_ERR_RUNTIME. */
int32_t rie_hip_k_moe_route(const float *logits, int32_t n_tok, int32_t n_exp, int32_t k, int32_t norm_topk, int32_t unit_weights,
                            int32_t *sel, float *wgt);
/* greedy argmax (sampler.rs:199-209) of n floats */
int32_t rie_hip_k_argmax(const float *x, int32_t n, uint32_t *out_idx);
/* The same argmax without allocating device memory.  No counterpart in the
 * reference: for callers that cannot call hipMalloc (code under HIP stream or
 * graph capture, tight serving loops, harnesses that forbid allocation).  The
 * partial maxima live in a fixed 8 KiB array of the library's static device
 * memory (one copy per GPU, held until the process ends), so n must be in
 * 1..1048576 (1024 partials of up to 1024 values); larger or empty inputs return
 * RIE_HIP_ERR_RUNTIME with the reason in err.  stream: a hipStream_t to launch on
 * (the call returns once the two kernels are queued, without synchronizing, so
 * it can be recorded under capture), or NULL: the null stream, and the call
 * returns after the result is written.  The first call on a device looks up the
 * array's address (hipGetSymbolAddress), so make it outside capture.  Calls that
 * overlap on one GPU (several streams or host threads) share that array and race. */
int32_t rie_hip_k_argmax_noalloc(const float *x, int32_t n, uint32_t *out_idx, void *stream, char *err, size_t err_len);

/* ---- batched serving: a cache of pages, attention over it and over packed prompts,
 * token log probabilities.  No counterpart in the reference, whose backends hold one
 * sequence each.  Everything but the structs themselves is device memory; nothing of it
 * is read by the host, so a call can be captured into a graph and replayed over new
 * contents.
 *
 * Types are ggml ids: 0 f32, 1 f16, 30 bf16.  Strides count elements.  Pointers and
 * strides of q, k, v, the pages and the outputs have to keep every row (of head_dim
 * consecutive values) 16-byte aligned; strides of rows, slots and heads go up to 2^26
 * bytes.  head_dim: 32, 64, 96, 128 or 256.  What a call writes may share no memory with
 * what it reads, and its rows none with one another: of the strides of what is written,
 * every one has to cover what the smaller ones span (refused otherwise).
 * The stride of a dimension with one entry (one row, head or page) is not looked at.
 *
 * stream: a hipStream_t of any device (NULL: the current device's null stream); the call
 * queues its kernels there and returns.  Pointers of host memory, or of another device
 * than the stream's, are refused.
 * No call allocates: ws is the caller's, of at least the bytes that the matching _ws
 * function names; two calls that may run at the same time (on two streams, or in two
 * graphs) need a workspace each. */

/* The sequences of a batch.  Rows starts[i]..starts[i+1] (ascending, starts[n_seq] ≤
 * n_rows) of the tensors hold sequence i's new tokens, which are the last of its lens[i]
 * positions; rows behind starts[n_seq] are neither read nor written.  A sequence may
 * bring no token; a token before position 0 (more new tokens than positions) is not
 * written to the cache and attends to nothing.  max_new and max_len bound the new tokens
 * and the positions of any one sequence: they choose kernels and splits, and of a
 * sequence that exceeds max_new only some rows may be computed, the others of its rows
 * holding anything. */
typedef struct rie_hip_seqs {
    int32_t n_seq, n_rows, max_new, max_len;
    const int32_t *starts; /* [n_seq + 1] */
    const int32_t *lens;   /* [n_seq] (packed attention ignores it) */
} rie_hip_seqs;

/* A layer's keys and values in pages: position p of sequence i lies in page
 * table[i*table_stride + p/page_size], slot p%page_size, and head h's values start at
 * page*page_stride + slot*slot_stride + h*head_stride of k and of v.  page_size: a power
 * of two, 16 to 4096.  Positions at and past table_cols*page_size, and those of a page id
 * outside 0..n_pages-1, are neither written nor seen (of a sequence whose length passes
 * its table, a token keeps its position and sees what the table holds).  Sequences may
 * share pages (a common prefix); where two new tokens come to the same slot, it holds
 * values of either. */
typedef struct rie_hip_pages {
    int32_t ty, head_dim, n_kv, n_pages, page_size, table_cols;
    void *k, *v;
    int64_t page_stride, slot_stride, head_stride;
    const int32_t *table;
    int64_t table_stride;
} rie_hip_pages;

/* Queries and outputs of an attention call, of the keys' type: row r, head h at
 * r*row_stride + h*head_stride.  Query head h reads KV head h / (n_head/n_kv).  scale:
 * positive.  window > 0: a token sees its own position and the window-1 before it.
 * softcap > 0: scores become softcap·tanh(score/softcap). */
typedef struct rie_hip_attn {
    int32_t n_head, window;
    float scale, softcap;
    const void *q;
    int64_t q_row_stride, q_head_stride;
    void *out;
    int64_t out_row_stride, out_head_stride;
} rie_hip_attn;

/* Writes the new tokens' keys and values (src_ty: f32, rounded to nearest, or the pages'
 * own type) to their pages. */
int32_t rie_hip_k_paged_append(const rie_hip_pages *pages, const rie_hip_seqs *seqs, int32_t src_ty, const void *k, const void *v,
                               int64_t row_stride, int64_t head_stride, void *stream, char *err, size_t err_len);
/* Causal attention of every sequence's new tokens over its pages, which already hold them:
 * chunks of prompts and single tokens in one batch.  A token that sees nothing, or nothing
 * that scores above −inf, gets zeros.  An infinite or NaN key or value reaches only the
 * tokens that see it (an infinite value as that infinity).  Finite values have finite
 * outputs (bf16: over up to 2^24 positions; bf16 values under 2^-94 may count as zeros).
 * Scores, the softmax's sums and the outputs are f32 sums.  With up to 32 query rows to a KV
 * head (max_new * n_head / n_kv) only the output is rounded to the keys' type; with more, and
 * in packed attention, so is each probability, once (2-norm against float64, bf16: 1.6e-3 and
 * 2.0e-3 to 2.3e-3; f16: 2.0e-4 and 2.3e-4 to 2.8e-4). */
size_t rie_hip_k_paged_attention_ws(const rie_hip_pages *pages, const rie_hip_seqs *seqs, const rie_hip_attn *attn);
int32_t rie_hip_k_paged_attention(const rie_hip_pages *pages, const rie_hip_seqs *seqs, const rie_hip_attn *attn, void *ws,
                                  size_t ws_bytes, void *stream, char *err, size_t err_len);
/* Causal attention within whole prompts packed one behind the other: keys and values are
 * rows beside the queries' (n_kv heads; slices of a fused projection, say). */
size_t rie_hip_k_packed_attention_ws(const rie_hip_seqs *seqs, int32_t ty, int32_t head_dim, int32_t n_kv, const rie_hip_attn *attn);
int32_t rie_hip_k_packed_attention(const rie_hip_seqs *seqs, int32_t ty, int32_t head_dim, int32_t n_kv, const void *k, const void *v,
                                   int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                                   const rie_hip_attn *attn, void *ws, size_t ws_bytes, void *stream, char *err, size_t err_len);

/* Of n rows of n_vocab logits (row_stride elements apart, any alignment of their type):
 * logprob[i] = ln p(targets[i]) (NaN for a target outside 0..n_vocab-1), the entropy of
 * the distribution in nats, and the n_top (≤ 64) most likely tokens in order, the lowest
 * index first among equals, with their log probabilities ([n][n_top]).  logprob with
 * targets, entropy, and top_ids with top_logprobs may be NULL.  −inf logits have
 * probability 0.  A row with a NaN or +inf logit, or nothing above −inf, has NaN for all
 * of its numbers (its top_ids rank NaN as −inf).  n_vocab ≤ 2^21. */
size_t rie_hip_k_token_logprobs_ws(int32_t n, int32_t n_vocab);
int32_t rie_hip_k_token_logprobs(int32_t ty, const void *logits, int32_t n, int32_t n_vocab, int64_t row_stride,
                                 const int32_t *targets, float *logprob, float *entropy, int32_t n_top, int32_t *top_ids,
                                 float *top_logprobs, void *ws, size_t ws_bytes, void *stream, char *err, size_t err_len);

#ifdef __cplusplus
}
#endif
#endif
