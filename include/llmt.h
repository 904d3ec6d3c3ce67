/* llmt.h — C ABI of the MI355X-native LoRA training step (libllmt.so).
 *
 * Two layers share one set of gfx950 kernels:
 *
 *  1. The compat layer: the reference's own step API with the same names,
 *     argument order and struct layouts, now `extern "C"`.  A train.cu-style
 *     driver links against it unchanged.  As in the reference, the compat
 *     functions report failures on stderr and exit(EXIT_FAILURE)
 *     (reference include/utils.h:10-28), run on the legacy default stream and
 *     synchronise only where the reference does (the loss read-back).
 *  2. The native layer (llmt_*): an explicit context, an explicit stream,
 *     batch > 1, int error codes (0 = success, <0 = error, message via
 *     llmt_last_error()) and one host synchronisation per step.
 *
 * All pointers are device pointers unless the parameter name ends in _host.
 * Matrices are row-major; frozen weights are [out, in] like the reference;
 * token ids are int32.  References are file:line in visheshnarayan/llm.cu.
 */
#ifndef LLMT_H
#define LLMT_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- model constants (reference include/config.h:5-21, include/lora.h:6-8) ---- */
#define LLMT_HIDDEN_SIZE       2048
#define LLMT_NUM_LAYERS        28
#define LLMT_NUM_HEADS         16
#define LLMT_NUM_KV_HEADS      8
#define LLMT_HEAD_DIM          128
#define LLMT_INTERMEDIATE_SIZE 6144
#define LLMT_VOCAB_SIZE        151936
#define LLMT_LORA_RANK         16
#define LLMT_LORA_ALPHA        32
#define LLMT_LORA_SCALE        2.0f
#define LLMT_RMS_NORM_EPS      1e-6f
#define LLMT_ROPE_THETA        1000000.0f

/* ======================================================================
 * 1. Compat layer — reference structs (include/lora.h:13-62, src/train.cu:10-24)
 * ====================================================================== */

/* include/lora.h:13-20 — one adapter: A [r, d_in], B [d_out, r], AdamW moments. */
typedef struct {
    float* A;
    float* B;
    float* mA; float* vA;
    float* mB; float* vB;
    int d_in, d_out;
} LoraAdapter;

/* include/lora.h:23-28 */
typedef struct {
    LoraAdapter wq[LLMT_NUM_LAYERS];
    LoraAdapter wk[LLMT_NUM_LAYERS];
    LoraAdapter wv[LLMT_NUM_LAYERS];
    LoraAdapter wo[LLMT_NUM_LAYERS];
} LoraWeights;

/* include/lora.h:31-34 */
typedef struct {
    float* dA;
    float* dB;
} LoraGrad;

/* include/lora.h:36-41 */
typedef struct {
    LoraGrad wq[LLMT_NUM_LAYERS];
    LoraGrad wk[LLMT_NUM_LAYERS];
    LoraGrad wv[LLMT_NUM_LAYERS];
    LoraGrad wo[LLMT_NUM_LAYERS];
} LoraGrads;

/* include/lora.h:44-62.  The layout is the reference's; the stashes
 * themselves are library-private (they live in the context, with the
 * softmax log-sum-exp in place of P), so lora_acts_alloc sets every slot to
 * NULL and the compat forward/backward never read or write them (the
 * reference's train.cu never reads acts either). */
typedef struct {
    float* layer_in[LLMT_NUM_LAYERS];
    float* attn_norm_out[LLMT_NUM_LAYERS];
    float* q_raw[LLMT_NUM_LAYERS];
    float* k_raw[LLMT_NUM_LAYERS];
    float* q_rope[LLMT_NUM_LAYERS];
    float* k_rope[LLMT_NUM_LAYERS];
    float* v_raw[LLMT_NUM_LAYERS];
    float* attn_w[LLMT_NUM_LAYERS];
    float* pre_o[LLMT_NUM_LAYERS];
    float* post_attn[LLMT_NUM_LAYERS];
    float* ffn_norm_out[LLMT_NUM_LAYERS];
    float* gate_raw[LLMT_NUM_LAYERS];
    float* up_raw[LLMT_NUM_LAYERS];
    float* hq[LLMT_NUM_LAYERS];
    float* hk[LLMT_NUM_LAYERS];
    float* hv[LLMT_NUM_LAYERS];
    float* ho[LLMT_NUM_LAYERS];
} LoraActs;

/* src/train.cu:10-17 (= src/kernels/lora_forward.cu:18-32).  The 21 pad slots
 * mirror src/main.cu:40-55: _pad[0..6] = fp16 (uint16 bits) copies of
 * wq, wk, wv, wo, w_gate, w_up, w_down; _pad[7..20] = (int8_t* q, float*
 * scale) pairs in the same order (q [out, in], scale fp32 [out], the
 * src/kernels/quantize.cu recipe).  Weight source, decided by layer 0: its
 * fp16 pads when set (fp16 weights; layers whose pads are NULL convert their
 * fp32 fields once); else its int8 pads when set (int8 weights, the scales
 * rounded to fp16 as the int8 GEMMs take them; layers whose int8 pads are
 * NULL quantise their fp32 fields); else the fp32 fields converted to fp16.
 * The fp32 weight fields may be NULL when the pads are supplied. */
typedef struct {
    float* attn_norm;
    float* ffn_norm;
    float* wq; float* wk; float* wv; float* wo;
    float* q_norm; float* k_norm;
    float* w_gate; float* w_up; float* w_down;
    void* _pad[21];
} LW;

/* src/train.cu:18-24.  _pad[0] = fp16 lm_head, _pad[1..2] = int8_t* lm_head
 * and its float* row scales (src/main.cu:63-64).  The head is read from the
 * fp16 pad, else the fp32 lm_head, else the int8 pair (as fp16 q * scale).
 * embed_table may be NULL when the lm_head is tied (the reference scripts
 * copy embed -> lm_head, scripts/run.sh:19); the gather then reads the
 * lm_head rows. */
typedef struct {
    float* embed_table;
    LW layers[LLMT_NUM_LAYERS];
    float* final_norm;
    float* lm_head;
    void* _pad[3];
} MW;

/* include/lora.h:66-90 */
void lora_weights_init(LoraWeights* lora);
void lora_weights_free(LoraWeights* lora);
void lora_grads_alloc(LoraGrads* grads, const LoraWeights* lora);
void lora_grads_free(LoraGrads* grads);
void lora_grads_zero(LoraGrads* grads);
void lora_acts_alloc(LoraActs* acts, int seq_len);
void lora_acts_free(LoraActs* acts, int seq_len);
/* src/kernels/lora.cu:181-202: y[seq, d_out] += 2 * (x A^T) B^T; h_buf = x A^T if non-NULL. */
void lora_forward_add(const float* x, const LoraAdapter* a, float* y, float* h_buf, int seq);
/* src/kernels/lora.cu:235-246 */
void adamw_step_lora(LoraWeights* lora, const LoraGrads* grads, float lr, float beta1,
                     float beta2, float eps, float wd, int step);
/* src/kernels/lora.cu:10-28 */
void scale_add_inplace(float* dst, const float* src, float scale, int n);
void gpu_zero(float* buf, int n);

/* src/kernels/lora_forward.cu:169-186.  The workspaces and acts are accepted
 * for ABI compatibility and not touched (the stashes live in the library's
 * context); logits receives the fp32 logits [seq, V].  Frozen weights are
 * uploaded (by the MW pad map above) on the first call for a given MW,
 * adapters on every call.  Any seq_len >= 2. */
void transformer_forward_lora(const int* token_ids, const MW* model, const LoraWeights* lora,
                              float* hidden, float* residual, float* norm_out,
                              float* q, float* k, float* v, float* k_exp, float* v_exp,
                              float* attn_out, float* gate_buf, float* up_buf,
                              float* logits, LoraActs* acts, int seq_len);
/* src/kernels/loss.cu:74-91: mean CE over the seq_len-1 rows with a target;
 * writes fp32 dlogits (row seq_len-1 zeroed); returns the loss (syncs). */
float cross_entropy_forward(const float* logits, const int* targets, float* dlogits, int seq_len);
/* src/kernels/lora_backward.cu:212-233.  Gradients are accumulated into
 * grads (callers zero them first, as src/train.cu:261 does). */
void transformer_backward_lora(const float* d_logits, const MW* model, const LoraWeights* lora,
                               const LoraActs* acts, LoraGrads* grads,
                               float* d_hidden, float* d_hidden2, float* d_norm,
                               float* d_q, float* d_k, float* d_v,
                               float* d_q_exp, float* d_k_exp, float* d_v_exp,
                               float* d_pre_o, float* d_gate, float* d_up,
                               float* dh_tmp, float* dx_lora, int seq_len);

/* ======================================================================
 * 2. Native layer
 * ====================================================================== */

typedef struct llmt_ctx llmt_ctx;

typedef struct {
    int hidden, n_layers, n_heads, n_kv_heads, head_dim, intermediate, vocab, rank;
    float alpha, eps, theta;
} llmt_dims;

typedef struct {
    float lr, beta1, beta2, eps, wd;
} llmt_hparams;

enum {
    LLMT_OK = 0,
    LLMT_ERR_ARG = -1,       /* bad argument / unsupported shape */
    LLMT_ERR_HIP = -2,       /* HIP runtime error */
    LLMT_ERR_IO = -3,        /* missing or short file */
    LLMT_ERR_STATE = -4      /* call order (e.g. backward before forward) */
};
enum { LLMT_WEIGHTS_F16 = 0, LLMT_WEIGHTS_I8 = 1 };
enum { LLMT_PROJ_Q = 0, LLMT_PROJ_K = 1, LLMT_PROJ_V = 2, LLMT_PROJ_O = 3 };
enum { LLMT_LORA_PARAM = 0, LLMT_LORA_GRAD = 1, LLMT_LORA_M = 2, LLMT_LORA_V = 3 };

const char* llmt_last_error(void);
void llmt_dims_qwen3_1_7b(llmt_dims* out);

/* Context for up to max_batch sequences of seq_len tokens (stashes and
 * workspaces are sized at creation).  stream may be NULL: the context then
 * creates its own stream, blocking with respect to the legacy default stream
 * (a captured HIP graph needs a non-default stream). */
int llmt_ctx_create(const llmt_dims* dims, int max_batch, int seq_len, int weight_format,
                    void* stream, llmt_ctx** out);
int llmt_ctx_destroy(llmt_ctx* ctx);
/* Bytes of device memory the context owns. */
size_t llmt_ctx_device_bytes(const llmt_ctx* ctx);

/* Frozen weights.  fp16 arguments are [out, in] fp16 device buffers; the
 * library copies them into its own packed, pre-transposed arena, so callers
 * may free theirs afterwards.  Norm weights are fp32 [n]. */
int llmt_set_layer_f16(llmt_ctx* ctx, int layer, const void* wq, const void* wk, const void* wv,
                       const void* wo, const void* w_gate, const void* w_up, const void* w_down,
                       const float* attn_norm, const float* ffn_norm, const float* q_norm,
                       const float* k_norm);
/* int8 [out, in] weights with fp16 per-output-row scales (the quantize.cu
 * recipe, produced e.g. by llmt_quantize_rows_i8).  A row whose fp16 scale is
 * 0 is taken as all zeros. */
int llmt_set_layer_i8(llmt_ctx* ctx, int layer, const int8_t* const q[7], const void* const scale[7],
                      const float* attn_norm, const float* ffn_norm, const float* q_norm,
                      const float* k_norm);
/* Tied embedding / lm_head [V, H] fp16 and the final norm [H] fp32.  Ties
 * the head to this embedding (again, after an llmt_set_lm_head_f16). */
int llmt_set_embed_f16(llmt_ctx* ctx, const void* embed_lm_head, const float* final_norm);
/* An untied lm_head [V, H] fp16 (the reference loads lm_head.weight.bin on its
 * own, src/train.cu:87-88): the logits and the head's dX use it, the token
 * gather keeps the embedding.  Allocates the head's packed copies on the
 * first call. */
int llmt_set_lm_head_f16(llmt_ctx* ctx, const void* lm_head);
/* Reference on-disk layout (src/train.cu:56-89, python/export_weights.py:19-26):
 * <dir>/<hf_param_name>.bin raw fp32 little-endian [out, in], no header.
 * lm_head.weight.bin is optional: absent or equal to the embedding means a
 * tied head, otherwise it is loaded as an untied head. */
int llmt_load_weights_dir(llmt_ctx* ctx, const char* dir);

/* Adapters live in one fp32 arena per kind (param, grad, m, v), ordered layer
 * by layer, q, k, v, o, A then B (A [r, d_in], B [d_out, r]). */
size_t llmt_lora_numel(const llmt_ctx* ctx);
size_t llmt_lora_offset(const llmt_ctx* ctx, int layer, int proj, int is_b);
/* Copy a whole arena to/from a caller device buffer (to_ctx: 1 = into ctx). */
int llmt_lora_copy(llmt_ctx* ctx, int kind, float* buf, int to_ctx);
/* Reference adapter files weights/lora_step{N}_layer{L}_{wq|wk|wv|wo}_{A|B}.bin
 * (src/train.cu:146-170) — raw fp32, A [16, d_in], B [d_out, 16]. */
int llmt_lora_save(llmt_ctx* ctx, const char* dir, int step);
int llmt_lora_load(llmt_ctx* ctx, const char* dir, int step);
/* AdamW moments for resuming a run (no counterpart in the reference, whose
 * driver cannot resume): <dir>/lora_step{N}_adamw.bin holds "LLMTADAM",
 * int32 version 1, int32 step, int64 numel, fp32 m, fp32 v.  After llmt_muon the
 * same file begins with "LLMTMUON": m is Muon's momentum, v unused. */
int llmt_lora_save_state(llmt_ctx* ctx, const char* dir, int step);
int llmt_lora_load_state(llmt_ctx* ctx, const char* dir, int step);
/* Seeded init on the device (the reference draws A with cuRAND, B = 0:
 * src/kernels/lora.cu:40-62; configs use A std a_std, B std b_std). */
int llmt_lora_init(llmt_ctx* ctx, uint64_t seed, float a_std, float b_std);

/* One training step (src/train.cu:251-288): forward, fused CE, backward,
 * AdamW with bias-correction step `step` (1-based).  tokens/targets: int32
 * device [batch, seq_len], any seq_len >= 2 and batch <= max_batch (the
 * kernels run on batch*seq_len rows rounded up to a multiple of 16; the pad
 * rows are zero and add nothing).  The loss is the mean over
 * batch*(seq_len-1) rows (src/kernels/loss.cu:86-90).  *loss_host is written
 * after the one host sync.  llmt_forward_backward runs everything but AdamW
 * (grads are left in the GRAD arena, overwritten, not accumulated). */
int llmt_step(llmt_ctx* ctx, const int* tokens, const int* targets, int batch,
              const llmt_hparams* hp, int step, float* loss_host);
int llmt_forward_backward(llmt_ctx* ctx, const int* tokens, const int* targets, int batch,
                          float* loss_host);
/* Capture llmt_step's device work into a HIP graph and replay it
 * (enable = 1); the graph is rebuilt when batch changes. */
int llmt_set_graph(llmt_ctx* ctx, int enable);
/* fp32 logits of the last forward: rows 0 .. batch*seq_len-1 in token order
 * (then the zero pad rows up to a multiple of 16), V wide. */
const float* llmt_logits(const llmt_ctx* ctx);
/* fp32 residual stream [batch*seq_len, H] at the input of `layer` (0..L-1)
 * from the last forward, the reference's LoraActs.layer_in[layer]
 * (include/lora.h:45, src/kernels/lora_forward.cu:205): layer 0's rows are
 * the gathered embedding rows E[token] (src/kernels/embed.cu:6-20).  NULL for
 * a layer outside the model. */
const float* llmt_layer_in(const llmt_ctx* ctx, int layer);

/* Single-layer forward/backward through layer `layer` (config C0): x, y, dy,
 * dx are fp32 [batch*seq_len, H], batch*seq_len a multiple of 16. The
 * backward writes the layer's adapter gradients into the GRAD arena and dx. */
int llmt_layer_forward(llmt_ctx* ctx, int layer, const float* x, float* y, int batch);
int llmt_layer_backward(llmt_ctx* ctx, int layer, const float* dy, float* dx, int batch);
/* AdamW over the whole arena (one multi-tensor launch). */
int llmt_adamw(llmt_ctx* ctx, const llmt_hparams* hp, int step);
/* Per-kernel timing of one llmt_step (no counterpart in the reference).  The
 * step (forward, CE, backward, AdamW: the adapters advance by this one step)
 * runs once eagerly with every kernel launch recorded; then the launches of
 * each kind (one kernel at one shape; a backward dX GEMM's name ends in
 * " dX") are replayed back to back, `reps`
 * times, as a HIP graph of their own and timed with HIP events on the
 * context's stream, so no events sit between kernels and no dependent-launch
 * gaps are counted (the kinds' totals sum to less than a step).  The
 * parameter and moment arenas are saved before the replays and restored
 * after; the GRAD arena and the stashes are left unspecified.  Per kind
 * k < *nkinds (<= max_kinds), in first-launch order: names[k] (owned by the
 * context, valid until its next llmt_profile_kernels or destroy), cats[k]
 * (0 forward GEMMs, 1 backward GEMMs, 2 lm_head GEMMs, 3 attention, 4 row
 * epilogues, 5 cross-entropy, 6 LoRA gradients, 7 AdamW), launches[k] per
 * step, us[k] = average launch duration in microseconds, flops[k] and
 * bytes[k] = algorithmic work of one launch: GEMMs 2 M N K and the streamed
 * weight bytes; attention the flops of its causal S x S x 128 products (two
 * forward, five backward) and no bytes; every other kernel no flops and the
 * bytes its interface reads and writes (split-K partials included). */
int llmt_profile_kernels(llmt_ctx* ctx, const int* tokens, const int* targets, int batch,
                         const llmt_hparams* hp, int step, int reps, int max_kinds, int* nkinds,
                         const char** names, int* cats, int* launches, float* us, double* flops,
                         double* bytes);

/* ---- standalone operators (stream may be NULL) ---- */

/* C = A B^T: A [M, K] fp16 (lda), B [N, K] fp16 (ldb), C [M, N] fp32 (ldc).
 * M % 16 == 0, K % 64 == 0. */
int llmt_gemm_f16(const void* A, int lda, const void* B, int ldb, float* C, int ldc,
                  int M, int N, int K, void* stream);
/* C = (A q^T) * scale[n]: q [N, K] int8, scale [N] fp16. */
int llmt_gemm_i8(const void* A, int lda, const int8_t* q, int ldq, const void* scale,
                 float* C, int ldc, int M, int N, int K, void* stream);
/* src/kernels/quantize.cu:8-44 bit-exact: q [rows, cols] int8, scale fp32 [rows]. */
int llmt_quantize_rows_i8(const float* w, int rows, int cols, int8_t* q, float* scale, void* stream);
/* Fused softmax + NLL + dlogits over rows of width V (src/kernels/loss.cu:13-71).
 * Row i is valid when (i % seq_len) < seq_len-1.  loss_rows [rows] (0 for
 * invalid rows), *loss_mean (device) = mean over valid rows, dlogits fp32
 * (may be NULL). */
int llmt_cross_entropy(const float* logits, const int* targets, int rows, int V, int seq_len,
                       float* dlogits, float* loss_rows, float* loss_mean, void* stream);
/* llmt_cross_entropy without any allocation: no counterpart in the reference;
 * for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops).  Same arguments, results and errors, plus
 * LLMT_ERR_ARG when rows * ceil(V / 8192) exceeds 262144 (the library's
 * built-in 2 MiB statistics scratch: 13,797 rows at V = 151936).  Calls that
 * overlap on one GPU share that scratch and race. */
int llmt_cross_entropy_noalloc(const float* logits, const int* targets, int rows, int V,
                               int seq_len, float* dlogits, float* loss_rows, float* loss_mean,
                               void* stream);
/* Config C1: logits = hidden W^T, fused CE, dlogits, dhidden = dlogits W.
 * hidden [T, H] fp16, W [V, H] fp16 row-major (packed into temporaries on
 * every call); outputs fp32; *loss_mean is a device float; dlogits may be
 * NULL.  T % 16 == 0, T % seq_len == 0. */
int llmt_lm_head_ce(const void* hidden, const void* W, const int* targets, int T, int seq_len,
                    int H, int V, float* loss_mean, float* dlogits, float* dhidden, void* stream);
/* Config C1 on a context's lm_head (already packed by llmt_set_embed_f16 /
 * llmt_set_lm_head_f16): hidden fp16 [batch*seq_len, H] (batch*seq_len a
 * multiple of 16), dlogits (may be NULL) and dhidden fp32 device buffers;
 * *loss_host after one host sync. */
int llmt_head_ce(llmt_ctx* ctx, const void* hidden16, const int* targets, int batch,
                 float* loss_host, float* dlogits, float* dhidden);
/* Causal GQA flash attention (config C3).  q [B,S,nq,128], k/v [B,S,nkv,128]
 * fp16, o fp16 [B,S,nq,128], lse fp32 [B,nq,S]. */
int llmt_attention_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                       int B, int S, int nq, int nkv, void* stream);
/* dq/dk/dv fp32 w.r.t. the attention inputs (post-norm, post-RoPE). do fp32. */
int llmt_attention_bwd(const void* q, const void* k, const void* v, const void* o,
                       const float* lse, const float* dout, float* dq, float* dk, float* dv,
                       int B, int S, int nq, int nkv, void* stream);
/* Config C3 end to end: raw (pre-QK-norm) q/k, v fp16; QK-RMSNorm (weights
 * q_norm/k_norm fp32 [128]) and RoPE(theta) forward, flash forward, then the
 * backward to dq_raw, dk_raw, dv (fp32). */
int llmt_attention_block_bwd(const void* q_raw, const void* k_raw, const void* v,
                             const float* q_norm, const float* k_norm, const void* dout,
                             float* dq_raw, float* dk_raw, float* dv,
                             int B, int S, int nq, int nkv, float theta, float eps, void* stream);

/* ---- tuning on preferences and rewards: operators on the caller's logits ----
 * No counterpart in the reference, whose only loss is the cross entropy.  They
 * allocate nothing: what they need beyond their outputs is the caller's
 * workspace (16-byte aligned, at least the bytes that the *_workspace function
 * gives for the same sizes; it may be NULL where that is 0), so a call can be
 * captured into a HIP graph.  A workspace belongs to one call at a time: two
 * streams, or two graphs that may run at once, take one each.  Results do not
 * depend on the workspace's contents and repeat bit for bit. */

enum { LLMT_F32 = 0, LLMT_F16 = 1, LLMT_BF16 = 2 };

/* Log-probabilities of target tokens.  logits [rows, V] of `dtype`, ld
 * elements from row to row (ld >= V; any alignment of whole elements), scaled
 * by inv_temp > 0 before the softmax:
 *   x = logits * inv_temp,  m = max x,  l = ln sum exp(x - m)
 *   logp[i] = x[target] - m - l,  stats[i] = (m, l),
 *   entropy[i] = -sum p ln p (may be NULL).
 * A row whose target is outside [0, V) (padding, a prompt token) is not read:
 * its outputs are 0.  An x of -inf has probability 0; a row of nothing but
 * -inf gives logp -inf, stats (-inf, 0), entropy 0.  Finite masks of any size
 * are logits like others: a row that they fill is uniform (where |m| exceeds
 * 2^29 each x is rounded to fp32 before m is subtracted); an x beyond fp32's
 * range is infinite, so masks of its lowest value are -inf at an inv_temp above
 * 1, and a row of nothing else is one of nothing but -inf.  A NaN or +inf makes
 * the outputs of its own row NaN.  rows may be 0. */
size_t llmt_token_logprobs_workspace(int rows, int V, int dtype);
int llmt_token_logprobs(const void* logits, int dtype, long long ld, const int* targets, int rows,
                        int V, float inv_temp, float* logp, float* stats, float* entropy,
                        void* workspace, size_t workspace_bytes, void* stream);
/* Its gradient: with p = exp(x - m - l) from the forward's stats,
 *   dlogits[j] = inv_temp (dlogp (1[j = target] - p_j)
 *                          - dentropy p_j (ln p_j + entropy)),
 * of the logits' type, rounded once.  dentropy may be NULL (entropy is then
 * not read).  Rows without a target, rows of nothing but -inf, and rows whose
 * dlogp and dentropy are both 0 are written as zeros and not read.  dlogits
 * may be logits itself (with ldd = ld); any other overlap is refused.  In fp16 a
 * probability times a small dlogp underflows: pass dlogp times a loss scale. */
int llmt_token_logprobs_bwd(const void* logits, int dtype, long long ld, const int* targets,
                            const float* stats, const float* entropy, const float* dlogp,
                            const float* dentropy, int rows, int V, float inv_temp, void* dlogits,
                            long long ldd, void* stream);

/* The same through a context's model: a forward that gives the log-probability
 * of every target, logp [batch * seq_len] (0 where the target is outside
 * [0, V): prompts, padding, the last position of a window), and the backward
 * of any function of them from dlogp, its gradient: the adapter gradients go
 * to the GRAD arena (overwritten), for llmt_adamw or llmt_muon.  The backward
 * takes the stashes of the last forward and fails with LLMT_ERR_STATE if that
 * was not llmt_forward_logprobs' or if weights or adapters have been set or
 * updated since; it may be called more than once.  tokens, targets, batch as
 * in llmt_step; one host synchronisation each.  They run on the context's
 * stream: what other streams write into their inputs has to be finished, or
 * ordered before that stream, when they are called. */
int llmt_forward_logprobs(llmt_ctx* ctx, const int* tokens, const int* targets, int batch,
                          float* logp);
int llmt_backward_logprobs(llmt_ctx* ctx, const float* dlogp);

/* Preference loss on n pairs of sequences.  Sequence s is tokens offsets[s] ..
 * offsets[s + 1] - 1 of the T (offsets int32 [2 n + 1], ascending); pair i
 * prefers sequence 2 i to sequence 2 i + 1.  logp, and ref_logp of the frozen
 * reference model (may be NULL: none), fp32 [T]; mask (bytes [T], may be NULL)
 * leaves tokens out.  With r = beta * sum over the kept tokens of
 * (logp - ref_logp), divided by their number with `average` (0 without any):
 *   z = r[2 i] - r[2 i + 1] - margin
 *   losses[i] = (1 - label_smoothing) f(z) + label_smoothing f(-z)
 * f: ln(1 + exp(-z)) (sigmoid), max(0, 1 - z) (hinge), (z - 1/2)^2 (square:
 * beta^2 times the identity-preference loss).  loss [1] is the mean of losses
 * [n], rewards [2 n] are r, dlogp [T] (may be NULL) the gradient of the mean:
 * 0 at tokens left out and at tokens of no sequence. */
enum { LLMT_PREF_SIGMOID = 0, LLMT_PREF_HINGE = 1, LLMT_PREF_SQUARE = 2 };
typedef struct {
    int kind, average;
    float beta, label_smoothing, margin;
} llmt_pref_params;
int llmt_preference_loss(const float* logp, const float* ref_logp, const unsigned char* mask,
                         const int* offsets, int T, int n, const llmt_pref_params* params,
                         float* loss, float* losses, float* rewards, float* dlogp, void* stream);

/* Clipped policy loss with a KL term over the tokens of n sequences (offsets
 * int32 [n + 1] as above).  Per kept token, with A its advantage (fp32 [T], or
 * [n] with adv_per_sequence), ratio = exp(logp - old_logp) (old_logp NULL: the
 * policy that sampled is this one, ratio 1) and d = ref_logp - logp:
 *   policy = -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A)
 *   kl     = exp(d) - d - 1                       (0 with ref_logp NULL)
 *   l      = policy + kl_coef kl - entropy_coef entropy   (entropy may be NULL)
 * A ratio beyond fp32 counts nothing at an advantage of 0; a logp of -inf has
 * ratio 0 (1 without old_logp) and a kl of +inf from a finite ref_logp; with
 * kl_coef 0 the kl, of any size, is only reported in stats.
 * loss [1] is the mean of l over all kept tokens (LLMT_MEAN_TOKEN), or the
 * mean over the n sequences of their kept tokens' means, a sequence without
 * any counting as 0 (LLMT_MEAN_SEQUENCE).  stats [3]: policy, kl and the share
 * of clipped tokens, averaged the same way.  dlogp, dentropy [T] (may be NULL):
 * the gradient of loss, 0 at tokens left out and at tokens of no sequence. */
enum { LLMT_MEAN_TOKEN = 0, LLMT_MEAN_SEQUENCE = 1 };
typedef struct {
    int mean, adv_per_sequence;
    float clip_low, clip_high, kl_coef, entropy_coef;
} llmt_policy_params;
size_t llmt_policy_loss_workspace(int T, int n);
int llmt_policy_loss(const float* logp, const float* old_logp, const float* ref_logp,
                     const float* advantages, const float* entropy, const unsigned char* mask,
                     const int* offsets, int T, int n, const llmt_policy_params* params,
                     float* loss, float* stats, float* dlogp, float* dentropy, void* workspace,
                     size_t workspace_bytes, void* stream);

/* ---- orthogonalised updates (no counterpart in the reference) ----
 * Newton-Schulz orthogonalisation of fp32 matrices whose short side is at most
 * 64 (adapters: their rank): X0 = X / (|X|_F + eps), then `steps` times
 * X <- 3.4445 X - 4.7750 (X X^T) X + 2.0315 (X X^T)^2 X (of the transpose for a
 * tall X), in fp64, rounded once.  A zero matrix gives zeros; a NaN or an
 * infinity makes its own matrix NaN.  count matrices [rows, cols], stride_x
 * elements from one to the next and ldx from row to row; out likewise, and may
 * be x itself with the same strides (any other overlap of the two is refused).  The
 * matrices of one argument must not overlap one another.  1 <= steps <= 20. */
size_t llmt_orthogonalize_workspace(int count, int rows, int cols);
int llmt_orthogonalize(const float* x, long long stride_x, long long ldx, float* out,
                       long long stride_out, long long ldo, int count, int rows, int cols,
                       int steps, float eps, void* workspace, size_t workspace_bytes, void* stream);

/* Muon on an arena of `layers` layers of nmat (<= 8) matrices, [rows_host[j],
 * cols_host[j]] each (host arrays), one behind another without gaps; p, g, m
 * fp32 arenas of that layout that do not overlap:
 *   m <- momentum m + g;   u = nesterov ? g + momentum m : m
 *   p <- p (1 - lr wd) - lr s orthogonalised(u)
 * with s = 0.2 sqrt(max(rows, cols)) (LLMT_MUON_SCALE_RMS: updates of AdamW's
 * size) or sqrt(max(1, rows / cols)) (LLMT_MUON_SCALE_SHAPE). */
enum { LLMT_MUON_SCALE_RMS = 0, LLMT_MUON_SCALE_SHAPE = 1 };
typedef struct {
    float lr, momentum, wd, eps;
    int steps, nesterov, scale;
} llmt_muon_params;
size_t llmt_muon_update_workspace(int layers, int nmat, const int* rows_host, const int* cols_host);
int llmt_muon_update(float* p, const float* g, float* m, int layers, int nmat,
                     const int* rows_host, const int* cols_host, const llmt_muon_params* params,
                     void* workspace, size_t workspace_bytes, void* stream);
/* Muon over a context's whole adapter arena from its GRAD arena (the M arena
 * holds the momentum, V is not used), in place of llmt_adamw; one host
 * synchronisation.  AdamW (llmt_step, llmt_adamw, llmt_profile_kernels) fails
 * with LLMT_ERR_STATE from then on, until M is set by llmt_lora_copy,
 * llmt_lora_load_state (of an AdamW state) or llmt_lora_init. */
int llmt_muon(llmt_ctx* ctx, const llmt_muon_params* params);

/* ---- training all weights on packed sequences (no counterpart in the reference) ----
 * Attention, embedding and AdamW on the caller's own tensors, for models that
 * train more than a context's adapters.  As the operators above they run on the
 * given stream, allocate nothing, repeat bit for bit and can be captured. */

/* Heads of tokens: element (t, h, i), i < head_dim, is p[t token + h head + i]
 * (strides in elements).  Any layout whose head_dim is contiguous: [T, heads, d],
 * a part of a fused projection's rows, [heads, T, d].  p is 16-byte aligned, the
 * strides are multiples of 8, token in [head_dim, 2^23], head in [0, 2^40], for
 * q, o, dout and dq (group - 1) head at most 2^28.  An output's elements must not
 * coincide with one another or with another argument's.  Parts of one buffer may lie
 * between one another ([T, heads, 2, d]) where they have the same strides; where
 * strides differ, they are taken as apart only if one lies behind the other, or
 * every token's heads do. */
typedef struct {
    void* p;
    long long token, head;
} llmt_heads;

/* Causal attention with grouped heads over n sequences packed one behind
 * another.  Sequence s has queries q_offsets[s] .. q_offsets[s + 1] - 1 of the
 * Tq tokens and keys k_offsets[s] .. k_offsets[s + 1] - 1 of the Tk (device int32
 * [n + 1], ascending; the same array where a sequence attends to itself).  Its
 * last query sees all of its keys: with ql queries and kl keys, query t sees keys
 * 0 .. t + kl - ql, so kl > ql continues a cache (ql = 1: a single new token), and
 * of ql > kl the first ql - kl queries see none.  Query head h reads KV head
 * h / (nq / nkv).
 *   o = softmax(scale q k^T) v,  lse = ln sum exp(scale q k^T)  (fp32 [Tq, nq])
 * A query without keys, and tokens of no sequence, have o 0 and lse -inf.  dtype
 * (q, k, v, o, the gradients): LLMT_F16 or LLMT_BF16; products accumulate in
 * fp32, probabilities are rounded to dtype before the second product (with few
 * rows or keys they enter it with their remainder: the result alone is rounded).
 * head_dim 64 or 128; nq at most 64 nkv; and, the launches' limit, the larger of
 * Tq nq / nkv and Tk at most 64 ((2^23 - 2^12) / nkv - n - 2).  Scores (scale q k) up to
 * 2^24 in magnitude; larger ones, and NaN or infinities in the inputs, spoil
 * results of their own sequence only. */
typedef struct {
    int dtype, nq, nkv, head_dim;
    int n, Tq, Tk;
    float scale;
    const int* q_offsets;
    const int* k_offsets;
} llmt_packed_dims;
size_t llmt_packed_attention_workspace(const llmt_packed_dims* dims);
int llmt_packed_attention(const llmt_packed_dims* dims, const llmt_heads* q, const llmt_heads* k,
                          const llmt_heads* v, const llmt_heads* o, float* lse, void* workspace,
                          size_t workspace_bytes, void* stream);
/* Its gradients, in dtype: dq of the queries, dk and dv of the keys (summed over
 * a group's query heads), from the forward's o and lse and dout = d o.  P, and dS =
 * P (dout v^T - rowsum(dout o)), are rounded to dtype before their products as the
 * forward's probabilities are.  (The
 * rounding of lse to fp32 is 2^-23 of its magnitude in every probability.)  Queries
 * without keys, keys without queries and tokens of no sequence get zeros. */
size_t llmt_packed_attention_bwd_workspace(const llmt_packed_dims* dims);
int llmt_packed_attention_bwd(const llmt_packed_dims* dims, const llmt_heads* q,
                              const llmt_heads* k, const llmt_heads* v, const llmt_heads* o,
                              const float* lse, const llmt_heads* dout, const llmt_heads* dq,
                              const llmt_heads* dk, const llmt_heads* dv, void* workspace,
                              size_t workspace_bytes, void* stream);

/* Embedding: out[i] = scale weight[tokens[i]], the product in fp32, rounded to the
 * output's type; zeros where the
 * token is outside [0, V) (padding).  weight [V, H], ldw elements from row to
 * row, out [T, H], ldo; LLMT_F32, LLMT_F16 or LLMT_BF16 each.  T at most 2^23, V
 * 2^30, H 2^20. */
int llmt_embedding(const int* tokens, int T, const void* weight, int wdtype, long long ldw, int V,
                   int H, float scale, void* out, int odtype, long long ldo, void* stream);
/* Its gradient: dweight[v] = scale sum of dout[i] over tokens[i] = v, or that
 * added to what dweight holds (accumulate; rows of no token are then not
 * touched).  Sums are fp32, in an order that the positions alone decide, rounded
 * once. */
size_t llmt_embedding_bwd_workspace(int T, int V, int H);
int llmt_embedding_bwd(const int* tokens, int T, const void* dout, int ddtype, long long ldd,
                       float scale, void* dweight, int wdtype, long long ldw, int V, int H,
                       int accumulate, void* workspace, size_t workspace_bytes, void* stream);

/* AdamW over a list of tensors (a host array of `count` descriptors; only the
 * pointers in it are the device's), as llmt_adamw's formula:
 *   g' = g grad_scale (one float on the device; NULL: 1)
 *   m = beta1 m + (1 - beta1) g',  v = beta2 v + ((1 - beta2) g') g'
 *   p = p (1 - lr wd) - lr (m / (1 - beta1^step)) / (sqrt(v / (1 - beta2^step)) + eps)
 * and copy, where not NULL, p rounded to copy_dtype (LLMT_F16, LLMT_BF16).  p is
 * fp32, g any type.  state_bits 32: m and v fp32 [n].  state_bits 8: m and v
 * bytes [n], m_exp and v_exp a byte for each 256 elements; all zero bytes are
 * moments of 0.  Under the block's scale 2^(exp - 127), the power of two that
 * brings its largest magnitude to at most 1.875, an m is sign, 4 exponent and 3
 * mantissa bits (the 15th binade that of the largest), a v 5 and 3 (the 31st), with
 * gradual underflow.  They are rounded up with the probability of their
 * remainder, from a generator's draws of (seed, step, the tensor's place in the
 * list, element), a v above 0 to at least its smallest code; p is updated from
 * the moments before that rounding.  A block with a NaN or an infinity (or
 * a magnitude beyond 1.875 2^126) becomes NaN.  Betas in [0, 1), eps at least 2^-126, count at most
 * 2^20, n 2^35.  No two written arrays may overlap, nor a written
 * one a gradient.  hp, step and seed are the call's: a captured call repeats
 * them. */
typedef struct {
    float* p;
    const void* g;
    void* m;
    void* v;
    unsigned char* m_exp;
    unsigned char* v_exp;
    void* copy;
    long long n;
    int g_dtype, copy_dtype;
} llmt_adam_tensor;
int llmt_adamw_update(const llmt_adam_tensor* tensors_host, int count, int state_bits,
                      const llmt_hparams* hp, int step, const float* grad_scale, uint64_t seed,
                      void* stream);
/* What 8-bit moments of n elements stand for, in fp32. */
int llmt_adamw_moments(const void* m, const void* v, const unsigned char* m_exp,
                       const unsigned char* v_exp, long long n, float* m32, float* v32,
                       void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LLMT_H */
