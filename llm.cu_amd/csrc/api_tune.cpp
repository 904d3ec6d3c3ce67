// api_tune.cpp — C ABI of the operators for tuning on preferences and rewards
// (token log-probabilities, the preference and policy losses) and of the
// orthogonalised updates.  Every entry point validates its arguments on the
// host before any launch; the standalone ones allocate nothing.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/llmt.h"
#include "ctx.h"

using namespace llmt;

#define TRY_ARG(cond, ...)    \
  do {                        \
    if (!(cond)) {            \
      set_error(__VA_ARGS__); \
      return LLMT_ERR_ARG;    \
    }                         \
  } while (0)

static int done(hipError_t e) {
  return e == hipSuccess ? LLMT_OK : e == hipErrorInvalidValue ? LLMT_ERR_ARG : LLMT_ERR_HIP;
}

static bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

// Matrices of one call, the long side of one (also a vocabulary), and a row or
// matrix stride: grids and indexes stay within 31 bits, offsets within 62.
constexpr int kMaxMatrices = 1 << 20, kMaxLong = 1 << 30;
constexpr long long kMaxStride = 1ll << 40;
static bool strides_fit(long long rows, long long ld) {
  return ld <= kMaxStride && (double)rows * (double)ld <= 1e18;
}

static size_t esize(int dtype) { return dtype == LLMT_F32 ? 4 : 2; }

// The checks that the log-probabilities' two directions share.
static int check_logits(const char* fn, const void* logits, int dtype, long long ld,
                        const int* targets, int rows, int V, float inv_temp) {
  TRY_ARG(dtype == LLMT_F32 || dtype == LLMT_F16 || dtype == LLMT_BF16, "%s: dtype %d", fn, dtype);
  TRY_ARG(rows >= 0 && V >= 1 && V <= kMaxLong && ld >= V && strides_fit(rows, ld),
          "%s: rows=%d V=%d ld=%lld (rows >= 0, V in [1, 2^30], ld >= V)", fn, rows, V, ld);
  TRY_ARG(inv_temp > 0.f && isfinite(inv_temp), "%s: inv_temp must be positive and finite", fn);
  TRY_ARG(rows == 0 || (logits && targets), "%s: NULL argument", fn);
  TRY_ARG(aligned(logits, esize(dtype)) && aligned(targets, 4), "%s: misaligned argument", fn);
  return LLMT_OK;
}

// Whether na floats at a and nb floats at b do not meet.
static bool apart(const void* a, long long na, const void* b, long long nb) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  return a0 + (size_t)na * 4 <= b0 || b0 + (size_t)nb * 4 <= a0;
}

static NsMat ns_matrix(int rows, int cols) {
  NsMat m{};
  m.tall = rows > cols;
  m.r = std::min(rows, cols);
  m.n = std::max(rows, cols);
  m.ld_in = m.ld_out = cols;
  m.lr = 0.f;
  return m;
}

// The layout of an arena of layers x nmat matrices.
static int muon_layout(const char* fn, int layers, int nmat, const int* rows, const int* cols,
                       NsArgs& a) {
  TRY_ARG(layers >= 1 && nmat >= 1 && nmat <= kNsMats && rows && cols,
          "%s: layers=%d nmat=%d (1 to %d matrices a layer)", fn, layers, nmat, kNsMats);
  TRY_ARG(layers <= kMaxMatrices / kNsMats, "%s: %d layers, at most %d", fn, layers,
          kMaxMatrices / kNsMats);
  a.layers = layers;
  a.nmat = nmat;
  long long off = 0;
  for (int j = 0; j < nmat; ++j) {
    TRY_ARG(rows[j] >= 1 && cols[j] >= 1 && std::min(rows[j], cols[j]) <= kNsMaxShort &&
                std::max(rows[j], cols[j]) <= kMaxLong,
            "%s: matrix %d is %d x %d (short side 1 to %d)", fn, j, rows[j], cols[j], kNsMaxShort);
    a.mat[j] = ns_matrix(rows[j], cols[j]);
    a.mat[j].off = off;
    off += (long long)rows[j] * cols[j];
  }
  a.in_stride = a.out_stride = off;
  return LLMT_OK;
}

static int muon_params(const char* fn, const llmt_muon_params* p, NsArgs& a) {
  TRY_ARG(p, "%s: NULL params", fn);
  TRY_ARG(isfinite(p->lr) && p->momentum >= 0.f && p->momentum < 1.f && isfinite(p->wd) &&
              p->eps > 0.f && isfinite(p->eps) && p->steps >= 1 && p->steps <= 20,
          "%s: momentum in [0, 1), eps positive, steps in [1, 20], finite lr and wd", fn);
  TRY_ARG(p->scale == LLMT_MUON_SCALE_RMS || p->scale == LLMT_MUON_SCALE_SHAPE, "%s: scale %d", fn,
          p->scale);
  a.mu = p->momentum;
  a.nesterov = p->nesterov != 0;
  a.steps = p->steps;
  a.eps = p->eps;
  a.decay = (float)(1.0 - (double)p->lr * p->wd);
  for (int j = 0; j < a.nmat; ++j) {
    const double r = a.mat[j].r, n = a.mat[j].n;
    const double s = p->scale == LLMT_MUON_SCALE_RMS ? 0.2 * sqrt(n) : a.mat[j].tall ? sqrt(n / r) : 1.0;
    a.mat[j].lr = (float)(p->lr * s);
  }
  return LLMT_OK;
}

extern "C" {

size_t llmt_token_logprobs_workspace(int rows, int V, int dtype) {
  return rows > 0 && V > 0 ? logprob_workspace(rows, V, dtype) : 0;
}

int llmt_token_logprobs(const void* logits, int dtype, long long ld, const int* targets, int rows,
                        int V, float inv_temp, float* logp, float* stats, float* entropy,
                        void* workspace, size_t workspace_bytes, void* stream) {
  set_error("");
  const int rc = check_logits("llmt_token_logprobs", logits, dtype, ld, targets, rows, V, inv_temp);
  if (rc) return rc;
  if (rows == 0) return LLMT_OK;
  TRY_ARG(logp && stats, "llmt_token_logprobs: NULL argument");
  TRY_ARG(aligned(logp, 4) && aligned(stats, 8) && aligned(entropy, 4),
          "llmt_token_logprobs: misaligned output (stats: 8 bytes)");
  const size_t need = logprob_workspace(rows, V, dtype);
  TRY_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
          "llmt_token_logprobs: workspace of %zu bytes, %zu needed (16-byte aligned)",
          workspace ? workspace_bytes : 0, need);
  LogprobArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.dtype = dtype;
  a.targets = targets;
  a.rows = rows;
  a.V = V;
  a.it = inv_temp;
  a.logp = logp;
  a.stats = stats;
  a.entropy = entropy;
  return done(logprob_fwd(a, workspace, (hipStream_t)stream));
}

int llmt_token_logprobs_bwd(const void* logits, int dtype, long long ld, const int* targets,
                            const float* stats, const float* entropy, const float* dlogp,
                            const float* dentropy, int rows, int V, float inv_temp, void* dlogits,
                            long long ldd, void* stream) {
  set_error("");
  const int rc =
      check_logits("llmt_token_logprobs_bwd", logits, dtype, ld, targets, rows, V, inv_temp);
  if (rc) return rc;
  TRY_ARG(ldd >= V && strides_fit(rows, ldd), "llmt_token_logprobs_bwd: ldd=%lld, V=%d", ldd, V);
  if (rows == 0) return LLMT_OK;
  TRY_ARG(stats && dlogp && dlogits && (!dentropy || entropy),
          "llmt_token_logprobs_bwd: NULL argument (dentropy needs entropy)");
  TRY_ARG(aligned(stats, 8) && aligned(dlogp, 4) && aligned(entropy, 4) && aligned(dentropy, 4) &&
              aligned(dlogits, esize(dtype)),
          "llmt_token_logprobs_bwd: misaligned argument (stats: 8 bytes)");
  if (dlogits == logits) {
    TRY_ARG(ldd == ld, "llmt_token_logprobs_bwd: in place with ldd=%lld, ld=%lld", ldd, ld);
  } else {
    const uintptr_t a0 = (uintptr_t)logits, b0 = (uintptr_t)dlogits;
    const uintptr_t a1 = a0 + ((size_t)(rows - 1) * ld + V) * esize(dtype);
    const uintptr_t b1 = b0 + ((size_t)(rows - 1) * ldd + V) * esize(dtype);
    TRY_ARG(a1 <= b0 || b1 <= a0, "llmt_token_logprobs_bwd: dlogits overlaps logits");
  }
  LogprobArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.dtype = dtype;
  a.targets = targets;
  a.rows = rows;
  a.V = V;
  a.it = inv_temp;
  a.stats = const_cast<float*>(stats);
  a.entropy = const_cast<float*>(entropy);
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  a.dlogits = dlogits;
  a.ldd = ldd;
  return done(logprob_bwd(a, (hipStream_t)stream));
}

int llmt_preference_loss(const float* logp, const float* ref_logp, const unsigned char* mask,
                         const int* offsets, int T, int n, const llmt_pref_params* p, float* loss,
                         float* losses, float* rewards, float* dlogp, void* stream) {
  set_error("");
  TRY_ARG(p && offsets && loss && losses && rewards && (logp || T == 0),
          "llmt_preference_loss: NULL argument");
  TRY_ARG(T >= 0 && n >= 1 && n <= (1 << 29), "llmt_preference_loss: T=%d n=%d", T, n);
  TRY_ARG(p->kind >= LLMT_PREF_SIGMOID && p->kind <= LLMT_PREF_SQUARE,
          "llmt_preference_loss: kind %d", p->kind);
  TRY_ARG(p->beta > 0.f && isfinite(p->beta) && isfinite(p->margin) &&
              p->label_smoothing >= 0.f && p->label_smoothing <= 0.5f,
          "llmt_preference_loss: beta must be positive, margin finite, label_smoothing in [0, 0.5]");
  TRY_ARG(aligned(logp, 4) && aligned(ref_logp, 4) && aligned(offsets, 4) && aligned(loss, 4) &&
              aligned(losses, 4) && aligned(rewards, 4) && aligned(dlogp, 4),
          "llmt_preference_loss: misaligned argument");
  PrefArgs a{};
  a.logp = logp;
  a.ref = ref_logp;
  a.mask = mask;
  a.offsets = offsets;
  a.T = T;
  a.n = n;
  a.kind = p->kind;
  a.average = p->average != 0;
  a.beta = p->beta;
  a.margin = p->margin;
  a.smooth = p->label_smoothing;
  a.losses = losses;
  a.rewards = rewards;
  a.mean = loss;
  a.dlogp = dlogp;
  return done(preference_loss(a, (hipStream_t)stream));
}

size_t llmt_policy_loss_workspace(int T, int n) {
  return T >= 0 && n >= 1 ? policy_workspace(T, n) : 0;
}

int llmt_policy_loss(const float* logp, const float* old_logp, const float* ref_logp,
                     const float* advantages, const float* entropy, const unsigned char* mask,
                     const int* offsets, int T, int n, const llmt_policy_params* p, float* loss,
                     float* stats, float* dlogp, float* dentropy, void* workspace,
                     size_t workspace_bytes, void* stream) {
  set_error("");
  // advantages a sequence are read for every sequence, without tokens too
  TRY_ARG(p && offsets && loss && stats && (logp || T == 0) &&
              (advantages || (T == 0 && !p->adv_per_sequence)),
          "llmt_policy_loss: NULL argument");
  TRY_ARG(T >= 0 && n >= 1 && n <= (1 << 29), "llmt_policy_loss: T=%d n=%d", T, n);
  TRY_ARG(p->mean == LLMT_MEAN_TOKEN || p->mean == LLMT_MEAN_SEQUENCE, "llmt_policy_loss: mean %d",
          p->mean);
  TRY_ARG(p->clip_low >= 0.f && p->clip_low <= 1.f && p->clip_high >= 0.f &&
              !isnan(p->clip_high) && isfinite(p->kl_coef) && isfinite(p->entropy_coef),
          "llmt_policy_loss: clip_low in [0, 1], clip_high >= 0, finite coefficients");
  TRY_ARG(!dentropy || entropy, "llmt_policy_loss: dentropy needs entropy");
  TRY_ARG(aligned(logp, 4) && aligned(old_logp, 4) && aligned(ref_logp, 4) &&
              aligned(advantages, 4) && aligned(entropy, 4) && aligned(offsets, 4) &&
              aligned(loss, 4) && aligned(stats, 4) && aligned(dlogp, 4) && aligned(dentropy, 4),
          "llmt_policy_loss: misaligned argument");
  const size_t need = policy_workspace(T, n);
  TRY_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
          "llmt_policy_loss: workspace of %zu bytes, %zu needed (16-byte aligned)",
          workspace ? workspace_bytes : 0, need);
  PolicyArgs a{};
  a.logp = logp;
  a.old = old_logp;
  a.ref = ref_logp;
  a.adv = advantages;
  a.entropy = entropy;
  a.mask = mask;
  a.offsets = offsets;
  a.T = T;
  a.n = n;
  a.adv_per_seq = p->adv_per_sequence != 0;
  a.seq_mean = p->mean == LLMT_MEAN_SEQUENCE;
  a.clip_low = p->clip_low;
  a.clip_high = p->clip_high;
  a.kl_coef = p->kl_coef;
  a.ent_coef = p->entropy_coef;
  a.loss = loss;
  a.stats = stats;
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  return done(policy_loss(a, workspace, (hipStream_t)stream));
}

size_t llmt_orthogonalize_workspace(int count, int rows, int cols) {
  if (count < 1 || count > kMaxMatrices || rows < 1 || cols < 1 ||
      std::min(rows, cols) > kNsMaxShort || std::max(rows, cols) > kMaxLong)
    return 0;
  NsArgs a{};
  a.layers = count;
  a.nmat = 1;
  a.mat[0] = ns_matrix(rows, cols);
  return ns_workspace(a);
}

int llmt_orthogonalize(const float* x, long long stride_x, long long ldx, float* out,
                       long long stride_out, long long ldo, int count, int rows, int cols,
                       int steps, float eps, void* workspace, size_t workspace_bytes,
                       void* stream) {
  set_error("");
  TRY_ARG(count >= 0 && rows >= 1 && cols >= 1, "llmt_orthogonalize: count=%d rows=%d cols=%d",
          count, rows, cols);
  TRY_ARG(std::min(rows, cols) <= kNsMaxShort && std::max(rows, cols) <= kMaxLong,
          "llmt_orthogonalize: %d x %d: the short side is at most %d", rows, cols, kNsMaxShort);
  TRY_ARG(count <= kMaxMatrices, "llmt_orthogonalize: %d matrices, at most %d", count, kMaxMatrices);
  TRY_ARG(steps >= 1 && steps <= 20 && eps > 0.f && isfinite(eps),
          "llmt_orthogonalize: steps in [1, 20], eps positive");
  const bool bounded = strides_fit(rows, ldx) && strides_fit(rows, ldo) &&
                       stride_x <= kMaxStride && stride_out <= kMaxStride;
  const long long span_x = bounded ? (long long)(rows - 1) * ldx + cols : 0;
  const long long span_o = bounded ? (long long)(rows - 1) * ldo + cols : 0;
  TRY_ARG(bounded && ldx >= cols && ldo >= cols &&
              (count <= 1 || (stride_x >= span_x && stride_out >= span_o)),
          "llmt_orthogonalize: ldx=%lld ldo=%lld stride_x=%lld stride_out=%lld", ldx, ldo, stride_x,
          stride_out);
  if (count == 0) return LLMT_OK;
  TRY_ARG(x && out, "llmt_orthogonalize: NULL argument");
  TRY_ARG(aligned(x, 4) && aligned(out, 4), "llmt_orthogonalize: misaligned argument");
  if (x == out)
    TRY_ARG(ldx == ldo && (count == 1 || stride_x == stride_out),
            "llmt_orthogonalize: in place with other strides");
  else
    TRY_ARG(apart(x, (count - 1) * stride_x + span_x, out, (count - 1) * stride_out + span_o),
            "llmt_orthogonalize: out overlaps x");
  NsArgs a{};
  a.x = x;
  a.out = out;
  a.in_stride = stride_x;
  a.out_stride = stride_out;
  a.layers = count;
  a.nmat = 1;
  a.mat[0] = ns_matrix(rows, cols);
  a.mat[0].ld_in = ldx;
  a.mat[0].ld_out = ldo;
  a.steps = steps;
  a.eps = eps;
  const size_t need = ns_workspace(a);
  TRY_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
          "llmt_orthogonalize: workspace of %zu bytes, %zu needed (16-byte aligned)",
          workspace ? workspace_bytes : 0, need);
  return done(newton_schulz(a, workspace, (hipStream_t)stream));
}

size_t llmt_muon_update_workspace(int layers, int nmat, const int* rows_host,
                                  const int* cols_host) {
  NsArgs a{};
  return muon_layout("", layers, nmat, rows_host, cols_host, a) == LLMT_OK ? ns_workspace(a) : 0;
}

int llmt_muon_update(float* p, const float* g, float* m, int layers, int nmat,
                     const int* rows_host, const int* cols_host, const llmt_muon_params* params,
                     void* workspace, size_t workspace_bytes, void* stream) {
  set_error("");
  NsArgs a{};
  int rc = muon_layout("llmt_muon_update", layers, nmat, rows_host, cols_host, a);
  if (rc) return rc;
  if ((rc = muon_params("llmt_muon_update", params, a))) return rc;
  TRY_ARG(p && g && m, "llmt_muon_update: NULL argument");
  TRY_ARG(aligned(p, 4) && aligned(g, 4) && aligned(m, 4), "llmt_muon_update: misaligned argument");
  const long long n = a.in_stride * layers;
  TRY_ARG(apart(p, n, g, n) && apart(p, n, m, n) && apart(g, n, m, n),
          "llmt_muon_update: p, g and m overlap");
  const size_t need = ns_workspace(a);
  TRY_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
          "llmt_muon_update: workspace of %zu bytes, %zu needed (16-byte aligned)",
          workspace ? workspace_bytes : 0, need);
  a.x = g;
  a.m = m;
  a.out = p;
  return done(newton_schulz(a, workspace, (hipStream_t)stream));
}

int llmt_muon(llmt_ctx* ctx, const llmt_muon_params* params) {
  set_error("");
  Ctx* c = reinterpret_cast<Ctx*>(ctx);
  TRY_ARG(c, "llmt_muon: NULL ctx");
  // a layer of the arena: q, k, v, o; A [rank, in] then B [out, rank]
  const int q = c->Q, kv = c->KV, h = c->H;
  const int in[4] = {h, h, h, q}, out[4] = {q, kv, kv, h};
  int rows[8], cols[8];
  for (int j = 0; j < 4; ++j) {
    rows[2 * j] = cols[2 * j + 1] = kRank;
    cols[2 * j] = in[j];
    rows[2 * j + 1] = out[j];
  }
  NsArgs a{};
  int rc = muon_layout("llmt_muon", c->L, 8, rows, cols, a);
  if (rc) return rc;
  if ((rc = muon_params("llmt_muon", params, a))) return rc;
  TRY_ARG((size_t)a.in_stride == c->lora_per_layer, "llmt_muon: the arena's layout");
  const size_t need = ns_workspace(a);
  if (need && !c->muon_ws) {
    c->muon_ws = c->alloc(need);
    if (!c->muon_ws) return LLMT_ERR_HIP;
  }
  a.x = c->lora_g;
  a.m = c->lora_m;
  a.out = c->lora_p;
  c->m_is_muon = true;
  hipError_t e = newton_schulz(a, c->muon_ws, c->st);
  if (e == hipSuccess) e = c->refresh_shadows();
  if (e == hipSuccess) e = hipStreamSynchronize(c->st);
  return done(e);
}

}  // extern "C"
