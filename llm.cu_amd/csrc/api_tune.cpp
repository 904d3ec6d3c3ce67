// api_tune.cpp — C ABI of the operators for tuning on preferences and rewards:
// token log-probabilities, the preference and policy losses.  Every entry
// point validates its arguments on the host before any launch and allocates
// nothing.
#include <math.h>
#include <stdint.h>

#include "../../include/llmt.h"
#include "ops.h"

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

static size_t esize(int dtype) { return dtype == LLMT_F32 ? 4 : 2; }

// The checks that the log-probabilities' two directions share.
static int check_logits(const char* fn, const void* logits, int dtype, long long ld,
                        const int* targets, int rows, int V, float inv_temp) {
  TRY_ARG(dtype == LLMT_F32 || dtype == LLMT_F16 || dtype == LLMT_BF16, "%s: dtype %d", fn, dtype);
  TRY_ARG(rows >= 0 && V >= 1 && ld >= V, "%s: rows=%d V=%d ld=%lld (rows >= 0, V >= 1, ld >= V)",
          fn, rows, V, ld);
  TRY_ARG(inv_temp > 0.f && isfinite(inv_temp), "%s: inv_temp must be positive and finite", fn);
  TRY_ARG(rows == 0 || (logits && targets), "%s: NULL argument", fn);
  TRY_ARG(aligned(logits, esize(dtype)) && aligned(targets, 4), "%s: misaligned argument", fn);
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
  TRY_ARG(ldd >= V, "llmt_token_logprobs_bwd: ldd=%lld < V=%d", ldd, V);
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
  TRY_ARG(p && offsets && loss && stats && ((logp && advantages) || T == 0),
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

}  // extern "C"
