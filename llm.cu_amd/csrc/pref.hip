// pref.hip — losses on token log-probabilities, with their gradients: the
// preference loss of pairs of sequences and the clipped policy loss with a
// KL term.
//
// Both work on flat arrays over T tokens; sequence s is the tokens
// offsets[s] .. offsets[s + 1] - 1 (clamped to [0, T], so malformed offsets
// read and write nothing outside the arrays).  A token of no sequence, or
// whose mask byte is 0, has no part in the loss, is not read and gets a
// gradient of 0.
//
// The arithmetic a token takes is done in fp64: a sum over a sequence of
// thousands of differences, a ratio that is compared with the clip borders
// and exp(d) - d - 1 of a small d all lose what matters in fp32, and at 12 to
// 25 bytes a token the kernels stay bound by their loads and launches.  Every
// sum has a fixed order.
#include <algorithm>

#include "../../include/llmt.h"
#include "ops.h"

namespace llmt {

namespace {

constexpr int NTH = 256;

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Sum over the block's waves; every thread gets it.  Contains barriers.
template <int NV>
__device__ __forceinline__ void block_sum_d(double (&v)[NV], double* red) {
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = wave_sum_d(v[i]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < NV; ++i) red[w * NV + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    double t = 0.0;
    for (int k = 0; k < nw; ++k) t += red[k * NV + i];
    v[i] = t;
  }
  __syncthreads();
}

struct Span {
  int b, e;
};
__device__ __forceinline__ Span span(const int* offsets, int s, int T) {
  const int b = min(max(offsets[s], 0), T);
  return {b, min(max(offsets[s + 1], b), T)};
}

// ------------------------------------------------------------------ preference loss

// f(z) and f'(z): softplus(-z), max(0, 1 - z) or (z - 1/2)^2.
__device__ __forceinline__ void pref_f(int kind, double z, double& f, double& df) {
  if (kind == LLMT_PREF_SIGMOID) {
    const double e = exp(-fabs(z));
    f = fmax(-z, 0.0) + log1p(e);
    df = -(z >= 0.0 ? e : 1.0) / (1.0 + e);
  } else if (kind == LLMT_PREF_HINGE) {
    f = fmax(1.0 - z, 0.0);
    df = z < 1.0 ? -1.0 : 0.0;
  } else {
    f = (z - 0.5) * (z - 0.5);
    df = 2.0 * z - 1.0;
  }
  if (z != z) f = df = z;
}

__global__ __launch_bounds__(NTH) void pref_kernel(const PrefArgs a) {
  __shared__ double red[NTH / 64 * 4];
  if (a.dlogp) {  // tokens before the first and behind the last sequence
    const int first = min(max(a.offsets[0], 0), a.T);
    const int last = min(max(a.offsets[2 * a.n], first), a.T);
    const long long step = (long long)gridDim.x * NTH;
    const long long id = (long long)blockIdx.x * NTH + threadIdx.x;
    for (long long t = id; t < first; t += step) a.dlogp[t] = 0.f;
    for (long long t = last + id; t < a.T; t += step) a.dlogp[t] = 0.f;
  }
  for (int pair = blockIdx.x; pair < a.n; pair += gridDim.x) {
    double v[4] = {0.0, 0.0, 0.0, 0.0};  // sum and count of the chosen, of the rejected
    Span sp[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sp[c] = span(a.offsets, 2 * pair + c, a.T);
      for (int t = sp[c].b + threadIdx.x; t < sp[c].e; t += NTH)
        if (!a.mask || a.mask[t]) {
          v[2 * c] += (double)a.logp[t] - (a.ref ? (double)a.ref[t] : 0.0);
          v[2 * c + 1] += 1.0;
        }
    }
    block_sum_d(v, red);
    const double wc = a.average ? 1.0 / fmax(v[1], 1.0) : 1.0;
    const double wr = a.average ? 1.0 / fmax(v[3], 1.0) : 1.0;
    const double rc = a.beta * (v[0] * wc), rr = a.beta * (v[2] * wr);
    const double z = rc - rr - a.margin;
    double fp, dp, fm, dm;
    pref_f(a.kind, z, fp, dp);
    pref_f(a.kind, -z, fm, dm);
    const double sm = a.smooth;
    const double loss = sm == 0.0 ? fp : (1.0 - sm) * fp + sm * fm;
    const double dz = sm == 0.0 ? dp : (1.0 - sm) * dp - sm * dm;
    if (threadIdx.x == 0) {
      a.losses[pair] = (float)loss;
      a.rewards[2 * pair] = (float)rc;
      a.rewards[2 * pair + 1] = (float)rr;
    }
    if (a.dlogp) {
      const double k = dz * a.beta / a.n;
      const float gc = (float)(k * wc), gr = (float)(-k * wr);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        for (int t = sp[c].b + threadIdx.x; t < sp[c].e; t += NTH)
          a.dlogp[t] = !a.mask || a.mask[t] ? (c ? gr : gc) : 0.f;
    }
  }
}

__global__ __launch_bounds__(1024) void pref_mean_kernel(const float* losses, int n, float* mean) {
  __shared__ double red[16];
  double v[1] = {0.0};
  for (int i = threadIdx.x; i < n; i += 1024) v[0] += (double)losses[i];
  block_sum_d(v, red);
  if (threadIdx.x == 0) *mean = (float)(v[0] / n);
}

// ------------------------------------------------------------------ policy loss

constexpr int kTile = 1024;    // tokens a workgroup of the main kernel
constexpr int kCountWg = 256;  // workgroups that count the kept tokens

// The sequence of token t: the last s with offsets[s] <= t, in [0, n).
__device__ __forceinline__ int seq_of(const int* offsets, int n, int t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (offsets[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ Span all_tokens(const PolicyArgs& a) {
  const int b = min(max(a.offsets[0], 0), a.T);
  return {b, min(max(a.offsets[a.n], b), a.T)};
}

// Kept tokens: of every sequence (counts[n], per_seq), or of kCountWg equal
// parts of all tokens (counts[kCountWg]).
__global__ __launch_bounds__(NTH) void policy_count_kernel(const PolicyArgs a, int per_seq) {
  __shared__ double red[NTH / 64];
  auto count = [&](Span s, int at) {
    double v[1] = {0.0};
    for (int t = s.b + threadIdx.x; t < s.e; t += NTH) v[0] += a.mask[t] ? 1.0 : 0.0;
    block_sum_d(v, red);
    if (threadIdx.x == 0) a.counts[at] = (int)v[0];
  };
  if (per_seq) {
    for (int s = blockIdx.x; s < a.n; s += gridDim.x) count(span(a.offsets, s, a.T), s);
  } else {
    const Span all = all_tokens(a);
    const int per = (int)(((long long)(all.e - all.b) + kCountWg - 1) / kCountWg);
    const int b = (int)min((long long)all.b + (long long)per * blockIdx.x, (long long)all.e);
    count({b, (int)min((long long)b + per, (long long)all.e)}, blockIdx.x);
  }
}

// One token: its terms and its derivative, not yet weighted.
struct Term {
  double pg, kl, clipped, loss, grad;
};
__device__ __forceinline__ Term policy_term(const PolicyArgs& a, double lp, double old, double ref,
                                            double adv, double ent) {
  Term r;
  const double ratio = exp(lp - old);
  const double lo = 1.0 - a.clip_low, hi = 1.0 + a.clip_high;
  const double s1 = ratio * adv, s2 = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv;
  const bool clip = s1 > s2;
  r.pg = -(clip ? s2 : s1);
  r.clipped = clip ? 1.0 : 0.0;
  r.grad = clip ? 0.0 : -s1;
  r.loss = r.pg;
  r.kl = 0.0;
  if (a.ref) {
    const double d = ref - lp, em = expm1(d);
    r.kl = em - d;
    r.loss += a.kl_coef * r.kl;
    r.grad -= a.kl_coef * em;
  }
  if (a.entropy) r.loss -= a.ent_coef * ent;
  return r;
}

// kTile tokens a workgroup; partial sums (loss, policy term, KL, clipped) of
// its tokens to parts[4 * blockIdx.x].
__global__ __launch_bounds__(NTH) void policy_kernel(const PolicyArgs a) {
  __shared__ double red[NTH / 64 * 4];
  const Span all = all_tokens(a);
  double inv = 0.0;
  if (!a.seq_mean) {
    double c[1] = {0.0};
    if (a.mask) {
      for (int i = threadIdx.x; i < kCountWg; i += NTH) c[0] += a.counts[i];
      block_sum_d(c, red);
    } else {
      c[0] = all.e - all.b;
    }
    inv = 1.0 / fmax(c[0], 1.0);
  }
  const bool need_seq = a.seq_mean || a.adv_per_seq;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  const long long t0 = (long long)blockIdx.x * kTile;
  for (long long i = threadIdx.x; i < kTile; i += NTH) {
    const long long tl = t0 + i;
    if (tl >= a.T) break;
    const int t = (int)tl;
    if (t < all.b || t >= all.e || (a.mask && !a.mask[t])) {
      if (a.dlogp) a.dlogp[t] = 0.f;
      if (a.dentropy) a.dentropy[t] = 0.f;
      continue;
    }
    const int s = need_seq ? seq_of(a.offsets, a.n, t) : 0;
    double w = inv;
    if (a.seq_mean) {
      int kept;
      if (a.mask) {
        kept = a.counts[s];
      } else {
        const Span sp = span(a.offsets, s, a.T);
        kept = sp.e - sp.b;
      }
      w = 1.0 / ((double)max(kept, 1) * a.n);
    }
    const double lp = a.logp[t];
    const Term r = policy_term(a, lp, a.old ? (double)a.old[t] : lp, a.ref ? a.ref[t] : 0.0,
                               a.adv[a.adv_per_seq ? s : t], a.entropy ? a.entropy[t] : 0.0);
    if (a.dlogp) a.dlogp[t] = (float)(r.grad * w);
    if (a.dentropy) a.dentropy[t] = (float)(-a.ent_coef * w);
    v[0] += r.loss * w;
    v[1] += r.pg * w;
    v[2] += r.kl * w;
    v[3] += r.clipped * w;
  }
  block_sum_d(v, red);
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) a.parts[4ll * blockIdx.x + i] = v[i];
}

__global__ __launch_bounds__(1024) void policy_final_kernel(const double* parts, int n, float* loss,
                                                            float* stats) {
  __shared__ double red[16 * 4];
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += 1024)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += parts[4ll * i + k];
  block_sum_d(v, red);
  if (threadIdx.x == 0) {
    *loss = (float)v[0];
    for (int k = 0; k < 3; ++k) stats[k] = (float)v[k + 1];
  }
}

int policy_tiles(int T) { return (int)(((long long)T + kTile - 1) / kTile); }

}  // namespace

hipError_t preference_loss(const PrefArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(pref_kernel, dim3(std::min(a.n, 1 << 20)), dim3(NTH), 0, st, a);
  LLMT_LAUNCH_CHECK();
  hipLaunchKernelGGL(pref_mean_kernel, dim3(1), dim3(1024), 0, st, a.losses, a.n, a.mean);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

// Kept-token counts (int, 16-byte rounded), then four partial sums a tile.
size_t policy_workspace(int T, int n) {
  const size_t counts = ((size_t)std::max(n, kCountWg) * 4 + 15) & ~(size_t)15;
  return counts + (size_t)policy_tiles(T) * 4 * sizeof(double);
}

hipError_t policy_loss(PolicyArgs a, void* workspace, hipStream_t st) {
  a.counts = (int*)workspace;
  a.parts = (double*)((char*)workspace + (((size_t)std::max(a.n, kCountWg) * 4 + 15) & ~(size_t)15));
  const int tiles = policy_tiles(a.T);
  if (a.mask) {
    hipLaunchKernelGGL(policy_count_kernel,
                       dim3(a.seq_mean ? std::min(a.n, 1 << 20) : kCountWg), dim3(NTH), 0, st, a,
                       a.seq_mean);
    LLMT_LAUNCH_CHECK();
  }
  if (tiles) {
    hipLaunchKernelGGL(policy_kernel, dim3(tiles), dim3(NTH), 0, st, a);
    LLMT_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(policy_final_kernel, dim3(1), dim3(1024), 0, st, a.parts, tiles, a.loss,
                     a.stats);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

}  // namespace llmt
