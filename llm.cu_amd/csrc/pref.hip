// pref.hip — losses on token log-probabilities, with their gradients: the
// preference loss of pairs of sequences and the clipped policy loss with a
// KL term.
//
// Both work on flat arrays over T tokens; sequence s is the tokens
// offsets[s] .. offsets[s + 1] - 1 (clamped to [0, T] and to one another, so
// malformed offsets read and write nothing outside the arrays).  A token of no
// sequence, or whose mask byte is 0, has no part in the loss and gets a
// gradient of 0, whatever the arrays hold there.
//
// The arithmetic a token takes is done in fp64: a sum over a sequence of
// thousands of differences, a ratio that is compared with the clip borders
// and exp(d) - d - 1 of a small d all lose what matters in fp32.  Small inputs
// are bound by memory round trips and launches: loads are issued before anything
// waits, four tokens a thread, and they take one launch.  Large ones move 1.4 to
// 1.6 TB/s in their first kernel, bound by each sequence's steps one after
// another and, in the policy loss, by the issue of its fp64 exp and expm1.
// Every sum has a fixed order.  Preference loss, 4 pairs of 417 tokens 5.8 us,
// 2048 pairs of 797 (14.7 MB) 12; policy loss, 8 x 139 tokens 6.8 us, 512 x 1025
// (15.2 MB) 12, in a graph.
#include <algorithm>

#include "../../include/llmt.h"
#include "ops.h"

namespace llmt {

namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int u1u __attribute__((aligned(1)));

// Sums over a wave without LDS (DPP rows, then lane swaps); every lane gets it.
template <int CTRL>
__device__ __forceinline__ double dpp16_d(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, 0xF, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double halves(unsigned lo, unsigned hi) {
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += dpp16_d<0xB1>(v);
  v += dpp16_d<0x4E>(v);
  v += dpp16_d<0x141>(v);
  v += dpp16_d<0x140>(v);
  unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  auto l = __builtin_amdgcn_permlane16_swap((unsigned)u, (unsigned)u, false, false);
  auto h = __builtin_amdgcn_permlane16_swap((unsigned)(u >> 32), (unsigned)(u >> 32), false, false);
  v = halves(l[0], h[0]) + halves(l[1], h[1]);
  u = __builtin_bit_cast(unsigned long long, v);
  l = __builtin_amdgcn_permlane32_swap((unsigned)u, (unsigned)u, false, false);
  h = __builtin_amdgcn_permlane32_swap((unsigned)(u >> 32), (unsigned)(u >> 32), false, false);
  return halves(l[0], h[0]) + halves(l[1], h[1]);
}
// Sums over a group of WAVES waves (1: no barrier; else the whole block);
// every thread gets them.
template <int WAVES, int NV>
__device__ __forceinline__ void group_sum(double (&v)[NV], double* red) {
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = wave_sum_d(v[i]);
  if constexpr (WAVES > 1) {
    __syncthreads();  // the last sum's readers are done with red
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < NV; ++i) red[(threadIdx.x >> 6) * NV + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      double t = 0.0;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) t += red[k * NV + i];
      v[i] = t;
    }
  }
}

// Four tokens of an array, `have` (<= 4) of them inside it.
__device__ __forceinline__ f4u load4(const float* p, long long t, int have) {
  if (have >= 4) return *reinterpret_cast<const f4u*>(p + t);
  f4u v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < have) v[e] = p[t + e];
  return v;
}
__device__ __forceinline__ void store4(float* p, long long t, f4u v, int have) {
  if (have >= 4) {
    *reinterpret_cast<f4u*>(p + t) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < have) p[t + e] = v[e];
}
// Bit e: token t + e exists and its mask byte is not 0.
__device__ __forceinline__ unsigned keep4(const unsigned char* mask, long long t, int have) {
  if (have <= 0) return 0;
  if (!mask) return have >= 4 ? 0xFu : (1u << have) - 1u;
  unsigned bits = 0;
  if (have >= 4) {
    const unsigned m = *reinterpret_cast<const u1u*>(mask + t);
#pragma unroll
    for (int e = 0; e < 4; ++e) bits |= (m >> (8 * e) & 0xFFu) ? 1u << e : 0u;
    return bits;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < have && mask[t + e]) bits |= 1u << e;
  return bits;
}

// Bytes of [b, e) of the mask that are not 0: a thread's share of a block of
// BLOCK threads, 16 at a time.
template <int BLOCK>
__device__ __forceinline__ int count_kept(const unsigned char* mask, long long b, long long e) {
  typedef unsigned int u4u __attribute__((ext_vector_type(4), aligned(1)));
  int n = 0;
  long long t = b + 16 * (int)threadIdx.x;
  for (; t + 16 <= e; t += 16 * BLOCK) {
    const u4u m = *reinterpret_cast<const u4u*>(mask + t);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // bit 7 of every byte that is not 0
      n += __popc((((m[i] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | m[i]) & 0x80808080u);
  }
  if (t < e)  // one thread has the last, shorter piece
    for (; t < e; ++t) n += mask[t] ? 1 : 0;
  return n;
}

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return min(max(v, lo), hi); }

// ------------------------------------------------------------------ preference loss

// WAVES waves a pair, whose two sequences are one stretch of tokens; BLOCK
// threads a workgroup.  A grid of one workgroup also writes the mean.
template <int WAVES, int BLOCK>
__global__ __launch_bounds__(BLOCK) void pref_kernel(const PrefArgs a) {
  constexpr int GROUP = 64 * WAVES, GROUPS = BLOCK / GROUP, STEP = 4 * GROUP;
  __shared__ double red[BLOCK / 64 * 4];
  const int id = threadIdx.x % GROUP;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / GROUP);
  double total = 0.0;
  for (int pair = blockIdx.x * GROUPS + group; pair < a.n; pair += gridDim.x * GROUPS) {
    const int b0 = clamped(a.offsets[2 * pair], 0, a.T);
    const int b1 = clamped(a.offsets[2 * pair + 1], b0, a.T);
    const int b2 = clamped(a.offsets[2 * pair + 2], b1, a.T);
    double v[4] = {0.0, 0.0, 0.0, 0.0};  // sum and count of the chosen, of the rejected
    unsigned keep0 = 0;                  // the first step's tokens, for the gradient
    for (long long t = (long long)b0 + 4 * id; t < b2; t += STEP) {
      const int have = (int)min((long long)b2 - t, 4ll);
      const f4u lp = load4(a.logp, t, have);
      f4u rf = {0.f, 0.f, 0.f, 0.f};
      if (a.ref) rf = load4(a.ref, t, have);
      const unsigned keep = keep4(a.mask, t, have);
      if (t < (long long)b0 + STEP) keep0 = keep;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (keep >> e & 1) {
          const int side = t + e < b1 ? 0 : 2;
          const double d = (double)lp[e] - (double)rf[e];
          v[0] += side ? 0.0 : d;
          v[2] += side ? d : 0.0;
          v[1] += side ? 0.0 : 1.0;
          v[3] += side ? 1.0 : 0.0;
        }
    }
    group_sum<WAVES>(v, red);
    const double wc = a.average ? 1.0 / fmax(v[1], 1.0) : 1.0;
    const double wr = a.average ? 1.0 / fmax(v[3], 1.0) : 1.0;
    const double rc = a.beta * (v[0] * wc), rr = a.beta * (v[2] * wr);
    const double z = rc - rr - a.margin, s = a.smooth;
    // dz = (1 - s) f'(z) - s f'(-z)
    double ez = 0.0, dz;
    if (a.kind == LLMT_PREF_SIGMOID) {
      ez = exp(-fabs(z));
      const double small = ez / (1.0 + ez), large = 1.0 / (1.0 + ez);  // sigma(-|z|), sigma(|z|)
      dz = z >= 0.0 ? s * large - (1.0 - s) * small : s * small - (1.0 - s) * large;
      if (s == 0.0) dz = z >= 0.0 ? -small : -large;
    } else if (a.kind == LLMT_PREF_HINGE) {
      dz = (s - 1.0) * (z < 1.0 ? 1.0 : 0.0) + s * (z > -1.0 ? 1.0 : 0.0);
    } else {
      dz = 2.0 * z - 1.0 + 2.0 * s;
    }
    if (z != z) dz = z;
    if (a.dlogp) {
      const double k = dz * a.beta / a.n;
      const float gc = (float)(k * wc), gr = (float)(-k * wr);
      for (long long t = (long long)b0 + 4 * id; t < b2; t += STEP) {
        const int have = (int)min((long long)b2 - t, 4ll);
        const unsigned keep = t < (long long)b0 + STEP ? keep0 : keep4(a.mask, t, have);
        f4u g;
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = keep >> e & 1 ? (t + e < b1 ? gc : gr) : 0.f;
        store4(a.dlogp, t, g, have);
      }
    }
    if (id == 0) {
      // f(z), f(-z)
      double fp, fm;
      if (a.kind == LLMT_PREF_SIGMOID) {
        const double l = log1p(ez);
        fp = fmax(-z, 0.0) + l;
        fm = fmax(z, 0.0) + l;
      } else if (a.kind == LLMT_PREF_HINGE) {
        fp = fmax(1.0 - z, 0.0);
        fm = fmax(1.0 + z, 0.0);
      } else {
        fp = (z - 0.5) * (z - 0.5);
        fm = (z + 0.5) * (z + 0.5);
      }
      double loss = s == 0.0 ? fp : (1.0 - s) * fp + s * fm;
      if (z != z) loss = z;
      a.losses[pair] = (float)loss;
      a.rewards[2 * pair] = (float)rc;
      a.rewards[2 * pair + 1] = (float)rr;
      total += loss;
    }
  }
  if (a.dlogp) {  // tokens before the first and behind the last sequence
    const int first = clamped(a.offsets[0], 0, a.T);
    const int last = clamped(a.offsets[2 * a.n], first, a.T);
    const long long step = (long long)gridDim.x * BLOCK;
    const long long at = (long long)blockIdx.x * BLOCK + threadIdx.x;
    for (long long t = at; t < first; t += step) a.dlogp[t] = 0.f;
    for (long long t = last + at; t < a.T; t += step) a.dlogp[t] = 0.f;
  }
  if (gridDim.x == 1) {
    double v[1] = {total};
    group_sum<BLOCK / 64>(v, red);
    if (threadIdx.x == 0) *a.mean = (float)(v[0] / a.n);
  }
}

constexpr int kMeanThreads = 256;
__global__ __launch_bounds__(kMeanThreads) void pref_mean_kernel(const float* losses, int n,
                                                                 float* mean) {
  __shared__ double red[kMeanThreads / 64];
  double v[1] = {0.0};
  for (long long i = 4 * threadIdx.x; i < n; i += 4 * kMeanThreads) {
    const f4u x = load4(losses, i, (int)min(n - i, 4ll));  // what is missing reads as 0
    v[0] += ((double)x[0] + (double)x[1]) + ((double)x[2] + (double)x[3]);
  }
  group_sum<kMeanThreads / 64>(v, red);
  if (threadIdx.x == 0) *mean = (float)(v[0] / n);
}

// ------------------------------------------------------------------ policy loss

// What four tokens need of the arrays, before the mask is looked at.
struct Quad {
  f4u lp, old, ref, adv, ent;
};
__device__ __forceinline__ Quad load_quad(const PolicyArgs& a, long long t, int have) {
  const f4u zero = {0.f, 0.f, 0.f, 0.f};
  Quad x;
  x.lp = load4(a.logp, t, have);
  x.old = a.old ? load4(a.old, t, have) : x.lp;
  x.ref = a.ref ? load4(a.ref, t, have) : zero;
  x.adv = a.adv_per_seq ? zero : load4(a.adv, t, have);
  x.ent = a.entropy ? load4(a.entropy, t, have) : zero;
  return x;
}

// Adds token e of the quad with weight w to the sums (loss, policy term, KL,
// clipped); returns the gradient by its log-probability.  Exponents end at 700:
// exp of it is 1e304, beyond fp32 times any number but 0, and 0 times 0 (exp's
// infinity times 0 is NaN).  A NaN stays NaN in the loss.  The guards cost six
// instructions a token, within the noise of every size; as selects on the results
// they were 2 to 7% of the call, which these kernels' issue rate bounds.
__device__ __forceinline__ float policy_token(const PolicyArgs& a, const Quad& x, int e,
                                              double adv, double w, double (&v)[4]) {
  // -inf less itself is 0: without an old policy the ratio is 1 there too
  const float lp = __builtin_elementwise_maximum(x.lp[e], -__FLT_MAX__);
  const float old = __builtin_elementwise_maximum(x.old[e], lp - 700.f);
  const double ratio = exp((double)lp - (double)old);
  const double lo = 1.0 - a.clip_low, hi = 1.0 + a.clip_high;
  const double s1 = ratio * adv, s2 = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv;
  const bool clip = s1 > s2;
  const double pg = -(clip ? s2 : s1);
  double grad = clip ? 0.0 : -s1, loss = pg, kl = 0.0;
  if (a.ref) {
    const double d = (double)x.ref[e] - (double)lp, em = expm1(fmin(d, 700.0));
    kl = em - d;
    // with a coefficient of 0 an infinite KL (d = -inf) is only reported
    loss += a.kl_coef * (a.kl_coef != 0.0 ? kl : em);
    grad -= a.kl_coef * em;
  }
  if (a.entropy) loss -= a.ent_coef * (double)x.ent[e];
  v[0] += loss * w;
  v[1] += pg * w;
  v[2] += kl * w;
  v[3] += clip ? w : 0.0;
  return (float)(grad * w);
}

// The last s in [0, n) with offsets[s] <= t (in LDS or in memory).
template <typename P>
__device__ __forceinline__ int seq_of(P offsets, int n, int t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (offsets[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void write_result(const PolicyArgs& a, const double (&v)[4]) {
  *a.loss = (float)v[0];
  for (int k = 0; k < 3; ++k) a.stats[k] = (float)v[k + 1];
}

// Few tokens: one workgroup, offsets, advantages and counts of the sequences in LDS.
constexpr int kOneTh = 1024, kOneQuads = 2, kOneTokens = 4 * kOneQuads * kOneTh, kOneSeqs = 2048;
__global__ __launch_bounds__(kOneTh) void policy_one_kernel(const PolicyArgs a) {
  __shared__ int off[kOneSeqs + 1], cnt[kOneSeqs];
  __shared__ float adv[kOneSeqs];
  __shared__ double red[kOneTh / 64 * 4];
  Quad x[kOneQuads];
  unsigned keep[kOneQuads];
  int seq[kOneQuads];
#pragma unroll
  for (int i = 0; i < kOneQuads; ++i) {
    const int t = 4 * (kOneTh * i + (int)threadIdx.x), have = min(a.T - t, 4);
    keep[i] = 0;
    if (have > 0) {
      x[i] = load_quad(a, t, have);
      keep[i] = keep4(a.mask, t, have);
    }
  }
  for (int s = threadIdx.x; s <= a.n; s += kOneTh) off[s] = a.offsets[s];
  for (int s = threadIdx.x; s < a.n; s += kOneTh) {
    cnt[s] = 0;
    if (a.adv_per_seq) adv[s] = a.adv[s];
  }
  __syncthreads();
  const int first = clamped(off[0], 0, a.T), last = clamped(off[a.n], first, a.T);
  const bool need_seq = a.seq_mean || a.adv_per_seq;
  int kept = 0;
#pragma unroll
  for (int i = 0; i < kOneQuads; ++i) {
    const int t = 4 * (kOneTh * i + (int)threadIdx.x);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t + e < first || t + e >= last) keep[i] &= ~(1u << e);
    kept += __popc(keep[i]);
    seq[i] = 0;
    if (need_seq && keep[i]) {
      int s = seq[i] = seq_of(off, a.n, t + __ffs(keep[i]) - 1);
      if (a.seq_mean)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (keep[i] >> e & 1) {
            while (s + 1 < a.n && off[s + 1] <= t + e) ++s;
            atomicAdd(&cnt[s], 1);
          }
    }
  }
  double inv = 0.0;
  if (a.seq_mean) {
    __syncthreads();
  } else {
    double c[1] = {(double)kept};
    group_sum<kOneTh / 64>(c, red);
    inv = 1.0 / fmax(c[0], 1.0);
  }
  double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < kOneQuads; ++i) {
    const int t = 4 * (kOneTh * i + (int)threadIdx.x), have = min(a.T - t, 4);
    if (have <= 0) break;
    f4u g = {0.f, 0.f, 0.f, 0.f}, ge = {0.f, 0.f, 0.f, 0.f};
    int s = seq[i];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (keep[i] >> e & 1) {
        if (need_seq)
          while (s + 1 < a.n && off[s + 1] <= t + e) ++s;
        const double w = a.seq_mean ? 1.0 / ((double)cnt[s] * a.n) : inv;
        g[e] = policy_token(a, x[i], e, a.adv_per_seq ? adv[s] : x[i].adv[e], w, v);
        ge[e] = (float)(-a.ent_coef * w);
      }
    if (a.dlogp) store4(a.dlogp, t, g, have);
    if (a.dentropy) store4(a.dentropy, t, ge, have);
  }
  group_sum<kOneTh / 64>(v, red);
  if (threadIdx.x == 0) write_result(a, v);
}

constexpr int NTH = 256;
constexpr int kTile = 4 * NTH;  // tokens a workgroup
constexpr int kCountWg = 256;   // workgroups that count the kept tokens

// Kept tokens of all sequences, counted in kCountWg equal parts.
__global__ __launch_bounds__(NTH) void policy_count_kernel(const PolicyArgs a) {
  __shared__ double red[NTH / 64];
  const int first = clamped(a.offsets[0], 0, a.T), last = clamped(a.offsets[a.n], first, a.T);
  const long long per = ((long long)last - first + kCountWg - 1) / kCountWg;
  const long long b = first + per * blockIdx.x, e = min(b + per, (long long)last);
  double v[1] = {(double)count_kept<NTH>(a.mask, b, e)};
  group_sum<NTH / 64>(v, red);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = (int)v[0];
}

// The mean over the tokens: a tile of the tokens a workgroup, its sums to
// parts[4 * blockIdx.x].  Of up to kCountHere tokens every workgroup counts the
// kept ones by itself, the mask's 64 KB at most read from the caches, which costs
// no more than the launch it saves (both ways, in a graph: 16 x 522 tokens 8.5
// and 10.3 us, 64 x 400 10.2 and 10.9, 100 x 576 10.6 and 10.6, 200 x 570 13.8
// and 11.7).
constexpr int kCountHere = 65536;
constexpr int kLdsSeqs = 4096;
__global__ __launch_bounds__(NTH) void policy_kernel(const PolicyArgs a) {
  __shared__ double red[NTH / 64 * 4];
  __shared__ int off[kLdsSeqs];
  const long long t = (long long)blockIdx.x * kTile + 4 * threadIdx.x;
  const int have = (int)min(max((long long)a.T - t, 0ll), 4ll);
  Quad x;
  unsigned keep = 0;
  if (have > 0) {
    x = load_quad(a, t, have);
    keep = keep4(a.mask, t, have);
  }
  const int first = clamped(a.offsets[0], 0, a.T), last = clamped(a.offsets[a.n], first, a.T);
  const bool lds = a.adv_per_seq && a.n <= kLdsSeqs;
  if (lds)
    for (int s = threadIdx.x; s < a.n; s += NTH) off[s] = a.offsets[s];
  double c[1] = {0.0};
  if (a.mask) {
    if (a.T <= kCountHere) c[0] = count_kept<NTH>(a.mask, first, last);
    else c[0] = threadIdx.x < kCountWg ? a.counts[threadIdx.x] : 0;
    group_sum<NTH / 64>(c, red);  // (its barriers also publish off)
  } else {
    c[0] = last - first;
    if (lds) __syncthreads();
  }
  const double w = 1.0 / fmax(c[0], 1.0);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (t + e < first || t + e >= last) keep &= ~(1u << e);
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  if (have > 0) {
    f4u g = {0.f, 0.f, 0.f, 0.f}, ge = {0.f, 0.f, 0.f, 0.f};
    int s = 0;
    if (a.adv_per_seq && keep) {
      const int from = (int)t + __ffs(keep) - 1;
      s = lds ? seq_of(off, a.n, from) : seq_of(a.offsets, a.n, from);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (keep >> e & 1) {
        if (a.adv_per_seq)
          while (s + 1 < a.n && (lds ? off[s + 1] : a.offsets[s + 1]) <= t + e) ++s;
        g[e] = policy_token(a, x, e, a.adv_per_seq ? a.adv[s] : x.adv[e], w, v);
        ge[e] = (float)(-a.ent_coef * w);
      }
    if (a.dlogp) store4(a.dlogp, t, g, have);
    if (a.dentropy) store4(a.dentropy, t, ge, have);
  }
  group_sum<NTH / 64>(v, red);
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) a.parts[4ll * blockIdx.x + i] = v[i];
}

// The mean over the sequences: WAVES waves a sequence; a workgroup's sums to
// parts[4 * blockIdx.x].
template <int WAVES>
__global__ __launch_bounds__(NTH) void policy_seq_kernel(const PolicyArgs a) {
  constexpr int GROUP = 64 * WAVES, GROUPS = NTH / GROUP, STEP = 4 * GROUP;
  __shared__ double red[NTH / 64 * 4];
  const int id = threadIdx.x % GROUP;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / GROUP);
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int s = blockIdx.x * GROUPS + group; s < a.n; s += gridDim.x * GROUPS) {
    const int b = clamped(a.offsets[s], 0, a.T), end = clamped(a.offsets[s + 1], b, a.T);
    const long long t0 = (long long)b + 4 * id;
    const int have0 = (int)min(max((long long)end - t0, 0ll), 4ll);
    // the first step's tokens are on their way while the kept ones are counted
    Quad x;
    if (have0 > 0) x = load_quad(a, t0, have0);
    const unsigned keep0 = keep4(a.mask, t0, have0);
    const double adv = a.adv_per_seq ? a.adv[s] : 0.f;
    double c[1] = {(double)__popc(keep0)};
    if (a.mask) {
      for (long long t = t0 + STEP; t < end; t += STEP)
        c[0] += __popc(keep4(a.mask, t, (int)min((long long)end - t, 4ll)));
      group_sum<WAVES>(c, red);
    } else {
      c[0] = end - b;
    }
    const double w = 1.0 / (fmax(c[0], 1.0) * a.n);
    for (long long t = t0; t < end; t += STEP) {
      const int have = (int)min((long long)end - t, 4ll);
      unsigned keep = keep0;
      if (t != t0) {
        x = load_quad(a, t, have);
        keep = keep4(a.mask, t, have);
      }
      f4u g = {0.f, 0.f, 0.f, 0.f}, ge = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (keep >> e & 1) {
          g[e] = policy_token(a, x, e, a.adv_per_seq ? adv : x.adv[e], w, v);
          ge[e] = (float)(-a.ent_coef * w);
        }
      if (a.dlogp) store4(a.dlogp, t, g, have);
      if (a.dentropy) store4(a.dentropy, t, ge, have);
    }
  }
  if (a.dlogp || a.dentropy) {  // tokens of no sequence
    const int first = clamped(a.offsets[0], 0, a.T), last = clamped(a.offsets[a.n], first, a.T);
    const long long step = (long long)gridDim.x * NTH;
    const long long at = (long long)blockIdx.x * NTH + threadIdx.x;
    auto clear = [&](long long b, long long e) {
      for (long long t = b + at; t < e; t += step) {
        if (a.dlogp) a.dlogp[t] = 0.f;
        if (a.dentropy) a.dentropy[t] = 0.f;
      }
    };
    clear(0, first);
    clear(last, a.T);
  }
  group_sum<NTH / 64>(v, red);
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) a.parts[4ll * blockIdx.x + i] = v[i];
}

__global__ __launch_bounds__(NTH) void policy_final_kernel(const PolicyArgs a, int n) {
  __shared__ double red[NTH / 64 * 4];
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += NTH)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += a.parts[4ll * i + k];
  group_sum<NTH / 64>(v, red);
  if (threadIdx.x == 0) write_result(a, v);
}

// Workgroups whose partial sums the final kernel adds: tiles of the tokens, or
// groups of sequences.
constexpr int kSeqWg = 2048;  // eight workgroups a CU
bool one_workgroup(int T, int n) { return T <= kOneTokens && n <= kOneSeqs; }
// A wave takes a sequence where it is one step of it (256 tokens on average:
// 2000 x 57 8.4 us, 17 with a workgroup each), or two and the sequences are
// more than the workgroups that the registers let run at once (2000 x 228:
// 11.5 and 17.9; 500 x 228: 9.5 and 8.5).
constexpr int kSeqResident = 768;
bool wave_a_sequence(int T, int n) { return T / n <= (n > kSeqResident ? 512 : 256); }
int policy_grid(int T, int n, int seq_mean) {
  if (!seq_mean) return (int)(((long long)T + kTile - 1) / kTile);
  const int per = wave_a_sequence(T, n) ? NTH / 64 : 1;
  return std::min((n + per - 1) / per, kSeqWg);
}
size_t counts_bytes() { return kCountWg * sizeof(int); }

}  // namespace

// Few and short pairs: one workgroup, a wave a pair, no second launch, which
// costs the caller 3 us (8 x 24 tokens 5.8 us, 6.3 in two; 16 x 345: 9.0 and
// 6.4; 16 x 919 would be 12.9 and 7.3).  Else a workgroup a pair while all can
// run at once (500 x 342: 6.9 us, 8.0 with a wave each), a wave a pair beyond
// (2048 x 342: 9.4, 12.0 with a workgroup each; 2048 x 797: 12.2 and 14.1), and
// twice the threads for long ones (100 x 2279: 7.8 and 9.2).
hipError_t preference_loss(const PrefArgs& a, hipStream_t st) {
  constexpr int kResident = 1024;
  const int len = a.T / a.n;  // tokens a pair on average
  auto go = [&](auto waves, auto block, int wgs) {
    constexpr int W = decltype(waves)::value, B = decltype(block)::value;
    const int grid = std::min(wgs, 1 << 16);
    hipLaunchKernelGGL((pref_kernel<W, B>), dim3(grid), dim3(B), 0, st, a);
    return grid;
  };
  using std::integral_constant;
  const int grid = a.n <= 16 && len <= 512
                       ? go(integral_constant<int, 1>(), integral_constant<int, 1024>(), 1)
                   : a.n > kResident && len <= 1024
                       ? go(integral_constant<int, 1>(), integral_constant<int, 256>(), (a.n + 3) / 4)
                   : len <= 2048
                       ? go(integral_constant<int, 4>(), integral_constant<int, 256>(), a.n)
                       : go(integral_constant<int, 8>(), integral_constant<int, 512>(), a.n);
  LLMT_LAUNCH_CHECK();
  if (grid > 1) {
    hipLaunchKernelGGL(pref_mean_kernel, dim3(1), dim3(kMeanThreads), 0, st, a.losses, a.n, a.mean);
    LLMT_LAUNCH_CHECK();
  }
  return hipSuccess;
}

// Kept-token counts, then four partial sums a workgroup (the larger of the two
// means' grids, whichever the call takes).
size_t policy_workspace(int T, int n) {
  if (one_workgroup(T, n)) return 0;
  return counts_bytes() +
         (size_t)std::max(policy_grid(T, n, 0), policy_grid(T, n, 1)) * 4 * sizeof(double);
}

hipError_t policy_loss(PolicyArgs a, void* workspace, hipStream_t st) {
  if (one_workgroup(a.T, a.n)) {
    hipLaunchKernelGGL(policy_one_kernel, dim3(1), dim3(kOneTh), 0, st, a);
    LLMT_LAUNCH_CHECK();
    return hipSuccess;
  }
  a.counts = (int*)workspace;
  a.parts = (double*)((char*)workspace + counts_bytes());
  const int grid = policy_grid(a.T, a.n, a.seq_mean);
  if (a.seq_mean) {
    if (wave_a_sequence(a.T, a.n))
      hipLaunchKernelGGL(policy_seq_kernel<1>, dim3(grid), dim3(NTH), 0, st, a);
    else
      hipLaunchKernelGGL(policy_seq_kernel<4>, dim3(grid), dim3(NTH), 0, st, a);
    LLMT_LAUNCH_CHECK();
  } else if (grid) {
    if (a.mask && a.T > kCountHere) {
      hipLaunchKernelGGL(policy_count_kernel, dim3(kCountWg), dim3(NTH), 0, st, a);
      LLMT_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(policy_kernel, dim3(grid), dim3(NTH), 0, st, a);
    LLMT_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(policy_final_kernel, dim3(1), dim3(NTH), 0, st, a, grid);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

}  // namespace llmt
