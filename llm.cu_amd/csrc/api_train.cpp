// api_train.cpp — C ABI of the operators for training all weights on packed
// sequences: packed attention, embedding, AdamW over a list of tensors.  Every
// entry point validates its arguments on the host before any launch and
// allocates nothing on the device.
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

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
static bool known(int dtype) { return dtype == LLMT_F32 || dtype == LLMT_F16 || dtype == LLMT_BF16; }
static size_t esize(int dtype) { return dtype == LLMT_F32 ? 4 : 2; }

constexpr int kMost = 1 << 30;  // tokens, rows of a group's heads, a vocabulary
constexpr int kMaxTokens = 1 << 23, kMaxWidth = 1 << 20;  // of an embedding: its grids
constexpr long long kMaxStride = 1ll << 40, kMaxElements = 1ll << 35;

// ---------------------------------------------------------------- packed attention

static bool dims_ok(const llmt_packed_dims* d) {
  if (!d || (d->dtype != LLMT_F16 && d->dtype != LLMT_BF16)) return false;
  if (d->head_dim != 64 && d->head_dim != 128) return false;
  if (d->nkv < 1 || d->nq < d->nkv || d->nq % d->nkv || d->nq > 4096 ||
      d->nq / d->nkv > 64)
    return false;
  if (d->n < 1 || d->n > (1 << 24) || d->Tq < 0 || d->Tk < 0 || d->Tk > kMost) return false;
  const long long rows = (long long)d->Tq * (d->nq / d->nkv);
  // A launch has less than 2^24 workgroups: one each 64 rows and each 64 keys, and
  // two a sequence, for each KV head, and up to 2^13 more where rows or keys are so
  // few that their blocks are smaller.
  return rows <= kMost &&
         (std::max<long long>(rows, d->Tk) / 64 + d->n + 2) * d->nkv * 2 < (1 << 24) - (1 << 13) &&
         (long long)d->Tq * d->nq <= 0x7fffffff;
}

struct View {
  const char* name;
  const llmt_heads* h;
  int T, heads;
  bool query, written;
};

static int check_view(const char* fn, const llmt_packed_dims* d, const View& x) {
  TRY_ARG(x.h, "%s: NULL %s", fn, x.name);
  if (x.T == 0) return LLMT_OK;
  const long long t = x.h->token, h = x.h->head, hd = d->head_dim;
  TRY_ARG(x.h->p && aligned(x.h->p, 16), "%s: %s must be given, 16-byte aligned", fn, x.name);
  TRY_ARG(t % 8 == 0 && h % 8 == 0 && t >= hd && t <= (1 << 23) && h >= 0 && h <= kMaxStride,
          "%s: %s has strides %lld (token) and %lld (head): multiples of 8, token in [%lld, 2^23]",
          fn, x.name, t, h, hd);
  const long long g = d->nq / d->nkv;
  TRY_ARG(!x.query || (g - 1) * h <= (1 << 28), "%s: %s has a head stride of %lld over %lld heads",
          fn, x.name, h, g);
  TRY_ARG(!x.written || x.heads == 1 || (h >= hd && t >= (x.heads - 1) * h + hd) ||
              h >= (x.T - 1) * t + hd,
          "%s: %s overlaps itself (strides %lld, %lld)", fn, x.name, t, h);
  return LLMT_OK;
}

// Pieces of `piece` bytes, n of them `stride` apart.
struct Comb {
  long long n, stride;
  long long width(long long piece) const { return (n - 1) * stride + piece; }
};
// Whether combs that begin at 0 and at `at` have no byte in common: one behind the
// other, or of one stride with pieces of the one between those of the other.
static bool combs_apart(const Comb& a, const Comb& b, long long at, long long piece) {
  if (at >= a.width(piece) || at + b.width(piece) <= 0) return true;
  const long long s = a.n == 1 ? b.stride : a.stride;
  if ((b.n > 1 && b.stride != s) || (a.n == 1 && b.n == 1) || s <= 0) return false;
  const long long d = ((at % s) + s) % s;
  return d >= piece && d + piece <= s;
}

// Whether two views have no element in common: apart from one another; or of the
// same stride from token to token (from head to head), with each token's heads
// (each head's tokens) inside one such stride and apart from the other view's
// there.  Other layouts may be apart as well: they are refused.
static bool views_apart(const View& a, const View& b, int hd) {
  if (a.T == 0 || b.T == 0) return true;
  const long long piece = hd * 2;
  const Comb ta = {a.T, a.h->token * 2}, ha = {a.heads, a.h->head * 2};
  const Comb tb = {b.T, b.h->token * 2}, hb = {b.heads, b.h->head * 2};
  const long long at = (intptr_t)b.h->p - (intptr_t)a.h->p;
  if (at >= ta.width(ha.width(piece)) || at + tb.width(hb.width(piece)) <= 0) return true;
  auto nested = [&](const Comb& oa, const Comb& ia, const Comb& ob, const Comb& ib) {
    if (oa.n == 1 && ob.n == 1) return combs_apart(ia, ib, at, piece);
    const long long s = oa.n == 1 ? ob.stride : oa.stride;
    if ((ob.n > 1 && ob.stride != s) || ia.width(piece) > s || ib.width(piece) > s) return false;
    // the row of b that begins in a's row at 0 ends in a's next one at the latest
    const long long d = ((at % s) + s) % s;
    return combs_apart(ia, ib, d, piece) && combs_apart(ia, ib, d - s, piece);
  };
  return nested(ta, ha, tb, hb) || nested(ha, ta, hb, tb);
}

static int check_packed(const char* fn, const llmt_packed_dims* d, const View* v, int nv,
                        const float* lse) {
  TRY_ARG(dims_ok(d), "%s: dtype f16 or bf16, head_dim 64 or 128, nq one to 64 times nkv, n in "
          "[1, 2^24], at most 2^24 workgroups", fn);
  TRY_ARG(d->scale > 0.f && isfinite(d->scale), "%s: scale must be positive and finite", fn);
  TRY_ARG(d->q_offsets && d->k_offsets && aligned(d->q_offsets, 4) && aligned(d->k_offsets, 4),
          "%s: offsets must be given, 4-byte aligned", fn);
  for (int i = 0; i < nv; ++i) {
    const int rc = check_view(fn, d, v[i]);
    if (rc) return rc;
  }
  TRY_ARG(d->Tq == 0 || (lse && aligned(lse, 4)), "%s: lse must be given, 4-byte aligned", fn);
  for (int i = 0; i < nv; ++i)
    for (int k = 0; k < nv; ++k)
      TRY_ARG(i == k || !v[i].written || views_apart(v[i], v[k], d->head_dim), "%s: %s overlaps %s",
              fn, v[i].name, v[k].name);
  return LLMT_OK;
}

static Heads heads(const llmt_heads* h) { return {h->p, h->token, h->head}; }

static PackArgs pack_args(const llmt_packed_dims* d) {
  PackArgs a{};
  a.qoff = d->q_offsets;
  a.koff = d->k_offsets;
  a.n = d->n;
  a.Tq = d->Tq;
  a.Tk = d->Tk;
  a.nq = d->nq;
  a.nkv = d->nkv;
  a.hd = d->head_dim;
  a.bf16 = d->dtype == LLMT_BF16;
  a.scale = d->scale;
  return a;
}

static int check_space(const char* fn, size_t need, const void* ws, size_t bytes) {
  TRY_ARG(need == 0 || (ws && bytes >= need && aligned(ws, 16)),
          "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", fn, ws ? bytes : 0, need);
  return LLMT_OK;
}

// ---------------------------------------------------------------- AdamW

// Whether no written array of the list meets another array of it (gradients may
// meet one another).  Lists in the order of one arena a kind, the usual case,
// are seen to be apart in one pass; others are sorted.
struct Extent {
  uintptr_t a, b;
  bool written;
};
constexpr int kKinds = 7;  // p, m, v, copy, the two exponents; the gradient last
static void extents(const llmt_adam_tensor& x, int bits, Extent (&e)[kKinds]) {
  const size_t n = (size_t)x.n, nb = (n + 255) / 256, ms = bits == 8 ? n : n * 4;
  const bool codes = bits == 8;
  auto put = [&](int k, const void* p, size_t bytes) {
    e[k] = {(uintptr_t)p, p ? (uintptr_t)p + bytes : 0, k < kKinds - 1};
  };
  put(0, x.p, n * 4);
  put(1, x.m, ms);
  put(2, x.v, ms);
  put(3, x.copy, n * 2);
  put(4, codes ? x.m_exp : nullptr, nb);
  put(5, codes ? x.v_exp : nullptr, nb);
  put(6, x.g, n * esize(x.g_dtype));
}
static bool list_apart(const llmt_adam_tensor* t, int count, int bits) {
  Extent e[kKinds];
  uintptr_t lo[kKinds], hi[kKinds];
  std::fill(lo, lo + kKinds, UINTPTR_MAX);
  std::fill(hi, hi + kKinds, (uintptr_t)0);
  bool ordered = true;
  for (int i = 0; i < count && ordered; ++i) {
    if (t[i].n == 0) continue;
    extents(t[i], bits, e);
    for (int k = 0; k < kKinds; ++k) {
      if (!e[k].a) continue;
      if (e[k].written && e[k].a < hi[k]) ordered = false;
      lo[k] = std::min(lo[k], e[k].a);
      hi[k] = std::max(hi[k], e[k].b);
    }
  }
  for (int k = 0; k < kKinds && ordered; ++k)
    for (int q = 0; q < k; ++q)
      if (lo[k] < hi[k] && lo[q] < hi[q] && lo[k] < hi[q] && lo[q] < hi[k]) ordered = false;
  if (ordered) return true;
  std::vector<Extent> x;
  x.reserve((size_t)count * kKinds);
  for (int i = 0; i < count; ++i) {
    if (t[i].n == 0) continue;
    extents(t[i], bits, e);
    for (const Extent& k : e)
      if (k.a) x.push_back(k);
  }
  std::sort(x.begin(), x.end(), [](const Extent& p, const Extent& q) { return p.a < q.a; });
  uintptr_t any = 0, written = 0;  // where what began earlier ends
  for (const Extent& k : x) {
    if (k.a < (k.written ? any : written)) return false;
    any = std::max(any, k.b);
    if (k.written) written = std::max(written, k.b);
  }
  return true;
}

extern "C" {

size_t llmt_packed_attention_workspace(const llmt_packed_dims* dims) {
  return dims_ok(dims) ? packed_fwd_workspace(pack_args(dims)) : 0;
}

int llmt_packed_attention(const llmt_packed_dims* d, const llmt_heads* q, const llmt_heads* k,
                          const llmt_heads* v, const llmt_heads* o, float* lse, void* workspace,
                          size_t workspace_bytes, void* stream) {
  set_error("");
  const char* const fn = "llmt_packed_attention";
  TRY_ARG(d, "%s: NULL dims", fn);
  const View views[4] = {{"q", q, d->Tq, d->nq, true, false},
                         {"k", k, d->Tk, d->nkv, false, false},
                         {"v", v, d->Tk, d->nkv, false, false},
                         {"o", o, d->Tq, d->nq, true, true}};
  int rc = check_packed(fn, d, views, 4, lse);
  if (rc) return rc;
  PackArgs a = pack_args(d);
  if ((rc = check_space(fn, packed_fwd_workspace(a), workspace, workspace_bytes))) return rc;
  a.q = heads(q);
  a.k = heads(k);
  a.v = heads(v);
  a.o = heads(o);
  a.lse = lse;
  return done(packed_fwd(a, workspace, (hipStream_t)stream));
}

size_t llmt_packed_attention_bwd_workspace(const llmt_packed_dims* dims) {
  return dims_ok(dims) ? packed_bwd_workspace(pack_args(dims)) : 0;
}

int llmt_packed_attention_bwd(const llmt_packed_dims* d, const llmt_heads* q, const llmt_heads* k,
                              const llmt_heads* v, const llmt_heads* o, const float* lse,
                              const llmt_heads* dout, const llmt_heads* dq, const llmt_heads* dk,
                              const llmt_heads* dv, void* workspace, size_t workspace_bytes,
                              void* stream) {
  set_error("");
  const char* const fn = "llmt_packed_attention_bwd";
  TRY_ARG(d, "%s: NULL dims", fn);
  const View views[8] = {{"q", q, d->Tq, d->nq, true, false},
                         {"k", k, d->Tk, d->nkv, false, false},
                         {"v", v, d->Tk, d->nkv, false, false},
                         {"o", o, d->Tq, d->nq, true, false},
                         {"dout", dout, d->Tq, d->nq, true, false},
                         {"dq", dq, d->Tq, d->nq, true, true},
                         {"dk", dk, d->Tk, d->nkv, false, true},
                         {"dv", dv, d->Tk, d->nkv, false, true}};
  int rc = check_packed(fn, d, views, 8, lse);
  if (rc) return rc;
  PackArgs a = pack_args(d);
  if ((rc = check_space(fn, packed_bwd_workspace(a), workspace, workspace_bytes))) return rc;
  a.q = heads(q);
  a.k = heads(k);
  a.v = heads(v);
  a.o = heads(o);
  a.lse = const_cast<float*>(lse);
  a.dout = heads(dout);
  a.dq = heads(dq);
  a.dk = heads(dk);
  a.dv = heads(dv);
  return done(packed_bwd(a, workspace, (hipStream_t)stream));
}

static int check_embed(const char* fn, const int* tokens, int T, const void* w, int wdtype,
                       long long ldw, int V, int H, float scale, const void* x, int xdtype,
                       long long ldx) {
  TRY_ARG(known(wdtype) && known(xdtype), "%s: dtypes %d and %d", fn, wdtype, xdtype);
  TRY_ARG(T >= 0 && T <= kMaxTokens && V >= 1 && V <= kMost && H >= 1 && H <= kMaxWidth,
          "%s: T=%d V=%d H=%d (at most 2^23, 2^30, 2^20)", fn, T, V, H);
  TRY_ARG(ldw >= H && ldw <= kMaxStride && ldx >= H && ldx <= kMaxStride &&
              (double)V * ldw <= 1e18 && (double)T * ldx <= 1e18,
          "%s: row strides %lld and %lld of rows of %d", fn, ldw, ldx, H);
  TRY_ARG(isfinite(scale), "%s: scale must be finite", fn);
  TRY_ARG(w && (T == 0 || (tokens && x)), "%s: NULL argument", fn);
  TRY_ARG(aligned(w, esize(wdtype)) && aligned(x, esize(xdtype)) && aligned(tokens, 4),
          "%s: misaligned argument", fn);
  const uintptr_t w0 = (uintptr_t)w, x0 = (uintptr_t)x;
  TRY_ARG(T == 0 || w0 + ((size_t)(V - 1) * ldw + H) * esize(wdtype) <= x0 ||
              x0 + ((size_t)(T - 1) * ldx + H) * esize(xdtype) <= w0,
          "%s: the rows overlap the table", fn);
  return LLMT_OK;
}

int llmt_embedding(const int* tokens, int T, const void* weight, int wdtype, long long ldw, int V,
                   int H, float scale, void* out, int odtype, long long ldo, void* stream) {
  set_error("");
  const int rc = check_embed("llmt_embedding", tokens, T, weight, wdtype, ldw, V, H, scale, out,
                             odtype, ldo);
  if (rc) return rc;
  EmbedArgs a{tokens, T, V, H, const_cast<void*>(weight), ldw, wdtype, out, ldo, odtype, scale, 0};
  return done(embed_fwd(a, (hipStream_t)stream));
}

size_t llmt_embedding_bwd_workspace(int T, int V, int H) {
  return T > 0 && T <= kMaxTokens && V >= 1 && V <= kMost && H >= 1 && H <= kMaxWidth
             ? embed_bwd_workspace(T, V, H) : 0;
}

int llmt_embedding_bwd(const int* tokens, int T, const void* dout, int ddtype, long long ldd,
                       float scale, void* dweight, int wdtype, long long ldw, int V, int H,
                       int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  set_error("");
  const char* const fn = "llmt_embedding_bwd";
  int rc = check_embed(fn, tokens, T, dweight, wdtype, ldw, V, H, scale, dout, ddtype, ldd);
  if (rc) return rc;
  const size_t need = T > 0 ? embed_bwd_workspace(T, V, H) : 0;
  if ((rc = check_space(fn, need, workspace, workspace_bytes))) return rc;
  EmbedArgs a{tokens, T, V, H, dweight, ldw, wdtype, const_cast<void*>(dout), ldd, ddtype, scale,
              accumulate != 0};
  return done(embed_bwd(a, workspace, (hipStream_t)stream));
}

int llmt_adamw_update(const llmt_adam_tensor* t, int count, int state_bits, const llmt_hparams* hp,
                      int step, const float* grad_scale, uint64_t seed, void* stream) {
  set_error("");
  const char* const fn = "llmt_adamw_update";
  TRY_ARG(count >= 0 && count <= (1 << 20) && (t || count == 0), "%s: %d tensors", fn, count);
  TRY_ARG(state_bits == 8 || state_bits == 32, "%s: moments of %d bits (8 or 32)", fn, state_bits);
  TRY_ARG(hp, "%s: NULL hp", fn);
  TRY_ARG(isfinite(hp->lr) && isfinite(hp->wd) && hp->beta1 >= 0.f && hp->beta1 < 1.f &&
              hp->beta2 >= 0.f && hp->beta2 < 1.f && hp->eps >= 0x1p-126f && isfinite(hp->eps) &&
              step >= 1,
          "%s: betas in [0, 1), eps from 2^-126, step from 1 on, finite lr and wd", fn);
  TRY_ARG(aligned(grad_scale, 4), "%s: misaligned grad_scale", fn);
  for (int i = 0; i < count; ++i) {
    const llmt_adam_tensor& x = t[i];
    TRY_ARG(x.n >= 0 && x.n <= kMaxElements, "%s: tensor %d has %lld elements", fn, i, x.n);
    TRY_ARG(known(x.g_dtype) && (!x.copy || x.copy_dtype == LLMT_F16 || x.copy_dtype == LLMT_BF16),
            "%s: tensor %d: gradient dtype %d, copy dtype %d (f16 or bf16)", fn, i, x.g_dtype,
            x.copy_dtype);
    if (x.n == 0) continue;
    TRY_ARG(x.p && x.g && x.m && x.v && (state_bits == 32 || (x.m_exp && x.v_exp)),
            "%s: tensor %d: NULL argument", fn, i);
    const size_t ms = state_bits == 8 ? 1 : 4;
    TRY_ARG(aligned(x.p, 4) && aligned(x.g, esize(x.g_dtype)) && aligned(x.m, ms) &&
                aligned(x.v, ms) && aligned(x.copy, 2),
            "%s: tensor %d: misaligned argument", fn, i);
  }
  try {
    TRY_ARG(list_apart(t, count, state_bits), "%s: a written array overlaps another", fn);
  } catch (const std::bad_alloc&) {
    TRY_ARG(false, "%s: out of host memory", fn);
  }
  static_assert(sizeof(AdamTensor) == sizeof(llmt_adam_tensor), "one layout");
  AdamStep k{};
  k.b1 = hp->beta1;
  k.b2 = hp->beta2;
  k.c1 = 1.0f - hp->beta1;
  k.c2 = 1.0f - hp->beta2;
  k.ib1 = (float)(1.0 / (1.0 - pow((double)hp->beta1, step)));
  const float ib2 = (float)(1.0 / (1.0 - pow((double)hp->beta2, step)));
  k.ib2_up = ib2 * 0x1p64f;
  k.ib2_down = ib2 * 0x1p-64f;
  k.decay = (float)(1.0 - (double)hp->lr * hp->wd);
  k.lr = hp->lr;
  k.eps = hp->eps;
  k.gscale = grad_scale;
  k.seed = seed;
  k.step = step;
  return done(adamw_list(reinterpret_cast<const AdamTensor*>(t), count, state_bits, k,
                         (hipStream_t)stream));
}

int llmt_adamw_moments(const void* m, const void* v, const unsigned char* m_exp,
                       const unsigned char* v_exp, long long n, float* m32, float* v32,
                       void* stream) {
  set_error("");
  const char* const fn = "llmt_adamw_moments";
  TRY_ARG(n >= 0 && n <= kMaxElements, "%s: n=%lld", fn, n);
  if (n == 0) return LLMT_OK;
  TRY_ARG(m && v && m_exp && v_exp && m32 && v32, "%s: NULL argument", fn);
  TRY_ARG(aligned(m32, 4) && aligned(v32, 4), "%s: misaligned argument", fn);
  return done(adamw_moments(m, v, m_exp, v_exp, n, m32, v32, (hipStream_t)stream));
}

}  // extern "C"
