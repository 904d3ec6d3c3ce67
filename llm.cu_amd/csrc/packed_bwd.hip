// packed_bwd.hip — backward of the packed attention, recomputing the
// probabilities from q, k and the forward's lse:
//   P = exp(scale q k^T - lse), dP = dO v^T, dS = P (dP - delta),
//   delta = rowsum(dO o), dQ = scale dS k, dK = scale dS^T q, dV = P^T dO.
// Two kinds of workgroups that share no outputs: dQ blocks (rows of one KV
// head's group, walking their keys) and dK/dV blocks (keys, walking the rows
// that see them: a sum over the whole group in registers, in a fixed order, no
// atomics).  Rows, tiles and offsets: packed_attn.h.
//
// Both kinds are in one launch (Mix), behind one that writes each row's lse and
// delta.  16 sequences of 8192 tokens together, 16 / 8 heads of 128 in bf16: 172
// us, 195 with a launch for each kind, which both ended with the tiles of the
// longest sequence; 1 x 512 tokens 21 and 28.  A long sequence is bound by issue:
// a matrix instruction of 16 x 16 x 32 takes a SIMD 17 cycles, and the
// exponentials and roundings of the other wave hardly run beside it (of the two
// alone, 272 and 174 cycles, together 420).  1 x 8192 tokens take 872 to
// 910 us, 755 to 788 TFLOP/s of the five products, up to 1100 of the seven computed
// (S and dP twice); a large library product reaches 1387.
//
// fp16.  dS spans many binades (a probability of one key in many times a small
// gradient), so it enters its product times a power of two that belongs to the
// accumulator's column (a row in dQ, a key in dK) and follows the largest value
// seen, as a running maximum does; when it changes the column is rescaled,
// exactly.  bf16 has the range.
#include <algorithm>
#include <type_traits>

#include "packed_attn.h"

namespace llmt {

namespace {

// Of each row in the order (KV head, token, head in the group): the base-2 lse,
// +inf for a row without keys (its probabilities are then 0), and delta.
struct RowVecs {
  float* lse2;
  float* delta;
};
__device__ __forceinline__ long long vec_at(const PackArgs& a, int G, int j, long long token) {
  return ((long long)j * a.Tq + token) * G;
}

// The running power of two of an accumulator column.  Returns the factor that
// brings what has been summed to the new scale.
struct ColScale {
  float s = 0x1p100f;
  __device__ __forceinline__ float follow(float amax) {
    // amax s in [2^14, 2^15) at most; a maximum of 0 asks for nothing, inf and
    // NaN keep what is there
    const int e = __builtin_amdgcn_frexp_expf(amax);
    const float want = amax > 0.f ? ldexpf(1.0f, min(100, 15 - e)) : s;
    const float n = fminf(s, want);
    const float f = n / s;
    s = n;
    return f;
  }
};

__device__ __forceinline__ float lse2_of(float lse) {
  return lse == -INFINITY ? INFINITY : lse * LOG2E;
}

// Sum over a row's 8 or 16 lanes.
template <int LR>
__device__ __forceinline__ float row_lanes_sum(float x) {
  x += dpp16<0xB1>(x);
  x += dpp16<0x4E>(x);
  x += dpp16<0x141>(x);
  return LR == 16 ? x + dpp16<0x140>(x) : x;
}

// The rows' lse2 and delta: HD / 8 lanes a row, in at most kDeltaWgs workgroups (a
// launch has less than 2^32 threads; the rows of one may be up to 2^29).
constexpr unsigned kDeltaWgs = 1 << 23;
template <class E, int HD>
__global__ __launch_bounds__(256) void packed_delta_kernel(const PackArgs a, int G, RowVecs rv) {
  typedef typename E::T T8 __attribute__((ext_vector_type(8)));
  constexpr int LR = HD / 8;
  const long long rows = (long long)a.Tq * a.nq;
  for (long long row = (long long)blockIdx.x * (256 / LR) + threadIdx.x / LR; row < rows;
       row += (long long)gridDim.x * (256 / LR)) {
    const long long t = row / a.nq;
    const int h = (int)(row - t * a.nq), d = threadIdx.x % LR * 8;
    const T8 x = *reinterpret_cast<const T8*>((const short*)a.dout.p + t * a.dout.token +
                                              h * a.dout.head + d);
    const T8 y = *reinterpret_cast<const T8*>((const short*)a.o.p + t * a.o.token + h * a.o.head + d);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf((float)x[e], (float)y[e], s);
    s = row_lanes_sum<LR>(s);
    if (d == 0) {
      const int j = h / G;
      const long long at = vec_at(a, G, j, t) + h - j * G;
      rv.lse2[at] = lse2_of(a.lse[row]);
      rv.delta[at] = s;
    }
  }
}

// The workgroups of one launch are of keys (dK, dV) and of rows (dQ): a quarter of
// those of keys, which take longest, then the others and those of rows in
// turn, so that all end together.
struct Mix {
  int nrows, nkeys;           // tiles a KV head
  unsigned long long share;  // of keys among what follows the quarter, times 2^32 (rounded up)
  // The tiles of keys before tile t of the launch.
  __device__ __forceinline__ int keys_before(int t) const {
    const int k0 = nkeys >> 2;
    return t < k0 ? t : k0 + (int)((t - k0) * share >> 32);
  }
};

// LDS of a workgroup: two buffers, each two tiles of 64 with two vectors, or that
// for two waves alone.
constexpr int NW = 4;
template <int HD>
constexpr int kBuf = 2 * BLK * HD + 4 * BLK * 2;

// Of one row's part in a lane (elements 32 ks + 8 g .. + 7 of df): its lse2 and
// delta, from the forward's o and lse.
template <class E, int KS>
__device__ __forceinline__ float delta_of(const short8v (&df)[KS], const short* orow, int g) {
  typedef typename E::T T8 __attribute__((ext_vector_type(8)));
  float s = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const T8 d8 = __builtin_bit_cast(T8, df[ks]);
    const T8 o8 = *reinterpret_cast<const T8*>(orow + 32 * ks + 8 * g);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf((float)d8[e], (float)o8[e], s);
  }
  return xg_sum(s);
}

// ---------------------------------------------------------------- dQ
// Four waves of 16 RW rows, against keys in tiles of 64, two halves one after
// the other.  (Two waves for each of two halves, as in dK/dV below, were slower
// at every size, 7% at 16 sequences of 8192 tokens.)  dS is rounded to the type
// once, here as P and dS in dK/dV: these blocks are bound by issue, and the remainder
// as a second operand would be a third (dQ) or half (dK, dV) more products.
template <class E, int HD, int RW, bool OWN>
__device__ __forceinline__ void dq_block(const PackArgs& a, Group gr, int j, int tile, Mix mix,
                                         RowVecs rv, short* buf0, short* buf1) {
  constexpr int QB = NW * RW * 16, KS = HD / 32, DT = HD / 16, TILE = BLK * HD;
  constexpr bool F = std::is_same_v<E, F16>;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int row = w * RW * 16;
  Tile x;
  if (!find<QB>(a, gr, tile, mix.nrows, mix.nrows + mix.nkeys, x)) return;
  const short* kbase = (const short*)a.k.p + x.kstart * a.k.token + j * a.k.head;
  const short* vbase = (const short*)a.v.p + x.kstart * a.v.token + j * a.v.head;
  const int nkb = (x.kmax + BLK - 1) / BLK;
  const int nfull = min(max((x.t0 + x.shift + 1) / BLK, 0), nkb);  // tiles that every row sees whole
  KeyDma<HD, NW, BLK> dk, dv;
  dk.init(a.k.token, w);
  dv.init(a.v.token, w);
  if (nkb > 0) {
    dk.issue(kbase, a.k.token, 0, x.klen, buf0, w);
    dv.issue(vbase, a.v.token, 0, x.klen, buf0 + TILE, w);
  }
  const int left = x.rows - x.row0 - row;  // rows from the wave's first on
  short8v qf[RW][KS], df[RW][KS];
  int lim[RW], at[RW], hq[RW];
  float lse2[RW], del[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int i = min(row + 16 * r + c, x.rows - 1 - x.row0);
    const int t = gr.div(x.rem + i), h = x.rem + i - t * gr.G;
    lim[r] = 16 * r + c < left ? x.t0 + t + x.shift : -1;
    at[r] = x.qstart + x.t0 + t;
    hq[r] = j * gr.G + h;
    const short* row = (const short*)a.q.p + at[r] * a.q.token + hq[r] * a.q.head;
    const short* dor = (const short*)a.dout.p + at[r] * a.dout.token + hq[r] * a.dout.head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[r][ks] = *reinterpret_cast<const short8v*>(row + 32 * ks + 8 * g);
      df[r][ks] = *reinterpret_cast<const short8v*>(dor + 32 * ks + 8 * g);
    }
    if constexpr (OWN) {
      const short* orow = (const short*)a.o.p + at[r] * a.o.token + hq[r] * a.o.head;
      del[r] = delta_of<E, KS>(df[r], orow, g);
      lse2[r] = lse2_of(a.lse[(long long)at[r] * a.nq + hq[r]]);
    } else {
      const long long vi = vec_at(a, gr.G, j, at[r]) + h;
      lse2[r] = rv.lse2[vi];
      del[r] = rv.delta[vi];
    }
  }
  const float sl2 = a.scale * LOG2E;
  floatx4 dqT[RW][DT];
  ColScale cs[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r)
#pragma unroll
    for (int i = 0; i < DT; ++i) dqT[r][i] = floatx4{0.f, 0.f, 0.f, 0.f};

  auto tile_step = [&](int kb, auto mask_tag, const short* Ks, short* nb) LLMT_INLINE {
    constexpr bool MASK = decltype(mask_tag)::value;
    wait_vm<0>();
    tile_barrier();
    if (kb + 1 < nkb) {
      dk.issue(kbase, a.k.token, (kb + 1) * BLK, x.klen, nb, w);
      dv.issue(vbase, a.v.token, (kb + 1) * BLK, x.klen, nb + TILE, w);
    }
    const short* Vs = Ks + TILE;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      floatx4 pt[RW][2], dp[RW][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          pt[r][u] = floatx4{0.f, 0.f, 0.f, 0.f};
          dp[r][u] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const short8v kf = frag_rm<HD>(Ks, (2 * jj + u) * 16, ks, lane);
          const short8v vf = frag_rm<HD>(Vs, (2 * jj + u) * 16, ks, lane);
#pragma unroll
          for (int r = 0; r < RW; ++r) {
            pt[r][u] = E::mfma(kf, qf[r][ks], pt[r][u]);
            dp[r][u] = E::mfma(vf, df[r][ks], dp[r][u]);
          }
        }
      }
      sched_reads_ahead<4 * KS, 4 * KS * RW, KS == 4 ? 6 : 4, 2 * RW, 2, 0>();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        float am = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float pv = __builtin_amdgcn_exp2f(fmaf(pt[r][u][v], sl2, -lse2[r]));
            if (MASK) pv = kb * BLK + (2 * jj + u) * 16 + 4 * g + v <= lim[r] ? pv : 0.f;
            dp[r][u][v] = pv * (dp[r][u][v] - del[r]);
            if (F) am = fmaxf(am, fabsf(dp[r][u][v]));
          }
        if constexpr (F) {
          const float f = cs[r].follow(xg_max(am));
          if (__ballot(f != 1.0f)) {
#pragma unroll
            for (int i = 0; i < DT; ++i) dqT[r][i] *= f;
          }
          dp[r][0] *= cs[r].s;
          dp[r][1] *= cs[r].s;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      short8v db[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) db[r] = pair_frag<E>(dp[r][0], dp[r][1]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const short8v kt = frag_tr<HD>(Ks, d * 16, jj, lane);
#pragma unroll
        for (int r = 0; r < RW; ++r) dqT[r][d] = E::mfma(kt, db[r], dqT[r][d]);
      }
      sched_reads_ahead<2 * DT, DT * RW, DT == 8 ? 6 : 4, RW, 2, 1>();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int kb = 0; kb + 1 < nfull; kb += 2) {
    tile_step(kb, std::false_type{}, buf0, buf1);
    tile_step(kb + 1, std::false_type{}, buf1, buf0);
  }
  for (int kb = nfull & ~1; kb < nkb; ++kb)
    tile_step(kb, std::true_type{}, (kb & 1) ? buf1 : buf0, (kb & 1) ? buf0 : buf1);
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    if (16 * r + c >= left) continue;
    const float f = F ? a.scale / cs[r].s : a.scale;
    short* dq = (short*)a.dq.p + at[r] * a.dq.token + hq[r] * a.dq.head;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<short4v*>(dq + d * 16 + 4 * g) = round4<E>(dqT[r][d] * f);
  }
}

// ---------------------------------------------------------------- dK, dV
// Four waves: 4 / JG groups of 16 keys, in registers; the rows that see them pass
// through LDS in tiles with their lse and delta, two halves one after the other
// (JG = 2: a wave takes one half, and the two groups' sums meet in LDS).  Row r sees key k where
// r >= (k - shift) G: only the first tiles take a mask.  Rows of zeros (past the
// end, or past the tile's whole tokens) add nothing by themselves, and keys
// past the end are not stored.
template <class E, int HD, int JG>
__device__ __forceinline__ void dkdv_block(const PackArgs& a, Group gr, int j, int tile, Mix mix,
                                           RowVecs rv, short* buf0, short* buf1,
                                           float (*scale)[16]) {
  constexpr int WG = NW / JG, KB = WG * 16, KS = HD / 32, DT = HD / 16, TILE = BLK * HD;
  constexpr bool F = std::is_same_v<E, F16>;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int jg = JG == 1 ? 0 : w / WG, wk = w - jg * WG;  // row group, key group
  int blk;
  SeqLens s;
  if (!pick_tile<false, KB>(a, gr.G, tile, mix.nkeys, mix.nrows + mix.nkeys, &s, &blk)) return;
  const Span qs = {s.qstart, s.ql}, ks = {s.kstart, s.kl};
  if (blk < 0 || blk >= (ks.len + KB - 1) / KB) return;
  const int shift = ks.len - qs.len;
  const int k0 = blk * KB, kw = k0 + wk * 16;
  const int tokens = 64 / gr.G, tr = tokens * gr.G;   // of a tile
  const int t0 = min(max(k0 - shift, 0), qs.len);     // the first token that sees a key
  const int niter = (qs.len - t0 + tokens - 1) / tokens;
  // tiles with a token that does not see the block's last key
  const int nmask = min(niter, (max(min(k0 + KB - 1 - shift, qs.len) - t0, 0) + tokens - 1) / tokens);
  const int key = kw + c;
  // the first row, counted from token t0, that sees the lane's key
  const int rmin = (min(max(key - shift, 0), qs.len) - t0) * gr.G;
  const short* qbase = (const short*)a.q.p + qs.start * a.q.token + j * gr.G * a.q.head;
  const short* dbase = (const short*)a.dout.p + qs.start * a.dout.token + j * gr.G * a.dout.head;
  const long long vbase = vec_at(a, gr.G, j, qs.start + t0);
  const int rows = (qs.len - t0) * gr.G;
  RowDma<HD, NW> dq_, dd_;
  dq_.init(a.q.token, a.q.head, gr, tr, w);
  dd_.init(a.dout.token, a.dout.head, gr, tr, w);
  auto issue = [&](int it, short* buf) LLMT_INLINE {
    const int t = t0 + it * tokens;
    dq_.issue(qbase, a.q.token, a.q.head, gr, t, qs.len, tokens, buf, w);
    dd_.issue(dbase, a.dout.token, a.dout.head, gr, t, qs.len, tokens, buf + TILE, w);
    float* vec = reinterpret_cast<float*>(buf + 2 * TILE);
    if (w == 0) dma_vec64(rv.lse2 + vbase, it * tr, min(rows, (it + 1) * tr), vec);
    if (w == NW - 1) dma_vec64(rv.delta + vbase, it * tr, min(rows, (it + 1) * tr), vec + BLK);
  };
  if (niter > 0) issue(0, buf0);
  const int tok = ks.start + min(key, ks.len - 1);
  short8v kf[KS], vf[KS];
  {
    const short* kr = (const short*)a.k.p + tok * a.k.token + j * a.k.head;
    const short* vr = (const short*)a.v.p + tok * a.v.token + j * a.v.head;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      kf[i] = *reinterpret_cast<const short8v*>(kr + 32 * i + 8 * g);
      vf[i] = *reinterpret_cast<const short8v*>(vr + 32 * i + 8 * g);
    }
  }
  const float sl2 = a.scale * LOG2E;
  floatx4 dkT[DT], dvT[DT];
  ColScale cs;
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    dkT[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    dvT[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  auto tile_step = [&](int it, auto mask_tag, const short* Qs, short* nb) LLMT_INLINE {
    constexpr bool MASK = decltype(mask_tag)::value;
    wait_vm<0>();
    tile_barrier();
    if (it + 1 < niter) issue(it + 1, nb);
    const short* Ds = Qs + TILE;
    const float* lse_s = reinterpret_cast<const float*>(Qs + 2 * TILE);
    const float* del_s = lse_s + BLK;
#pragma unroll
    for (int h = 0; h < 2 / JG; ++h) {
      const int jj = JG == 1 ? h : jg;
      floatx4 p[2], ds[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int m0 = (2 * jj + u) * 16;
        p[u] = floatx4{0.f, 0.f, 0.f, 0.f};
        ds[u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          p[u] = E::mfma(frag_rm<HD>(Qs, m0, i, lane), kf[i], p[u]);
          ds[u] = E::mfma(frag_rm<HD>(Ds, m0, i, lane), vf[i], ds[u]);
        }
      }
      sched_reads_ahead<4 * KS, 4 * KS, KS == 4 ? 6 : 4, 2, 2, 0>();
      __builtin_amdgcn_sched_barrier(0);
      float am = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i0 = (2 * jj + u) * 16 + 4 * g;
        const floatx4 ls = *reinterpret_cast<const floatx4*>(lse_s + i0);
        const floatx4 dl = *reinterpret_cast<const floatx4*>(del_s + i0);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float pv = __builtin_amdgcn_exp2f(fmaf(p[u][v], sl2, -ls[v]));
          if (MASK) pv = it * tr + i0 + v >= rmin ? pv : 0.f;
          ds[u][v] = pv * (ds[u][v] - dl[v]);
          p[u][v] = F ? pv * (float)(1 << E::PSH) : pv;
          if (F) am = fmaxf(am, fabsf(ds[u][v]));
        }
      }
      if constexpr (F) {
        const float f = cs.follow(xg_max(am));
        if (__ballot(f != 1.0f)) {
#pragma unroll
          for (int i = 0; i < DT; ++i) dkT[i] *= f;
        }
        ds[0] *= cs.s;
        ds[1] *= cs.s;
      }
      __builtin_amdgcn_sched_barrier(0);
      const short8v pb = pair_frag<E>(p[0], p[1]), db = pair_frag<E>(ds[0], ds[1]);
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        dvT[i] = E::mfma(frag_tr<HD>(Ds, i * 16, jj, lane), pb, dvT[i]);
        dkT[i] = E::mfma(frag_tr<HD>(Qs, i * 16, jj, lane), db, dkT[i]);
      }
      sched_reads_ahead<4 * DT, 2 * DT, 8, 2, 4, 1>();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto step_rt = [&](int it, auto mask_tag) LLMT_INLINE {
    tile_step(it, mask_tag, (it & 1) ? buf1 : buf0, (it & 1) ? buf0 : buf1);
  };
  int it = 0;
  for (; it < nmask; ++it) step_rt(it, std::true_type{});
  // in pairs with statically named buffers: the reads of a tile are then not
  // made to wait for the next one's DMA
  if (it < niter && (it & 1)) step_rt(it++, std::false_type{});
  for (; it < niter; it += 2) {
    tile_step(it, std::false_type{}, buf0, buf1);
    if (it + 1 < niter) tile_step(it + 1, std::false_type{}, buf1, buf0);
  }
  if constexpr (JG == 2) {  // [register][lane], where the tiles were
    auto room = [&](int i) LLMT_INLINE { return reinterpret_cast<floatx4*>(i ? buf1 : buf0); };
    static_assert(2 * DT * 64 * 16 <= kBuf<HD> * 2, "a wave's sums fit a buffer");
    __syncthreads();
    if (jg == 1) {
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        room(wk)[i * 64 + lane] = dkT[i];
        room(wk)[(DT + i) * 64 + lane] = dvT[i];
      }
      if (g == 0) scale[wk][c] = F ? cs.s : 1.f;
    }
    __syncthreads();
    if (jg == 1) return;
    const float f = F ? cs.s / scale[wk][c] : 1.f;  // a power of two
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      dkT[i] += room(wk)[i * 64 + lane] * f;
      dvT[i] += room(wk)[(DT + i) * 64 + lane];
    }
  }
  if (key < ks.len) {
    const float fk = F ? a.scale / cs.s : a.scale;
    const float fv = 1.0f / (float)(1 << E::PSH);
    short* dkr = (short*)a.dk.p + tok * a.dk.token + j * a.dk.head;
    short* dvr = (short*)a.dv.p + tok * a.dv.token + j * a.dv.head;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      *reinterpret_cast<short4v*>(dkr + i * 16 + 4 * g) = round4<E>(dkT[i] * fk);
      *reinterpret_cast<short4v*>(dvr + i * 16 + 4 * g) = round4<E>(dvT[i] * fv);
    }
  }
}

// ---------------------------------------------------------------- few tiles
// Where the blocks above would leave CUs idle, their chains of tiles, each
// waiting for its own loads, are the time: blocks of 16 rows (16 keys) whose
// four waves take the tiles of 32 in turn, each through LDS of its own, without
// a barrier in the loop; the waves' sums meet in LDS and are added in order.
// They wait for loads, not for the matrix units, so P and dS enter in two parts
// (pair_split), and nothing but the result is rounded to the type.
template <class E, int HD, bool OWN>
__device__ __forceinline__ void dq_split_block(const PackArgs& a, Group gr, int j, int tile,
                                               Mix mix, RowVecs rv, short* buf0, short* buf1,
                                               float (*scale)[16]) {
  constexpr int QB = 16, KT = 32, KS = HD / 32, DT = HD / 16;
  constexpr bool F = std::is_same_v<E, F16>;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  Tile x;
  if (!find<QB>(a, gr, tile, mix.nrows, mix.nrows + mix.nkeys, x)) return;
  const short* kbase = (const short*)a.k.p + x.kstart * a.k.token + j * a.k.head;
  const short* vbase = (const short*)a.v.p + x.kstart * a.v.token + j * a.v.head;
  const int nkt = (x.kmax + KT - 1) / KT;
  auto room = [&](int u) LLMT_INLINE { return (u & 2 ? buf1 : buf0) + (u & 1) * 2 * KT * HD; };
  short* const Ks = room(w);
  short* const Vs = Ks + KT * HD;
  KeyDma<HD, 1, KT> dk, dv;
  dk.init(a.k.token, 0);
  dv.init(a.v.token, 0);
  auto issue = [&](int kt) LLMT_INLINE {
    dk.issue(kbase, a.k.token, kt * KT, x.klen, Ks, 0);
    dv.issue(vbase, a.v.token, kt * KT, x.klen, Vs, 0);
  };
  if (w < nkt) issue(w);
  const int left = x.rows - x.row0;
  const int t = gr.div(x.rem + min(c, left - 1)), h = x.rem + min(c, left - 1) - t * gr.G;
  const int lim = c < left ? x.t0 + t + x.shift : -1, at = x.qstart + x.t0 + t, hq = j * gr.G + h;
  short8v qf[KS], df[KS];
  {
    const short* row = (const short*)a.q.p + at * a.q.token + hq * a.q.head;
    const short* dor = (const short*)a.dout.p + at * a.dout.token + hq * a.dout.head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = *reinterpret_cast<const short8v*>(row + 32 * ks + 8 * g);
      df[ks] = *reinterpret_cast<const short8v*>(dor + 32 * ks + 8 * g);
    }
  }
  float lse2, del;
  if constexpr (OWN) {
    del = delta_of<E, KS>(df, (const short*)a.o.p + at * a.o.token + hq * a.o.head, g);
    lse2 = lse2_of(a.lse[(long long)at * a.nq + hq]);
  } else {
    const long long vi = vec_at(a, gr.G, j, at) + h;
    lse2 = rv.lse2[vi];
    del = rv.delta[vi];
  }
  const float sl2 = a.scale * LOG2E;
  floatx4 dqT[DT];
  ColScale cs;
#pragma unroll
  for (int i = 0; i < DT; ++i) dqT[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int kt = w; kt < nkt; kt += NW) {
    wait_vm<0>();  // the wave's own tile
    asm volatile("" ::: "memory");
    floatx4 p[2], dp[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      p[u] = floatx4{0.f, 0.f, 0.f, 0.f};
      dp[u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        p[u] = E::mfma(frag_rm<HD>(Ks, u * 16, ks, lane), qf[ks], p[u]);
        dp[u] = E::mfma(frag_rm<HD>(Vs, u * 16, ks, lane), df[ks], dp[u]);
      }
    }
    float am = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float pv = __builtin_amdgcn_exp2f(fmaf(p[u][v], sl2, -lse2));
        pv = kt * KT + u * 16 + 4 * g + v <= lim ? pv : 0.f;
        dp[u][v] = pv * (dp[u][v] - del);
        if (F) am = fmaxf(am, fabsf(dp[u][v]));
      }
    if constexpr (F) {
      const float f = cs.follow(xg_max(am));
#pragma unroll
      for (int i = 0; i < DT; ++i) dqT[i] *= f;
      dp[0] *= cs.s;
      dp[1] *= cs.s;
    }
    short8v db, dl;
    pair_split<E>(dp[0], dp[1], db, dl);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const short8v kt = frag_tr<HD>(Ks, d * 16, 0, lane);
      dqT[d] = E::mfma(kt, db, E::mfma(kt, dl, dqT[d]));
    }
    if (kt + NW < nkt) {  // refill once this tile's reads have returned
      wait_lds();
      asm volatile("" ::: "memory");
      issue(kt + NW);
    }
  }
  // the waves' sums, each in its own column scale, go where its tiles were
  floatx4* const mine = reinterpret_cast<floatx4*>(Ks);
  static_assert(DT * 64 * 16 <= 2 * KT * HD * 2, "a wave's sums fit its tiles");
  wait_lds();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int d = 0; d < DT; ++d) mine[d * 64 + lane] = dqT[d];
  if (g == 0) scale[w][c] = F ? cs.s : 1.f;
  __syncthreads();
  // wave w takes a quarter of the dims
#pragma unroll
  for (int d0 = 0; d0 < DT / NW; ++d0) {
    const int d = w * (DT / NW) + d0;
    floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const floatx4 y = reinterpret_cast<const floatx4*>(room(u))[d * 64 + lane];
      s += y * (a.scale / scale[u][c]);
    }
    if (c < left)
      *reinterpret_cast<short4v*>((short*)a.dq.p + at * a.dq.token + hq * a.dq.head + d * 16 +
                                  4 * g) = round4<E>(s);
  }
}

template <class E, int HD, bool OWN>
__device__ __forceinline__ void dkdv_split_block(const PackArgs& a, Group gr, int j, int tile,
                                                 Mix mix, RowVecs rv, short* buf0, short* buf1,
                                                 float (*scale)[16]) {
  constexpr int KB = 16, QT = 32, KS = HD / 32, DT = HD / 16, TILE = QT * HD;
  constexpr int BUF = 2 * TILE + 2 * 64 * 2;  // a wave's Q and dO tile, lse and delta
  constexpr bool F = std::is_same_v<E, F16>;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  int blk;
  SeqLens s;
  if (!pick_tile<false, KB>(a, gr.G, tile, mix.nkeys, mix.nrows + mix.nkeys, &s, &blk)) return;
  if (blk < 0 || blk >= (s.kl + KB - 1) / KB) return;
  const int shift = s.kl - s.ql, key = blk * KB + c;
  const int tokens = QT / gr.G, tr = tokens * gr.G;
  const int t0 = min(max(blk * KB - shift, 0), s.ql);
  const int niter = (s.ql - t0 + tokens - 1) / tokens, rows = (s.ql - t0) * gr.G;
  const int rmin = (min(max(key - shift, 0), s.ql) - t0) * gr.G;
  const short* qbase = (const short*)a.q.p + s.qstart * a.q.token + j * gr.G * a.q.head;
  const short* dbase = (const short*)a.dout.p + s.qstart * a.dout.token + j * gr.G * a.dout.head;
  const short* obase = (const short*)a.o.p + s.qstart * a.o.token + j * gr.G * a.o.head;
  auto room = [&](int u) LLMT_INLINE { return (u & 2 ? buf1 : buf0) + (u & 1) * BUF; };
  static_assert(2 * BUF <= kBuf<HD>, "two waves a buffer");
  short* const Qs = room(w);
  short* const Ds = Qs + TILE;
  float* const lse_s = reinterpret_cast<float*>(Qs + 2 * TILE);
  float* const del_s = lse_s + 64;
  RowDma<HD, 1, QT> dq_, dd_;
  dq_.init(a.q.token, a.q.head, gr, tr, 0);
  dd_.init(a.dout.token, a.dout.head, gr, tr, 0);
  const long long vbase = vec_at(a, gr.G, j, s.qstart + t0);
  // OWN: o's pieces of 8 of the tile's rows, HD / 8 lanes a row, and (lanes below QT) its lse
  constexpr int LR = HD / 8, RL = 64 / LR, NO = QT / RL;
  typedef typename E::T T8 __attribute__((ext_vector_type(8)));
  T8 ov[NO];
  float lv = 0.f;
  auto issue = [&](int it) LLMT_INLINE {
    const int t = t0 + it * tokens;
    dq_.issue(qbase, a.q.token, a.q.head, gr, t, s.ql, tokens, Qs, 0);
    dd_.issue(dbase, a.dout.token, a.dout.head, gr, t, s.ql, tokens, Ds, 0);
    if constexpr (OWN) {
      const int here = min(tr, rows - it * tr);
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const int r = min(RL * i + lane / LR, here - 1), u = gr.div(r);
        ov[i] = *reinterpret_cast<const T8*>(obase + (t + u) * a.o.token +
                                             (r - u * gr.G) * a.o.head + lane % LR * 8);
      }
      const int r = min(lane, here - 1), u = gr.div(r);
      lv = a.lse[(long long)(s.qstart + t + u) * a.nq + j * gr.G + r - u * gr.G];
    } else {
      dma_vec64(rv.lse2 + vbase, it * tr, min(rows, (it + 1) * tr), lse_s);
      dma_vec64(rv.delta + vbase, it * tr, min(rows, (it + 1) * tr), del_s);
    }
  };
  if (w < niter) issue(w);
  const int tok = s.kstart + min(key, s.kl - 1);
  short8v kf[KS], vf[KS];
  {
    const short* kr = (const short*)a.k.p + tok * a.k.token + j * a.k.head;
    const short* vr = (const short*)a.v.p + tok * a.v.token + j * a.v.head;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      kf[i] = *reinterpret_cast<const short8v*>(kr + 32 * i + 8 * g);
      vf[i] = *reinterpret_cast<const short8v*>(vr + 32 * i + 8 * g);
    }
  }
  const float sl2 = a.scale * LOG2E;
  floatx4 dkT[DT], dvT[DT];
  ColScale cs;
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    dkT[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    dvT[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  for (int it = w; it < niter; it += NW) {
    wait_vm<0>();  // the wave's own tile
    asm volatile("" ::: "memory");
    if constexpr (OWN) {
      // rows of zeros (past the tile's tokens, or past the end) have no probabilities
      const int here = rows - it * tr < tr ? rows - it * tr : tr;
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const int r = RL * i + lane / LR;
        const T8 d8 = *reinterpret_cast<const T8*>(Ds + toff<HD>(r, lane % LR));
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaf((float)d8[e], (float)ov[i][e], x);
        x = row_lanes_sum<LR>(x);
        if (lane % LR == 0) del_s[r] = r < here ? x : 0.f;
      }
      if (lane < QT) lse_s[lane] = lane < here ? lse2_of(lv) : INFINITY;
    }
    floatx4 p[2], ds[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      p[u] = floatx4{0.f, 0.f, 0.f, 0.f};
      ds[u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        p[u] = E::mfma(frag_rm<HD>(Qs, u * 16, i, lane), kf[i], p[u]);
        ds[u] = E::mfma(frag_rm<HD>(Ds, u * 16, i, lane), vf[i], ds[u]);
      }
    }
    float am = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i0 = u * 16 + 4 * g;
      const floatx4 ls = *reinterpret_cast<const floatx4*>(lse_s + i0);
      const floatx4 dl = *reinterpret_cast<const floatx4*>(del_s + i0);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float pv = __builtin_amdgcn_exp2f(fmaf(p[u][v], sl2, -ls[v]));
        pv = it * tr + i0 + v >= rmin ? pv : 0.f;
        ds[u][v] = pv * (ds[u][v] - dl[v]);
        p[u][v] = F ? pv * (float)(1 << E::PSH) : pv;
        if (F) am = fmaxf(am, fabsf(ds[u][v]));
      }
    }
    if constexpr (F) {
      const float f = cs.follow(xg_max(am));
#pragma unroll
      for (int i = 0; i < DT; ++i) dkT[i] *= f;
      ds[0] *= cs.s;
      ds[1] *= cs.s;
    }
    short8v pb, pl, db, dl;
    pair_split<E>(p[0], p[1], pb, pl);
    pair_split<E>(ds[0], ds[1], db, dl);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const short8v x = frag_tr<HD>(Ds, i * 16, 0, lane), y = frag_tr<HD>(Qs, i * 16, 0, lane);
      dvT[i] = E::mfma(x, pb, E::mfma(x, pl, dvT[i]));
      dkT[i] = E::mfma(y, db, E::mfma(y, dl, dkT[i]));
    }
    if (it + NW < niter) {
      wait_lds();
      asm volatile("" ::: "memory");
      issue(it + NW);
    }
  }
  floatx4* const mine = reinterpret_cast<floatx4*>(Qs);
  static_assert(2 * DT * 64 * 16 <= BUF * 2, "a wave's sums fit its tiles");
  wait_lds();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    mine[i * 64 + lane] = dkT[i];
    mine[(DT + i) * 64 + lane] = dvT[i];
  }
  if (g == 0) scale[w][c] = F ? cs.s : 1.f;
  __syncthreads();
  const float fv = 1.0f / (float)(1 << E::PSH);
#pragma unroll
  for (int d0 = 0; d0 < DT / NW; ++d0) {
    const int d = w * (DT / NW) + d0;
    floatx4 sk = {0.f, 0.f, 0.f, 0.f}, sv = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const floatx4* y = reinterpret_cast<const floatx4*>(room(u));
      sk += y[d * 64 + lane] * (a.scale / scale[u][c]);
      sv += y[(DT + d) * 64 + lane];
    }
    if (key < s.kl) {
      *reinterpret_cast<short4v*>((short*)a.dk.p + tok * a.dk.token + j * a.dk.head + d * 16 +
                                  4 * g) = round4<E>(sk);
      *reinterpret_cast<short4v*>((short*)a.dv.p + tok * a.dv.token + j * a.dv.head + d * 16 +
                                  4 * g) = round4<E>(sv * fv);
    }
  }
}

template <class E, int HD, int ROWS, int KEYS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void packed_bwd_kernel(const PackArgs a, Group gr, Mix mix, RowVecs rv) {
  __shared__ __attribute__((aligned(1024))) short buf0[kBuf<HD>];
  __shared__ __attribute__((aligned(1024))) short buf1[kBuf<HD>];
  __shared__ float scale[NW][16];
  const int j = blockIdx.x % a.nkv, t = blockIdx.x / a.nkv;
  const int kt = mix.keys_before(t);
  if (mix.keys_before(t + 1) > kt) {
    if constexpr (KEYS <= 1)
      dkdv_split_block<E, HD, KEYS == 0>(a, gr, j, kt, mix, rv, buf0, buf1, scale);
    else
      dkdv_block<E, HD, KEYS == 2 ? 2 : 1>(a, gr, j, kt, mix, rv, buf0, buf1, scale);
  } else {
    if constexpr (ROWS == 0)
      dq_split_block<E, HD, KEYS == 0>(a, gr, j, t - kt, mix, rv, buf0, buf1, scale);
    else
      dq_block<E, HD, ROWS, KEYS == 0>(a, gr, j, t - kt, mix, rv, buf0, buf1);
  }
}

// The blocks' kinds.  rows: 0 keys over a workgroup's waves, else 16 times that a wave;
// keys: 0 and 1 the rows over a workgroup's waves, 2 over its two halves, 3 not;
// with 0 every block works out the rows' delta for itself.
//
// Fewer and longer chains of tiles against idle CUs, us of a call in a graph with
// changing inputs, bf16, the kind of smaller blocks first:
//   rows 0 or 1, with keys 1: one head of 128, 1 x 8000 117 / 140; 16 / 8 heads of 128,
//     1 x 512 25.1 / 22.2, 6 x 250 45 / 35; 32 / 8 of 64, 4 x 250 29.4 / 21.4
//   keys 1 or 2, with rows 1: 16 / 8 of 128, 1 x 512 22.2 / 25.4, 6 x 250 34.9 / 29.2;
//     32 / 8 of 64, 4 x 250 21.4 / 23.4
//   rows 1 or 2: 16 / 8 of 128, 6 x 417 53 / 47, 4 x 1000 106 / 97
//   keys 2 or 3, with rows 2: 16 / 8 of 128, 6 x 417, just below that border, 47 / 43, 4 x
//     1000 97 / 89; 32 / 8 of 64, 4 x 1000 91 / 94, 8 x 1024 181 / 169
// keys 0 saves the launch before and is longer by tile: with rows 1, 16 / 8 of 128, 8 x 77
// 14.9 / 15.8, with rows 0, 4 / 4 heads of 128, 2 x 500 19.9 / 17.6, one head 1 x 2000
// 45 / 28.
struct BwdPlan {
  int rows, keys;
};
BwdPlan bwd_plan(const PackArgs& a) {
  const long long rows = (long long)a.Tq * (a.nq / a.nkv), blocks = (long long)a.Tk / 16 * a.nkv;
  const bool far = a.Tk / a.n >= 1024, half = a.hd == 64;
  BwdPlan p{};
  p.rows = rows / 16 * a.nkv <= (far ? 512 : 256) ? 0 : rows / 128 * a.nkv >= 256 ? 2 : 1;
  p.keys = blocks <= (far ? 768 : half ? 512 : 384) && a.nq / a.nkv <= 32
               ? (rows / a.n <= 256 ? 0 : 1)
               : (blocks <= (half ? 3000 : 1280) ? 2 : 3);
  if (p.keys == 0 && p.rows == 2) p.rows = 1;
  return p;
}

template <class E, int HD>
hipError_t launch(const PackArgs& a, void* ws, hipStream_t st) {
  const Group gr = group_of(a);
  const long long R = (long long)a.Tq * a.nq;
  RowVecs rv = {(float*)ws, (float*)ws + R};
  if (a.Tq == 0 && a.Tk == 0) return hipSuccess;
  const BwdPlan p = bwd_plan(a);
  const int kr = p.rows, kk = p.keys;
  if (a.Tq && kk) {
    constexpr int RB = 256 / (HD / 8);
    const unsigned wgs = (unsigned)std::min<long long>((R + RB - 1) / RB, kDeltaWgs);
    hipLaunchKernelGGL((packed_delta_kernel<E, HD>), dim3(wgs), dim3(256), 0, st, a, gr.G, rv);
    LLMT_LAUNCH_CHECK();
  }
  Mix mix{};
  if (a.Tq) mix.nrows = row_tiles(a, kr == 0 ? 16 : 64 * kr);
  if (a.Tk) mix.nkeys = key_tiles(a, kk < 2 ? 16 : 16 << (kk - 1));
  const int nt = mix.nrows + mix.nkeys, k0 = mix.nkeys >> 2;
  mix.share = (((unsigned long long)(mix.nkeys - k0) << 32) + nt - k0 - 1) / (nt - k0);
  const auto kernel =
      kr == 0   ? (kk == 0   ? packed_bwd_kernel<E, HD, 0, 0>
                   : kk == 1 ? packed_bwd_kernel<E, HD, 0, 1>
                   : kk == 2 ? packed_bwd_kernel<E, HD, 0, 2>
                             : packed_bwd_kernel<E, HD, 0, 3>)
      : kr == 1 ? (kk == 0   ? packed_bwd_kernel<E, HD, 1, 0>
                   : kk == 1 ? packed_bwd_kernel<E, HD, 1, 1>
                   : kk == 2 ? packed_bwd_kernel<E, HD, 1, 2>
                             : packed_bwd_kernel<E, HD, 1, 3>)
                : (kk <= 1   ? packed_bwd_kernel<E, HD, 2, 1>
                   : kk == 2 ? packed_bwd_kernel<E, HD, 2, 2>
                             : packed_bwd_kernel<E, HD, 2, 3>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)nt * a.nkv), dim3(256), 0, st, a, gr, mix, rv);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

}  // namespace

size_t packed_bwd_workspace(const PackArgs& a) {
  return bwd_plan(a).keys ? (size_t)a.Tq * a.nq * 8 : 0;
}

hipError_t packed_bwd(const PackArgs& a, void* ws, hipStream_t st) {
  if (a.hd == 128) return a.bf16 ? launch<B16, 128>(a, ws, st) : launch<F16, 128>(a, ws, st);
  return a.bf16 ? launch<B16, 64>(a, ws, st) : launch<F16, 64>(a, ws, st);
}

}  // namespace llmt
