// packed_fwd.hip — forward of the packed attention: o = softmax(scale q k^T) v
// over the keys that a query may see, and the log of each row's sum of
// exponentials.  Rows, tiles and offsets: packed_attn.h.
//
// Query t of a sequence with ql queries and kl keys sees keys 0 .. t + kl - ql
// (its own position where the two are equally long); below 0 it sees none, its
// output is 0 and its lse -inf.  One pass over the keys with the running
// maximum and sum; the scores never leave registers.
//
// Long sequences are bound by issue: a wave's tile of 64 keys and 32 rows takes
// 64 matrix instructions of 17 cycles and some 250 vector ones, which hardly
// overlap those of the other wave on the SIMD.  1 x 8192 tokens, 16 / 8 heads of
// 128 in bf16: 270 to 277 us, 990 to 1015 TFLOP/s (a large library product reaches
// 1387); 1 x 16384, 32 / 8 heads of 64 in fp16, twice the exponentials a product: 1240
// to 1265 us, 870 to 885.  Many sequences end with the longest one's chain of tiles: 16 of 8192 tokens
// together 58 us, 630.  Single tokens wait for their keys: 8 tokens of 9001 keys
// 13.5 us in a graph with the join, 32 of 32000 31, 4.2 TB/s.
#include <algorithm>
#include <type_traits>

#include "packed_attn.h"

namespace llmt {

namespace {

// A tile of 32 keys of the running softmax for RW 16-row tiles of a wave:
// st holds raw scores (rows key, column row) and on return probabilities
// relative to the running maximum, times 2^PSH.  lim: the last key a lane's
// row sees.
template <class E, int RW, int DT, bool MASK>
__device__ __forceinline__ void softmax_tile(floatx4 (&st)[RW][2], float (&m)[RW], float (&l)[RW],
                                             floatx4 (&ot)[RW][DT], float sl2, int key0,
                                             const int (&lim)[RW], int lane) {
  const int g = lane >> 4;
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    float bm = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float s = st[r][mt][v];
        if (MASK) {
          s = key0 + mt * 16 + 4 * g + v <= lim[r] ? s : -INFINITY;
          st[r][mt][v] = s;
        }
        bm = fmaxf(bm, s);
      }
    bm = xg_max(bm);
    const float mn = fmaxf(m[r], bm * sl2);  // sl2 > 0: the maximum commutes with the scale
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m[r] - mu);
    m[r] = mn;
    const float shift = mu - E::PSH;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        st[r][mt][v] = __builtin_amdgcn_exp2f(fmaf(st[r][mt][v], sl2, -shift));
    float ps[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
      ps[mt] = (st[r][mt][0] + st[r][mt][1]) + (st[r][mt][2] + st[r][mt][3]);
    l[r] = l[r] * alpha + (ps[0] + ps[1]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) ot[r][dt] *= alpha;
  }
}

// The keys that the wave's rows do not see leave the scores of a tile.
template <int RW, int MT>
__device__ __forceinline__ void mask_tile(floatx4 (&st)[RW][MT], int key0, const int (&lim)[RW],
                                          int g) {
#pragma unroll
  for (int r = 0; r < RW; ++r)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        st[r][mt][v] = key0 + mt * 16 + 4 * g + v <= lim[r] ? st[r][mt][v] : -INFINITY;
}

// NW waves of 16 RW rows each walk all keys of the workgroup's rows, K and V
// in LDS tiles of 64 keys.  A wave's tiles are a pipeline of two stages in one
// straight block, so that matrix and vector instructions run side by side: the
// scores of tile i + 1 beside the exponentials, sums and roundings of tile i,
// then its output beside the maxima of tile i + 1.
//
// The maximum that a row's exponentials refer to follows the running one only
// when some row of the wave has left it by more than 2^kGrow: rescaling the
// output is then a branch that few tiles take, and what it saves in range is
// in the types.  Base-2 scores of 2^24 and more are even numbers in fp32, where
// m + 7 is a tie that rounds up for every other m, so that a maximum of m + 8 would
// not be followed; with the score's own rounding P times 2^PSH would reach 2^17,
// beyond fp16.  m + 6 is exact up to 2^25, and fp16's P 2^PSH stays at or below 2^15.
template <class E>
constexpr float kGrow = E::PSH ? 6.f : 7.f;

// Slower: 16 rows a wave at 16 sequences of 8192 tokens (71 us, 62 with 32), 64
// rows a wave, two groups of waves on halves of the keys, a third tile in flight.

template <class E, int HD, int NW, int RW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2)))
void packed_fwd_kernel(const PackArgs a, Group gr, int ntiles) {
  constexpr int QB = NW * RW * 16, KS = HD / 32, DT = HD / 16, TILE = BLK * HD;
  __shared__ __attribute__((aligned(1024))) short kbuf0[TILE];
  __shared__ __attribute__((aligned(1024))) short kbuf1[TILE];
  __shared__ __attribute__((aligned(1024))) short vbuf0[TILE];
  __shared__ __attribute__((aligned(1024))) short vbuf1[TILE];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int j = blockIdx.x % a.nkv;
  Tile x;
  if (!find<QB>(a, gr, blockIdx.x / a.nkv, ntiles, ntiles, x)) return;

  const short* kbase = (const short*)a.k.p + x.kstart * a.k.token + j * a.k.head;
  const short* vbase = (const short*)a.v.p + x.kstart * a.v.token + j * a.v.head;
  const int nkb = (x.kmax + BLK - 1) / BLK;
  KeyDma<HD, NW, BLK> dk, dv;
  dk.init(a.k.token, w);
  dv.init(a.v.token, w);
  if (nkb > 0) dk.issue(kbase, a.k.token, 0, x.klen, kbuf0, w);
  const int left = x.rows - x.row0 - w * RW * 16;  // rows from the wave's first on
  const int nfull = (x.t0 + x.shift + 1) / BLK;  // tiles that every row sees whole
  short8v qf[RW][KS];
  int lim[RW];
  int at[RW], hq[RW];  // token and query head
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int i = min(w * RW * 16 + 16 * r + c, x.rows - 1 - x.row0);
    const int t = gr.div(x.rem + i), h = x.rem + i - t * gr.G;
    lim[r] = 16 * r + c < left ? x.t0 + t + x.shift : -1;
    at[r] = x.qstart + x.t0 + t;
    hq[r] = j * gr.G + h;
    const short* row = (const short*)a.q.p + at[r] * a.q.token + hq[r] * a.q.head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[r][ks] = *reinterpret_cast<const short8v*>(row + 32 * ks + 8 * g);
  }
  const float sl2 = a.scale * LOG2E;
  floatx4 ot[RW][DT], sa[RW][4], sb[RW][4];
  float m[RW], l[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) ot[r][i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  auto scores = [&](floatx4 (&st)[RW][4], const short* Ks) LLMT_INLINE {
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
      for (int r = 0; r < RW; ++r) st[r][mt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const short8v kf = frag_rm<HD>(Ks, mt * 16, ks, lane);
#pragma unroll
        for (int r = 0; r < RW; ++r) st[r][mt] = E::mfma(kf, qf[r][ks], st[r][mt]);
      }
    }
  };
  auto maxima = [&](const floatx4 (&st)[RW][4], float (&bm)[RW]) LLMT_INLINE {
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      bm[r] = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int v = 0; v < 4; ++v) bm[r] = fmaxf(bm[r], st[r][mt][v]);
      bm[r] = xg_max(bm[r]) * sl2;  // sl2 > 0: the maximum commutes with the scale
    }
  };
  auto follow = [&](const float (&bm)[RW]) LLMT_INLINE {
    bool grow = false;
#pragma unroll
    for (int r = 0; r < RW; ++r) grow = grow || bm[r] > m[r] + kGrow<E>;
    if (__ballot(grow)) {
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        const float mn = fmaxf(m[r], bm[r]);
        const float alpha = __builtin_amdgcn_exp2f(m[r] - (mn == -INFINITY ? 0.f : mn));
        m[r] = mn;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < DT; ++i) ot[r][i] *= alpha;
      }
    }
  };
  // probabilities of the scores st as operands, and their sums
  auto probs = [&](floatx4 (&st)[RW][4], short8v (&pb)[RW][2]) LLMT_INLINE {
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const float shift = (m[r] == -INFINITY ? 0.f : m[r]) - E::PSH;
      float ps[4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          st[r][mt][v] = __builtin_amdgcn_exp2f(fmaf(st[r][mt][v], sl2, -shift));
        ps[mt] = (st[r][mt][0] + st[r][mt][1]) + (st[r][mt][2] + st[r][mt][3]);
      }
      l[r] += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      pb[r][0] = pair_frag<E>(st[r][0], st[r][1]);
      pb[r][1] = pair_frag<E>(st[r][2], st[r][3]);
    }
  };
  auto output = [&](const short8v (&pb)[RW][2], const short* Vs) LLMT_INLINE {
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const short8v vf = frag_tr<HD>(Vs, dt * 16, jj, lane);
#pragma unroll
        for (int r = 0; r < RW; ++r) ot[r][dt] = E::mfma(vf, pb[r][jj], ot[r][dt]);
      }
  };
  // iteration i: K(i + 1) and V(i) have landed, K(i + 2) and V(i + 1) set out
  auto land = [&](int i, short* K0, short* V1) LLMT_INLINE {
    wait_vm<0>();
    tile_barrier();
    if (i + 2 < nkb) dk.issue(kbase, a.k.token, (i + 2) * BLK, x.klen, K0, w);
    if (i + 1 < nkb) dv.issue(vbase, a.v.token, (i + 1) * BLK, x.klen, V1, w);
  };
  // tile i where tile i + 1 takes no mask
  auto stage = [&](int i, floatx4 (&st)[RW][4], floatx4 (&nx)[RW][4], short* K0, short* K1,
                   short* V0, short* V1) LLMT_INLINE {
    land(i, K0, V1);
    short8v pb[RW][2];
    scores(nx, K1);
    probs(st, pb);
    float bm[RW];
    output(pb, V0);
    maxima(nx, bm);
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int u = 0; u < 2 * KS * RW; ++u) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      if (u % RW == 0 && u < 4 * KS * RW / 2 - 2 * RW) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      if (u >= 2 * KS * RW - 4) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, KS == 4 ? 5 : 10, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, KS == 4 ? 2 : 4, 0);
    }
#pragma unroll
    for (int u = 0; u < 2 * DT - 4; ++u) {
      __builtin_amdgcn_sched_group_barrier(0x008, RW, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4 * RW, 0);
    __builtin_amdgcn_sched_barrier(0);
    follow(bm);
  };
  if (nkb > 0) {
    wait_vm<0>();
    tile_barrier();
    if (nkb > 1) dk.issue(kbase, a.k.token, BLK, x.klen, kbuf1, w);
    dv.issue(vbase, a.v.token, 0, x.klen, vbuf0, w);
    scores(sa, kbuf0);
    if (nfull < 1) mask_tile<RW, 4>(sa, 0, lim, g);
    float bm[RW];
    maxima(sa, bm);
    follow(bm);
    // in pairs, so that the buffers are named statically
    int i = 0;
    for (; i + 2 < nfull; i += 2) {
      stage(i, sa, sb, kbuf0, kbuf1, vbuf0, vbuf1);
      stage(i + 1, sb, sa, kbuf1, kbuf0, vbuf1, vbuf0);
    }
    // the rest, masked: i is even
    for (; i < nkb; ++i) {
      const bool odd = i & 1;
      wait_lds();  // the reads of the tiles that the next ones replace have returned
      land(i, odd ? kbuf1 : kbuf0, odd ? vbuf0 : vbuf1);
      short8v pb[RW][2];
      probs(sa, pb);
      output(pb, odd ? vbuf1 : vbuf0);
      if (i + 1 < nkb) {
        scores(sa, odd ? kbuf0 : kbuf1);
        mask_tile<RW, 4>(sa, (i + 1) * BLK, lim, g);
        maxima(sa, bm);
        follow(bm);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const float lr = xg_sum(l[r]);
    const float inv = lr > 0.f || lr != lr ? 1.0f / lr : 0.f;
    if (16 * r + c < left) {
      short* o = (short*)a.o.p + at[r] * a.o.token + hq[r] * a.o.head;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<short4v*>(o + dt * 16 + 4 * g) = round4<E>(ot[r][dt] * inv);
      if (g == 0) a.lse[(long long)at[r] * a.nq + hq[r]] = (m[r] + (__log2f(lr) - E::PSH)) * LN2;
    }
  }
}

// Few rows: a workgroup takes 16 RW rows and one of nsplit parts of their keys,
// in 32-key tiles that its four or eight waves take in turn, each through LDS of its own
// and without a barrier in the loop; the waves' results meet in LDS.  It waits
// for loads, not for the matrix units, so probabilities enter the product in two
// parts (pair_split), and nothing but the result is rounded to the type.  With
// several parts the result goes to the workspace as (max, sum) and the
// unnormalised output, for packed_join_kernel.
constexpr int FS_KEYS = 32;
struct Parts {
  int nsplit;
  float* o;    // [nsplit][Tq nq][hd]
  float2* ml;  // [nsplit][Tq nq]: base-2 maximum, sum
};

template <class E, int HD, int RW, int NW>
__global__ __launch_bounds__(NW * 64, 2) void packed_fwd_split_kernel(const PackArgs a, Group gr,
                                                                      int ntiles, Parts parts) {
  constexpr int QB = RW * 16, KS = HD / 32, DT = HD / 16, FT = FS_KEYS * HD;
  // a wave's K and V tile; later its output, 16 rows x HD fp32 each
  __shared__ __attribute__((aligned(1024))) short kbuf[NW * FT];
  __shared__ __attribute__((aligned(1024))) short vbuf[NW * FT];
  __shared__ float2 ml[NW][QB];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int j = blockIdx.x % a.nkv;
  const int part = blockIdx.y;
  Tile x;
  if (!find<QB>(a, gr, blockIdx.x / a.nkv, ntiles, ntiles, x)) return;
  const short* kbase = (const short*)a.k.p + x.kstart * a.k.token + j * a.k.head;
  const short* vbase = (const short*)a.v.p + x.kstart * a.v.token + j * a.v.head;
  const int nkt_all = (x.kmax + FS_KEYS - 1) / FS_KEYS;
  const int per = (nkt_all + parts.nsplit - 1) / parts.nsplit;
  const int kt0 = part * per + w, nkt = min(nkt_all, (part + 1) * per);
  short* const Ks = kbuf + w * FT;
  short* const Vs = vbuf + w * FT;
  using Dma = KeyDma<HD, 1, FS_KEYS>;
  Dma dk, dv;
  dk.init(a.k.token, 0);
  dv.init(a.v.token, 0);
  if (kt0 < nkt) {
    dk.issue(kbase, a.k.token, kt0 * FS_KEYS, x.klen, Ks, 0);
    dv.issue(vbase, a.v.token, kt0 * FS_KEYS, x.klen, Vs, 0);
  }
  const int left = x.rows - x.row0;
  const int wfirst = x.t0 + x.shift;
  short8v qf[RW][KS];
  int lim[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int i = min(16 * r + c, left - 1);
    const int t = gr.div(x.rem + i), h = x.rem + i - t * gr.G;
    lim[r] = 16 * r + c < left ? x.t0 + t + x.shift : -1;
    const short* row = (const short*)a.q.p + (long long)(x.qstart + x.t0 + t) * a.q.token +
                       (j * gr.G + h) * a.q.head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[r][ks] = *reinterpret_cast<const short8v*>(row + 32 * ks + 8 * g);
  }
  const float sl2 = a.scale * LOG2E;
  floatx4 ot[RW][DT];
  float m[RW], l[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) ot[r][i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  for (int kt = kt0; kt < nkt; kt += NW) {
    const bool next = kt + NW < nkt;
    if (kt != kt0) wait_vm<Dma::CH>();  // this K tile (the V tile may be in flight)
    else wait_vm<0>();
    asm volatile("" ::: "memory");
    floatx4 st[RW][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int r = 0; r < RW; ++r) st[r][mt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const short8v kf = frag_rm<HD>(Ks, mt * 16, ks, lane);
#pragma unroll
        for (int r = 0; r < RW; ++r) st[r][mt] = E::mfma(kf, qf[r][ks], st[r][mt]);
      }
    }
    wait_lds();  // the reads of the K tile have returned
    asm volatile("" ::: "memory");
    if (next) dk.issue(kbase, a.k.token, (kt + NW) * FS_KEYS, x.klen, Ks, 0);
    if (kt * FS_KEYS + FS_KEYS - 1 <= wfirst && left >= QB)
      softmax_tile<E, RW, DT, false>(st, m, l, ot, sl2, kt * FS_KEYS, lim, lane);
    else
      softmax_tile<E, RW, DT, true>(st, m, l, ot, sl2, kt * FS_KEYS, lim, lane);
    short8v pb[RW], pl[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) pair_split<E>(st[r][0], st[r][1], pb[r], pl[r]);
    if (next) wait_vm<Dma::CH>();  // this V tile (the next K tile may be in flight)
    else wait_vm<0>();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const short8v vf = frag_tr<HD>(Vs, dt * 16, 0, lane);
#pragma unroll
      for (int r = 0; r < RW; ++r) ot[r][dt] = E::mfma(vf, pb[r], E::mfma(vf, pl[r], ot[r][dt]));
    }
    wait_lds();
    asm volatile("" ::: "memory");
    if (next) dv.issue(vbase, a.v.token, (kt + NW) * FS_KEYS, x.klen, Vs, 0);
  }

  // the waves' outputs meet: the first 16 rows where the wave's K tile was, the
  // second where its V tile was, 16-byte pieces swizzled by the row; wave w then
  // takes rows 4 w .. 4 w + 3 of each sixteen, 16 lanes a row
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    float* const xo = reinterpret_cast<float*>(r ? vbuf : kbuf) + (w * 16 + c) * HD;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<floatx4*>(xo + (((4 * dt + g) ^ c) << 2)) = ot[r][dt];
    const float lw = xg_sum(l[r]);
    if (g == 0) ml[w][16 * r + c] = make_float2(m[r], lw);
  }
  __syncthreads();
  if (w >= 4) return;
  constexpr int PC = HD / 64;  // 16-byte pieces a lane
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const float* const xo = reinterpret_cast<const float*>(r ? vbuf : kbuf);
    const int qi = 4 * w + g, i = 16 * r + qi;
    float M = -INFINITY;
#pragma unroll
    for (int u = 0; u < NW; ++u) M = fmaxf(M, ml[u][i].x);
    const float mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    floatx4 o[PC];
#pragma unroll
    for (int e = 0; e < PC; ++e) o[e] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float2 p = ml[u][i];
      const float f = __builtin_amdgcn_exp2f(p.x - mu);
      L = fmaf(p.y, f, L);
      const float* row = xo + (u * 16 + qi) * HD;
#pragma unroll
      for (int e = 0; e < PC; ++e)
        o[e] += *reinterpret_cast<const floatx4*>(row + (((PC * c + e) ^ qi) << 2)) * f;
    }
    if (i < left) {
      const int t = gr.div(x.rem + i), h = j * gr.G + x.rem + i - t * gr.G;
      const long long tok = x.qstart + x.t0 + t;
      if (parts.nsplit > 1) {
        const long long at = (long long)part * a.Tq * a.nq + tok * a.nq + h;
#pragma unroll
        for (int e = 0; e < PC; ++e)
          *reinterpret_cast<floatx4*>(parts.o + at * HD + (PC * c + e) * 4) = o[e];
        if (c == 0) parts.ml[at] = make_float2(M, L);
      } else {
        const float inv = L > 0.f || L != L ? 1.0f / L : 0.f;
        short* op = (short*)a.o.p + tok * a.o.token + h * a.o.head;
#pragma unroll
        for (int e = 0; e < PC; ++e)
          *reinterpret_cast<short4v*>(op + (PC * c + e) * 4) = round4<E>(o[e] * inv);
        if (c == 0) a.lse[tok * a.nq + h] = (M + (__log2f(L) - E::PSH)) * LN2;
      }
    }
  }
}

// The parts of a row joined in their order: HD / 4 lanes a row; GR groups of so
// many lanes take every GR-th part, and their sums meet in LDS.
template <class E, int HD, int GR>
__global__ __launch_bounds__(256) void packed_join_kernel(const PackArgs a, Parts parts) {
  constexpr int LR = HD / 4, RB = 256 / LR / GR;
  __shared__ float ml[GR * RB][2];
  __shared__ __attribute__((aligned(16))) float sums[GR > 1 ? GR * RB * HD : 1];
  const long long R = (long long)a.Tq * a.nq;
  const int grp = threadIdx.x / LR, q = grp % GR, d = (threadIdx.x % LR) * 4;
  const long long row = (long long)blockIdx.x * RB + grp / GR;
  const bool on = row < R;
  float M = -INFINITY, L = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  if (on) {
#pragma unroll 8
    for (int s = q; s < parts.nsplit; s += GR) M = fmaxf(M, parts.ml[s * R + row].x);
    const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll 8
    for (int s = q; s < parts.nsplit; s += GR) {
      const float2 p = parts.ml[s * R + row];
      const float f = __builtin_amdgcn_exp2f(p.x - mu);
      L = fmaf(p.y, f, L);
      o += *reinterpret_cast<const floatx4*>(parts.o + (s * R + row) * HD + d) * f;
    }
  }
  if constexpr (GR > 1) {
    if (d == 0) {
      ml[grp][0] = M;
      ml[grp][1] = L;
    }
    *reinterpret_cast<floatx4*>(sums + grp * HD + d) = o;
    __syncthreads();
    if (q > 0) return;
#pragma unroll
    for (int u = 0; u < GR; ++u) M = fmaxf(M, ml[grp + u][0]);
    const float mu = M == -INFINITY ? 0.f : M;
    L = 0.f;
    o = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < GR; ++u) {
      const float f = __builtin_amdgcn_exp2f(ml[grp + u][0] - mu);
      L = fmaf(ml[grp + u][1], f, L);
      o += *reinterpret_cast<const floatx4*>(sums + (grp + u) * HD + d) * f;
    }
  }
  if (!on) return;
  const long long t = row / a.nq, h = row - t * a.nq;
  const float inv = L > 0.f || L != L ? 1.0f / L : 0.f;
  *reinterpret_cast<short4v*>((short*)a.o.p + t * a.o.token + h * a.o.head + d) =
      round4<E>(o * inv);
  if (d == 0) a.lse[row] = (M + (__log2f(L) - E::PSH)) * LN2;
}

// The kernel and its split.
struct FwdPlan {
  int nw, rw;  // nw 0: packed_fwd_split_kernel
  int nsplit, sw;  // its parts and waves
};
FwdPlan fwd_plan(const PackArgs& a) {
  const long long rows = (long long)a.Tq * (a.nq / a.nkv);
  const long long n = std::min(a.n, a.Tq);
  // 32 rows a wave where that gives every CU two workgroups, 16 where those do (us in a
  // graph with changing inputs, 32 / 16: 32 / 8 heads of 64, 4 x 1000 tokens 39 / 38, 16 / 8
  // of 128, 16 x 512 46 / 58, 4 x 1000, a little below that border, 33 / 37)
  if (rows / 128 * a.nkv >= 512) return {4, 2, 1, 0};
  if (rows / 64 * a.nkv >= 256) return {4, 1, 1, 0};
  // tiles of 16 rows, or of 32 where that many workgroups would not run at once
  const int rw = rows / 16 * a.nkv > 512 ? 2 : 1;
  const long long wgs = std::max<long long>(1, std::max(rows / (16 * rw), n) * a.nkv);
  const long long keys = a.Tk / std::max<long long>(1, n);
  const long long most = std::min<long long>(64, std::max<long long>(1, keys / 128));
  // A CU for each workgroup and few keys: eight waves, no parts.  us in a graph with
  // changing inputs, four waves in parts / eight: single tokens of 500 keys 9.1 / 7.8, of
  // 1000 10.4 / 15.5, 8 of 1000 14.6 / 17.0 (32 of 1000, where every CU has a workgroup
  // without parts, 34 / 25); whole tiles, whose parts are larger: 4 heads, 2 x 500 15.9 /
  // 8.1, 16 / 8 heads, 128 tokens behind 900 19.6 / 12.1, one head, 1 x 4000 (the same
  // inputs) 25.1 / 21.1
  const long long seen = keys - a.Tq / std::max<long long>(1, n) / 2;
  if (rw == 1 && wgs <= 256 && seen <= (rows / 16 >= n ? 2048 : 768)) return {0, 1, 1, 8};
  return {0, rw, (int)std::min(most, std::max<long long>(1, 768 / wgs)), 4};
}

template <class E, int HD>
hipError_t launch(const PackArgs& a, void* ws, hipStream_t st) {
  const FwdPlan p = fwd_plan(a);
  const Group gr = group_of(a);
  if (p.nw) {
    const int nt = row_tiles(a, p.nw * p.rw * 16);
    const dim3 grid((unsigned)nt * a.nkv);
    if (p.rw == 2)
      hipLaunchKernelGGL((packed_fwd_kernel<E, HD, 4, 2>), grid, dim3(256), 0, st, a, gr, nt);
    else
      hipLaunchKernelGGL((packed_fwd_kernel<E, HD, 4, 1>), grid, dim3(256), 0, st, a, gr, nt);
    LLMT_LAUNCH_CHECK();
    return hipSuccess;
  }
  Parts parts = {p.nsplit, nullptr, nullptr};
  const long long R = (long long)a.Tq * a.nq;
  if (p.nsplit > 1) {
    parts.o = (float*)ws;
    parts.ml = (float2*)(parts.o + p.nsplit * R * HD);
  }
  const int nt = row_tiles(a, 16 * p.rw);
  const dim3 grid((unsigned)nt * a.nkv, p.nsplit);
  if (p.rw == 2)
    hipLaunchKernelGGL((packed_fwd_split_kernel<E, HD, 2, 4>), grid, dim3(256), 0, st, a, gr, nt, parts);
  else if (p.sw == 8)
    hipLaunchKernelGGL((packed_fwd_split_kernel<E, HD, 1, 8>), grid, dim3(512), 0, st, a, gr, nt, parts);
  else
    hipLaunchKernelGGL((packed_fwd_split_kernel<E, HD, 1, 4>), grid, dim3(256), 0, st, a, gr, nt, parts);
  LLMT_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    // few rows and many parts: a workgroup a row (one token of 8000 keys, 62 parts: 15.7
    // us, 28.2 with a row's lanes walking all of them)
    constexpr int G = 256 / (HD / 4);
    if (p.nsplit >= 4)
      hipLaunchKernelGGL((packed_join_kernel<E, HD, G>), dim3((unsigned)R), dim3(256), 0, st, a, parts);
    else
      hipLaunchKernelGGL((packed_join_kernel<E, HD, 1>), dim3((unsigned)((R + G - 1) / G)), dim3(256),
                         0, st, a, parts);
    LLMT_LAUNCH_CHECK();
  }
  return hipSuccess;
}

}  // namespace

size_t packed_fwd_workspace(const PackArgs& a) {
  if (a.Tq == 0) return 0;
  const FwdPlan p = fwd_plan(a);
  return p.nsplit > 1 ? (size_t)p.nsplit * a.Tq * a.nq * (a.hd * 4 + 8) : 0;
}

hipError_t packed_fwd(const PackArgs& a, void* ws, hipStream_t st) {
  if (a.Tq == 0) return hipSuccess;
  if (a.hd == 128) return a.bf16 ? launch<B16, 128>(a, ws, st) : launch<F16, 128>(a, ws, st);
  return a.bf16 ? launch<B16, 64>(a, ws, st) : launch<F16, 64>(a, ws, st);
}

}  // namespace llmt
