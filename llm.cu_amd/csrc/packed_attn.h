// packed_attn.h — shared pieces of the packed attention (packed_fwd.hip,
// packed_bwd.hip): causal attention with grouped heads over sequences packed
// one behind another, fp16 or bf16, head_dim 64 or 128.
//
// Rows.  For KV head j a sequence's queries are rows r = G t + i: token t, i
// the query head within j's group of G = nq / nkv.  A tile is a run of rows, so
// the K and V that a tile reads serve the whole group, and a group's dK and dV
// are one sum over rows, whatever G is.
//
// Tiles.  The sequences' lengths are on the device only.  Sequence s starts at
// row e_s and has ceil(rows / QB) tiles of QB rows; giving it the tile numbers
// from floor(e_s / QB) + s on leaves room for them and makes the start of each
// sequence known without a sum over the ones before, so a workgroup finds its
// sequence by a search over the offsets, no list is built, and a launch has
// floor(rows / QB) + sequences tiles, of which those behind a sequence's end
// leave at once.  Tokens before the first and behind the last sequence are two
// more sequences, whose queries have no keys.  Offsets are clamped to [0, T]:
// whatever they hold, no access leaves the arrays.
//
// The MFMA conventions, the 64-row LDS tiles with their swizzle and the DMA
// into them are those of attn_common.h, for both widths.
#pragma once

#include "ops.h"

namespace llmt {

namespace {

constexpr int BLK = 64;  // rows per LDS tile
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) void lds_void;

// The two element types.  PSH: probabilities enter the second product times
// 2^PSH.  An fp16 below 2^-14 loses bits, which a probability of one key in
// many is; times 2^8 the largest, 2^7 in the forward, is still in range.
struct F16 {
  typedef _Float16 T;
  static constexpr int PSH = 8;
  __device__ static __forceinline__ floatx4 mfma(short8v a, short8v b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a),
                                                  __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
};
struct B16 {
  typedef __bf16 T;
  static constexpr int PSH = 0;
  __device__ static __forceinline__ floatx4 mfma(short8v a, short8v b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  }
};

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }  // lgkmcnt(0)

__device__ __forceinline__ void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr int kRsrcWord3 = 0x00020000;  // raw buffer, 32-bit data format
__device__ __forceinline__ void buffer_lds16(__amdgpu_buffer_rsrc_t rs, void* lds, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)lds, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void buffer_lds4(__amdgpu_buffer_rsrc_t rs, void* lds, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)lds, 4, off, 0, 0, 0);
}
// A buffer of `bytes` from p (a size that the host's bounds keep below 2^31).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, kRsrcWord3);
}

// Offset (elements) of elements 8 p .. 8 p + 7 of tile row r: the 16-byte
// piece p sits in slot p ^ (r mod pieces a row).
template <int HD>
__device__ __forceinline__ int toff(int r, int p) {
  return r * HD + ((p ^ (r & (HD / 8 - 1))) << 3);
}

// Tile rows into LDS, 1 KB a wave instruction: chunk ch holds RPC rows, lane l
// fills slot l % P of row RPC ch + l / P.  Rows past the end arrive as zeros.
template <int HD, int NW, int ROWS>
struct KeyDma {  // rows `token` elements apart: keys, values
  static constexpr int P = HD / 8, RPC = 64 / P, CH = ROWS / RPC / NW;
  unsigned off[CH];
  __device__ __forceinline__ void init(long long token, int w) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int r = RPC * (w + NW * i) + lane / P;
      off[i] = (unsigned)(r * (int)token * 2 + (((lane & (P - 1)) ^ (r & (P - 1))) << 4));
    }
  }
  // rows r0 .. of the n rows at src
  __device__ __forceinline__ void issue(const short* src, long long token, int r0, int n,
                                        short* tile, int w) const {
    const int left = min(n - r0, ROWS);
    const __amdgpu_buffer_rsrc_t rs =
        buffer_of(src + (long long)r0 * token, left > 0 ? ((left - 1) * (int)token + HD) * 2 : 0);
#pragma unroll
    for (int i = 0; i < CH; ++i) buffer_lds16(rs, tile + (w + NW * i) * 512, off[i]);
  }
};

// Quotient by G of a row below 2^16.
struct Group {
  int G;
  unsigned magic;  // ceil(2^32 / G); 0 for G = 1
  __device__ __forceinline__ int div(int x) const {
    return magic ? (int)__umulhi((unsigned)x, magic) : x;
  }
};

// Query-side rows (token t, head i of the group at t * token + i * head) in
// tiles of whole tokens, TR = ROWS / G * G rows: a lane's offsets are then the
// same in every tile.  Tile rows from TR on, and rows past the end, are zeros.
template <int HD, int NW, int ROWS = BLK>
struct RowDma {
  static constexpr int P = HD / 8, RPC = 64 / P, CH = ROWS / RPC / NW;
  unsigned off[CH];
  __device__ __forceinline__ void init(long long token, long long head, Group gr, int tr, int w) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int r = RPC * (w + NW * i) + lane / P;
      const int t = gr.div(r), h = r - t * gr.G;
      off[i] = r < tr ? (unsigned)((t * (int)token + h * (int)head) * 2 +
                                   (((lane & (P - 1)) ^ (r & (P - 1))) << 4))
                      : 0x80000000u;
    }
  }
  // tokens t0 .. t0 + tokens - 1 of the n tokens at src
  __device__ __forceinline__ void issue(const short* src, long long token, long long head, Group gr,
                                        int t0, int n, int tokens, short* tile, int w) const {
    const int left = min(n - t0, tokens);
    const __amdgpu_buffer_rsrc_t rs =
        buffer_of(src + (long long)t0 * token,
                  left > 0 ? ((left - 1) * (int)token + (gr.G - 1) * (int)head + HD) * 2 : 0);
    if (left < tokens) {  // heads may lie further apart than tokens: a token past the end inside
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int r = RPC * (w + NW * i) + (int)(threadIdx.x & 63) / P;
        buffer_lds16(rs, tile + (w + NW * i) * 512, r < left * gr.G ? off[i] : 0x80000000u);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) buffer_lds16(rs, tile + (w + NW * i) * 512, off[i]);
  }
};

// src[i0 .. i0 + 63] (fp32, zeros past n) into LDS by one wave.
__device__ __forceinline__ void dma_vec64(const float* src, int i0, int n, float* dst) {
  const int left = min(n - i0, 64);
  buffer_lds4(buffer_of(src + i0, left > 0 ? left * 4 : 0), dst, (threadIdx.x & 63) * 4);
}

// Row fragment: rows m0 + c, elements 32 ks + 8 g .. + 7.
template <int HD>
__device__ __forceinline__ short8v frag_rm(const short* t, int m0, int ks, int lane) {
  return *reinterpret_cast<const short8v*>(t + toff<HD>(m0 + (lane & 15), 4 * ks + (lane >> 4)));
}
// Column fragment for the paired-accumulator k order: lane (c, g) gets
// tile[32 j + 4 g + i][d0 + c] (i < 4) and tile[32 j + 16 + 4 g + i - 4][d0 + c].
template <int HD>
__device__ __forceinline__ short8v frag_tr(const short* t, int d0, int j, int lane) {
  const int jl = lane & 15;
  const int r = 32 * j + 4 * (lane >> 4) + (jl >> 2);
  const int col = d0 + 4 * (jl & 3), off = col & 7;
  const short4v lo =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(t + toff<HD>(r, col >> 3) + off));
  const short4v hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(t + toff<HD>(r + 16, col >> 3) + off));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// B fragment of two accumulator tiles, rounded to nearest.
template <class E>
__device__ __forceinline__ short8v pair_frag(const floatx4& a, const floatx4& b) {
  typedef typename E::T T8 __attribute__((ext_vector_type(8)));
  T8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = (typename E::T)a[i];
    r[4 + i] = (typename E::T)b[i];
  }
  return __builtin_bit_cast(short8v, r);
}
// The same in two parts, the rounded value and what it left out: twice the bits.
template <class E>
__device__ __forceinline__ void pair_split(const floatx4& a, const floatx4& b, short8v& hi,
                                           short8v& lo) {
  typedef typename E::T T8 __attribute__((ext_vector_type(8)));
  T8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = i < 4 ? a[i & 3] : b[i & 3];
    h[i] = (typename E::T)x;
    l[i] = (typename E::T)(x - (float)h[i]);
  }
  hi = __builtin_bit_cast(short8v, h);
  lo = __builtin_bit_cast(short8v, l);
}
template <class E>
__device__ __forceinline__ short4v round4(const floatx4& a) {
  typedef typename E::T T4 __attribute__((ext_vector_type(4)));
  T4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (typename E::T)a[i];
  return __builtin_bit_cast(short4v, r);
}

// One side's span in sequence s of 0 .. n + 1 (0 and n + 1: the tokens before
// the first and behind the last sequence).
__device__ __forceinline__ int clamp_off(const int* off, int i, int T) {
  return min(max(off[i], 0), T);
}
struct Span {
  int start, len;
};
__device__ __forceinline__ Span span_of(const int* off, int s, int n, int T) {
  const int a = s == 0 ? 0 : clamp_off(off, s - 1, T);
  const int b = s == n + 1 ? T : clamp_off(off, s, T);
  return {a, max(b - a, 0)};
}

// The sequence of tile t and the tile's number in it, `per` rows a token.
template <int QB>
__device__ __forceinline__ int find_tile(const int* off, int n, int T, int per, int t, int* block) {
  const int lane = threadIdx.x & 63;
  auto first = [&](int s) {  // the sequence's first tile
    const int e = s == 0 ? 0 : clamp_off(off, s - 1, T);
    return (int)((unsigned)e * (unsigned)per / QB) + s;
  };
  int lo = 0, hi = n + 2;  // first(lo) <= t < first(hi)
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64;
    const int s = lo + lane * step;
    const bool le = s < hi && first(s) <= t;
    const int k = max(1, (int)__popcll(__ballot(le)));
    lo += (k - 1) * step;
    hi = min(hi, lo + step);
  }
  const int s = lo + lane;
  const bool le = s < hi && first(s) <= t;
  const int k = max(1, (int)__popcll(__ballot(le)));
  lo = __builtin_amdgcn_readfirstlane(lo + k - 1);
  *block = __builtin_amdgcn_readfirstlane(t - first(lo));
  return lo;
}

// Longest first.  A workgroup's time follows the number of keys its last row
// sees (rows that see its first key, in dK/dV), and the sequences' lengths
// differ: workgroup t takes the t-th tile in falling order of that number, in
// steps of 64.  Up to kOrdered sequences a wave holds them all, so it finds the
// step by bisection over the count of tiles above it, then the sequence among
// those that have tiles of the step (contiguous blocks in each).  More sequences
// than that are as good in any order: find_tile.
constexpr int kOrderedRegs = 4, kOrdered = 64 * kOrderedRegs - 2;

__device__ __forceinline__ int wave_isum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);
  auto r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  v = (int)(r[0] + r[1]);
  r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane((int)(r[0] + r[1]));
}

// Inclusive sums over the lanes.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15: rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31: rows 2, 3
  return v;
}
__device__ __forceinline__ int wave_max_int(int v) {
  auto up = [](int x, int y) { return x > y ? x : y; };
  v = up(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
  v = up(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
  v = up(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
  v = up(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
  auto r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  v = up((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane(up((int)r[0], (int)r[1]));
}

// Blocks of a sequence with more than x of what they walk (x < 0: all).  ROWS:
// blocks of QB rows walking keys, the last blocks the longest; else blocks of QB
// keys walking tokens, the first ones the longest.
struct SeqLens {
  int ql, kl, qstart, kstart;
};
template <bool ROWS, int QB>
__device__ __forceinline__ int blocks_above(SeqLens s, int G, int x) {
  const int nb = ((ROWS ? s.ql * G : s.kl) + QB - 1) / QB;
  if (x < 0) return nb;
  if constexpr (ROWS) {
    const int y = x - (s.kl - s.ql);  // tokens from y on see more than x keys
    return y >= s.ql ? 0 : y < 0 ? nb : nb - (int)((unsigned)(y * G) / QB);
  } else {
    return s.ql <= x ? 0 : min(nb, max(s.kl - x + QB - 1, 0) / QB);
  }
}

// The t-th tile: its sequence's spans and its block in it; false behind the
// last.  level and top: its step and the bound of all.
template <bool ROWS, int QB>
__device__ __forceinline__ bool nth_longest(const PackArgs& a, int G, int t, SeqLens* seq,
                                            int* block, int* level, int* top) {
  const int lane = threadIdx.x & 63;
  SeqLens s[kOrderedRegs];
  int longest = 0;
#pragma unroll
  for (int u = 0; u < kOrderedRegs; ++u) {
    const int i = 64 * u + lane;
    s[u] = {0, 0, 0, 0};
    if (64 * u < a.n + 2 && i < a.n + 2) {
      const bool in = i > 0 && i <= a.n;
      const Span q = span_of(a.qoff, i, a.n, a.Tq), k = span_of(a.koff, i, a.n, a.Tk);
      // the tokens outside of all sequences walk nothing
      s[u] = {ROWS || in ? q.len : 0, !ROWS || in ? k.len : 0, q.start, k.start};
    }
    longest = max(longest, ROWS ? s[u].kl : s[u].ql);
  }
  auto above = [&](int k) {  // tiles above step k: x = -1, 0, 64, 128, ..
    const int x = k == 0 ? -1 : 64 * (k - 1);
    int n = 0;
#pragma unroll
    for (int u = 0; u < kOrderedRegs; ++u)
      if (64 * u < a.n + 2) n += blocks_above<ROWS, QB>(s[u], G, x);
    return wave_isum(n);
  };
  longest = wave_max_int(longest);
  int lo = 0, hi = (longest + 63) / 64 + 1;  // above(lo) > t >= above(hi)
  *top = hi;
  if (above(0) <= t) return false;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (above(mid) > t) lo = mid;
    else hi = mid;
  }
  *level = lo;
  int r = t - above(hi);
  const int x0 = lo == 0 ? -1 : 64 * (lo - 1), x1 = 64 * lo;
#pragma unroll
  for (int u = 0; u < kOrderedRegs; ++u) {
    if (64 * u >= a.n + 2) break;
    const int c0 = blocks_above<ROWS, QB>(s[u], G, x0), c1 = blocks_above<ROWS, QB>(s[u], G, x1);
    const int sum = wave_scan(c0 - c1);
    const unsigned long long past = __ballot(sum > r);
    if (past) {
      const int l = __ffsll(past) - 1;
      const int i = r - (sum - (c0 - c1));
      const int nb = ((ROWS ? s[u].ql * G : s[u].kl) + QB - 1) / QB;
      *seq = {__builtin_amdgcn_readlane(s[u].ql, l), __builtin_amdgcn_readlane(s[u].kl, l),
              __builtin_amdgcn_readlane(s[u].qstart, l), __builtin_amdgcn_readlane(s[u].kstart, l)};
      *block = __builtin_amdgcn_readlane(ROWS ? nb - c0 + i : c1 + i, l);
      return true;
    }
    r -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;  // (of malformed offsets)
}

// A wave of a long tile goes before its neighbours': the launch ends with the
// longest tile.
__device__ __forceinline__ void set_priority(int level, int top) {
  if (4 * level >= 3 * top) __builtin_amdgcn_s_setprio(3);
  else if (2 * level >= top) __builtin_amdgcn_s_setprio(2);
  else if (4 * level >= top) __builtin_amdgcn_s_setprio(1);
}

// The tiles of few rows run at once: any order.  Up to 62 sequences a wave holds
// them all, and one load finds the t-th tile (numbered as in find_tile) and its
// spans; its block may lie behind the sequence's end.
template <bool ROWS, int QB>
__device__ __forceinline__ void any_tile(const PackArgs& a, int G, int t, SeqLens* seq, int* block) {
  const int i = threadIdx.x & 63, last = a.n + 1;
  const bool in = i > 0 && i < last;
  Span q = {0, 0}, k = {0, 0};
  if (i <= last) {
    if (ROWS || in) q = span_of(a.qoff, i, a.n, a.Tq);
    if (!ROWS || in) k = span_of(a.koff, i, a.n, a.Tk);
  }
  const int first = (int)((ROWS ? (unsigned)q.start * G : (unsigned)k.start) / QB) + i;
  const int l = max(1, (int)__popcll(__ballot(i <= last && first <= t))) - 1;
  *seq = {__builtin_amdgcn_readlane(q.len, l), __builtin_amdgcn_readlane(k.len, l),
          __builtin_amdgcn_readlane(q.start, l), __builtin_amdgcn_readlane(k.start, l)};
  *block = t - __builtin_amdgcn_readlane(first, l);
}

// Tile t of nt in a launch of `all` a KV head: the spans of its sequence and
// its block in it, which may lie behind the sequence's end (or, with malformed
// offsets, before it).
template <bool ROWS, int QB>
__device__ __forceinline__ bool pick_tile(const PackArgs& a, int G, int t, int nt, int all,
                                          SeqLens* seq, int* block) {
  if (all * a.nkv > 512 && a.n <= kOrdered) {
    int level, top;
    if (!nth_longest<ROWS, QB>(a, G, t, seq, block, &level, &top)) return false;
    set_priority(level, top);
    return true;
  }
  const int at = ROWS ? nt - 1 - t : t;
  if (a.n <= 62) {
    any_tile<ROWS, QB>(a, G, at, seq, block);
    return true;
  }
  const int s = ROWS ? find_tile<QB>(a.qoff, a.n, a.Tq, G, at, block)
                     : find_tile<QB>(a.koff, a.n, a.Tk, 1, at, block);
  const bool in = s > 0 && s <= a.n;  // the tokens outside of all sequences: no other side
  const Span none = {0, 0};
  const Span q = ROWS || in ? span_of(a.qoff, s, a.n, a.Tq) : none;
  const Span k = !ROWS || in ? span_of(a.koff, s, a.n, a.Tk) : none;
  *seq = {q.len, k.len, q.start, k.start};
  return true;
}

// What a workgroup works on: QB rows from row0 of a sequence, for KV head j.
struct Tile {
  int qstart, rows, row0, shift, kstart, klen, kmax;
  int t0, rem;  // the first row's token and head in the group
};
template <int QB>
__device__ __forceinline__ bool find(const PackArgs& a, Group gr, int t, int ntiles, int all, Tile& x) {
  int blk;
  SeqLens s;
  if (!pick_tile<true, QB>(a, gr.G, t, ntiles, all, &s, &blk)) return false;
  x.qstart = s.qstart;
  x.rows = s.ql * gr.G;
  if (blk < 0 || blk >= (x.rows + QB - 1) / QB) return false;
  x.row0 = blk * QB;
  x.shift = s.kl - s.ql;
  x.kstart = s.kstart;
  x.klen = s.kl;
  x.t0 = x.row0 / gr.G;
  x.rem = x.row0 - x.t0 * gr.G;
  const int last = x.t0 + gr.div(x.rem + min(QB, x.rows - x.row0) - 1);
  x.kmax = min(max(last + x.shift + 1, 0), x.klen);
  return true;
}

// Scheduling of a straight-line block of NR LDS reads feeding NM MFMAs: RA
// reads issued ahead, then groups of MP MFMAs each followed by the next DP
// reads, then the remaining MFMAs.  The default schedule waits on each read
// right before its MFMA.
template <int NR, int NM, int RA, int MP, int DP, int ID>
__device__ __forceinline__ void sched_reads_ahead() {
  static_assert(RA <= NR && (NR - RA) % DP == 0 && (NR - RA) / DP * MP <= NM, "schedule shape");
  __builtin_amdgcn_sched_group_barrier(0x100, RA, ID);
#pragma unroll
  for (int i = 0; i < (NR - RA) / DP; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, MP, ID);
    __builtin_amdgcn_sched_group_barrier(0x100, DP, ID);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, NM - (NR - RA) / DP * MP, ID);
}

#define LLMT_INLINE __attribute__((always_inline))

Group group_of(const PackArgs& a) {
  const int G = a.nq / a.nkv;
  return {G, G == 1 ? 0u : (unsigned)((0x100000000ull + G - 1) / G)};
}
// Tiles of qb rows, of kb keys.
int row_tiles(const PackArgs& a, int qb) {
  return (int)((long long)a.Tq * (a.nq / a.nkv) / qb) + a.n + 2;
}
int key_tiles(const PackArgs& a, int kb) { return a.Tk / kb + a.n + 2; }

}  // namespace

}  // namespace llmt
