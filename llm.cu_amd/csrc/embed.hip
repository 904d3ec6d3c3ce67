// embed.hip — embedding lookup with scaling, out[i] = scale w[tok[i]], and its
// gradient, dw[v] (+)= scale sum over tok[i] = v of dout[i].
//
// The gradient adds every token's rows in an order that the positions alone
// decide: positions are sorted by token (stable), the sorted list
// is cut into chunks, a group of lanes sums the runs of equal tokens of its
// chunk in fp32, and a run that spans chunks is joined from their partial sums
// in an order of their number alone.  No atomics, and a frequent token's rows are shared by as many
// groups as it has chunks.  Few positions need no sort: a workgroup for each
// looks whether it is its token's first and gathers the others.  Where the
// table is written whole, its zeros ride in the sorting launches, which leave
// the memory idle.
//
// Memory-bound where large: the lookup of 16384 rows of 1037 fp32 in 17.9 us, 5.1 TB/s
// (the odd width takes single elements); the gradient of 32768 rows of 1024 bf16
// into a table of 50257 fp32 rows in 78 us of kernels (88 a call whose inputs change), of
// which the sorting launches with the 206 MB of zeros take 46, the sums 24 (its 67 MB
// gathered, 41 written) and the join 8; a copy would take 56 for all of it.  Few
// tokens cost a launch: 128 rows 2.6 us, the gradient of 300 added to the table 5.0.
#include <algorithm>

#include "ops.h"

namespace llmt {

namespace {

constexpr int NTH = 256;

template <class T>
struct Bits;  // 16-byte pieces and single elements of a type
template <>
struct Bits<float> {
  static constexpr int N = 4;
};
template <>
struct Bits<_Float16> {
  static constexpr int N = 8;
};
template <>
struct Bits<__bf16> {
  static constexpr int N = 8;
};

// N elements at p (one aligned access where VEC), as fp32.
template <class T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&x)[N]) {
  typedef T TN __attribute__((ext_vector_type(N)));
  if constexpr (N == 1) {
    x[0] = (float)*p;
  } else if constexpr (N * sizeof(T) <= 16) {
    const TN v = *reinterpret_cast<const TN*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
  } else {  // fp32 beside a 16-bit type: 8 elements are two pieces
    float a[N / 2], b[N / 2];
    load_n<T, N / 2>(p, a);
    load_n<T, N / 2>(p + N / 2, b);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      x[i] = a[i];
      x[N / 2 + i] = b[i];
    }
  }
}
template <class T, int N>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N]) {
  typedef T TN __attribute__((ext_vector_type(N)));
  if constexpr (N == 1) {
    *p = (T)x[0];
  } else if constexpr (N * sizeof(T) <= 16) {
    TN v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    *reinterpret_cast<TN*>(p) = v;
  } else {
    float a[N / 2], b[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      a[i] = x[i];
      b[i] = x[N / 2 + i];
    }
    store_n<T, N / 2>(p, a);
    store_n<T, N / 2>(p + N / 2, b);
  }
}

// Lanes a row (a power of two up to 256) for H columns in pieces of N.
int lanes_for(int H, int N) {
  int l = 1;
  while (l < NTH && l * N < H) l *= 2;
  return l;
}

// lpr lanes a row, NTH / lpr rows a workgroup.
template <class TW, class TX, int N>
__global__ __launch_bounds__(NTH) void embed_kernel(const EmbedArgs a, int lpr) {
  const int i = blockIdx.x * (NTH / lpr) + threadIdx.x / lpr;
  if (i >= a.T) return;
  const int t = a.tok[i];
  const bool ok = (unsigned)t < (unsigned)a.V;
  const TW* w = (const TW*)a.w + (ok ? t : 0) * a.ldw;
  TX* x = (TX*)a.x + i * a.ldx;
  // U pieces in flight
  constexpr int U = N == 1 ? 8 : 2;
  for (int c0 = (threadIdx.x % lpr) * N; c0 < a.H; c0 += U * lpr * N) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * lpr * N;
      if (ok && c < a.H) load_n<TW, N>(w + c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * lpr * N;
      if (c >= a.H) break;
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] = ok ? v[u][e] * a.scale : 0.f;
      store_n<TX, N>(x + c, v[u]);
    }
  }
}

// ---------------------------------------------------------------- zeros
// Rows v0 .. v1 - 1 of the table, by the workgroups from `first` on of a launch.
struct Zeros {
  void* w;
  long long ldw;
  int v0, v1, H, es, vec;  // es: bytes an element; vec: 16-byte pieces
  unsigned first;
};
__device__ __forceinline__ void zero_rows(const Zeros& z) {
  const int per = z.vec ? 16 : z.es, n = z.H * z.es / per;  // pieces a row
  const int lanes = n >= NTH ? NTH : n >= 64 ? 64 : n >= 16 ? 16 : 4;
  const int groups = NTH / lanes;
  for (long long v = z.v0 + (long long)(blockIdx.x - z.first) * groups + threadIdx.x / lanes;
       v < z.v1; v += (long long)(gridDim.x - z.first) * groups) {
    char* row = (char*)z.w + v * z.ldw * z.es;
    for (int c = threadIdx.x % lanes; c < n; c += lanes) {
      if (z.vec) *reinterpret_cast<u32x4*>(row + c * 16ll) = u32x4{0, 0, 0, 0};
      else if (z.es == 4) *reinterpret_cast<unsigned*>(row + c * 4ll) = 0;
      else *reinterpret_cast<unsigned short*>(row + c * 2ll) = 0;
    }
  }
}
__global__ __launch_bounds__(NTH) void embed_zero_kernel(const Zeros z) { zero_rows(z); }

// ---------------------------------------------------------------- sorting
// Sort key of a position: its token, V where that is outside [0, V).
__device__ __forceinline__ int key_of(const int* tok, int i, int V) {
  const int t = tok[i];
  return (unsigned)t < (unsigned)V ? t : V;
}

// Up to kRankMost positions: a position's place is the number of positions in
// front of it, counted by 16 lanes over all of them (T^2 comparisons: at 3500
// positions 9 us less than the launches of a radix sort, at 5000 3 more, at 16000 120).
constexpr int kRankMost = 4096;
__global__ __launch_bounds__(NTH) void embed_rank_kernel(const int* tok, int T, int V, int* skey,
                                                         int* spos, const Zeros z) {
  constexpr int LPI = 16;
  if (blockIdx.x >= z.first) return zero_rows(z);
  const int sub = threadIdx.x % LPI;
  const int i = blockIdx.x * (NTH / LPI) + threadIdx.x / LPI;
  const int ki = i < T ? key_of(tok, i, V) : V;
  int n = 0;
#pragma unroll 4
  for (int k = sub; k < T; k += LPI) {
    const int kk = key_of(tok, k, V);
    n += kk < ki + (k < i ? 1 : 0) ? 1 : 0;
  }
#pragma unroll
  for (int d = 1; d < LPI; d *= 2) n += __shfl_xor(n, d, LPI);
  if (i < T && sub == 0) {
    skey[n] = ki;
    spos[n] = i;
  }
}

// More positions: least significant digit first, RB bits a pass, each pass a
// count and a stable placement.  A workgroup's four waves take `per` positions
// each, 64 at a time in order.
constexpr int RB = 9, BINS = 1 << RB, SORT_WAVES = NTH / 64;

// The lanes of the wave whose digit is this lane's (valid lanes only).
__device__ __forceinline__ unsigned long long same_digit(int d, bool valid) {
  unsigned long long m = __ballot(valid);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const unsigned long long set = __ballot(d >> b & 1);
    m &= d >> b & 1 ? set : ~set;
  }
  return m;
}

struct SortArgs {
  const int* key;  // NULL on the first pass: the tokens themselves, in order
  const int* pos;
  const int* tok;
  int T, V, shift, per, wgs;
  int* hist;  // [workgroups][BINS]
  int* key_out;
  int* pos_out;
};

__global__ __launch_bounds__(NTH) void embed_count_kernel(const SortArgs a, const Zeros z) {
  __shared__ int h[BINS];
  if (blockIdx.x >= z.first) return zero_rows(z);
  for (int i = threadIdx.x; i < BINS; i += NTH) h[i] = 0;
  __syncthreads();
  const int n = a.per * SORT_WAVES, i0 = blockIdx.x * n;
  for (int i = i0 + threadIdx.x; i < min(a.T, i0 + n); i += NTH) {
    const int k = a.key ? a.key[i] : key_of(a.tok, i, a.V);
    atomicAdd(&h[k >> a.shift & (BINS - 1)], 1);  // counts: the order is of no account
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NTH) a.hist[blockIdx.x * BINS + i] = h[i];
}

__global__ __launch_bounds__(NTH) void embed_place_kernel(const SortArgs a, const Zeros z) {
  __shared__ int at[SORT_WAVES][BINS];  // counts, then the next place
  __shared__ int sums[NTH];
  if (blockIdx.x >= z.first) return zero_rows(z);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < SORT_WAVES * BINS; i += NTH) (&at[0][0])[i] = 0;
  const int i0 = (blockIdx.x * SORT_WAVES + w) * a.per;
  const int end = min(a.T, i0 + a.per);
  volatile int* mine = at[w];
  auto key_at = [&](int i) { return i >= end ? 0 : a.key ? a.key[i] : key_of(a.tok, i, a.V); };
  auto pos_at = [&](int i) { return i >= end ? 0 : a.pos ? a.pos[i] : i; };
  // the wave's first 256 positions in registers: their loads wait once
  constexpr int R = 4;
  int key[R], pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    key[r] = key_at(i0 + 64 * r + lane);
    pos[r] = pos_at(i0 + 64 * r + lane);
  }
  // a digit's first place: the positions of lower digits, then those of earlier
  // workgroups.  Thread t has digits 2 t and 2 t + 1.
  static_assert(BINS == 2 * NTH, "two digits a thread");
  int before[2] = {0, 0}, total[2] = {0, 0};
#pragma unroll 32
  for (int b = 0; b < a.wgs; ++b) {
    const int2 x = *reinterpret_cast<const int2*>(a.hist + b * BINS + 2 * threadIdx.x);
    if (b < (int)blockIdx.x) {
      before[0] += x.x;
      before[1] += x.y;
    }
    total[0] += x.x;
    total[1] += x.y;
  }
  sums[threadIdx.x] = total[0] + total[1];
  __syncthreads();
  for (int d = 1; d < NTH; d *= 2) {  // inclusive sums
    const int v = threadIdx.x >= d ? sums[threadIdx.x - d] : 0;
    __syncthreads();
    sums[threadIdx.x] += v;
    __syncthreads();
  }
  const int lower = sums[threadIdx.x] - total[0] - total[1];
  auto count = [&](int i, int k) {
    const bool ok = i < end;
    const int d = k >> a.shift & (BINS - 1);
    const unsigned long long m = same_digit(d, ok);
    if (ok && (m & ((1ull << lane) - 1)) == 0) mine[d] = mine[d] + (int)__popcll(m);
  };
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (i0 + 64 * r < end) count(i0 + 64 * r + lane, key[r]);
  for (int r = i0 + 64 * R; r < end; r += 64) count(r + lane, key_at(r + lane));
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int d = 2 * threadIdx.x + u;
    int p = lower + (u ? total[0] : 0) + before[u];
    for (int x = 0; x < SORT_WAVES; ++x) {
      const int c = at[x][d];
      at[x][d] = p;
      p += c;
    }
  }
  __syncthreads();
  auto place = [&](int i, int k, int q) {
    const bool ok = i < end;
    const int d = k >> a.shift & (BINS - 1);
    const unsigned long long m = same_digit(d, ok), lower_lanes = m & ((1ull << lane) - 1);
    const int first = ok ? mine[d] : 0;
    if (ok) {
      const int p = first + (int)__popcll(lower_lanes);
      a.key_out[p] = k;
      a.pos_out[p] = q;
      if (lower_lanes == 0) mine[d] = first + (int)__popcll(m);
    }
  };
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (i0 + 64 * r < end) place(i0 + 64 * r + lane, key[r], pos[r]);
  for (int r = i0 + 64 * R; r < end; r += 64) place(r + lane, key_at(r + lane), pos_at(r + lane));
}

// ---------------------------------------------------------------- sums
struct SumArgs {
  const int* skey;
  const int* spos;
  int T, V, H, C, nchunks;
  const void* x;
  long long ldx;
  void* dw;
  long long ldw;
  float scale;
  int add;
  float* part;  // [nchunks][2][H]: of a run from an earlier chunk, of one that goes on
};

template <class TW, int N>
__device__ __forceinline__ void put_row(const SumArgs& a, int v, int c, const float (&s)[N]) {
  TW* w = (TW*)a.dw + v * a.ldw + c;
  float y[N];
  if (a.add) {
    load_n<TW, N>(w, y);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] += s[e] * a.scale;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = s[e] * a.scale;
  }
  store_n<TW, N>(w, y);
}

// Chunk k: sorted entries k C .. (C up to 32); lpr >= 32 lanes a chunk,
// blockIdx.y: columns.  A lane holds an entry's token and position, so that the
// rows' loads, eight at a time, wait for nothing else.
template <class TX, class TW, int N>
__global__ __launch_bounds__(NTH) void embed_sum_kernel(const SumArgs a, int lpr) {
  const int k = blockIdx.x * (NTH / lpr) + threadIdx.x / lpr;
  const int c = (blockIdx.y * lpr + threadIdx.x % lpr) * N;
  if (k >= a.nchunks) return;
  const int i0 = k * a.C, end = min(a.T, i0 + a.C), n = end - i0;
  const int mine = i0 + min((int)(threadIdx.x % 32), n - 1);
  const int ekey = a.skey[mine], epos = a.spos[mine];
  const int before = i0 > 0 ? a.skey[i0 - 1] : -1, behind = end < a.T ? a.skey[end] : -1;
  const bool on = c < a.H;  // the lanes of a group leave together: they hold its entries
  int run = __shfl(ekey, 0, 32);
  bool cont = before == run;  // from an earlier chunk
  float s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = 0.f;
  for (int i = 0; i < n && run < a.V; i += 8) {
    int key[8];
    float x[8][N];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      key[u] = i + u < n ? __shfl(ekey, (i + u) & 31, 32) : a.V;
      const int pos = __shfl(epos, (i + u) & 31, 32);
      if (on && key[u] < a.V) load_n<TX, N>((const TX*)a.x + pos * a.ldx + c, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (i + u >= n) break;
      if (key[u] != run) {
        if (on) {
          if (cont) store_n<float, N>(a.part + (long long)(2 * k) * a.H + c, s);
          else put_row<TW, N>(a, run, c, s);
        }
        cont = false;
        run = key[u];
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] = 0.f;
      }
      if (run >= a.V) break;
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] += x[u][e];
    }
  }
  if (run >= a.V || !on) return;
  if (cont)
    store_n<float, N>(a.part + (long long)(2 * k) * a.H + c, s);
  else if (behind == run)
    store_n<float, N>(a.part + (long long)(2 * k + 1) * a.H + c, s);
  else
    put_row<TW, N>(a, run, c, s);
}

// Runs that begin in chunk k and go on behind it: a workgroup for each chunk and
// 32 N columns, whose eight groups of lanes take every eighth partial sum.
constexpr int JG = NTH / 32;
template <class TW, int N>
__global__ __launch_bounds__(NTH) void embed_join_kernel(const SumArgs a) {
  __shared__ float sums[JG][32 * N];
  const int k = blockIdx.x, lane = threadIdx.x % 32, grp = threadIdx.x / 32;
  const int c = (blockIdx.y * 32 + lane) * N;
  const int i0 = k * a.C, end = i0 + a.C;
  const int first = a.skey[i0], run = a.skey[end - 1], next = a.skey[end];
  const int before = i0 > 0 ? a.skey[i0 - 1] : -1;
  if (run >= a.V || next != run || (first == run && before == run)) return;  // or begins earlier
  int m = k + 1;  // behind the chunks that it fills from their start
  for (;;) {
    const int at = m + (int)threadIdx.x;
    const int n = __syncthreads_count(at < a.nchunks && a.skey[(long long)at * a.C] == run);
    m += n;
    if (n < NTH) break;
  }
  const int total = m - k;
  float s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = 0.f;
  for (int i = grp; i < total && c < a.H; i += 8 * JG) {
    float x[8][N];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = i + u * JG;  // the first partial sum is of a run that goes on
      if (p < total)
        load_n<float, N>(a.part + (long long)(2 * (k + p) + (p ? 0 : 1)) * a.H + c, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * JG < total) {
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += x[u][e];
      }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) sums[grp][e * 32 + lane] = s[e];
  __syncthreads();
  if (grp || c >= a.H) return;
#pragma unroll
  for (int u = 1; u < JG; ++u)
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += sums[u][e * 32 + lane];
  put_row<TW, N>(a, run, c, s);
}

// Up to kFewMost positions: workgroup (i, columns) of position i.  If no earlier
// position has its token, the positions that have it are listed in order, each
// wave sums a quarter of the list, and the quarters are added in order.
constexpr int kFewMost = 1024;
template <class TX, class TW, int N>
__global__ __launch_bounds__(NTH) void embed_few_kernel(const SumArgs a, const int* tok) {
  __shared__ int list[kFewMost];
  __shared__ int count[NTH / 64];
  __shared__ float part[3][64 * N];
  const int i = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int t = tok[i];
  if ((unsigned)t >= (unsigned)a.V) return;
  // wave w looks at positions w P ..
  constexpr int P = kFewMost / 4, R = P / 64;
  unsigned long long hit[R];
  int n = 0;
  bool earlier = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = w * P + r * 64 + lane;
    const bool same = p < a.T && tok[p] == t;
    earlier = earlier || (same && p < i);
    hit[r] = __ballot(same);
    n += (int)__popcll(hit[r]);
  }
  if (lane == 0) count[w] = n;
  if (__syncthreads_or(earlier)) return;
  int at = 0;
  for (int k = 0; k < w; ++k) at += count[k];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (hit[r] >> lane & 1)
      list[at + (int)__popcll(hit[r] & ((1ull << lane) - 1))] = w * P + r * 64 + lane;
    at += (int)__popcll(hit[r]);
  }
  __syncthreads();
  const int total = count[0] + count[1] + count[2] + count[3], per = (total + 3) / 4;
  const int c = (blockIdx.y * 64 + lane) * N;
  const bool on = c < a.H;
  float s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = 0.f;
  for (int k = w * per; on && k < min(total, (w + 1) * per); k += 8) {
    float x[8][N];
    const int left = min(total, (w + 1) * per) - k;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u < left) load_n<TX, N>((const TX*)a.x + list[k + u] * a.ldx + c, x[u]);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u < left) {
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += x[u][e];
      }
  }
  if (total == 1) {
    if (w == 0 && on) put_row<TW, N>(a, t, c, s);
    return;
  }
  if (w > 0) {
#pragma unroll
    for (int e = 0; e < N; ++e) part[w - 1][e * 64 + lane] = s[e];
  }
  __syncthreads();
  if (w > 0 || !on) return;
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += part[k][e * 64 + lane];
  put_row<TW, N>(a, t, c, s);
}

bool pieces(const void* p, long long ld, int H, size_t es, int N) {
  return (uintptr_t)p % std::min<size_t>(16, N * es) == 0 && (ld * es) % 16 == 0 && H % N == 0;
}

size_t size_of(int type) { return type == kF32 ? 4 : 2; }

// Entries of a chunk: more chunks feed more CUs and leave more partial sums (us of a call
// in a row, 50257 fp32 rows of 1024 written whole, with 16 / 32: 4096 positions 55 / 64,
// 32768 79 / 84, 65536 133 / 122; added to the table 28 / 36, 58 / 64, 97 / 91).
int chunk_of(int T) { return T >= 65536 ? 32 : T >= 4096 ? 16 : 8; }

// The workspace: sorted keys and positions (twice for the radix passes), the
// passes' counts, the partial sums.
struct Space {
  size_t keys, hist, part, total;
};
// Positions a wave of the radix passes: about sqrt(T / 32) workgroups, since
// every one reads the counts of all of them (32768 positions: a placement takes
// 20 us with 128 workgroups).
int sort_per(int T) {
  int wgs = 16;
  while (wgs < 256 && (long long)wgs * wgs * 32 < T) wgs += 16;
  return (T + wgs * 256 - 1) / (wgs * 256) * 64;
}
int sort_wgs(int T) { return (T + sort_per(T) * SORT_WAVES - 1) / (sort_per(T) * SORT_WAVES); }
Space space(int T, int H) {
  Space s{};
  if (T <= kFewMost) return s;
  const size_t n = ((size_t)T + 3) & ~(size_t)3;
  const bool radix = T > kRankMost;
  s.keys = 0;
  s.hist = n * 4 * (radix ? 4 : 2);
  s.part = s.hist + (radix ? (size_t)sort_wgs(T) * BINS * 4 : 0);
  const size_t chunks = ((size_t)T + chunk_of(T) - 1) / chunk_of(T);
  s.total = s.part + chunks * 2 * (((size_t)H + 3) & ~(size_t)3) * 4;
  return s;
}

template <class F>
hipError_t with_type(int type, F&& f) {
  return type == kF32 ? f((float*)nullptr) : type == kF16 ? f((_Float16*)nullptr) : f((__bf16*)nullptr);
}

}  // namespace

hipError_t embed_fwd(const EmbedArgs& a, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  return with_type(a.wtype, [&](auto* tw) {
    using TW = std::remove_pointer_t<decltype(tw)>;
    return with_type(a.xtype, [&](auto* tx) -> hipError_t {
      using TX = std::remove_pointer_t<decltype(tx)>;
      constexpr int N = Bits<TW>::N > Bits<TX>::N ? Bits<TW>::N : Bits<TX>::N;
      const bool vec = pieces(a.w, a.ldw, a.H, sizeof(TW), N) && pieces(a.x, a.ldx, a.H, sizeof(TX), N);
      const int lpr = lanes_for(a.H, vec ? N : 1), rpb = NTH / lpr;
      const dim3 grid((unsigned)((a.T + rpb - 1) / rpb));
      if (vec)
        hipLaunchKernelGGL((embed_kernel<TW, TX, N>), grid, dim3(NTH), 0, st, a, lpr);
      else
        hipLaunchKernelGGL((embed_kernel<TW, TX, 1>), grid, dim3(NTH), 0, st, a, lpr);
      LLMT_LAUNCH_CHECK();
      return hipSuccess;
    });
  });
}

size_t embed_bwd_workspace(int T, int V, int H) { return space(T, H).total; }

// Sorted keys and positions, the zeros of the table in the same launches.
static hipError_t sort_tokens(const EmbedArgs& a, const Space& sp, void* ws, Zeros z, int** key,
                              int** pos, hipStream_t st) {
  const size_t n = ((size_t)a.T + 3) & ~(size_t)3;
  int* const k0 = (int*)ws;
  const int V = a.V;
  if (a.T <= kRankMost) {
    *key = k0;
    *pos = k0 + n;
    constexpr int per = NTH / 16;
    z.first = (unsigned)((a.T + per - 1) / per);
    z.v1 = a.add ? 0 : V;
    const dim3 grid(z.first + (a.add ? 0 : 2048));
    hipLaunchKernelGGL(embed_rank_kernel, grid, dim3(NTH), 0, st, a.tok, a.T, V, *key, *pos, z);
    LLMT_LAUNCH_CHECK();
    return hipSuccess;
  }
  SortArgs s{};
  s.tok = a.tok;
  s.T = a.T;
  s.V = V;
  s.per = sort_per(a.T);
  s.wgs = sort_wgs(a.T);
  s.hist = (int*)((char*)ws + sp.hist);
  int passes = 1;
  while (passes * RB < 31 && (V >> (passes * RB)) > 0) ++passes;
  int* buf[2][2] = {{k0, k0 + n}, {k0 + 2 * n, k0 + 3 * n}};
  z.first = (unsigned)s.wgs;
  const dim3 grid(z.first + (a.add ? 0 : 2048));
  for (int p = 0; p < passes; ++p) {
    s.shift = p * RB;
    s.key_out = buf[p & 1][0];
    s.pos_out = buf[p & 1][1];
    for (int half = 0; half < 2; ++half) {
      // a launch's share of the rows: a quarter beside a count, the rest beside a placement
      z.v0 = (int)((long long)V * (4 * p + half) / (4 * passes));
      z.v1 = (int)((long long)V * (4 * p + (half ? 4 : 1)) / (4 * passes));
      if (half == 0)
        hipLaunchKernelGGL(embed_count_kernel, grid, dim3(NTH), 0, st, s, z);
      else
        hipLaunchKernelGGL(embed_place_kernel, grid, dim3(NTH), 0, st, s, z);
      LLMT_LAUNCH_CHECK();
    }
    s.key = *key = s.key_out;
    s.pos = *pos = s.pos_out;
  }
  return hipSuccess;
}

hipError_t embed_bwd(const EmbedArgs& a, void* ws, hipStream_t st) {
  const Space sp = space(a.T, a.H);
  const int es = (int)size_of(a.wtype);
  Zeros z{(void*)a.w, a.ldw, 0, a.V, a.H, es, 0, 0};
  z.vec = (uintptr_t)a.w % 16 == 0 && a.ldw * es % 16 == 0 && (long long)a.H * es % 16 == 0;
  int *key = nullptr, *pos = nullptr;
  if (a.T <= kFewMost) {
    if (!a.add) {
      hipLaunchKernelGGL(embed_zero_kernel, dim3(4096), dim3(NTH), 0, st, z);
      LLMT_LAUNCH_CHECK();
    }
    if (a.T == 0) return hipSuccess;
  } else {
    const hipError_t e = sort_tokens(a, sp, ws, z, &key, &pos, st);
    if (e != hipSuccess) return e;
  }
  return with_type(a.wtype, [&](auto* tw) {
    using TW = std::remove_pointer_t<decltype(tw)>;
    return with_type(a.xtype, [&](auto* tx) -> hipError_t {
      using TX = std::remove_pointer_t<decltype(tx)>;
      constexpr int N = Bits<TX>::N;
      const bool vec = pieces(a.w, a.ldw, a.H, sizeof(TW), N) && pieces(a.x, a.ldx, a.H, sizeof(TX), N);
      SumArgs s{key, pos, a.T, a.V, a.H, chunk_of(a.T), 0, a.x, a.ldx, (void*)a.w, a.ldw, a.scale,
                a.add, (float*)((char*)ws + sp.part)};
      if (a.T <= kFewMost) {
        const int cols = 64 * (vec ? N : 1);
        const dim3 grid((unsigned)a.T, (unsigned)((a.H + cols - 1) / cols));
        if (vec)
          hipLaunchKernelGGL((embed_few_kernel<TX, TW, N>), grid, dim3(NTH), 0, st, s, a.tok);
        else
          hipLaunchKernelGGL((embed_few_kernel<TX, TW, 1>), grid, dim3(NTH), 0, st, s, a.tok);
        LLMT_LAUNCH_CHECK();
        return hipSuccess;
      }
      s.nchunks = (a.T + s.C - 1) / s.C;
      const int lpr = std::max(32, lanes_for(a.H, vec ? N : 1)), gpb = NTH / lpr;
      const int cols = lpr * (vec ? N : 1);
      const dim3 grid((unsigned)((s.nchunks + gpb - 1) / gpb), (unsigned)((a.H + cols - 1) / cols));
      const int jcols = 32 * (vec ? N : 1);
      const dim3 join((unsigned)(s.nchunks - 1), (unsigned)((a.H + jcols - 1) / jcols));
      if (vec) {
        hipLaunchKernelGGL((embed_sum_kernel<TX, TW, N>), grid, dim3(NTH), 0, st, s, lpr);
        LLMT_LAUNCH_CHECK();
        if (s.nchunks > 1)
          hipLaunchKernelGGL((embed_join_kernel<TW, N>), join, dim3(NTH), 0, st, s);
      } else {
        hipLaunchKernelGGL((embed_sum_kernel<TX, TW, 1>), grid, dim3(NTH), 0, st, s, lpr);
        LLMT_LAUNCH_CHECK();
        if (s.nchunks > 1)
          hipLaunchKernelGGL((embed_join_kernel<TW, 1>), join, dim3(NTH), 0, st, s);
      }
      LLMT_LAUNCH_CHECK();
      return hipSuccess;
    });
  });
}

}  // namespace llmt
