// embed.hip — embedding lookup with scaling, out[i] = scale w[tok[i]], and its
// gradient, dw[v] (+)= scale sum over tok[i] = v of dout[i].
//
// The gradient adds every token's rows in the order of their positions,
// whatever the launch: positions are sorted by token (stable), the sorted list
// is cut into chunks, a group of lanes sums the runs of equal tokens of its
// chunk in fp32, and a run that spans chunks is joined from their partial sums
// in order.  No atomics, and a frequent token's rows are shared by as many
// groups as it has chunks.
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
  for (int c = (threadIdx.x % lpr) * N; c < a.H; c += lpr * N) {
    float v[N];
    if (ok) load_n<TW, N>(w + c, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = ok ? v[e] * a.scale : 0.f;
    store_n<TX, N>(x + c, v);
  }
}

// ---------------------------------------------------------------- sorting
// Sort key of a position: its token, V where that is outside [0, V).
__device__ __forceinline__ int key_of(const int* tok, int i, int V) {
  const int t = tok[i];
  return (unsigned)t < (unsigned)V ? t : V;
}

// Up to kRankMost positions: a position's place is the number of positions in
// front of it, counted by LPI lanes over all of them (T^2 comparisons: at 4096
// positions fewer than the launches of a radix sort would wait for).
constexpr int kRankMost = 16384;
template <int LPI>
__global__ __launch_bounds__(NTH) void embed_rank_kernel(const int* tok, int T, int V, int* skey,
                                                         int* spos) {
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
  int T, V, shift, per;
  int* hist;  // [workgroups][BINS]
  int* key_out;
  int* pos_out;
};

__global__ __launch_bounds__(NTH) void embed_count_kernel(const SortArgs a) {
  __shared__ int h[BINS];
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

__global__ __launch_bounds__(NTH) void embed_place_kernel(const SortArgs a) {
  __shared__ int at[SORT_WAVES][BINS];  // counts, then the next place
  __shared__ int sums[NTH];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < SORT_WAVES * BINS; i += NTH) (&at[0][0])[i] = 0;
  // a digit's first place: the positions of lower digits, then those of earlier
  // workgroups.  Thread t has digits 2 t and 2 t + 1.
  static_assert(BINS == 2 * NTH, "two digits a thread");
  int before[2] = {0, 0}, total[2] = {0, 0};
  for (int b = 0; b < (int)gridDim.x; ++b) {
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
  const int i0 = (blockIdx.x * SORT_WAVES + w) * a.per;
  const int end = min(a.T, i0 + a.per);
  volatile int* mine = at[w];
  for (int r = i0; r < i0 + a.per; r += 64) {
    const int i = r + lane;
    const bool ok = i < end;
    const int k = ok ? (a.key ? a.key[i] : key_of(a.tok, i, a.V)) : 0;
    const int d = k >> a.shift & (BINS - 1);
    const unsigned long long m = same_digit(d, ok);
    if (ok && (m & ((1ull << lane) - 1)) == 0) mine[d] = mine[d] + (int)__popcll(m);
  }
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
  for (int r = i0; r < i0 + a.per; r += 64) {
    const int i = r + lane;
    const bool ok = i < end;
    const int k = ok ? (a.key ? a.key[i] : key_of(a.tok, i, a.V)) : 0;
    const int d = k >> a.shift & (BINS - 1);
    const unsigned long long m = same_digit(d, ok), lower_lanes = m & ((1ull << lane) - 1);
    const int first = ok ? mine[d] : 0;
    if (ok) {
      const int p = first + (int)__popcll(lower_lanes);
      a.key_out[p] = k;
      a.pos_out[p] = a.pos ? a.pos[i] : i;
      if (lower_lanes == 0) mine[d] = first + (int)__popcll(m);
    }
  }
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

// Chunk k: sorted entries k C ..; lpr lanes a chunk, blockIdx.y: columns.
template <class TX, class TW, int N>
__global__ __launch_bounds__(NTH) void embed_sum_kernel(const SumArgs a, int lpr) {
  const int k = blockIdx.x * (NTH / lpr) + threadIdx.x / lpr;
  const int c = (blockIdx.y * lpr + threadIdx.x % lpr) * N;
  if (k >= a.nchunks || c >= a.H) return;
  const int i0 = k * a.C, end = min(a.T, i0 + a.C);
  int run = a.skey[i0];
  bool cont = i0 > 0 && a.skey[i0 - 1] == run;  // from an earlier chunk
  float s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = 0.f;
  for (int i = i0; i < end && run < a.V; i += 4) {
    int key[4];
    float x[4][N];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      key[u] = i + u < end ? a.skey[i + u] : a.V;
      if (key[u] < a.V) load_n<TX, N>((const TX*)a.x + a.spos[i + u] * a.ldx + c, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u >= end) break;
      if (key[u] != run) {
        if (cont) {
          store_n<float, N>(a.part + (long long)(2 * k) * a.H + c, s);
          cont = false;
        } else {
          put_row<TW, N>(a, run, c, s);
        }
        run = key[u];
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] = 0.f;
      }
      if (run >= a.V) break;
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] += x[u][e];
    }
  }
  if (run >= a.V) return;
  if (cont)
    store_n<float, N>(a.part + (long long)(2 * k) * a.H + c, s);
  else if (end < a.T && a.skey[end] == run)
    store_n<float, N>(a.part + (long long)(2 * k + 1) * a.H + c, s);
  else
    put_row<TW, N>(a, run, c, s);
}

// Runs that begin in chunk k and go on behind it.
template <class TW, int N>
__global__ __launch_bounds__(NTH) void embed_join_kernel(const SumArgs a, int lpr) {
  const int k = blockIdx.x * (NTH / lpr) + threadIdx.x / lpr;
  const int c = (blockIdx.y * lpr + threadIdx.x % lpr) * N;
  if (k >= a.nchunks - 1 || c >= a.H) return;
  const int i0 = k * a.C, end = i0 + a.C;
  const int run = a.skey[end - 1];
  if (run >= a.V || a.skey[end] != run) return;
  if (a.skey[i0] == run && i0 > 0 && a.skey[i0 - 1] == run) return;  // begins earlier
  float s[N];
  load_n<float, N>(a.part + (long long)(2 * k + 1) * a.H + c, s);
  for (int m = k + 1; m < a.nchunks; m += 4) {
    float x[4][N];
    bool in[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      in[u] = m + u < a.nchunks && a.skey[(m + u) * a.C] == run;
      if (in[u]) load_n<float, N>(a.part + (long long)(2 * (m + u)) * a.H + c, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (in[u]) {
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += x[u][e];
      }
    if (!in[3]) break;
  }
  put_row<TW, N>(a, run, c, s);
}

// Zeros in every row.
template <class TW, int N>
__global__ __launch_bounds__(NTH) void embed_zero_kernel(TW* w, long long ldw, int V, int H,
                                                         int lpr) {
  float z[N];
#pragma unroll
  for (int e = 0; e < N; ++e) z[e] = 0.f;
  for (long long v = (long long)blockIdx.x * (NTH / lpr) + threadIdx.x / lpr; v < V;
       v += (long long)gridDim.x * (NTH / lpr))
    for (int c = (threadIdx.x % lpr) * N; c < H; c += lpr * N) store_n<TW, N>(w + v * ldw + c, z);
}

bool pieces(const void* p, long long ld, int H, size_t es, int N) {
  return (uintptr_t)p % std::min<size_t>(16, N * es) == 0 && (ld * es) % 16 == 0 && H % N == 0;
}

size_t size_of(int type) { return type == kF32 ? 4 : 2; }

int chunk_of(int T) { return T >= 16384 ? 32 : T >= 2048 ? 16 : 4; }

// The workspace: sorted keys and positions (twice for the radix passes), its
// counts, the partial sums.
struct Space {
  size_t keys, hist, part, total;
};
int sort_per(int T) { return T <= 262144 ? 512 : 2048; }
Space space(int T, int H) {
  const size_t n = ((size_t)T + 3) & ~(size_t)3;
  const bool radix = T > kRankMost;
  const int wgs = (T + sort_per(T) * SORT_WAVES - 1) / (sort_per(T) * SORT_WAVES);
  Space s;
  s.keys = 0;
  s.hist = n * 4 * (radix ? 4 : 2);
  s.part = s.hist + (radix ? (size_t)wgs * BINS * 4 : 0);
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

size_t embed_bwd_workspace(int T, int V, int H) { return T > 0 ? space(T, H).total : 0; }

hipError_t embed_bwd(const EmbedArgs& a, void* ws, hipStream_t st) {
  const Space sp = space(std::max(a.T, 1), a.H);
  const size_t n = ((size_t)a.T + 3) & ~(size_t)3;
  int* const k0 = (int*)ws;
  int *key = k0, *pos = k0 + n;
  if (a.T > kRankMost) {
    SortArgs s{};
    s.tok = a.tok;
    s.T = a.T;
    s.V = a.V;
    s.per = sort_per(a.T);
    s.hist = (int*)((char*)ws + sp.hist);
    const unsigned wgs = (unsigned)((a.T + s.per * SORT_WAVES - 1) / (s.per * SORT_WAVES));
    int* buf[2][2] = {{k0, k0 + n}, {k0 + 2 * n, k0 + 3 * n}};
    int cur = 0;
    for (s.shift = 0; s.shift == 0 || (s.shift < 31 && (a.V >> s.shift) > 0); s.shift += RB) {
      s.key_out = buf[cur][0];
      s.pos_out = buf[cur][1];
      hipLaunchKernelGGL(embed_count_kernel, dim3(wgs), dim3(NTH), 0, st, s);
      LLMT_LAUNCH_CHECK();
      hipLaunchKernelGGL(embed_place_kernel, dim3(wgs), dim3(NTH), 0, st, s);
      LLMT_LAUNCH_CHECK();
      s.key = key = s.key_out;
      s.pos = pos = s.pos_out;
      cur ^= 1;
    }
  } else if (a.T > 0) {
    if (a.T <= 8192)
      hipLaunchKernelGGL(embed_rank_kernel<16>, dim3((unsigned)((a.T + 15) / 16)), dim3(NTH), 0, st,
                         a.tok, a.T, a.V, key, pos);
    else
      hipLaunchKernelGGL(embed_rank_kernel<8>, dim3((unsigned)((a.T + 31) / 32)), dim3(NTH), 0, st,
                         a.tok, a.T, a.V, key, pos);
    LLMT_LAUNCH_CHECK();
  }
  return with_type(a.wtype, [&](auto* tw) {
    using TW = std::remove_pointer_t<decltype(tw)>;
    return with_type(a.xtype, [&](auto* tx) -> hipError_t {
      using TX = std::remove_pointer_t<decltype(tx)>;
      constexpr int N = Bits<TX>::N;
      const bool vec = pieces(a.w, a.ldw, a.H, sizeof(TW), N) && pieces(a.x, a.ldx, a.H, sizeof(TX), N);
      const int lpr = lanes_for(a.H, vec ? N : 1), gpb = NTH / lpr;
      if (!a.add) {
        const unsigned wgs = (unsigned)std::min<long long>(((long long)a.V + gpb - 1) / gpb, 8192);
        if (vec)
          hipLaunchKernelGGL((embed_zero_kernel<TW, N>), dim3(wgs), dim3(NTH), 0, st, (TW*)a.w, a.ldw,
                             a.V, a.H, lpr);
        else
          hipLaunchKernelGGL((embed_zero_kernel<TW, 1>), dim3(wgs), dim3(NTH), 0, st, (TW*)a.w, a.ldw,
                             a.V, a.H, lpr);
        LLMT_LAUNCH_CHECK();
      }
      if (a.T == 0) return hipSuccess;
      SumArgs s{key, pos, a.T, a.V, a.H, chunk_of(a.T), 0, a.x, a.ldx, (void*)a.w, a.ldw, a.scale,
                a.add, (float*)((char*)ws + sp.part)};
      s.nchunks = (a.T + s.C - 1) / s.C;
      const int cols = lpr * (vec ? N : 1);
      const dim3 grid((unsigned)((s.nchunks + gpb - 1) / gpb), (unsigned)((a.H + cols - 1) / cols));
      if (vec) {
        hipLaunchKernelGGL((embed_sum_kernel<TX, TW, N>), grid, dim3(NTH), 0, st, s, lpr);
        LLMT_LAUNCH_CHECK();
        hipLaunchKernelGGL((embed_join_kernel<TW, N>), grid, dim3(NTH), 0, st, s, lpr);
      } else {
        hipLaunchKernelGGL((embed_sum_kernel<TX, TW, 1>), grid, dim3(NTH), 0, st, s, lpr);
        LLMT_LAUNCH_CHECK();
        hipLaunchKernelGGL((embed_join_kernel<TW, 1>), grid, dim3(NTH), 0, st, s, lpr);
      }
      LLMT_LAUNCH_CHECK();
      return hipSuccess;
    });
  });
}

}  // namespace llmt
