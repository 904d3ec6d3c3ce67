// logprob.hip — log-probabilities of target tokens over a vocabulary, and
// their gradient, on logits that the caller has (fp32, fp16 or bf16).
//
// With x = logits * it (it the inverse temperature), m = max x and
// s = sum exp(x - m):
//   logp = (x_t - m) - ln s             stats = (m, ln s)
//   H    = ln s - sum exp(x - m) (x - m) / s
// and with p = exp((x - m) - ln s), the gradients of logp and H given:
//   dlogits_j = it (dlogp (1[j = t] - p_j) - dH p_j (ln p_j + H)).
// m and ln s stay apart: their sum rounded to fp32 would move every p by
// |m + ln s| 2^-24.  A row without a target (an id outside [0, V)) is not
// read; its outputs and its gradient are zeros.
//
// Both are bound by HBM: the forward reads the logits once, the backward
// reads them and writes their gradient.  4096 x 151936 fp32, a quarter of the
// rows without a target: forward 283 us in a row, 6.6 TB/s (295 in a graph).  1000
// x 151936 fp32:
// backward 194 us, 6.3 TB/s (a plain copy 4.8-5.1).
#include <algorithm>

#include "ops.h"

namespace llmt {

namespace {

constexpr int NTH = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e4f;  // exp of it is 0
constexpr float kLeast = -0x1p30f;

// Rows whose largest x is beyond 2^29 (all of a row masked with a large finite
// value, say): there an fma's x - m keeps the rounding of m, which is more
// than such logits can differ by without differing altogether.  Their x are
// rounded before m is subtracted, as m itself was.
constexpr float kFarRow = 0x1p29f;
__device__ __forceinline__ bool far_row(float m) { return fabsf(m) > kFarRow && fabsf(m) < INFINITY; }
__device__ __forceinline__ float far_diff(float logit, float it, float m) {
#pragma clang fp contract(off)
  const float x = logit * it;
  return x - m;
}

// 16-byte pieces at any alignment of the element: gfx950 takes unaligned
// global accesses, so rows of an odd length need no peeling.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int N = 4;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Piece<_Float16> {
  static constexpr int N = 8;
  typedef _Float16 V __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Piece<__bf16> {
  static constexpr int N = 8;
  typedef __bf16 V __attribute__((ext_vector_type(8), aligned(2)));
};

// The statistics are kept in base 2: with y = logits * c, c = it log2 e,
// (m, s, u) are the largest y, sum 2^(y - m) and sum 2^(y - m) (y - m), each
// y - m one fma; x is the largest logit itself.  16-bit logits are bound by the
// VALU as much as by HBM, and this is the fewest instructions an element.  The
// roundings of m and c are common to a row's terms; finish takes them out of
// its m, and the rounding of c leaves 2^-24 of each y - m.  m starts at kLeast
// and only rises: logits below it (-inf, finite masks) add nothing, every m is
// finite, and where m >= kLeast the rounding of m moves an exponent by at most
// 64.  The empty set is (kLeast, 0, 0), -inf.
struct Stat {
  float m, s, u, x;
};
__device__ __forceinline__ Stat empty_stat() { return {kLeast, 0.f, 0.f, -INFINITY}; }
template <bool ENT>
__device__ __forceinline__ void merge(Stat& a, const Stat& b) {
  const float m2 = b.m, s2 = b.s, u2 = b.u;
  const float mn = fmaxf(a.m, m2);
  const float d1 = a.m - mn, d2 = m2 - mn;
  const float f1 = __builtin_amdgcn_exp2f(d1), f2 = __builtin_amdgcn_exp2f(d2);
  if constexpr (ENT) a.u = f1 * fmaf(a.s, d1, a.u) + f2 * fmaf(s2, d2, u2);
  a.s = a.s * f1 + s2 * f2;
  a.m = mn;
  a.x = fmaxf(a.x, b.x);
}

// Adds NV logits to a thread's statistics: one rescale.
template <bool ENT, int NV>
__device__ __forceinline__ void add(Stat& a, const float (&x)[NV], float c) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) mx = fmaxf(mx, x[i]);
  const float m = fmaxf(a.m, mx * c);
  const float d = a.m - m, f = __builtin_amdgcn_exp2f(d);
  float s = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float z = fmaf(x[i], c, -m);
    const float e = __builtin_amdgcn_exp2f(z);
    s += e;
    if constexpr (ENT) u = fmaf(e, fmaxf(z, kFar), u);  // a logit of -inf adds nothing
  }
  if constexpr (ENT) a.u = fmaf(f, fmaf(a.s, d, a.u), u);
  a.s = fmaf(a.s, f, s);
  a.m = m;
  a.x = fmaxf(a.x, mx);
}

template <bool ENT>
__device__ __forceinline__ Stat wave_merge(Stat a) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const Stat b = {__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64),
                    ENT ? __shfl_xor(a.u, o, 64) : 0.f, __shfl_xor(a.x, o, 64)};
    merge<ENT>(a, b);
  }
  return a;
}

// A thread's share of columns [j0, j1) of a row, `nth` threads a row, BATCH
// logits at a time.  FAR: of what far_diff makes of them.
template <bool ENT, bool NT, int BATCH = 16, bool FAR = false, typename T>
__device__ __forceinline__ void scan(Stat& a, const T* row, int j0, int j1, int tid, int nth,
                                     float c, float it = 1.f, float m = 0.f) {
  auto of = [&](T v) { return FAR ? far_diff((float)v, it, m) : (float)v; };
  constexpr int N = Piece<T>::N, U = BATCH / N;
  typedef typename Piece<T>::V Vec;
  const int np = (j1 - j0) / N;
  int k = tid;
  for (; k + (U - 1) * nth < np; k += U * nth) {
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      auto* p = reinterpret_cast<const Vec*>(row + j0 + (long long)N * (k + u * nth));
      if constexpr (NT) v[u] = __builtin_nontemporal_load(p);
      else v[u] = *p;
    }
    float x[U * N];
#pragma unroll
    for (int i = 0; i < U * N; ++i) x[i] = of(v[i / N][i % N]);
    add<ENT, U * N>(a, x, c);
  }
  for (; k < np; k += nth) {
    const Vec v = *reinterpret_cast<const Vec*>(row + j0 + (long long)N * k);
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = of(v[e]);
    add<ENT, N>(a, x, c);
  }
  const int j = j0 + N * np + tid;
  if (j < j1) {
    const float x[1] = {of(row[j])};
    add<ENT, 1>(a, x, c);
  }
}

// The row's outputs from its statistics; all lanes of a wave, with the same `a`.
template <bool ENT, typename T>
__device__ __forceinline__ void finish(Stat a, const T* x, int t, int V, float it, long long row,
                                       float* logp, float2* stats, float* entropy) {
  const int lane = threadIdx.x & 63;
  const float m = a.x * it, xt = (float)x[t];
  const bool far = far_row(m);
  if (far) {
    a = empty_stat();
    scan<ENT, false, Piece<T>::N, true>(a, x, 0, V, lane, 64, kLog2e, it, m);
    a = wave_merge<ENT>(a);
  }
  if (lane) return;
  if (m == -INFINITY && a.s == 0.f) {  // every x is -inf: nothing has any probability
    logp[row] = -INFINITY;
    stats[row] = make_float2(-INFINITY, 0.f);
    if constexpr (ENT) entropy[row] = 0.f;
    return;
  }
  const float ls = logf(a.s);
  float l = ls;
  if (far) {
    logp[row] = far_diff(xt, it, m) - l;
  } else {
    // the offset a.m of the sums in natural units, by the c that they took
    l += (float)((double)a.m * ((double)it / (double)(it * kLog2e)) - m);
    logp[row] = fmaf(xt, it, -m) - l;
  }
  stats[row] = make_float2(m, l);
  if constexpr (ENT) entropy[row] = fmaf(-0.69314718f, a.u / a.s, ls);
}

// Outputs of a row without a target.
template <bool ENT>
__device__ __forceinline__ void no_target(long long row, float* logp, float2* stats,
                                          float* entropy) {
  logp[row] = 0.f;
  stats[row] = make_float2(0.f, 0.f);
  if constexpr (ENT) entropy[row] = 0.f;
}

// The block's statistics, in its first wave.  Contains a barrier.
template <bool ENT, int BLOCK>
__device__ __forceinline__ Stat block_merge(Stat a, Stat* part) {
  a = wave_merge<ENT>(a);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x < 64)
    for (int w = 1; w < BLOCK / 64; ++w) merge<ENT>(a, part[w]);
  return a;
}

// A workgroup of BLOCK threads a row, BATCH logits at a time.
template <bool ENT, bool NT, int BLOCK, int BATCH, typename T>
__global__ __launch_bounds__(BLOCK) void logprob_row_kernel(const T* __restrict__ logits,
                                                          long long ld,
                                                          const int* __restrict__ targets, int rows,
                                                          int V, float it, float* __restrict__ logp,
                                                          float2* __restrict__ stats,
                                                          float* __restrict__ entropy) {
  __shared__ Stat part[BLOCK / 64];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const int t = targets[row];
    if (t < 0 || t >= V) {
      if (threadIdx.x == 0) no_target<ENT>(row, logp, stats, entropy);
      continue;
    }
    const T* x = logits + row * ld;
    Stat a = empty_stat();
    scan<ENT, NT, BATCH>(a, x, 0, V, threadIdx.x, BLOCK, it * kLog2e);
    a = block_merge<ENT, BLOCK>(a, part);
    if (threadIdx.x < 64) finish<ENT>(a, x, t, V, it, row, logp, stats, entropy);
    __syncthreads();
  }
}

// A wave a row, for short ones.
template <bool ENT, bool NT, typename T>
__global__ __launch_bounds__(NTH) void logprob_wave_kernel(const T* __restrict__ logits,
                                                           long long ld,
                                                           const int* __restrict__ targets,
                                                           int rows, int V, float it,
                                                           float* __restrict__ logp,
                                                           float2* __restrict__ stats,
                                                           float* __restrict__ entropy) {
  const int lane = threadIdx.x & 63, wave = blockIdx.x * (NTH / 64) + (threadIdx.x >> 6);
  for (long long row = wave; row < rows; row += (long long)gridDim.x * (NTH / 64)) {
    const int t = targets[row];
    if (t < 0 || t >= V) {
      if (lane == 0) no_target<ENT>(row, logp, stats, entropy);
      continue;
    }
    const T* x = logits + row * ld;
    Stat a = empty_stat();
    scan<ENT, NT>(a, x, 0, V, lane, 64, it * kLog2e);
    a = wave_merge<ENT>(a);
    finish<ENT>(a, x, t, V, it, row, logp, stats, entropy);
  }
}

// Few rows: a workgroup a (row, chunk), its statistics to parts[row][chunk];
// then a wave a row merges them.
template <bool ENT, typename T>
__global__ __launch_bounds__(NTH) void logprob_part_kernel(const T* __restrict__ logits,
                                                           long long ld,
                                                           const int* __restrict__ targets, int V,
                                                           float it, int chunks, int width,
                                                           float4* __restrict__ parts) {
  __shared__ Stat part[NTH / 64];
  const int row = blockIdx.x / chunks, ch = blockIdx.x - row * chunks;
  const int t = targets[row];
  if (t < 0 || t >= V) return;
  const int j0 = (int)min((long long)ch * width, (long long)V), j1 = min(V - j0, width) + j0;
  Stat a = empty_stat();
  scan<ENT, false>(a, logits + row * ld, j0, j1, threadIdx.x, NTH, it * kLog2e);
  a = block_merge<ENT, NTH>(a, part);
  if (threadIdx.x == 0) parts[blockIdx.x] = make_float4(a.m, a.s, a.u, a.x);
}

template <bool ENT, typename T>
__global__ __launch_bounds__(64) void logprob_merge_kernel(const T* __restrict__ logits,
                                                           long long ld,
                                                           const int* __restrict__ targets, int V,
                                                           float it, int chunks,
                                                           const float4* __restrict__ parts,
                                                           float* __restrict__ logp,
                                                           float2* __restrict__ stats,
                                                           float* __restrict__ entropy) {
  const int row = blockIdx.x, t = targets[row];
  if (t < 0 || t >= V) {
    if (threadIdx.x == 0) no_target<ENT>(row, logp, stats, entropy);
    return;
  }
  Stat a = empty_stat();
  for (int c = threadIdx.x; c < chunks; c += 64) {
    const float4 p = parts[(long long)row * chunks + c];
    merge<ENT>(a, Stat{p.x, p.y, p.z, p.w});
  }
  a = wave_merge<ENT>(a);
  finish<ENT>(a, logits + row * ld, t, V, it, row, logp, stats, entropy);
}

// 16-byte pieces a lane of the backward: fp32 logits stream best with one
// (1000 x 151936: 202 us, 213 with two, 233 with four), 16-bit ones with two
// (1000 x 50257: 31.3, 26.6, 28.1).
template <typename T>
constexpr int kBwdPieces = sizeof(T) == 4 ? 1 : 2;
// A wave a (row, chunk of BU pieces a lane); a workgroup a chunk is no faster
// at any length and leaves threads idle on short rows (8192 x 1000 fp16: 8.3
// against 13.4 us).  NT: gradients beyond the 256 MB last-level cache are
// stored nontemporal (1000 x 151936 fp32: 194 us, 201 without), smaller ones
// stay there for the next kernel.
// TO: the type written.  FACTOR: the rows are written for dlogp = -1 times
// kGradLogitScale (the lm_head dX GEMM's operand) and factor[row] gets
// what they lack of the gradient, -dlogp; rows from `rows` to `factor_rows`
// get a factor of 0.
template <bool ENT, bool NT, typename T, typename TO = T, bool FACTOR = false>
__global__ __launch_bounds__(NTH) void logprob_bwd_kernel(
    const T* logits, long long ld, const int* __restrict__ targets,
    const float2* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ dlogp, const float* __restrict__ dentropy, int rows, int V, float it,
    int chunks, TO* dlogits, long long ldd, float* __restrict__ factor, int factor_rows) {
  typedef typename Piece<T>::V Vec;
  typedef TO VecO __attribute__((ext_vector_type(Piece<T>::N), aligned(sizeof(TO))));
  constexpr int N = Piece<T>::N, BU = kBwdPieces<T>, WAVES = NTH / 64;
  const long long items = (long long)rows * chunks;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (long long w = (long long)blockIdx.x * WAVES + wave; w < items;
       w += (long long)gridDim.x * WAVES) {
    const int row = (int)(w / chunks), ch = (int)(w - (long long)row * chunks);
    const int t = targets[row];
    float g = dlogp[row] * it;
    if constexpr (FACTOR) {
      if (ch == 0 && lane == 0) factor[row] = t < 0 || t >= V ? 0.f : -g;
      g = g == 0.f ? 0.f : -kGradLogitScale;
    }
    const float h = ENT ? dentropy[row] * it : 0.f;
    const float2 st = stats[row];
    const bool zero = t < 0 || t >= V || (g == 0.f && h == 0.f) ||
                      (st.x == -INFINITY && st.y == 0.f);
    const float gh = ENT ? -fmaf(h, entropy[row], g) : -g;
    const long long start = (long long)ch * (BU * N * 64);
    const int j0 = (int)start, j1 = (int)min((long long)V, start + BU * N * 64);
    const T* x = logits + row * ld;
    TO* d = dlogits + row * ldd;
    // exp is 0 far below, and 0 * z has to stay 0
    auto log_p = [&](float diff) { return ENT && diff - st.y < kFar ? kFar : diff - st.y; };
    auto value_of = [&](float z) {
      return __builtin_amdgcn_exp2f(z * kLog2e) * (ENT ? fmaf(-h, z, gh) : gh);
    };
    auto target_of = [&](float z) {  // g (1 - p) without the cancellation
      const float p = __builtin_amdgcn_exp2f(z * kLog2e), dg = -g * expm1f(z);
      return ENT ? fmaf(-h * p, z + entropy[row], dg) : dg;
    };
    auto value = [&](float xv) { return value_of(log_p(fmaf(xv, it, -st.x))); };
    auto at_target = [&](float xv) { return target_of(log_p(fmaf(xv, it, -st.x))); };
    if (!FACTOR && !zero && far_row(st.x)) {
      for (int j = j0 + lane; j < j1; j += 64) {
        const float z = log_p(far_diff((float)x[j], it, st.x));
        d[j] = (TO)(j == t ? target_of(z) : value_of(z));
      }
      continue;
    }
    const int np = (j1 - j0) / N;
    Vec v[BU];
    if (!zero)
#pragma unroll
      for (int u = 0; u < BU; ++u)
        if (lane + u * 64 < np)
          v[u] = *reinterpret_cast<const Vec*>(x + j0 + N * (lane + u * 64));
#pragma unroll
    for (int u = 0; u < BU; ++u) {
      const int k = lane + u * 64;
      if (k < np) {
        const int j = j0 + N * k;
        VecO o;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = zero ? (TO)0.f : (TO)value((float)v[u][e]);
        if (!zero && (unsigned)(t - j) < (unsigned)N)
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (t == j + e) o[e] = (TO)at_target((float)v[u][e]);
        auto* to = reinterpret_cast<VecO*>(d + j);
        if constexpr (NT) __builtin_nontemporal_store(o, to);
        else *to = o;
      }
    }
    const int j = j0 + N * np + lane;
    if (j < j1) d[j] = zero ? (TO)0.f : (TO)(j == t ? at_target((float)x[j]) : value((float)x[j]));
  }
  if constexpr (FACTOR)
    for (int r = rows + blockIdx.x * NTH + threadIdx.x; r < factor_rows; r += gridDim.x * NTH)
      factor[r] = 0.f;
}

}  // namespace

// Rows up to kWaveV logits take a wave each: 8192 x 1000 bf16 7.2 us, 14.2
// with a workgroup each; from there on the two are level (8192 x 2000 fp32
// 14.6 and 15.4) or the workgroups ahead (300 x 3000: 3.9 against 4.5).
constexpr int kWaveV = 2048;

// Fewer rows than the chip has CUs (256) take the wide workgroups: a row is
// one CU's loads and exponentials (1 x 151936 fp32 9.6 us, 15.9 with 256
// threads and 16 logits at a time; 128 x 50257 5.8 and 8.0).  From there on
// the narrow ones, which share CUs, stream better (8192 x 4000: 25.2 and 29.6).
//
// Rows too long for one CU are split into chunks, as many as make four
// workgroups a CU and at least one batch of loads a thread, and merged by a
// second launch, which costs a caller from Python 4 us: worth 192 K logits off a
// workgroup's share (one row of 262144 bf16, a call and its wait: split 25 us,
// unsplit 31), up to half a row a CU (200 x 262144 bf16: split 20.6, unsplit
// 17.9).  The rule follows such calls.  In a graph a split would be worth it from
// fewer logits on; 151936, split and unsplit, us:
//   rows             1          8          32         64         128
//   fp32 graph    5.9  9.3   6.4  9.7   7.0 10.0  10.6 13.8  16.7 16.9
//   bf16 graph    5.7  9.4   6.2  9.7   7.0  9.9   7.8  9.9  11.2 11.9
// while a call in a row is 4 us longer split at each of these sizes, and one with
// its wait level (fp32, 64 rows: 2.7 us shorter split).  50257 is slower split
// either way (fp32 graph, 1 and 128 rows: 5.8 and 5.3, 7.9 and 7.0).
constexpr int kCus = 256, kSplitLogits = 192 << 10;
static int fwd_chunks(int rows, int V, int dtype) {
  if (rows > kCus / 2) return 1;
  const long long batch = NTH * 4 * (dtype == kF32 ? 4 : 8);
  const long long chunks = std::min((V + batch - 1) / batch, (long long)(4 * kCus / rows));
  return V * (chunks - 1) >= kSplitLogits * chunks ? (int)chunks : 1;
}

size_t logprob_workspace(int rows, int V, int dtype) {
  const int chunks = fwd_chunks(rows, V, dtype);
  return chunks > 1 ? (size_t)rows * chunks * sizeof(float4) : 0;
}

template <typename F>
static hipError_t with_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f((float*)nullptr);
    case kF16: return f((_Float16*)nullptr);
    default: return f((__bf16*)nullptr);
  }
}

// Logits beyond the 256 MB last-level cache stream past it (4096 x 151936 fp32,
// a quarter of the rows skipped: 283 us nontemporal, 321 not; 1000 x 151936 with
// the backward behind it 290 and 303); smaller ones stay for the backward
// (256 x 151936 with it 79 us, 90 nontemporal).
static bool beyond_cache(const LogprobArgs& a, size_t esize) {
  return (double)a.rows * a.V * esize > 256.0 * (1 << 20);
}

template <bool ENT, bool NT, typename T>
static hipError_t launch_fwd(const LogprobArgs& a, float4* parts, hipStream_t st) {
  const T* x = (const T*)a.logits;
  float2* stats = (float2*)a.stats;
  const int chunks = fwd_chunks(a.rows, a.V, a.dtype);
  if (chunks > 1) {
    constexpr int N = Piece<T>::N;  // chunks start at whole pieces
    const int width = (int)(((long long)a.V + chunks - 1) / chunks + N - 1) / N * N;
    hipLaunchKernelGGL((logprob_part_kernel<ENT, T>), dim3(a.rows * chunks), dim3(NTH), 0, st, x,
                       a.ld, a.targets, a.V, a.it, chunks, width, parts);
    LLMT_LAUNCH_CHECK();
    hipLaunchKernelGGL((logprob_merge_kernel<ENT, T>), dim3(a.rows), dim3(64), 0, st, x, a.ld,
                       a.targets, a.V, a.it, chunks, parts, a.logp, stats, a.entropy);
  } else if (a.V <= kWaveV) {
    hipLaunchKernelGGL((logprob_wave_kernel<ENT, NT, T>),
                       dim3(std::min(((long long)a.rows + NTH / 64 - 1) / (NTH / 64), 1ll << 20)), dim3(NTH), 0,
                       st, x, a.ld, a.targets, a.rows, a.V, a.it, a.logp, stats, a.entropy);
  } else if (a.rows < kCus) {
    hipLaunchKernelGGL((logprob_row_kernel<ENT, NT, 512, 32, T>), dim3(a.rows), dim3(512), 0, st, x,
                       a.ld, a.targets, a.rows, a.V, a.it, a.logp, stats, a.entropy);
  } else {
    hipLaunchKernelGGL((logprob_row_kernel<ENT, NT, NTH, 16, T>), dim3(std::min(a.rows, 1 << 20)),
                       dim3(NTH), 0, st, x, a.ld, a.targets, a.rows, a.V, a.it, a.logp, stats,
                       a.entropy);
  }
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

hipError_t logprob_fwd(const LogprobArgs& a, void* workspace, hipStream_t st) {
  return with_type(a.dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    float4* ws = (float4*)workspace;
    if (beyond_cache(a, sizeof(T)))
      return a.entropy ? launch_fwd<true, true, T>(a, ws, st) : launch_fwd<false, true, T>(a, ws, st);
    return a.entropy ? launch_fwd<true, false, T>(a, ws, st) : launch_fwd<false, false, T>(a, ws, st);
  });
}

template <bool ENT, bool NT, typename T>
static hipError_t launch_bwd(const LogprobArgs& a, hipStream_t st) {
  const int per = kBwdPieces<T> * Piece<T>::N * 64;
  const int chunks = (int)(((long long)a.V + per - 1) / per);
  const long long wgs = ((long long)a.rows * chunks + NTH / 64 - 1) / (NTH / 64);
  hipLaunchKernelGGL((logprob_bwd_kernel<ENT, NT, T>), dim3(std::min(wgs, 1ll << 22)), dim3(NTH), 0,
                     st, (const T*)a.logits, a.ld, a.targets, (const float2*)a.stats, a.entropy,
                     a.dlogp, a.dentropy, a.rows, a.V, a.it, chunks, (T*)a.dlogits, a.ldd,
                     (float*)nullptr, 0);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

hipError_t logprob_bwd(const LogprobArgs& a, hipStream_t st) {
  return with_type(a.dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (beyond_cache(a, sizeof(T)))
      return a.dentropy ? launch_bwd<true, true, T>(a, st) : launch_bwd<false, true, T>(a, st);
    return a.dentropy ? launch_bwd<true, false, T>(a, st) : launch_bwd<false, false, T>(a, st);
  });
}

// ------------------------------------------------------------------ in a context

namespace {
// A wave a row: the (max, sum exp(x - max)) pairs of the logits GEMM's column
// tiles, in a fixed order, into the row's statistics.
__global__ __launch_bounds__(64) void logprob_pairs_kernel(const float2* __restrict__ pairs,
                                                           int ntiles,
                                                           const float* __restrict__ logits,
                                                           const int* __restrict__ targets, int V,
                                                           float* __restrict__ logp,
                                                           float2* __restrict__ stats) {
  const int row = blockIdx.x, t = targets[row];
  if (t < 0 || t >= V) {
    if (threadIdx.x == 0) no_target<false>(row, logp, stats, nullptr);
    return;
  }
  const float xt = logits[(long long)row * V + t];
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x; i < ntiles; i += 64) {
    const float2 p = pairs[(long long)row * ntiles + i];
    softmax_merge(m, s, p.x, p.y);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
    softmax_merge(m, s, m2, s2);
  }
  if (threadIdx.x == 0) {
    const float l = logf(s);
    logp[row] = (xt - m) - l;
    stats[row] = make_float2(m, l);
  }
}
}  // namespace

hipError_t logprob_from_pairs(const float2* pairs, int ntiles, const float* logits,
                              const int* targets, int rows, int V, float* logp, float2* stats,
                              hipStream_t st) {
  hipLaunchKernelGGL(logprob_pairs_kernel, dim3(rows), dim3(64), 0, st, pairs, ntiles, logits,
                     targets, V, logp, stats);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

hipError_t logprob_grad16(const float* logits, const int* targets, const float2* stats,
                          const float* dlogp, int rows, int V, _Float16* grad16, float* factor,
                          int factor_rows, hipStream_t st) {
  constexpr int per = kBwdPieces<float> * Piece<float>::N * 64;
  const int chunks = (V + per - 1) / per;
  const long long wgs = ((long long)rows * chunks + NTH / 64 - 1) / (NTH / 64);
  hipLaunchKernelGGL((logprob_bwd_kernel<false, false, float, _Float16, true>),
                     dim3(std::min(wgs, 1ll << 22)), dim3(NTH), 0, st, logits, (long long)V,
                     targets, stats, (const float*)nullptr, dlogp, (const float*)nullptr, rows, V,
                     1.0f, chunks, grad16, (long long)V, factor, factor_rows);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

}  // namespace llmt
