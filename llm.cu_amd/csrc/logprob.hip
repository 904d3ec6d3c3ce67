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
// reads them and writes their gradient.
#include <algorithm>

#include "ops.h"

namespace llmt {

namespace {

constexpr int NTH = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e4f;  // exp of it is 0

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

// (m, s, u): max x, sum exp(x - m), sum exp(x - m) (x - m).  The empty set is
// (-inf, 0, 0).
struct Stat {
  float m, s, u;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }
template <bool ENT>
__device__ __forceinline__ void merge(Stat& a, float m2, float s2, float u2) {
  const float mn = fmaxf(a.m, m2), ref = finite_ref(mn);
  const float d1 = a.m - ref, d2 = m2 - ref;
  const float f1 = __builtin_amdgcn_exp2f(d1 * kLog2e), f2 = __builtin_amdgcn_exp2f(d2 * kLog2e);
  if constexpr (ENT) {
    // far below, the factor is 0 and s d has to stay finite (a mask of the
    // type's lowest value, or an empty side's d = -inf)
    const float e1 = fmaxf(d1, kFar), e2 = fmaxf(d2, kFar);
    a.u = f1 * fmaf(a.s, e1, a.u) + f2 * fmaf(s2, e2, u2);
  }
  a.s = a.s * f1 + s2 * f2;
  a.m = mn;
}

// Adds NV values x (already read) to a thread's statistics: one rescale.
template <bool ENT, int NV>
__device__ __forceinline__ void add(Stat& a, const float (&x)[NV], float it) {
  float m = a.m;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, x[i] * it);
  const float ref = finite_ref(m);
  const float d = a.m - ref, f = __builtin_amdgcn_exp2f(d * kLog2e);
  float s = a.s * f, u = 0.f;
  if constexpr (ENT) u = f * fmaf(a.s, fmaxf(d, kFar), a.u);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float z = fmaf(x[i], it, -ref);
    const float e = __builtin_amdgcn_exp2f(z * kLog2e);
    s += e;
    if constexpr (ENT) u = fmaf(e, fmaxf(z, kFar), u);  // a logit of -inf adds nothing
  }
  a.m = m;
  a.s = s;
  a.u = u;
}

template <bool ENT>
__device__ __forceinline__ Stat wave_merge(Stat a) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(a.m, o, 64), s2 = __shfl_xor(a.s, o, 64);
    const float u2 = ENT ? __shfl_xor(a.u, o, 64) : 0.f;
    merge<ENT>(a, m2, s2, u2);
  }
  return a;
}

// A thread's share of columns [j0, j1) of a row, `nth` threads a row.
template <bool ENT, typename T>
__device__ __forceinline__ void scan(Stat& a, const T* row, int j0, int j1, int tid, int nth,
                                     float it) {
  constexpr int N = Piece<T>::N, U = 4;
  const int np = (j1 - j0) / N;
  int k = tid;
  for (; k + (U - 1) * nth < np; k += U * nth) {
    typename Piece<T>::V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const typename Piece<T>::V*>(row + j0 + (long long)N * (k + u * nth));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = (float)v[u][e];
      add<ENT, N>(a, x, it);
    }
  }
  for (; k < np; k += nth) {
    const typename Piece<T>::V v =
        *reinterpret_cast<const typename Piece<T>::V*>(row + j0 + (long long)N * k);
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (float)v[e];
    add<ENT, N>(a, x, it);
  }
  const int j = j0 + N * np + tid;
  if (j < j1) {
    const float x[1] = {(float)row[j]};
    add<ENT, 1>(a, x, it);
  }
}

// The row's outputs from its statistics (one thread).
template <bool ENT>
__device__ __forceinline__ void finish(const Stat& a, float xt, float it, long long row, float* logp,
                                       float2* stats, float* entropy) {
  if (a.m == -INFINITY && a.s == 0.f) {  // every logit is -inf: nothing has any probability
    logp[row] = -INFINITY;
    stats[row] = make_float2(-INFINITY, 0.f);
    if constexpr (ENT) entropy[row] = 0.f;
    return;
  }
  const float ls = logf(a.s);
  logp[row] = fmaf(xt, it, -a.m) - ls;
  stats[row] = make_float2(a.m, ls);
  if constexpr (ENT) entropy[row] = ls - a.u / a.s;
}

template <bool ENT, typename T>
__global__ __launch_bounds__(NTH) void logprob_row_kernel(const T* __restrict__ logits,
                                                          long long ld,
                                                          const int* __restrict__ targets, int rows,
                                                          int V, float it, float* __restrict__ logp,
                                                          float2* __restrict__ stats,
                                                          float* __restrict__ entropy) {
  __shared__ Stat part[NTH / 64];
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const int t = targets[row];
    if (t < 0 || t >= V) {
      if (threadIdx.x == 0) {
        logp[row] = 0.f;
        stats[row] = make_float2(0.f, 0.f);
        if constexpr (ENT) entropy[row] = 0.f;
      }
      continue;
    }
    const T* x = logits + row * ld;
    Stat a{-INFINITY, 0.f, 0.f};
    scan<ENT>(a, x, 0, V, threadIdx.x, NTH, it);
    a = wave_merge<ENT>(a);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < NTH / 64; ++w) merge<ENT>(a, part[w].m, part[w].s, part[w].u);
      finish<ENT>(a, (float)x[t], it, row, logp, stats, entropy);
    }
    __syncthreads();
  }
}

// A workgroup a (row, chunk of U pieces a thread).
constexpr int BU = 2;
template <bool ENT, typename T>
__global__ __launch_bounds__(NTH) void logprob_bwd_kernel(
    const T* logits, long long ld, const int* __restrict__ targets,
    const float2* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ dlogp, const float* __restrict__ dentropy, int rows, int V, float it,
    int chunks, T* dlogits, long long ldd) {
  constexpr int N = Piece<T>::N;
  const long long items = (long long)rows * chunks;
  for (long long w = blockIdx.x; w < items; w += gridDim.x) {
    const int row = (int)(w / chunks), ch = (int)(w - (long long)row * chunks);
    const int t = targets[row];
    const float g = dlogp[row] * it, h = ENT ? dentropy[row] * it : 0.f;
    const float2 st = stats[row];
    const bool zero = t < 0 || t >= V || (g == 0.f && h == 0.f) ||
                      (st.x == -INFINITY && st.y == 0.f);
    const float gh = ENT ? -fmaf(h, entropy[row], g) : -g;
    const int j0 = ch * (BU * N * NTH), j1 = min(V, j0 + BU * N * NTH);
    const T* x = logits + row * ld;
    T* d = dlogits + row * ldd;
    auto value = [&](float xv, int j) {
      float z = fmaf(xv, it, -st.x) - st.y;
      z = z < kFar ? kFar : z;  // exp is 0 there, and 0 * z has to stay 0
      const float p = __builtin_amdgcn_exp2f(z * kLog2e);
      if (j == t) {  // g (1 - p) without the cancellation
        const float dg = -g * expm1f(z);
        return ENT ? fmaf(-h * p, z + (entropy[row]), dg) : dg;
      }
      return p * (ENT ? fmaf(-h, z, gh) : gh);
    };
    const int np = (j1 - j0) / N;
    typename Piece<T>::V v[BU];
    if (!zero)
#pragma unroll
      for (int u = 0; u < BU; ++u)
        if ((int)threadIdx.x + u * NTH < np)
          v[u] = *reinterpret_cast<const typename Piece<T>::V*>(
              x + j0 + N * ((int)threadIdx.x + u * NTH));
#pragma unroll
    for (int u = 0; u < BU; ++u) {
      const int k = threadIdx.x + u * NTH;
      if (k < np) {
        const int j = j0 + N * k;
        typename Piece<T>::V o;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = zero ? (T)0.f : (T)value((float)v[u][e], j + e);
        *reinterpret_cast<typename Piece<T>::V*>(d + j) = o;
      }
    }
    const int j = j0 + N * np + threadIdx.x;
    if (j < j1) d[j] = zero ? (T)0.f : (T)value((float)x[j], j);
  }
}

}  // namespace

size_t logprob_workspace(int rows, int V, int dtype) { return 0; }

template <typename F>
static hipError_t with_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f((float*)nullptr);
    case kF16: return f((_Float16*)nullptr);
    default: return f((__bf16*)nullptr);
  }
}

hipError_t logprob_fwd(const LogprobArgs& a, void* workspace, hipStream_t st) {
  return with_type(a.dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const unsigned grid = (unsigned)std::min(a.rows, 1 << 20);
    if (a.entropy)
      hipLaunchKernelGGL((logprob_row_kernel<true, T>), dim3(grid), dim3(NTH), 0, st,
                         (const T*)a.logits, a.ld, a.targets, a.rows, a.V, a.it, a.logp,
                         (float2*)a.stats, a.entropy);
    else
      hipLaunchKernelGGL((logprob_row_kernel<false, T>), dim3(grid), dim3(NTH), 0, st,
                         (const T*)a.logits, a.ld, a.targets, a.rows, a.V, a.it, a.logp,
                         (float2*)a.stats, a.entropy);
    LLMT_LAUNCH_CHECK();
    return hipSuccess;
  });
}

hipError_t logprob_bwd(const LogprobArgs& a, hipStream_t st) {
  return with_type(a.dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const int per = BU * Piece<T>::N * NTH, chunks = (a.V + per - 1) / per;
    const unsigned grid = (unsigned)std::min<long long>((long long)a.rows * chunks, 1 << 22);
    if (a.dentropy)
      hipLaunchKernelGGL((logprob_bwd_kernel<true, T>), dim3(grid), dim3(NTH), 0, st,
                         (const T*)a.logits, a.ld, a.targets, (const float2*)a.stats, a.entropy,
                         a.dlogp, a.dentropy, a.rows, a.V, a.it, chunks, (T*)a.dlogits, a.ldd);
    else
      hipLaunchKernelGGL((logprob_bwd_kernel<false, T>), dim3(grid), dim3(NTH), 0, st,
                         (const T*)a.logits, a.ld, a.targets, (const float2*)a.stats, a.entropy,
                         a.dlogp, a.dentropy, a.rows, a.V, a.it, chunks, (T*)a.dlogits, a.ldd);
    LLMT_LAUNCH_CHECK();
    return hipSuccess;
  });
}

}  // namespace llmt
