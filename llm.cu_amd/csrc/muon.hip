// muon.hip — orthogonalising an update by Newton-Schulz products, and the
// Muon step on an arena of matrices.
//
// X0 = U / (|U| + eps) (Frobenius norm), then `steps` times
//   X <- a X + b (X X^T) X + c (X X^T)^2 X,   (a, b, c) = (3.4445, -4.7750, 2.0315),
// which carries every singular value toward 1 and leaves the vectors.  One
// side of an adapter is its rank r: with G = X X^T on that side and
// p(G) = a I + b G + c G^2, the iterate is a polynomial of G times X0,
//   X_k = P_k X0,  P <- p(G) P,  G <- p(G)^2 G,
// so the matrix is read once for G0 = U U^T / (|U| + eps)^2 (|U|^2 is its
// trace) and once for the product P U, and the iteration itself is r x r.
// That trades 2 steps (4 r^2 n + 2 r^3) flops and as many passes for two.
//
// G holds the squares of the singular values, and a small one is amplified by
// up to 3.4445^2 a step: in fp32 the rounding of G (2^-24 of the largest
// square) would come out of five steps 2e5 times larger.  G, the iteration
// and the product are therefore fp64 on v_mfma_f64_16x16x4 (inputs are exact
// there), rounded once to fp32.
//
// All matrices of the iteration are symmetric and commute.  A lane of an f64
// MFMA result holds rows 4 v + l / 16 (v = 0..3) of column l % 16; read by
// symmetry the same registers are a first operand with row l % 16 and a
// second operand with column l % 16, their k in the same order, so a product
// takes its operands as the last product left them.
#include <algorithm>

#include "ops.h"

namespace llmt {

namespace {

constexpr int NTH = 256;
constexpr int KT = 64;  // long-axis elements a stage
constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;

typedef double doublex4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ doublex4 mfma64(double a, double b, doublex4 c) {
  return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

// Tile (i, j), i <= j, of an upper triangle of NT x NT tiles.
__host__ __device__ constexpr int tri(int nt, int i, int j) { return i * nt - i * (i - 1) / 2 + j - i; }
__host__ __device__ constexpr int ntri(int nt) { return nt * (nt + 1) / 2; }

// Four elements of U (or of a stream beside it): along the long axis of a
// wide matrix [r, n], along the short one of a tall matrix [n, r].  `have` of
// them exist.
__device__ __forceinline__ floatx4 load4(const float* p, int have) {
  if (have >= 4) {
    const f4u v = *reinterpret_cast<const f4u*>(p);
    return floatx4{v[0], v[1], v[2], v[3]};
  }
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < have) v[e] = p[e];
  return v;
}
__device__ __forceinline__ void store4(float* p, floatx4 v, int have) {
  if (have >= 4) {
    f4u o = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f4u*>(p) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < have) p[e] = v[e];
}

// Piece `idx` of the stage at k0: its place in LDS (long index k, short index
// s, step of its four elements), how many of them exist and its offset from
// the matrix's start.
template <int NT>
struct Place {
  int k, s, have;
  long long at;
  bool tall;
  __device__ __forceinline__ Place(const NsMat& mt, long long ld, int k0, int k1, int idx) {
    tall = mt.tall;
    if (tall) {
      k = idx / (4 * NT);
      s = 4 * (idx - k * (4 * NT));
      have = k0 + k < k1 ? mt.r - s : 0;
      at = (k0 + k) * ld + s;
    } else {
      s = idx >> 4;
      k = 4 * (idx & 15);
      have = s < mt.r ? k1 - (k0 + k) : 0;
      at = s * ld + k0 + k;
    }
  }
  template <int LD>
  __device__ __forceinline__ void put(float (*S)[LD], floatx4 v) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) tall ? S[k][s + e] = v[e] : S[k + e][s] = v[e];
  }
  template <int LD>
  __device__ __forceinline__ floatx4 get(float (*S)[LD]) const {
    floatx4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = tall ? S[k][s + e] : S[k + e][s];
    return v;
  }
};

// The momentum update of four elements: m <- mu m + g and the update u.
__device__ __forceinline__ floatx4 momentum(const NsArgs& a, floatx4 g, floatx4& m) {
  floatx4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = fmaf(a.mu, m[e], g[e]);
    u[e] = a.nesterov ? fmaf(a.mu, m[e], g[e]) : m[e];
  }
  return u;
}

// Block b of a matrix's `splits`: k range in whole stages.
__device__ __forceinline__ void k_range(int n, int splits, int b, int& k0, int& k1) {
  const int stages = (n + KT - 1) / KT, per = (stages + splits - 1) / splits;
  k0 = (int)min((long long)b * per * KT, (long long)n);
  k1 = (int)min((long long)k0 + per * KT, (long long)n);
}

// G partials of one k range of a matrix: ws.gram[matrix][split][tile][v][lane].
template <int NT, bool MUON>
__global__ __launch_bounds__(NTH) void ns_gram_kernel(const NsArgs a) {
  constexpr int LD = 16 * NT + 1;
  __shared__ float S[KT][LD];
  __shared__ double red[ntri(NT)][256];
  const int mat = blockIdx.x / a.splits, split = blockIdx.x - mat * a.splits;
  const int layer = mat / a.nmat;
  const NsMat mt = a.mat[mat - layer * a.nmat];
  const long long in0 = layer * a.in_stride + mt.off, ld = mt.ld_in;
  int k0, k1;
  k_range(mt.n, a.splits, split, k0, k1);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4, c = lane & 15;
  doublex4 acc[ntri(NT)];
#pragma unroll
  for (int i = 0; i < ntri(NT); ++i) acc[i] = doublex4{0, 0, 0, 0};
  for (int k = k0; k < k1; k += KT) {
    floatx4 x[NT], m[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const Place<NT> pl(mt, ld, k, k1, threadIdx.x + NTH * i);
      x[i] = load4(a.x + in0 + pl.at, pl.have);
      if constexpr (MUON) m[i] = load4(a.m + in0 + pl.at, pl.have);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const Place<NT> pl(mt, ld, k, k1, threadIdx.x + NTH * i);
      if constexpr (MUON) {
        x[i] = momentum(a, x[i], m[i]);
        store4(a.m + in0 + pl.at, m[i], pl.have);
      }
      pl.put(S, x[i]);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      double v[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) v[i] = S[16 * w + 4 * s + q][16 * i + c];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = i; j < NT; ++j) acc[tri(NT, i, j)] = mfma64(v[i], v[j], acc[tri(NT, i, j)]);
    }
  }
  for (int t = 0; t < NTH / 64; ++t) {  // the waves' shares, in wave order
    if (w == t)
#pragma unroll
      for (int i = 0; i < ntri(NT); ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          red[i][64 * v + lane] = t ? red[i][64 * v + lane] + acc[i][v] : acc[i][v];
    __syncthreads();
  }
  double* out = a.gram + ((long long)mat * a.splits + split) * ntri(NT) * 256;
  for (int i = threadIdx.x; i < ntri(NT) * 256; i += NTH) out[i] = red[i >> 8][i & 255];
}

// X = M1 M2, tile (i, j) of it: operands as fragments [tile row][tile col][v][lane].
template <int NT>
__device__ __forceinline__ doublex4 product(const double* m1, const double* m2, int i, int j,
                                            int lane) {
  doublex4 x = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 4; ++v)
      x = mfma64(m1[(t * NT + i) * 256 + 64 * v + lane], m2[(t * NT + j) * 256 + 64 * v + lane], x);
  return x;
}

// The iteration of one matrix, a wave a tile: the split partials into G0, then
// P, scaled for the product with U: ws.proj[matrix][tile row][tile col][v][lane].
template <int NT>
__global__ __launch_bounds__(64 * NT * NT) void ns_solve_kernel(const NsArgs a) {
  __shared__ double sG[NT * NT * 256], sB[NT * NT * 256], sP[NT * NT * 256];
  __shared__ double tr[NT];
  const int mat = blockIdx.x;
  const NsMat mt = a.mat[mat % a.nmat];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = w / NT, j = w - i * NT;
  const int q = lane >> 4, c = lane & 15;
  const double* part = a.gram + (long long)mat * a.splits * ntri(NT) * 256;
  doublex4 G = {0, 0, 0, 0};
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    // below the diagonal: the transposed element of tile (j, i)
    const int at = i <= j ? tri(NT, i, j) * 256 + 64 * v + lane
                          : tri(NT, j, i) * 256 + 64 * (c >> 2) + 16 * (c & 3) + 4 * v + q;
    for (int s = 0; s < a.splits; ++s) G[v] += part[(long long)s * ntri(NT) * 256 + at];
  }
  doublex4 I;
#pragma unroll
  for (int v = 0; v < 4; ++v) I[v] = i == j && 4 * v + q == c ? 1.0 : 0.0;
  double t = 0.0;
#pragma unroll
  for (int v = 0; v < 4; ++v) t += I[v] != 0.0 ? G[v] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if (i == j && lane == 0) tr[i] = t;
  __syncthreads();
  t = 0.0;
#pragma unroll
  for (int k = 0; k < NT; ++k) t += tr[k];
  const double inv = 1.0 / (sqrt(t) + a.eps);
  G *= inv * inv;
  doublex4 P = I;
  auto put = [&](double* m, doublex4 x) {
#pragma unroll
    for (int v = 0; v < 4; ++v) m[w * 256 + 64 * v + lane] = x[v];
  };
  for (int step = 0; step < a.steps; ++step) {
    put(sG, G);
    put(sP, P);
    __syncthreads();
    const doublex4 B = kB * G + kC * product<NT>(sG, sG, i, j, lane);
    put(sB, B);
    __syncthreads();
    P = kA * P + product<NT>(sB, sP, i, j, lane);
    if (step + 1 == a.steps) break;
    const doublex4 Y = kA * G + product<NT>(sB, sG, i, j, lane);  // p(G) G
    __syncthreads();
    put(sG, Y);
    __syncthreads();
    G = kA * Y + product<NT>(sB, sG, i, j, lane);
    __syncthreads();
  }
  P *= inv;
  double* out = a.proj + (long long)mat * NT * NT * 256;
#pragma unroll
  for (int v = 0; v < 4; ++v) out[w * 256 + 64 * v + lane] = P[v];
}

// P U of one k range of a matrix, and with MUON the parameters' update by it.
template <int NT, bool MUON>
__global__ __launch_bounds__(NTH) void ns_apply_kernel(const NsArgs a) {
  constexpr int LD = 16 * NT + 1;
  __shared__ float S[KT][LD];
  const int mat = blockIdx.x / a.splits, split = blockIdx.x - mat * a.splits;
  const int layer = mat / a.nmat;
  const NsMat mt = a.mat[mat - layer * a.nmat];
  const long long in0 = layer * a.in_stride + mt.off, out0 = layer * a.out_stride + mt.off;
  int k0, k1;
  k_range(mt.n, a.splits, split, k0, k1);
  if (k0 >= k1) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4, c = lane & 15;
  const double* proj = a.proj + (long long)mat * NT * NT * 256;
  doublex4 P[NT][NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) P[i][j][v] = proj[(i * NT + j) * 256 + 64 * v + lane];
  for (int k = k0; k < k1; k += KT) {
    floatx4 x[NT], m[NT], p[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const Place<NT> pl(mt, mt.ld_in, k, k1, threadIdx.x + NTH * i);
      if constexpr (MUON) {
        m[i] = load4(a.m + in0 + pl.at, pl.have);  // already updated
        if (a.nesterov) x[i] = load4(a.x + in0 + pl.at, pl.have);
        p[i] = load4(a.out + in0 + pl.at, pl.have);
      } else {
        x[i] = load4(a.x + in0 + pl.at, pl.have);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const Place<NT> pl(mt, mt.ld_in, k, k1, threadIdx.x + NTH * i);
      if constexpr (MUON)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = a.nesterov ? fmaf(a.mu, m[i][e], x[i][e]) : m[i][e];
      pl.put(S, x[i]);
    }
    __syncthreads();
    doublex4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = doublex4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const double u = S[16 * w + c][16 * i + 4 * v + q];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = mfma64(u, P[i][j][v], acc[j]);
      }
    // a wave reads and writes its own 16 rows of the stage
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) S[16 * w + 4 * v + q][16 * j + c] = (float)acc[j][v];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const Place<NT> pl(mt, mt.ld_out, k, k1, threadIdx.x + NTH * i);
      floatx4 o = pl.get(S);
      if constexpr (MUON)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(-mt.lr, o[e], p[i][e] * a.decay);
      store4(a.out + out0 + pl.at, o, pl.have);
    }
  }
}

constexpr int kTargetWg = 1024;  // workgroups of the gram and apply launches

int splits_for(const NsArgs& a) {
  int n = 1;
  for (int j = 0; j < a.nmat; ++j) n = std::max(n, a.mat[j].n);
  const int stages = (n + KT - 1) / KT, mats = a.layers * a.nmat;
  const int want = std::min(std::max(1, kTargetWg / mats), stages);
  const int per = (stages + want - 1) / want;  // stages a block
  return (stages + per - 1) / per;
}

size_t gram_bytes(const NsArgs& a, int nt) {
  return (size_t)a.layers * a.nmat * splits_for(a) * ntri(nt) * 256 * sizeof(double);
}
size_t class_bytes(const NsArgs& a, int nt) {
  return gram_bytes(a, nt) + (size_t)a.layers * a.nmat * nt * nt * 256 * sizeof(double);
}

// The matrices of `all` whose short side takes nt tiles of 16.
NsArgs class_of(const NsArgs& all, int nt) {
  NsArgs a = all;
  a.nmat = 0;
  for (int j = 0; j < all.nmat; ++j)
    if ((all.mat[j].r + 15) / 16 == nt) a.mat[a.nmat++] = all.mat[j];
  return a;
}

template <int NT, bool MUON>
hipError_t launch(NsArgs a, void* ws, hipStream_t st) {
  a.splits = splits_for(a);
  a.gram = (double*)ws;
  a.proj = (double*)((char*)ws + gram_bytes(a, NT));
  const unsigned mats = (unsigned)(a.layers * a.nmat);
  hipLaunchKernelGGL((ns_gram_kernel<NT, MUON>), dim3(mats * a.splits), dim3(NTH), 0, st, a);
  LLMT_LAUNCH_CHECK();
  hipLaunchKernelGGL((ns_solve_kernel<NT>), dim3(mats), dim3(64 * NT * NT), 0, st, a);
  LLMT_LAUNCH_CHECK();
  hipLaunchKernelGGL((ns_apply_kernel<NT, MUON>), dim3(mats * a.splits), dim3(NTH), 0, st, a);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

}  // namespace

size_t ns_workspace(const NsArgs& all) {
  size_t most = 0;
  for (int nt = 1; nt <= kNsMaxShort / 16; ++nt) {
    const NsArgs a = class_of(all, nt);
    if (a.nmat) most = std::max(most, class_bytes(a, nt));
  }
  return most;
}

hipError_t newton_schulz(const NsArgs& all, void* ws, hipStream_t st) {
  for (int nt = 1; nt <= kNsMaxShort / 16; ++nt) {
    const NsArgs a = class_of(all, nt);
    if (!a.nmat) continue;
    auto go = [&](auto n) {
      constexpr int NT = decltype(n)::value;
      return a.m ? launch<NT, true>(a, ws, st) : launch<NT, false>(a, ws, st);
    };
    using std::integral_constant;
    hipError_t e = nt == 1   ? go(integral_constant<int, 1>())
                   : nt == 2 ? go(integral_constant<int, 2>())
                   : nt == 3 ? go(integral_constant<int, 3>())
                             : go(integral_constant<int, 4>());
    LLMT_HIP_TRY(e);
  }
  return hipSuccess;
}

}  // namespace llmt
