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
// That trades steps x (4 r^2 n + 2 r^3) flops in as many passes over the matrix
// for 4 r^2 n + 8 steps r^3 in two.
//
// G holds the squares of the singular values, and a small one is amplified by
// up to 3.4445^2 a step: in fp32 the rounding of G (2^-24 of the largest
// square) would come out of five steps 2e5 times larger.  G, the iteration
// and the product are therefore fp64 on v_mfma_f64_16x16x4 (inputs are exact
// there), rounded once to fp32.
//
// Bound by HBM where the short side is 16 and matrices are many (the 28-layer
// Muon step, 128 MB: 26.7 us, 4.8 TB/s, a copy's rate), by the fp64 matrix rate
// above (28 x 12288 x 64: 4.5 GFLOP, gram 34 us, iteration 42, product 56), by
// launches and memory round trips for few matrices (1 x 16 x 2048: 10.3 us).
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

constexpr int NTH = 256, NW = NTH / 64;
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

// A stage is what a wave fetches at once, KW long-axis elements by 16 NT: it
// puts them into its own LDS rows [KW][LD] and nobody else reads those, so
// the loops below have no barriers and a wave's loads fly while it multiplies.
template <int NT>
struct Stage {
  static constexpr int KW = NT == 1 ? 64 : NT == 2 ? 32 : 16;
  static constexpr int PC = KW * NT / 16;  // 16-byte pieces a lane
  static constexpr int LD = 16 * NT + 1;
};

// A lane's pieces of a stage: piece i's place in LDS (its first element, and
// `step` to the next), its offset from the stage's first element in memory,
// and where the matrix ends.  A stage of all KW elements takes plain 16-byte
// accesses where the short side is all of 16 NT, 16-byte ones or none where it
// is whole pieces; the others count elements.
template <int NT>
struct Lane {
  static constexpr int PC = Stage<NT>::PC, LD = Stage<NT>::LD, KW = Stage<NT>::KW;
  int lane, step, r;
  bool tall;
  long long ld;
  __device__ __forceinline__ Lane(const NsMat& mt, long long ld_, int lane_)
      : lane(lane_), step(mt.tall ? 1 : LD), r(mt.r), tall(mt.tall), ld(ld_) {}
  __device__ __forceinline__ int kk(int i) const {
    const int idx = lane + 64 * i;
    return tall ? idx / (4 * NT) : 4 * (idx % (KW / 4));
  }
  __device__ __forceinline__ int sh(int i) const {
    const int idx = lane + 64 * i;
    return tall ? 4 * (idx % (4 * NT)) : idx / (KW / 4);
  }
  __device__ __forceinline__ long long at(int i) const {
    return tall ? kk(i) * ld + sh(i) : sh(i) * ld + kk(i);
  }
  __device__ __forceinline__ int lds(int i) const { return kk(i) * LD + sh(i); }
  // Offset of the stage at k from the matrix's start.
  __device__ __forceinline__ long long base(int k) const { return tall ? k * ld : k; }
  // Elements of piece i of the stage at k.
  __device__ __forceinline__ int have(int i, int k, int k1) const {
    return tall ? (k + kk(i) < k1 ? r - sh(i) : 0) : (sh(i) < r ? k1 - (k + kk(i)) : 0);
  }
  // f(i, elements) for every piece of the stage at k.
  template <typename F>
  __device__ __forceinline__ void pieces(int k, int k1, F&& f) const {
    const bool all = k + KW <= k1;
    if (all && r == 16 * NT) {
#pragma unroll
      for (int i = 0; i < PC; ++i) f(i, 4);
    } else if (all && r % 4 == 0) {
#pragma unroll
      for (int i = 0; i < PC; ++i) f(i, sh(i) < r ? 4 : 0);
    } else {
#pragma unroll
      for (int i = 0; i < PC; ++i) f(i, have(i, k, k1));
    }
  }
  __device__ __forceinline__ void load(floatx4 (&x)[PC], const float* p, int k, int k1) const {
    p += base(k);
    pieces(k, k1, [&](int i, int n) { x[i] = load4(p + at(i), n); });
  }
  __device__ __forceinline__ void store(float* p, const floatx4 (&x)[PC], int k, int k1) const {
    p += base(k);
    pieces(k, k1, [&](int i, int n) { store4(p + at(i), x[i], n); });
  }
  __device__ __forceinline__ void put(float (*S)[LD], const floatx4 (&x)[PC]) const {
#pragma unroll
    for (int i = 0; i < PC; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[0][lds(i) + e * step] = x[i][e];
  }
  __device__ __forceinline__ void get(floatx4 (&x)[PC], float (*S)[LD]) const {
#pragma unroll
    for (int i = 0; i < PC; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = S[0][lds(i) + e * step];
  }
};

// What the lanes of a wave wrote to LDS is read by its other lanes.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

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

// A stage of U, or of the gradient and the momentum, on its way into LDS.
template <int NT, bool MUON>
struct Fetch {
  floatx4 x[Stage<NT>::PC], m[Stage<NT>::PC];
  __device__ __forceinline__ void load(const NsArgs& a, const Lane<NT>& ln, long long in0, int k,
                                       int k1) {
    ln.load(x, a.x + in0, k, k1);
    if constexpr (MUON) ln.load(m, a.m + in0, k, k1);
  }
  // With MUON the momentum is updated and stored.
  __device__ __forceinline__ void put(const NsArgs& a, const Lane<NT>& ln, long long in0, int k,
                                      int k1, float (*S)[Stage<NT>::LD]) {
    if constexpr (MUON) {
#pragma unroll
      for (int i = 0; i < Stage<NT>::PC; ++i) x[i] = momentum(a, x[i], m[i]);
      ln.store(a.m + in0, m, k, k1);
    }
    ln.put(S, x);
  }
};

// The stage's part of G.
template <int NT>
__device__ __forceinline__ void gram_stage(float (*S)[Stage<NT>::LD], doublex4 (&acc)[ntri(NT)],
                                           int q, int c) {
#pragma unroll
  for (int s = 0; s < Stage<NT>::KW / 4; ++s) {
    double v[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) v[i] = S[4 * s + q][16 * i + c];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = i; j < NT; ++j) acc[tri(NT, i, j)] = mfma64(v[i], v[j], acc[tri(NT, i, j)]);
  }
}

// The stage times P, in its place, rounded.
template <int NT, typename TP>
__device__ __forceinline__ void apply_stage(float (*S)[Stage<NT>::LD],
                                            const TP& P, int q, int c) {
#pragma unroll
  for (int k = 0; k < Stage<NT>::KW; k += 16) {
    doublex4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = doublex4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const double u = S[k + c][16 * i + 4 * v + q];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = mfma64(u, P(i, j, v), acc[j]);
      }
    wave_fence();
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) S[k + 4 * v + q][16 * j + c] = (float)acc[j][v];
  }
}

// The product out of LDS to its place, or the parameters' update by it.
template <int NT, bool MUON>
__device__ __forceinline__ void store_stage(const NsArgs& a, const Lane<NT>& ln, float lr,
                                            long long out0, int k, int k1,
                                            float (*S)[Stage<NT>::LD],
                                            const floatx4 (&p)[Stage<NT>::PC]) {
  floatx4 o[Stage<NT>::PC];
  ln.get(o, S);
  if constexpr (MUON)
#pragma unroll
    for (int i = 0; i < Stage<NT>::PC; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = fmaf(-lr, o[i][e], p[i][e] * a.decay);
  ln.store(a.out + out0, o, k, k1);
}

// Block b of a matrix's `splits`: a k range in whole stages a wave.
template <int NT>
__device__ __forceinline__ void k_range(int n, int splits, int b, int& k0, int& k1) {
  constexpr int KG = Stage<NT>::KW * NW;
  const int groups = (n + KG - 1) / KG, per = (groups + splits - 1) / splits;
  k0 = (int)min((long long)b * per * KG, (long long)n);
  k1 = (int)min((long long)k0 + per * KG, (long long)n);
}

// G partials of one k range of a matrix: ws.gram[matrix][split][tile][v][lane].
template <int NT, bool MUON>
__global__ __launch_bounds__(NTH, 2) void ns_gram_kernel(const NsArgs a) {
  constexpr int KW = Stage<NT>::KW, LD = Stage<NT>::LD;
  __shared__ float S_[NW][KW][LD];
  __shared__ double red[ntri(NT)][256];
  const int mat = blockIdx.x / a.splits, split = blockIdx.x - mat * a.splits;
  const int layer = mat / a.nmat;
  const NsMat mt = a.mat[mat - layer * a.nmat];
  const long long in0 = layer * a.in_stride + mt.off;
  int k0, k1;
  k_range<NT>(mt.n, a.splits, split, k0, k1);
  const int lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float(*S)[LD] = S_[w];
  doublex4 acc[ntri(NT)];
#pragma unroll
  for (int i = 0; i < ntri(NT); ++i) acc[i] = doublex4{0, 0, 0, 0};
  const Lane<NT> ln(mt, mt.ld_in, lane);
  Fetch<NT, MUON> f;
  int k = k0 + KW * w;
  if (k < k1) f.load(a, ln, in0, k, k1);
  for (; k < k1; k += KW * NW) {
    wave_fence();
    f.put(a, ln, in0, k, k1, S);
    wave_fence();
    if (k + KW * NW < k1) f.load(a, ln, in0, k + KW * NW, k1);
    gram_stage<NT>(S, acc, q, c);
  }
  for (int t = 0; t < NW; ++t) {  // the waves' shares, in wave order
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

// Lane l's elements of the identity: rows 4 v + l / 16 of column l % 16.
__device__ __forceinline__ doublex4 identity(int lane) {
  doublex4 x;
#pragma unroll
  for (int v = 0; v < 4; ++v) x[v] = 4 * v + (lane >> 4) == (lane & 15) ? 1.0 : 0.0;
  return x;
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// X = M1 M2 of 16 x 16 matrices in a wave's registers.
__device__ __forceinline__ doublex4 product16(doublex4 m1, doublex4 m2) {
  doublex4 x = {0, 0, 0, 0};
#pragma unroll
  for (int v = 0; v < 4; ++v) x = mfma64(m1[v], m2[v], x);
  return x;
}

// P / (|U| + eps) of a 16 x 16 Gram matrix U U^T in a wave's registers: four
// products a step (three in the first, two in the last).
__device__ __forceinline__ doublex4 solve16(doublex4 G, int steps, double eps, int lane) {
  const doublex4 I = identity(lane);
  double t = 0.0;
#pragma unroll
  for (int v = 0; v < 4; ++v) t += I[v] != 0.0 ? G[v] : 0.0;
  const double inv = 1.0 / (sqrt(wave_sum_d(t)) + eps);
  G *= inv * inv;
  doublex4 B = kB * G + kC * product16(G, G);
  doublex4 P = kA * I + B;
  for (int step = 1; step < steps; ++step) {
    const doublex4 Y = kA * G + product16(B, G);  // p(G) G
    G = kA * Y + product16(B, Y);
    B = kB * G + kC * product16(G, G);
    P = kA * P + product16(B, P);
  }
  return P * inv;
}

// Element `at` of a matrix's G partials summed over the splits, in their
// order; eight loads in flight.
__device__ __forceinline__ double sum_splits(const double* part, int splits, long long step) {
  double t = 0.0;
  int s = 0;
  for (; s + 8 <= splits; s += 8) {
    double v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = part[(s + i) * step];
#pragma unroll
    for (int i = 0; i < 8; ++i) t += v[i];
  }
  for (; s < splits; ++s) t += part[s * step];
  return t;
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

// The iteration of one matrix, a wave a tile of the upper triangle (the lower one
// is written, not computed): the split partials into G0, then P, scaled for the
// product with U: ws.proj[matrix][tile row][tile col][v][lane].  Of 42 us at 28
// matrices of short side 64 the matrix instructions are 18 (22 on the fullest
// SIMD) and bank conflicts of the transposed tiles 11; the splits are summed before.
template <int NT>
__global__ __launch_bounds__(64 * ntri(NT)) void ns_solve_kernel(const NsArgs a) {
  constexpr int M = NT * NT * 256;
  __shared__ double sG[M], sY[M], sB[M], sP[M], tr[NT];
  const int mat = blockIdx.x;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4, c = lane & 15;
  int i = 0, j = w;  // wave w's tile
  while (j >= NT - i) j -= NT - i, ++i;
  j += i;
  const double* part = a.gram + (long long)mat * a.splits * ntri(NT) * 256 + w * 256 + lane;
  doublex4 G;
#pragma unroll
  for (int v = 0; v < 4; ++v) G[v] = sum_splits(part + 64 * v, a.splits, ntri(NT) * 256);
  const doublex4 I = i == j ? identity(lane) : doublex4{0, 0, 0, 0};
  double t = 0.0;
#pragma unroll
  for (int v = 0; v < 4; ++v) t += I[v] != 0.0 ? G[v] : 0.0;
  t = wave_sum_d(t);
  if (i == j && lane == 0) tr[i] = t;
  __syncthreads();
  t = 0.0;
#pragma unroll
  for (int k = 0; k < NT; ++k) t += tr[k];
  const double inv = 1.0 / (sqrt(t) + a.eps);
  G *= inv * inv;
  auto put = [&](double* m, doublex4 x) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      m[(i * NT + j) * 256 + 64 * v + lane] = x[v];
      // row 4 v + q, column c of tile (i, j) is row c, column 4 v + q of (j, i)
      if (i != j) m[(j * NT + i) * 256 + 64 * (c >> 2) + 16 * (c & 3) + 4 * v + q] = x[v];
    }
  };
  put(sG, G);
  __syncthreads();
  doublex4 B = kB * G + kC * product<NT>(sG, sG, i, j, lane);
  doublex4 P = kA * I + B;
  put(sB, B);
  __syncthreads();
  // three barriers a step: a buffer is written a barrier after its last reader
  for (int step = 1; step < a.steps; ++step) {
    const doublex4 Y = kA * G + product<NT>(sB, sG, i, j, lane);  // p(G) G
    if (step > 1) P = kA * P + product<NT>(sB, sP, i, j, lane);
    put(sY, Y);
    __syncthreads();
    G = kA * Y + product<NT>(sB, sY, i, j, lane);
    put(sG, G);
    put(sP, P);
    __syncthreads();
    B = kB * G + kC * product<NT>(sG, sG, i, j, lane);
    put(sB, B);
    __syncthreads();
  }
  if (a.steps > 1) P = kA * P + product<NT>(sB, sP, i, j, lane);
  put(a.proj + (long long)mat * NT * NT * 256, P * inv);
}

// P U of one k range of a matrix, and with MUON the parameters' update by it
// (the momentum is already updated).  NT = 1: every workgroup iterates by
// itself (2 us, during which its first loads arrive), which is less than the
// launch that it saves.  Else P is read from LDS as it is used: in registers it
// left one or two waves a SIMD (28 layers at rank 64: 214 us, 259 so).
template <int NT, bool MUON>
__global__ __launch_bounds__(NTH, 2) void ns_apply_kernel(const NsArgs a) {
  constexpr int KW = Stage<NT>::KW, LD = Stage<NT>::LD, PC = Stage<NT>::PC;
  __shared__ float S_[NW][KW][LD];
  const int mat = blockIdx.x / a.splits, split = blockIdx.x - mat * a.splits;
  const int layer = mat / a.nmat;
  const NsMat mt = a.mat[mat - layer * a.nmat];
  const long long in0 = layer * a.in_stride + mt.off, out0 = layer * a.out_stride + mt.off;
  int k0, k1;
  k_range<NT>(mt.n, a.splits, split, k0, k1);
  const int lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float(*S)[LD] = S_[w];
  int k = k0 + KW * w;
  if (k0 >= k1) return;
  const Lane<NT> ln(mt, mt.ld_in, lane), lo(mt, mt.ld_out, lane);
  floatx4 x[PC], m[PC], p[PC];
  auto load = [&](int at) {
    if constexpr (MUON) ln.load(m, a.m + in0, at, k1);
    if (!MUON || a.nesterov) ln.load(x, a.x + in0, at, k1);
  };
  if (k < k1) {
    load(k);
    if constexpr (MUON) lo.load(p, a.out + out0, k, k1);
  }
  __shared__ double red[NT * NT * 256];  // P; NT = 1: first the sum over the splits
  doublex4 P1;
  if constexpr (NT == 1) {
    red[threadIdx.x] = sum_splits(a.gram + (long long)mat * a.splits * 256 + threadIdx.x, a.splits,
                                  256);
    __syncthreads();
    if (w == 0) {
      doublex4 G;
#pragma unroll
      for (int v = 0; v < 4; ++v) G[v] = red[64 * v + lane];
      G = solve16(G, a.steps, a.eps, lane);
#pragma unroll
      for (int v = 0; v < 4; ++v) red[64 * v + lane] = G[v];
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v) P1[v] = red[64 * v + lane];
  } else {
    const double* proj = a.proj + (long long)mat * NT * NT * 256;
#pragma unroll
    for (int i = 0; i < NT * NT; ++i) red[256 * i + threadIdx.x] = proj[256 * i + threadIdx.x];
    __syncthreads();
  }
  auto P = [&](int i, int j, int v) {
    return NT == 1 ? P1[v] : red[(i * NT + j) * 256 + 64 * v + lane];
  };
  for (; k < k1; k += KW * NW) {
    wave_fence();
    if constexpr (MUON)
#pragma unroll
      for (int i = 0; i < PC; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = a.nesterov ? fmaf(a.mu, m[i][e], x[i][e]) : m[i][e];
    ln.put(S, x);
    wave_fence();
    const int next = k + KW * NW;
    if (next < k1) load(next);
    apply_stage<NT>(S, P, q, c);
    wave_fence();
    store_stage<NT, MUON>(a, lo, mt.lr, out0, k, k1, S, p);
    if constexpr (MUON)
      if (next < k1) lo.load(p, a.out + out0, next, k1);
  }
}

// A whole matrix of short side <= 16 in one workgroup: U is read once into LDS,
// its Gram matrix summed over the waves, wave 0 iterates, and every wave
// multiplies the stages that it fetched.
constexpr int FTH = 512, FW = FTH / 64, FKW = Stage<1>::KW, FLD = Stage<1>::LD;
constexpr int kLdsBytes = 160 * 1024;
__host__ __device__ constexpr int fused_rows(int n) { return (n + FKW - 1) / FKW * FKW; }
constexpr size_t fused_lds(int n) {
  return (size_t)fused_rows(n) * FLD * sizeof(float) + FW * 256 * sizeof(double);
}


template <bool MUON>
__global__ __launch_bounds__(FTH) void ns_fused_kernel(const NsArgs a) {
  extern __shared__ double lds[];
  double* red = lds;  // [FW][256], then P
  float(*S)[FLD] = reinterpret_cast<float(*)[FLD]>(lds + FW * 256);
  const int mat = blockIdx.x, layer = mat / a.nmat;
  const NsMat mt = a.mat[mat - layer * a.nmat];
  const long long in0 = layer * a.in_stride + mt.off, out0 = layer * a.out_stride + mt.off;
  const int lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  doublex4 acc[1] = {{0, 0, 0, 0}};
  const Lane<1> ln(mt, mt.ld_in, lane), lo(mt, mt.ld_out, lane);
  Fetch<1, MUON> f;
  int k = FKW * w;
  if (k < mt.n) f.load(a, ln, in0, k, mt.n);
  for (; k < mt.n; k += FKW * FW) {
    f.put(a, ln, in0, k, mt.n, S + k);
    wave_fence();
    if (k + FKW * FW < mt.n) f.load(a, ln, in0, k + FKW * FW, mt.n);
    gram_stage<1>(S + k, acc, q, c);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) red[256 * w + 64 * v + lane] = acc[0][v];
  // the first parameters are fetched before the iteration
  floatx4 p[Stage<1>::PC];
  k = FKW * w;
  if constexpr (MUON)
    if (k < mt.n) lo.load(p, a.out + out0, k, mt.n);
  __syncthreads();
  if (w == 0) {
    doublex4 G = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < FW; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) G[v] += red[256 * t + 64 * v + lane];
    const doublex4 P = solve16(G, a.steps, a.eps, lane);
#pragma unroll
    for (int v = 0; v < 4; ++v) red[64 * v + lane] = P[v];
  }
  __syncthreads();
  doublex4 P1;
#pragma unroll
  for (int v = 0; v < 4; ++v) P1[v] = red[64 * v + lane];
  auto P = [&](int, int, int v) { return P1[v]; };
  for (; k < mt.n; k += FKW * FW) {
    apply_stage<1>(S + k, P, q, c);
    wave_fence();
    store_stage<1, MUON>(a, lo, mt.lr, out0, k, mt.n, S + k, p);
    if constexpr (MUON)
      if (k + FKW * FW < mt.n) lo.load(p, a.out + out0, k + FKW * FW, mt.n);
  }
}

// Workgroups of the gram and apply launches: two a CU (28 x 12288 x 64: 130 us,
// 134 with one a CU, 139 with four; 20 x 4096 x 32: 30.4, 30.7, 33.6).
constexpr int kTargetWg = 512;

// k ranges a matrix, in groups of a stage a wave.
int splits_for(const NsArgs& a, int nt) {
  int n = 1;
  for (int j = 0; j < a.nmat; ++j) n = std::max(n, a.mat[j].n);
  const int group = (nt == 1 ? Stage<1>::KW : nt == 2 ? Stage<2>::KW : Stage<3>::KW) * NW;
  const int groups = (n + group - 1) / group, mats = a.layers * a.nmat;
  const int want = std::min(std::max(1, kTargetWg / mats), groups);
  const int per = (groups + want - 1) / want;  // groups a block
  return (groups + per - 1) / per;
}

size_t gram_bytes(const NsArgs& a, int nt) {
  return (size_t)a.layers * a.nmat * splits_for(a, nt) * ntri(nt) * 256 * sizeof(double);
}
size_t class_bytes(const NsArgs& a, int nt) {
  return gram_bytes(a, nt) + (size_t)a.layers * a.nmat * nt * nt * 256 * sizeof(double);
}

// The matrices of `all` whose short side takes nt tiles of 16; 0: those that
// the one-workgroup kernel takes, which the others then leave out.  It is one
// launch, but one CU's fp64 rate and memory lanes a matrix: long sides of up to
// 1024 take it at any count (in a graph, 1 x 16 x 512: 8.7 us, 10.2 in two
// launches; 1 x 16 x 1024: 11.5 and 10.6, level with the second launch's cost
// to a caller), longer ones from kFusedMats matrices on (2048: 17.1 and 10.5
// for one, 19.1 and 18.1 for 128, 20.6 and 26.3 for 224; Muon, 64 matrices 21.7
// and 17.4, 128 23.4 and 25.1, 224 27.7 and 37).  All matrices of a call that
// fit go one way.
constexpr int kFusedLong = 1024, kFusedMats = 112;
NsArgs class_of(const NsArgs& all, int nt) {
  auto fits = [](const NsMat& m) { return m.r <= 16 && fused_lds(m.n) <= kLdsBytes; };
  int longest = 0, count = 0;
  for (int j = 0; j < all.nmat; ++j)
    if (fits(all.mat[j])) longest = std::max(longest, all.mat[j].n), count += all.layers;
  const bool fuse = longest <= kFusedLong || count >= kFusedMats;
  NsArgs a = all;
  a.nmat = 0;
  for (int j = 0; j < all.nmat; ++j) {
    const bool one = fuse && fits(all.mat[j]);
    if (nt == 0 ? one : !one && (all.mat[j].r + 15) / 16 == nt) a.mat[a.nmat++] = all.mat[j];
  }
  return a;
}

template <bool MUON>
hipError_t launch_fused(const NsArgs& a, hipStream_t st) {
  size_t lds = 0;
  for (int j = 0; j < a.nmat; ++j) lds = std::max(lds, fused_lds(a.mat[j].n));
  hipLaunchKernelGGL(ns_fused_kernel<MUON>, dim3((unsigned)(a.layers * a.nmat)), dim3(FTH), lds, st,
                     a);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

template <int NT, bool MUON>
hipError_t launch(NsArgs a, void* ws, hipStream_t st) {
  a.splits = splits_for(a, NT);
  a.gram = (double*)ws;
  a.proj = (double*)((char*)ws + gram_bytes(a, NT));
  const unsigned mats = (unsigned)(a.layers * a.nmat);
  hipLaunchKernelGGL((ns_gram_kernel<NT, MUON>), dim3(mats * a.splits), dim3(NTH), 0, st, a);
  LLMT_LAUNCH_CHECK();
  if constexpr (NT > 1) {
    hipLaunchKernelGGL((ns_solve_kernel<NT>), dim3(mats), dim3(64 * ntri(NT)), 0, st, a);
    LLMT_LAUNCH_CHECK();
  }
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
  for (int nt = 0; nt <= kNsMaxShort / 16; ++nt) {
    const NsArgs a = class_of(all, nt);
    if (!a.nmat) continue;
    auto go = [&](auto n) {
      constexpr int NT = decltype(n)::value;
      return a.m ? launch<NT, true>(a, ws, st) : launch<NT, false>(a, ws, st);
    };
    using std::integral_constant;
    hipError_t e = nt == 0   ? (a.m ? launch_fused<true>(a, st) : launch_fused<false>(a, st))
                   : nt == 1 ? go(integral_constant<int, 1>())
                   : nt == 2 ? go(integral_constant<int, 2>())
                   : nt == 3 ? go(integral_constant<int, 3>())
                             : go(integral_constant<int, 4>());
    LLMT_HIP_TRY(e);
  }
  return hipSuccess;
}

}  // namespace llmt
