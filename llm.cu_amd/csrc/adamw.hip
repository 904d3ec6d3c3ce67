// adamw.hip — one AdamW step over a list of tensors, moments in 32 or 8 bits.
//
//   g' = g f (f a factor on the device, or 1)
//   m = b1 m + (1 - b1) g';  v = b2 v + ((1 - b2) g') g'
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
// and p rounded to the working copy.  m and v are computed as written, each
// operation rounded (no contraction), so that 8-bit codes are defined to the
// bit; p takes the fp32 moments, before they are rounded to codes.
//
// 8-bit moments are floats of their own: blocks of 256 share a power-of-two
// scale 2^(e - 127) (a byte e), under which an m has a sign, 4 exponent and 3
// mantissa bits, a v 5 and 3, both with gradual underflow.  A power of two
// costs no precision under a float code, and 31 binades of v keep every step
// that the block's largest does not drown.  Rounding is stochastic: an average
// with b2 = 0.999 moves by less than half a step, which rounding to nearest
// would never let happen.  A v above 0 stays above 0, so that no denominator
// collapses.  In bits: y = |x| 2^(127 - e) 2^-112 (m; 2^-96 for v) is the float
// whose upper 12 bits are the code, and the rounding adds a 16-bit draw below.
//
// Memory-bound: 26 bytes an element with fp32 moments, 14 with 8-bit ones (a
// 16-bit gradient, plus 2 for a copy).  50.3 M parameters with copies: 266 us,
// 5.3 TB/s; 100.7 M with 8-bit moments 325 us, 5.0 TB/s, and the decoding of those
// moments into fp32 (adamw_moments_kernel) 227, 4.4.  200 tensors of up to 5000: three launches of 3.8 us.  A wave takes a
// block of 256 elements at a time, a workgroup one piece of one tensor.  The
// list is cut into launches of as many descriptors as travel in 4 KB of kernel
// arguments.
#include <algorithm>
#include <type_traits>

#include "ops.h"

namespace llmt {

namespace {

constexpr int NTH = 256, BLOCK = 256;
// Elements of a workgroup's piece: U blocks a wave, one after another.
template <int U>
constexpr int kPiece = NTH / 64 * BLOCK * U;

struct AdamDev32 {
  float* p;
  const void* g;
  void* m;
  void* v;
  void* copy;
  long long n;
  int first;               // its first workgroup
  unsigned index : 24;     // its place in the list
  unsigned gtype : 2;
  unsigned ctype : 2;      // kF32: no copy
  unsigned vec : 1;        // whole aligned accesses
};
struct AdamDev8 : AdamDev32 {
  unsigned char* mexp;
  unsigned char* vexp;
};
template <int BITS>
struct AdamBatch {
  using Dev = std::conditional_t<BITS == 8, AdamDev8, AdamDev32>;
  static constexpr int kMost = 3968 / sizeof(Dev);  // 70, and 55 with 8-bit moments
  Dev t[kMost];
  int count;
};

// 4 elements: consecutive and aligned (vec), or 64 apart.
template <class T>
__device__ __forceinline__ void load4(const T* p, bool vec, const bool (&ok)[4], float (&x)[4]) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  if (vec && ok[3]) {
    const T4 v = *reinterpret_cast<const T4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ok[i] ? (float)p[vec ? i : 64 * i] : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store4(T* p, bool vec, const bool (&ok)[4], const float (&x)[4]) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  if (vec && ok[3]) {
    T4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)x[i];
    *reinterpret_cast<T4*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ok[i]) p[vec ? i : 64 * i] = (T)x[i];
  }
}
__device__ __forceinline__ void load4_codes(const unsigned char* p, bool vec, const bool (&ok)[4],
                                            unsigned (&x)[4]) {
  if (vec && ok[3]) {
    const unsigned v = *reinterpret_cast<const unsigned*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v >> 8 * i & 255;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ok[i] ? p[vec ? i : 64 * i] : 0;
  }
}
__device__ __forceinline__ void store4_codes(unsigned char* p, bool vec, const bool (&ok)[4],
                                             const unsigned (&x)[4]) {
  if (vec && ok[3]) {
    *reinterpret_cast<unsigned*>(p) = x[0] | x[1] << 8 | x[2] << 16 | x[3] << 24;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ok[i]) p[vec ? i : 64 * i] = (unsigned char)x[i];
  }
}

// The largest over the wave, as bits (a NaN is above infinity).
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
  auto step = [](unsigned x, unsigned y) { return x > y ? x : y; };
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = step(r[0], r[1]);
  r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return step(r[0], r[1]);
}

// TOP: the code's exponent field of [1, 2) under the block's scale; m 15, v 31.
template <int TOP>
__device__ __forceinline__ float decode(unsigned c, unsigned e) {
  const float y = __uint_as_float((TOP == 15 ? c & 127 : c) << 20) *
                  __uint_as_float((unsigned)(254 - TOP) << 23);  // 2^(127 - TOP)
  const float x = y * __uint_as_float(min(e, 254u) << 23);
  const float s = TOP == 15 && c >= 128 ? -x : x;
  return e == 255 ? __uint_as_float(0x7fc00000u) : s;
}
// The exponent byte of a block whose largest magnitude has these bits: the
// largest stays at or below 1.875; 255 (infinite, NaN, or beyond 1.875 2^126) is a
// block of NaN.
__device__ __forceinline__ unsigned block_exp(unsigned amax) {
  const unsigned e = (amax >> 23) + ((amax & 0x7FFFFF) > 0x700000 ? 1 : 0);
  return e >= 254 ? 255 : e < 1 ? 1 : e;
}
template <int TOP>
__device__ __forceinline__ unsigned encode(float x, unsigned e, unsigned draw) {
  if (e == 255) return 0;
  const float y = (fabsf(x) * __uint_as_float((254 - e) << 23)) * __uint_as_float((unsigned)TOP << 23);
  unsigned c = (__float_as_uint(y) + (draw << 4)) >> 20;
  if (TOP == 15) return c | (x < 0.f ? 128u : 0u);
  return x > 0.f && c == 0 ? 1u : c;
}

__host__ __device__ __forceinline__ unsigned long long mix(unsigned long long x) {  // SplitMix64
  x += 0x9E3779B97F4A7C15ull;
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

__device__ __forceinline__ void moments(const AdamStep& k, float g, float& m, float& v) {
#pragma clang fp contract(off)
  const float gm = k.c1 * g, bm = k.b1 * m;
  m = bm + gm;
  const float gv = k.c2 * g, gg = gv * g, bv = k.b2 * v;
  v = bv + gg;
}

// (seven waves a SIMD: with six, two layers of 8-bit moments and their values take 572 us for 554)
template <int BITS, int U>
__global__ __launch_bounds__(NTH, 7) void adamw_list_kernel(const AdamBatch<BITS> b, const AdamStep k) {
  const int lane = threadIdx.x & 63;
  // a row of workgroups a tensor; or one row of all, in which this workgroup's
  // tensor is the last that begins at or before it
  const bool rows = gridDim.y > 1;
  int ti = rows ? blockIdx.y : 0;
  for (int hi = rows ? 0 : b.count; hi - ti > 1;) {
    const int mid = (ti + hi) / 2;
    if (b.t[mid].first <= (int)blockIdx.x) ti = mid;
    else hi = mid;
  }
  const auto& t = b.t[ti];
  const int piece = blockIdx.x - (rows ? 0 : t.first);
  const bool vec = t.vec;
  const float gs = k.gscale ? *k.gscale : 1.f;
  const unsigned long long key =
      BITS == 8 ? mix(k.seed ^ (((unsigned long long)(unsigned)k.step << 32) + t.index)) : 0;
  const long long base = (long long)piece * kPiece<U> + (threadIdx.x >> 6) * (U * BLOCK);
  for (int u = 0; u < U; ++u) {
    const long long i0 = base + u * BLOCK;
    if (i0 >= t.n) return;
    const long long at = i0 + (vec ? 4 * lane : lane);
    bool ok[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ok[e] = at + (vec ? e : 64 * e) < t.n;
    float p[4], g[4], m[4], v[4];
    load4(t.p + at, vec, ok, p);
    if (t.gtype == kF32) load4((const float*)t.g + at, vec, ok, g);
    else if (t.gtype == kF16) load4((const _Float16*)t.g + at, vec, ok, g);
    else load4((const __bf16*)t.g + at, vec, ok, g);
    if constexpr (BITS == 32) {
      load4((const float*)t.m + at, vec, ok, m);
      load4((const float*)t.v + at, vec, ok, v);
    } else {
      unsigned mc[4], vc[4];
      load4_codes((const unsigned char*)t.m + at, vec, ok, mc);
      load4_codes((const unsigned char*)t.v + at, vec, ok, vc);
      const unsigned me = t.mexp[i0 / BLOCK], ve = t.vexp[i0 / BLOCK];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = decode<15>(mc[e], me);
        v[e] = decode<31>(vc[e], ve);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gg = k.gscale ? g[e] * gs : g[e];
      moments(k, gg, m[e], v[e]);
      // the root's instruction takes a subnormal for 0, and v / (1 - b2^t) may leave fp32
      // where v does not: v below 1 at 2^64 times its size, others at 2^-64
      const bool low = v[e] < 1.f;
      const float root = __builtin_amdgcn_sqrtf(v[e] * (low ? k.ib2_up : k.ib2_down));
      const float denom = root * (low ? 0x1p-32f : 0x1p32f) + k.eps;
      p[e] = p[e] * k.decay - k.lr * (m[e] * k.ib1 * __builtin_amdgcn_rcpf(denom));
    }
    store4(t.p + at, vec, ok, p);
    if (t.ctype == kF16) store4((_Float16*)t.copy + at, vec, ok, p);
    else if (t.ctype == kBF16) store4((__bf16*)t.copy + at, vec, ok, p);
    if constexpr (BITS == 32) {
      store4((float*)t.m + at, vec, ok, m);
      store4((float*)t.v + at, vec, ok, v);
    } else {
      unsigned am = 0, av = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned x = __float_as_uint(m[e]) & 0x7FFFFFFF, y = __float_as_uint(v[e]) & 0x7FFFFFFF;
        am = ok[e] && x > am ? x : am;
        av = ok[e] && y > av ? y : av;
      }
      const unsigned me = block_exp(wave_umax(am)), ve = block_exp(wave_umax(av));
      unsigned mc[4], vc[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long long i = at + (vec ? e : 64 * e);
        const unsigned long long d = mix(key + (unsigned long long)(i >> 1));
        const unsigned h = (unsigned)(i & 1 ? d >> 32 : d);
        mc[e] = encode<15>(m[e], me, h & 0xFFFF);
        vc[e] = encode<31>(v[e], ve, h >> 16);
      }
      store4_codes((unsigned char*)t.m + at, vec, ok, mc);
      store4_codes((unsigned char*)t.v + at, vec, ok, vc);
      if (lane == 0) {
        t.mexp[i0 / BLOCK] = (unsigned char)me;
        t.vexp[i0 / BLOCK] = (unsigned char)ve;
      }
    }
  }
}

__global__ __launch_bounds__(NTH) void adamw_moments_kernel(const unsigned char* m,
                                                            const unsigned char* v,
                                                            const unsigned char* mexp,
                                                            const unsigned char* vexp, long long n,
                                                            float* m32, float* v32, bool vec) {
  const int lane = threadIdx.x & 63;
  for (long long i0 = (long long)blockIdx.x * kPiece<1> + (threadIdx.x >> 6) * BLOCK; i0 < n;
       i0 += (long long)gridDim.x * kPiece<1>) {
    const long long at = i0 + (vec ? 4 * lane : lane);
    bool ok[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ok[e] = at + (vec ? e : 64 * e) < n;
    unsigned mc[4], vc[4];
    load4_codes(m + at, vec, ok, mc);
    load4_codes(v + at, vec, ok, vc);
    const unsigned me = mexp[i0 / BLOCK], ve = vexp[i0 / BLOCK];
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = decode<15>(mc[e], me);
      y[e] = decode<31>(vc[e], ve);
    }
    store4(m32 + at, vec, ok, x);
    store4(v32 + at, vec, ok, y);
  }
}

constexpr long long kMostWgs = 1 << 24;  // of a launch (2^32 threads)
bool at4(const void* p, size_t es) { return (uintptr_t)p % (4 * es) == 0; }
size_t esize(int type) { return type == kF32 ? 4 : 2; }

}  // namespace

template <int BITS, int U>
static hipError_t launch_list(const AdamTensor* ts, int count, const AdamStep& k, hipStream_t st) {
  AdamBatch<BITS> b;
  for (int i = 0; i < count;) {
    long long wgs = 0, most = 0;
    b.count = 0;
    for (; i < count && b.count < AdamBatch<BITS>::kMost; ++i) {
      const AdamTensor& t = ts[i];
      if (t.n == 0) continue;
      const long long w = (t.n + kPiece<U> - 1) / kPiece<U>;
      if (b.count && wgs + w >= kMostWgs) break;
      auto& d = b.t[b.count++];
      d.p = t.p;
      d.g = t.g;
      d.m = t.m;
      d.v = t.v;
      d.copy = t.copy;
      d.n = t.n;
      d.first = (int)wgs;
      d.index = (unsigned)i;
      d.gtype = (unsigned)t.gtype;
      d.ctype = t.copy ? (unsigned)t.ctype : (unsigned)kF32;
      const size_t ms = BITS == 8 ? 1 : 4;
      d.vec = at4(t.p, 4) && at4(t.g, esize(t.gtype)) && at4(t.m, ms) && at4(t.v, ms) &&
              (!t.copy || at4(t.copy, 2));
      if constexpr (BITS == 8) {
        d.mexp = t.mexp;
        d.vexp = t.vexp;
      }
      wgs += w;
      most = std::max(most, w);
    }
    if (!b.count) break;
    // small tensors of like sizes: no search (3.4 us a launch, 5.1 with it);
    // elsewhere workgroups without work would cost more
    const bool rows = U == 1 && most * b.count <= 2 * wgs + 1024;
    const dim3 grid((unsigned)(rows ? most : wgs), rows ? b.count : 1);
    hipLaunchKernelGGL((adamw_list_kernel<BITS, U>), grid, dim3(NTH), 0, st, b, k);
    LLMT_LAUNCH_CHECK();
  }
  return hipSuccess;
}

hipError_t adamw_list(const AdamTensor* ts, int count, int bits, const AdamStep& k0,
                      hipStream_t st) {
  AdamStep k = k0;
  k.seed = mix(k0.seed);
  // few elements: a block a wave, so that none waits for a second (200 tensors
  // of up to 5000 elements: 13.9 us a call, 24.8 with four)
  long long n = 0;
  for (int i = 0; i < count; ++i) n += ts[i].n;
  const bool few = n <= 2048 * kPiece<1>;
  if (bits == 8)
    return few ? launch_list<8, 1>(ts, count, k, st) : launch_list<8, 4>(ts, count, k, st);
  return few ? launch_list<32, 1>(ts, count, k, st) : launch_list<32, 4>(ts, count, k, st);
}

hipError_t adamw_moments(const void* m, const void* v, const unsigned char* mexp,
                         const unsigned char* vexp, long long n, float* m32, float* v32,
                         hipStream_t st) {
  if (n == 0) return hipSuccess;
  const bool vec = at4(m, 1) && at4(v, 1) && at4(m32, 4) && at4(v32, 4);
  const long long wgs = std::min<long long>((n + kPiece<1> - 1) / kPiece<1>, 1 << 23);
  hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)wgs), dim3(NTH), 0, st,
                     (const unsigned char*)m, (const unsigned char*)v, mexp, vexp, n, m32, v32, vec);
  LLMT_LAUNCH_CHECK();
  return hipSuccess;
}

}  // namespace llmt
