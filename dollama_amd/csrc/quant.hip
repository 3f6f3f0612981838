// Rows in 8 bits for gfx950: quantisation, the norms that end in it, and the
// way back.  No counterpart in the reference, whose linears are fp16 only
// (src/kernels/gemm.cu:425-434) and whose norms write fp16
// (src/kernels/layernorm.cu:78-126).
//
// A row v of K values becomes q[k] = round(127 v[k] / a) with a = max |v|,
// rounded to the nearest integer (halves to the even one), and scale =
// a / 127, so that v ~ q * scale.  The three sources of v:
//   quantise    v = x
//   RMS norm    h = x + residual, v = h gamma / sqrt(mean(h^2) + eps).  The
//               root cancels in q, so q is formed from h gamma / max|h gamma|
//               and only the scale sees it: the largest magnitude and the sum
//               of squares come out of one pass over the row.
//   LayerNorm   v = (h - mean) / sqrt(var + eps) gamma + beta, the variance from
//               the differences (rows whose mean is far from 0 keep theirs)
//
// Rounding.  127 v / a is formed as v * (127 * rcp(a)) in fp32, which is off by
// 2.3e-5 at most (relative errors of 2^-23 and 2^-24 on values up to 127).
// Quotients within 2^-15 of a half (one in 16,000) are decided again by comparing
// 254 v with (2k + 1) a in fp64, where both products are exact.  So q is the
// quotient's nearest integer whatever the launch looks like: exactly for fp16 rows
// (and fp16 gamma) of the first two kinds and for fp32 rows of the first, where v is
// exact in fp32.  An fp32 row's products with gamma are exact in fp64, and are that;
// so are LayerNorm's statistics and values, whose quotients come out to 2^-38.  (In
// fp32 one integer in 8 million of the former fell on the other side of a half, one in
// a million of the latter, 15 in a million where the mean is 40 times the spread; and
// the squares of rows beyond 1e19 or below 1e-19 were lost.)  fp64 instructions run at
// fp32's rate here; the values take twice the registers, which many rows notice:
// LayerNorm 8192x1280 11.8 -> 13.3 us, 8192x640 7.3 -> 7.7, RMS norm of 8192x640 in
// fp32 7.4 -> 8.6, with residual 12.2 -> 12.3.
//
// What bounds them: memory, one pass.  A row stays in registers between its
// statistics and its output, in 8 to 512 threads by its length.  Measured (graph
// replays, inputs that no cache holds): quantise 8192x1280 fp16 8.2 us (3.8 TB/s,
// of which the launch is 2 us), RMS norm with residual 13.5 us (5.4 TB/s; fp32
// 27.2 us, 5.0), LayerNorm 13.4 us (2.3 TB/s: some 16 VALU instructions a value
// and three reductions in a chain; with residual 15.3 us, 4.8 TB/s; fp32 14.9 and
// 27.5); a 1 GiB copy reaches 5.15 TB/s.  One row: 2.3 us, 2.9 and 3.2.
#include <algorithm>

#include "common.hpp"

namespace dlm {
namespace {

enum RowKind { kQuant, kRms, kLayer };

struct RowArgs {
  const void* x;
  const void* res;  // may be NULL
  void* h;          // x + res, or NULL
  const f16* gamma;
  const f16* beta;
  int8_t* q;
  float* scale;
  long long ldx, ldr, ldh, ldq;
  int rows, K;
  float eps;
  double inv_k;
};

// What a row's statistics, and its values on their way to q, are held in: fp64
// where fp32 would round them.
template <class T, RowKind KIND>
using Wide = std::conditional_t<KIND == kLayer || (KIND == kRms && sizeof(T) == 4), double, float>;

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef double f64x8 __attribute__((ext_vector_type(8)));
template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

// Eight elements at any element-aligned address: one 16-byte access (two for
// fp32), which the hardware takes at any alignment.
template <class T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& v) {
  __builtin_memcpy(p, &v, sizeof(v));
}
// Largest magnitude, NaN where one of the two is NaN (v_maximum3_f32 for two
// values at a time).
__device__ __forceinline__ float max_abs(float m, float v) { return __builtin_elementwise_maximum(m, fabsf(v)); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// fp64 has no such instruction: these pass NaN over, and `Top` remembers it.
__device__ __forceinline__ double max_abs(double m, double v) { return __builtin_fmax(m, __builtin_fabs(v)); }
__device__ __forceinline__ double max_nan(double a, double b) { return __builtin_fmax(a, b); }

// Running maximum of |v|; infinite or NaN once a value was.
template <class W>
struct Top {
  W top = 0, zero = 0;  // zero: 0 times every value
  __device__ __forceinline__ void add(W v) {
    top = max_abs(top, v);
    if constexpr (sizeof(W) == 8) zero = __builtin_fma(v, 0.0, zero);
  }
  __device__ __forceinline__ W get() const { return sizeof(W) == 8 && !(zero == 0) ? (W)INFINITY : top; }
};

// What a row's values are multiplied by on their way to q.
template <class W>
struct RowScale {
  W r;         // 127 / (a m), 0 for rows without a finite positive maximum
  W a;         // a m
  float m;     // fp32 rows: a power of two that keeps 127 / a and its reciprocal normal numbers; else 1
  W unit;      // a / 127, NaN for a row that holds an infinity or NaN
};
// a: max |v|, not finite if a value is not.  Values of fp16 rows are no smaller
// than 2^-48 where they are not 0.
template <class T>
__device__ __forceinline__ RowScale<float> row_scale(float a, bool bad) {
  RowScale<float> s;
  bad = bad || !(a < INFINITY);
  s.m = sizeof(T) == 2 ? 1.0f : a < 0x1p-100f ? 0x1p100f : a > 0x1p100f ? 0x1p-100f : 1.0f;
  s.a = a * s.m;
  s.r = bad || a == 0.0f ? 0.0f : 127.0f * __builtin_amdgcn_rcpf(s.a);
  s.unit = bad ? __uint_as_float(0x7fc00000u) : a / 127.0f;
  return s;
}
// fp64 values, of at least 2^-240 where they are not 0 (2^-149 over the root of
// the largest eps, times fp16's least gamma).  v_rcp_f64 and one step of Newton's
// iteration, 1 / a to 2^-48, and 127 2^-45 more (see quant8).
template <class T>
__device__ __forceinline__ RowScale<double> row_scale(double a, bool bad) {
  RowScale<double> s;
  bad = bad || !(a < INFINITY);
  s.a = a;
  const double r = __builtin_amdgcn_rcp(a);
  s.r = bad || a == 0.0 ? 0.0 : (127.0 + 127.0 * 0x1p-45) * __builtin_fma(__builtin_fma(-a, r, 1.0), r, r);
  const double unit = a * (1.0 / 127.0);
  s.unit = bad ? __builtin_nan("") : __builtin_fma(__builtin_fma(-unit, 127.0, a), 1.0 / 127.0, unit);
  return s;
}

// Eight values to eight bytes.  Adding 1.5 * 2^23 rounds to an integer (ties
// to even) and leaves it in the low byte.
constexpr float kRound = 12582912.0f;
__device__ __forceinline__ u32x2 pack8(const unsigned (&u)[8], bool none) {
  u32x2 o;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const unsigned lo = __builtin_amdgcn_perm(u[4 * j + 1], u[4 * j], 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(u[4 * j + 3], u[4 * j + 2], 0x04000c0cu);
    o[j] = none ? 0u : lo | hi;  // zeros, or a row with an infinity or NaN
  }
  return o;
}
template <class T, RowKind KIND>
__device__ __forceinline__ u32x2 quant8(const f32x8& v, const RowScale<float>& s) {
  float far = 0.0f, x[8];
  unsigned u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = sizeof(T) == 4 ? v[i] * s.m : v[i];
    const float t = __builtin_fmaf(x[i], s.r, kRound);
    u[i] = __float_as_uint(t);
    far = max_abs(far, __builtin_fmaf(x[i], s.r, -(t - kRound)));
  }
  if (far > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = __uint_as_float(u[i]) - kRound;
      const float d = __builtin_fmaf(x[i], s.r, -n);
      if (fabsf(d) > 0.5f - 0x1p-15f) {
        const float k = d > 0.0f ? n : n - 1.0f;  // between k and k + 1
        const double e = 254.0 * (double)x[i] - (double)(2.0f * k + 1.0f) * (double)s.a;
        const bool up = e > 0.0 || (e == 0.0 && ((int)k & 1));
        u[i] = __float_as_uint((up ? k + 1.0f : k) + kRound);
      }
    }
  }
  return pack8(u, s.r == 0.0f);
}
// The same from fp64 values, whose quotients come out to 2^-38 and a little large:
// adding 1.5 * 2^52 leaves the nearest integer.  What is half an integer exactly,
// 254 v = (2k + 1) a, takes k = 63 or an a that 127 divides: either v = a / 2, and
// 63.5 goes to the even 64 as a little more than it does, or a / 127 is exact, and
// the products decide (exact for the RMS norm's 35 bits).  LayerNorms, of whose
// values only beta alone is exact, ask whether a is an fp32 value, which is known
// earlier (5% at 512x16384).
constexpr double kRound64 = 6755399441055744.0;
template <class T, RowKind KIND>
__device__ __forceinline__ u32x2 quant8(const f64x8& v, const RowScale<double>& s) {
  unsigned u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = (unsigned)__double2loint(__builtin_fma(v[i], s.r, kRound64));
  const bool ties = KIND == kLayer ? (__double2loint(s.a) & 0x1fffffff) == 0 : __builtin_fma(s.unit, -127.0, s.a) == 0.0;
  if (ties) {  // uniform in a row
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double n = (double)(int)u[i], d = __builtin_fma(v[i], s.r, -n);
      if (__builtin_fabs(d) > 0.5 - 0x1p-34) {
        const double k = d > 0.0 ? n : n - 1.0;  // between k and k + 1
        const double e = 254.0 * v[i] - (2.0 * k + 1.0) * s.a;
        u[i] = (unsigned)(int)(e > 0.0 || (e == 0.0 && ((int)k & 1)) ? k + 1.0 : k);
      }
    }
  }
  return pack8(u, s.r == 0.0);
}

// Reductions over the TPR threads of a row: 8, 16 or 32 lanes of a wave, a wave,
// or the waves of a workgroup through LDS (`lds`: another part of it for each
// use).  All lanes have to take part.
template <int TPR, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, Op op, V* lds) {
  if constexpr (TPR >= 64 && sizeof(V) == 4) {
    v = wave_reduce(v, op);
  } else {
    // the same steps; of what fp64 has no DPP form, the moves need no old value
    constexpr int W = sizeof(V) / 4;
    auto dpp = [&](auto ctrl) {
      unsigned w[W];
      V o;
      __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
      for (int i = 0; i < W; ++i)
        w[i] = (unsigned)__builtin_amdgcn_mov_dpp((int)w[i], decltype(ctrl)::value, 0xF, 0xF, true);
      __builtin_memcpy(&o, w, sizeof(V));
      v = op(v, o);
    };
    auto swap = [&](auto sw) {
      unsigned w[W], x[W], y[W];
      V a, b;
      __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const auto s = sw(w[i]);
        x[i] = s[0];
        y[i] = s[1];
      }
      __builtin_memcpy(&a, x, sizeof(V));
      __builtin_memcpy(&b, y, sizeof(V));
      v = op(a, b);
    };
    dpp(std::integral_constant<int, kDppXor1>{});
    dpp(std::integral_constant<int, kDppXor2>{});
    dpp(std::integral_constant<int, kDppHalfMirror>{});
    if constexpr (TPR > 8) dpp(std::integral_constant<int, kDppMirror>{});
    if constexpr (TPR >= 32) swap([](unsigned u) { return __builtin_amdgcn_permlane16_swap(u, u, false, false); });
    if constexpr (TPR >= 64) swap([](unsigned u) { return __builtin_amdgcn_permlane32_swap(u, u, false, false); });
  }
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = op(v, lds[i]);
  }
  return v;
}
constexpr auto kSum = [](auto a, auto b) { return a + b; };
constexpr auto kMax = [](auto a, auto b) { return max_nan(a, b); };

// sum / K: the product with 1 / K and one step of Newton's division, so that the
// mean of equal values is that value.
__device__ __forceinline__ double mean_of(double sum, int K, double inv_k) {
  const double m = sum * inv_k;
  return __builtin_fma(__builtin_fma(-m, (double)K, sum), inv_k, m);
}
template <class S>
__device__ __forceinline__ S add_square(S s, S v) {
  if constexpr (sizeof(S) == 8) return __builtin_fma(v, v, s);
  return __builtin_fmaf(v, v, s);
}
// 1 / sqrt(mean of squares + eps)
__device__ __forceinline__ float root_of(float sq, const RowArgs& p) { return rsqrtf(sq * (float)p.inv_k + p.eps); }
__device__ __forceinline__ double root_of(double sq, const RowArgs& p) {
  return rsqrt(__builtin_fma(sq, p.inv_k, (double)p.eps));
}

// A row in the registers of TPR threads, VPT vectors of eight values each
// (K >= 8).  Vector j of a thread starts at 8 (thread + TPR j); the row's last
// one starts at K - 8 and repeats values of the one before, which sums leave
// out and whose results are the same bytes.  All loads are issued before any
// is used, at addresses inside the row.
template <class T, RowKind KIND, int TPR, int VPT>
__global__ void __launch_bounds__(TPR < 128 ? 256 : TPR) row_q8_kernel(RowArgs p) {
  constexpr int ROWS = TPR < 128 ? 256 / TPR : 1;  // of a workgroup
  typedef Wide<T, KIND> W;
  constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;  // of a row
  constexpr bool APART = KIND == kLayer && (TPR == 64 ? VPT > 2 : TPR == 128), HALVES = TPR == 32 && VPT > 1;
  __shared__ W red[2][WAVES * (APART ? VPT : 1)];
  __shared__ W red_top[WAVES];
  const int t = ROWS == 1 ? threadIdx.x : threadIdx.x & (TPR - 1);
  const int row_at = ROWS == 1 ? (int)blockIdx.x : (int)blockIdx.x * ROWS + (int)threadIdx.x / TPR;
  const int row = min(row_at, p.rows - 1);  // lanes past the last row repeat it, and store nothing
  const int K = p.K, S = (K + 7) >> 3;
  const bool ragged = K & 7;
  const T* x = (const T*)p.x + (size_t)row * p.ldx;
  const T* res = (const T*)p.res + (size_t)row * p.ldr;
  Vec8<T> h[VPT], r[VPT];
  f16x8 g[VPT], b[VPT];
  int at[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    at[j] = min(min(t + TPR * j, S - 1) * 8, K - 8);
    h[j] = load8(x + at[j]);
    if (KIND != kQuant && p.res) r[j] = load8(res + at[j]);
    if (KIND != kQuant) g[j] = (f16)1.0f;
    if (KIND == kLayer) b[j] = (f16)0.0f;
    if (KIND != kQuant && p.gamma) g[j] = load8(p.gamma + at[j]);
    if (KIND == kLayer && p.beta) b[j] = load8(p.beta + at[j]);
  }
  if (KIND != kQuant && p.res) {
    // in T: the sum of two fp16 values rounded once, as through fp32
#pragma unroll
    for (int j = 0; j < VPT; ++j) h[j] = h[j] + r[j];
  }
  // sum over the row's values, each once: f(sum, j, i) adds value i of vector j.
  // Threads that hold the vectors of twice to four times as many (LayerNorms of
  // many rows) add them up as those would, so that the sum does not depend on the
  // kernel: a wave as several waves, each of which adds 64 vectors in a row, half
  // a wave as the halves of a wave.
  auto row_sum = [&](auto f, W* lds) {
    W sum = 0, odd = 0, parts[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      W part = 0;
      if (ragged) {
        const int skip = (t + TPR * j) * 8 - at[j];
#pragma unroll
        for (int i = 0; i < 8; ++i) part = i >= skip ? f(part, j, i) : part;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) part = f(part, j, i);
      }
      part = t + TPR * j < S ? part : (W)0;
      if constexpr (APART) parts[j] = row_reduce<64>(part, kSum, lds);
      if (HALVES && (j & 1))
        odd = j == 1 ? part : odd + part;
      else
        sum = j == 0 ? part : sum + part;
    }
    if constexpr (APART) {
      if constexpr (TPR > 64) {
        if ((t & 63) == 0) {
#pragma unroll
          for (int j = 0; j < VPT; ++j) lds[j * WAVES + (t >> 6)] = parts[j];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VPT * WAVES; ++i) sum = i == 0 ? lds[0] : sum + lds[i];
      } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) sum = j == 0 ? parts[0] : sum + parts[j];
      }
      return sum;
    }
    if constexpr (HALVES) return row_reduce<TPR>(sum, kSum, lds) + row_reduce<TPR>(odd, kSum, lds);
    return row_reduce<TPR>(sum, kSum, lds);
  };
  typedef W W8 __attribute__((ext_vector_type(8)));
  W8 y[VPT];
  W rstd = 1;
  bool bad = false;
  if constexpr (KIND == kQuant) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) y[j] = __builtin_convertvector(h[j], f32x8);
  } else if constexpr (KIND == kRms) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] = (W)h[j][i] * (W)g[j][i];
    const W ss = row_sum([&](W s, int j, int i) { return add_square<W>(s, h[j][i]); }, red[0]);
    bad = !(ss < INFINITY);
    rstd = root_of(ss, p);
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j) y[j] = __builtin_convertvector(h[j], f64x8);
    const double mean = mean_of(row_sum([&](double s, int j, int i) { return s + y[j][i]; }, red[0]), K, p.inv_k);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] = y[j][i] - mean;
    const double sq = row_sum([&](double s, int j, int i) { return __builtin_fma(y[j][i], y[j][i], s); }, red[1]);
    bad = !(sq < INFINITY);
    const double rs = root_of(sq, p);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[j][i] = __builtin_fma(y[j][i], rs * (double)g[j][i], (double)b[j][i]);
  }
  Top<W> top;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) top.add(y[j][i]);
  const RowScale<W> s = row_scale<T>(row_reduce<TPR>(top.get(), kMax, red_top), bad);
  if (ROWS > 1 && row_at >= p.rows) return;
  int8_t* q = p.q + (size_t)row * p.ldq;
  T* ho = (T*)p.h + (size_t)row * p.ldh;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (t + TPR * j >= S) continue;
    if (KIND != kQuant && p.h) store8(ho + at[j], h[j]);
    const u32x2 o = quant8<T, KIND>(y[j], s);
    __builtin_memcpy(q + at[j], &o, 8);
  }
  if (t == 0) p.scale[row] = s.unit == 0 ? 0.0f : (float)(rstd * s.unit);
}

// Rows of more values than the registers of a workgroup hold: one workgroup a
// row, which reads it again for every statistic (from the L2).  With a
// residual the sums are read back from h where the caller takes them, from x
// and the residual otherwise.  h may be either of them, so each value is read
// and replaced by one thread: vectors of eight, and the row's last values one
// by one.
template <class T, RowKind KIND>
__global__ void __launch_bounds__(1024) row_q8_long_kernel(RowArgs p) {
  constexpr int NT = 1024;
  typedef Wide<T, KIND> W;
  typedef W W8 __attribute__((ext_vector_type(8)));
  __shared__ W red[2][NT / 64];
  __shared__ W red_top[NT / 64];
  const int row = blockIdx.x, t = threadIdx.x;
  const int K = p.K, S = K >> 3, tail = S * 8 + t;
  const T* x = (const T*)p.x + (size_t)row * p.ldx;
  const T* res = (const T*)p.res + (size_t)row * p.ldr;
  T* ho = (T*)p.h + (size_t)row * p.ldh;
  const bool add = KIND != kQuant && p.res;
  bool first = true;
  // f(values, gamma, beta, n, k) for each of the row's vectors
  auto each = [&](auto f) {
    for (int s = t; s < S; s += NT) {
      const int k = s * 8;
      const bool back = add && p.h && !first;
      Vec8<T> v = load8(back ? ho + k : x + k);
      if (add && !back) {
        v = v + load8(res + k);
        if (p.h) store8(ho + k, v);
      }
      f16x8 g = (f16)1.0f, b = (f16)0.0f;
      if (KIND != kQuant && p.gamma) g = load8(p.gamma + k);
      if (KIND == kLayer && p.beta) b = load8(p.beta + k);
      f(__builtin_convertvector(v, f32x8), __builtin_convertvector(g, f32x8), __builtin_convertvector(b, f32x8), 8, k);
    }
    if (tail < K) {
      const bool back = add && p.h && !first;
      T v = back ? ho[tail] : x[tail];
      if (add && !back) {
        v = v + res[tail];
        if (p.h) ho[tail] = v;
      }
      f32x8 v8{}, g = 1.0f, b = 0.0f;
      v8[0] = (float)v;
      if (KIND != kQuant && p.gamma) g[0] = (float)p.gamma[tail];
      if (KIND == kLayer && p.beta) b[0] = (float)p.beta[tail];
      f(v8, g, b, 1, tail);
    }
    first = false;
  };
  W rstd = 1, mean = 0, rs = 1;
  bool bad = false;
  auto value = [&](float v, float g, float b) -> W {
    if constexpr (KIND == kRms) return (W)v * (W)g;
    if constexpr (KIND == kLayer) return __builtin_fma(v - mean, rs * g, (double)b);
    return v;
  };
  Top<W> top;
  if constexpr (KIND == kLayer) {
    // Both sums in one pass, over the differences from the row's first value: its
    // own square is among those that the variance sums, so that taking
    // K (mean difference)^2 away again leaves the variance to 2 K 2^-53.
    float v0 = (float)(T)(add ? x[0] + res[0] : x[0]);
    asm volatile("" : "+v"(v0));  // here by now: behind the barrier the sum may replace it
    __syncthreads();
    const double first_value = v0;
    double sum = 0.0, sq = 0.0;
    each([&](const f32x8& v, const f32x8&, const f32x8&, int n, int) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double d = i < n ? v[i] - first_value : 0.0;
        sum += d;
        sq = __builtin_fma(d, d, sq);
      }
    });
    sum = row_reduce<NT>(sum, kSum, red[0]);
    sq = row_reduce<NT>(sq, kSum, red[1]);
    bad = !(sq < INFINITY);
    mean = sum * p.inv_k;
    rs = root_of(__builtin_fmax(__builtin_fma(-sum, mean, sq), 0.0), p);
    mean += first_value;
    each([&](const f32x8& v, const f32x8& g, const f32x8& b, int n, int) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) top.add(value(v[i], g[i], b[i]));
    });
  } else {
    W ss = 0;
    each([&](const f32x8& v, const f32x8& g, const f32x8& b, int n, int) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss = add_square<W>(ss, v[i]);
        top.add(value(v[i], g[i], b[i]));  // past n: zeros
      }
    });
    if constexpr (KIND == kRms) {
      ss = row_reduce<NT>(ss, kSum, red[0]);
      bad = !(ss < INFINITY);
      rstd = root_of(ss, p);
    }
  }
  const RowScale<W> s = row_scale<T>(row_reduce<NT>(top.get(), kMax, red_top), bad);
  int8_t* q = p.q + (size_t)row * p.ldq;
  each([&](const f32x8& v, const f32x8& g, const f32x8& b, int n, int k) {
    W8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = value(v[i], g[i], b[i]);
    const u32x2 o = quant8<T, KIND>(y, s);
    if (n == 8)
      __builtin_memcpy(q + k, &o, 8);
    else
      q[k] = (int8_t)(o[0] & 0xff);
  });
  if (t == 0) p.scale[row] = s.unit == 0 ? 0.0f : (float)(rstd * s.unit);
}

// Rows of fewer than eight values: a thread a row.
template <class T, RowKind KIND>
__global__ void __launch_bounds__(256) row_q8_short_kernel(RowArgs p) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= p.rows) return;
  const T* x = (const T*)p.x + (size_t)row * p.ldx;
  typedef Wide<T, KIND> W;
  typedef W W8 __attribute__((ext_vector_type(8)));
  W8 y{};
  W sum = 0, sq = 0, rstd = 1, mean = 0;
  Top<W> top;
#pragma unroll
  for (int k = 0; k < 7; ++k) {
    if (k >= p.K) break;
    T v = x[k];
    if (KIND != kQuant && p.res) v = v + ((const T*)p.res)[(size_t)row * p.ldr + k];
    if (KIND != kQuant && p.h) ((T*)p.h)[(size_t)row * p.ldh + k] = v;
    y[k] = (W)v;
    sum += y[k];
  }
  if constexpr (KIND == kLayer) mean = mean_of(sum, p.K, p.inv_k);
#pragma unroll
  for (int k = 0; k < 7; ++k) sq += k < p.K ? ((W)y[k] - mean) * ((W)y[k] - mean) : (W)0;
  const bool bad = KIND != kQuant && !(sq < INFINITY);
  const W rs = root_of(sq, p);
  if (KIND == kRms) rstd = rs;
#pragma unroll
  for (int k = 0; k < 7; ++k) {
    if (k >= p.K) break;
    const float g = KIND != kQuant && p.gamma ? (float)p.gamma[k] : 1.0f;
    if constexpr (KIND == kRms) y[k] = y[k] * g;
    if constexpr (KIND == kLayer) y[k] = __builtin_fma(y[k] - mean, rs * g, p.beta ? (double)p.beta[k] : 0.0);
    top.add(y[k]);
  }
  const RowScale<W> s = row_scale<T>(top.get(), bad);
  const u32x2 o = quant8<T, KIND>(y, s);
  int8_t* q = p.q + (size_t)row * p.ldq;
#pragma unroll
  for (int k = 0; k < 7; ++k)
    if (k < p.K) q[k] = (int8_t)(o[k >> 2] >> (8 * (k & 3)));
  p.scale[row] = s.unit == 0 ? 0.0f : (float)(rstd * s.unit);
}

// y = q * scale, sixteen values a thread (K >= 16: the last vector of a row
// ends with it and repeats values of the one before), single values below.
template <class T, int V>
__global__ void __launch_bounds__(256)
dequant_kernel(const int8_t* __restrict__ q, long long ldq, const float* __restrict__ scale, T* __restrict__ y,
               long long ldy, int rows, int K) {
  const int S = (K + V - 1) / V;
  const long long n = (long long)rows * S;
  GRID_STRIDE(i, n) {
    // a 64-bit division takes as long as everything else here
    const int row = n >> 32 ? (int)((unsigned long long)i / (unsigned)S) : (int)((unsigned)i / (unsigned)S);
    const int at = min((int)(i - (long long)row * S) * V, K - V);
    int8_t b[V];
    __builtin_memcpy(b, q + (size_t)row * ldq + at, V);
    const float s = scale[row];
    T o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v = (float)b[e] * s;
      asm("" : "+v"(v));  // rounded to fp32 before T, not merged into one instruction
      o[e] = (T)v;
    }
    __builtin_memcpy(y + (size_t)row * ldy + at, o, sizeof(o));
  }
}

template <class T, RowKind KIND, int TPR, int VPT>
void launch_rows(const RowArgs& a, hipStream_t s) {
  static const std::string name = std::string("row_q8_kernel<") + (sizeof(T) == 2 ? "_Float16" : "float") + ", " +
                                  std::to_string((int)KIND) + ", " + std::to_string(TPR) + ", " +
                                  std::to_string(VPT) + ">";
  constexpr int ROWS = TPR < 128 ? 256 / TPR : 1;
  DLM_LAUNCH(name.c_str(), (row_q8_kernel<T, KIND, TPR, VPT>), dim3((a.rows + ROWS - 1) / ROWS),
             dim3(TPR < 128 ? 256 : TPR), 0, s, a);
}

// Rows of 1025-16384 values that are fp64 on their way.  Their instructions are the
// longest part, or nearly, so they take as many threads as leave few of them idle:
// 192 or 384 with one vector each, 256 or 512 with three (LayerNorm 975x1283 5.1 ->
// 4.8 us against 256, 2048x5120 16.9 -> 12.6 and 1024x12000 20.3 -> 13.6 against 512
// with two and four; RMS norm 8192x1280 13.3 -> 11.7, with residual 26.9 -> 27.2, and
// 1024x12000 18.0 -> 13.1).  LayerNorms of many rows share what a row has to do once
// among fewer threads: a wave with three vectors (fp16 3000x1280 7.4 -> 6.6 us, 1536
// rows the same, fp32 rows 7.6 -> 7.8) or four (16384x2048 36 -> 31; below 4096 rows
// nothing), two waves with three (2048x2560 10.0 -> 8.5; 512 rows 4.4 -> 5.0).  RMS
// norms do not take 256 with three: 2048x5120 12.7 -> 12.1, but 28.2 -> 29.7 with a
// residual.
template <class T, RowKind KIND>
void wide_rows(const RowArgs& a, hipStream_t s) {
  constexpr bool LAYER = KIND == kLayer;
  const int S = (a.K + 7) / 8;  // vectors a row
  if constexpr (LAYER && sizeof(T) == 2) {
    if (a.rows >= 2048 && S <= 192) return launch_rows<T, KIND, 64, 3>(a, s);
    if (a.rows >= 4096 && S <= 256) return launch_rows<T, KIND, 64, 4>(a, s);
  }
  if (S <= 192) return launch_rows<T, KIND, 192, 1>(a, s);
  if (S <= 256) return launch_rows<T, KIND, 256, 1>(a, s);
  if constexpr (LAYER) {
    if (a.rows >= 1024 && S <= 384) return launch_rows<T, KIND, 128, 3>(a, s);
  }
  if (S <= 384) return launch_rows<T, KIND, 384, 1>(a, s);
  if (S <= 512) return launch_rows<T, KIND, 256, 2>(a, s);
  if constexpr (LAYER) {
    if (S <= 768) return launch_rows<T, KIND, 256, 3>(a, s);
  }
  if (S <= 1024) return launch_rows<T, KIND, 512, 2>(a, s);
  return S <= 1536 ? launch_rows<T, KIND, 512, 3>(a, s) : launch_rows<T, KIND, 512, 4>(a, s);
}

// Threads a row by its length: each holds one to four vectors.  Rows of 1025-2048
// values take a workgroup (8192x1280 quantise 8.2 us, RMS norm 13.5; with a wave
// each 8.4 and 13.9, and 2.8 against 3.8 us for 256 rows).  Many fp16 LayerNorms of
// 513-768 values take half a wave each (8192x640 9.2 -> 7.7 us; the other kinds lose
// 2-6%).
template <class T, RowKind KIND>
void row_q8(const RowArgs& a, hipStream_t s) {
  const int K = a.K;
  if (K < 8)
    DLM_LAUNCH("row_q8_short_kernel", (row_q8_short_kernel<T, KIND>), dim3((a.rows + 255) / 256), dim3(256), 0, s, a);
  else if (K <= 64)
    launch_rows<T, KIND, 8, 1>(a, s);
  else if (K <= 128)
    launch_rows<T, KIND, 16, 1>(a, s);
  else if (K <= 256)
    launch_rows<T, KIND, 32, 1>(a, s);
  else if (K <= 512)
    launch_rows<T, KIND, 64, 1>(a, s);
  else if (K <= 1024) {
    if constexpr (KIND == kLayer && sizeof(T) == 2) {
      if (a.rows >= 4096 && K <= 768) return launch_rows<T, KIND, 32, 3>(a, s);
    }
    launch_rows<T, KIND, 64, 2>(a, s);
  } else if (K > 16384)
    DLM_LAUNCH("row_q8_long_kernel", (row_q8_long_kernel<T, KIND>), dim3(a.rows), dim3(1024), 0, s, a);
  else if constexpr (sizeof(Wide<T, KIND>) == 8)
    wide_rows<T, KIND>(a, s);
  else if (K <= 2048)
    launch_rows<T, KIND, 256, 1>(a, s);
  else if (K <= 4096)
    launch_rows<T, KIND, 256, 2>(a, s);
  else if (K <= 8192)
    launch_rows<T, KIND, 512, 2>(a, s);
  else
    launch_rows<T, KIND, 512, 4>(a, s);
}

// A launch counts its threads in 32 bits: more rows than 2^21 go in parts.
template <class T>
int row_parts(RowKind kind, RowArgs a, hipStream_t s) {
  constexpr int kPart = 1 << 21;
  for (int left = a.rows; left > 0; left -= kPart) {
    a.rows = std::min(left, kPart);
    switch (kind) {
      case kQuant: row_q8<T, kQuant>(a, s); break;
      case kRms: row_q8<T, kRms>(a, s); break;
      case kLayer: row_q8<T, kLayer>(a, s); break;
    }
    DLM_LAUNCH_CHECK();
    a.x = (const T*)a.x + kPart * a.ldx;
    if (a.res) a.res = (const T*)a.res + kPart * a.ldr;
    if (a.h) a.h = (T*)a.h + kPart * a.ldh;
    a.q += kPart * a.ldq;
    a.scale += kPart;
  }
  return DLM_OK;
}

// ---------------------------------------------------------------------------
// Argument checks shared by the entry points.
// ---------------------------------------------------------------------------
// The sum may be x or the residual where it is the same tensor (same address and
// row stride); otherwise an output overlaps neither inputs nor other outputs.
template <class T>
int row_entry(RowKind kind, const char* fn, const RowArgs& a, hipStream_t s) {
  auto bad = [&](const std::string& m) { return fail(DLM_ERR_INVALID_ARG, std::string(fn) + ": " + m); };
  if (!a.x || !a.q || !a.scale) return bad("NULL pointer");
  if (a.ldx < a.K || a.ldq < a.K || (a.res && a.ldr < a.K) || (a.h && a.ldh < a.K)) return bad("row stride below K");
  if (a.h && !a.res) return bad("a sum is written only with a residual");
  if ((uintptr_t)a.x % sizeof(T) || (uintptr_t)a.res % sizeof(T) || (uintptr_t)a.h % sizeof(T) ||
      (uintptr_t)a.gamma % 2 || (uintptr_t)a.beta % 2 || (uintptr_t)a.scale % 4)
    return bad("pointer not aligned to its element");
  if (!(a.eps >= 0.0f)) return bad("eps is negative or NaN");
  const int e = (int)sizeof(T);
  const Span in[] = {{"x", a.x, a.ldx, a.rows, a.K, e},
                     {"residual", a.res, a.ldr, a.rows, a.K, e},
                     {"gamma", a.gamma, a.K, 1, a.K, 2},
                     {"beta", a.beta, a.K, 1, a.K, 2}};
  const Span out[] = {{"q", a.q, a.ldq, a.rows, a.K, 1},
                      {"scale", a.scale, 1, a.rows, 1, 4},
                      {"sum", a.h, a.ldh, a.rows, a.K, e}};
  for (int o = 0; o < 3; ++o) {
    for (int i = 0; i < 4; ++i) {
      const bool in_place = o == 2 && i < 2 && in[i].p == a.h && in[i].ld == a.ldh;
      if (!in_place && overlap(out[o], in[i])) return bad(std::string(out[o].name) + " overlaps " + in[i].name);
    }
    for (int u = 0; u < o; ++u)
      if (overlap(out[o], out[u])) return bad(std::string(out[o].name) + " overlaps " + out[u].name);
  }
  return row_parts<T>(kind, a, s);
}

template <class T>
int dequant(const char* fn, const void* q, int ldq, const float* scale, void* y, int ldy, int rows, int K,
            hipStream_t s) {
  auto bad = [&](const std::string& m) { return fail(DLM_ERR_INVALID_ARG, std::string(fn) + ": " + m); };
  if (!q || !scale || !y) return bad("NULL pointer");
  if (ldq < K || ldy < K) return bad("row stride below K");
  if ((uintptr_t)y % sizeof(T) || (uintptr_t)scale % 4) return bad("pointer not aligned to its element");
  const Span out{"y", y, ldy, rows, K, (int)sizeof(T)};
  for (const Span& i : {Span{"q", q, ldq, rows, K, 1}, Span{"scale", scale, 1, rows, 1, 4}})
    if (overlap(out, i)) return bad(std::string("y overlaps ") + i.name);
  if (K >= 16)
    DLM_LAUNCH("dequant_kernel<16>", (dequant_kernel<T, 16>), dim3(grid_for((long long)rows * ((K + 15) / 16))),
               dim3(256), 0, s, (const int8_t*)q, (long long)ldq, scale, (T*)y, (long long)ldy, rows, K);
  else
    DLM_LAUNCH("dequant_kernel<1>", (dequant_kernel<T, 1>), dim3(grid_for((long long)rows * K)), dim3(256), 0, s,
               (const int8_t*)q, (long long)ldq, scale, (T*)y, (long long)ldy, rows, K);
  DLM_LAUNCH_CHECK();
  return DLM_OK;
}

}  // namespace
}  // namespace dlm

using namespace dlm;

extern "C" {

int dlm_quantize_rows_fp16(const void* x, int ldx, void* q, int ldq, float* scale, int rows, int K, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<f16>(kQuant, __func__,
                        RowArgs{x, nullptr, nullptr, nullptr, nullptr, (int8_t*)q, scale, ldx, 0, 0, ldq, rows, K, 0.0f, 0.0},
                        (hipStream_t)stream);
}

int dlm_quantize_rows_f32(const float* x, int ldx, void* q, int ldq, float* scale, int rows, int K, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<float>(
      kQuant, __func__,
      RowArgs{x, nullptr, nullptr, nullptr, nullptr, (int8_t*)q, scale, ldx, 0, 0, ldq, rows, K, 0.0f, 0.0},
      (hipStream_t)stream);
}

int dlm_rms_norm_q8_fp16(const void* x, int ldx, const void* R, int ldr, void* H, int ldh, const void* gamma, void* q,
                         int ldq, float* scale, int rows, int K, float eps, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<f16>(
      kRms, __func__,
      RowArgs{x, R, H, (const f16*)gamma, nullptr, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps, 1.0 / K},
      (hipStream_t)stream);
}

int dlm_rms_norm_q8_f32(const float* x, int ldx, const float* R, int ldr, float* H, int ldh, const void* gamma,
                        void* q, int ldq, float* scale, int rows, int K, float eps, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<float>(
      kRms, __func__,
      RowArgs{x, R, H, (const f16*)gamma, nullptr, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps, 1.0 / K},
      (hipStream_t)stream);
}

int dlm_layer_norm_q8_fp16(const void* x, int ldx, const void* R, int ldr, void* H, int ldh, const void* gamma,
                           const void* beta, void* q, int ldq, float* scale, int rows, int K, float eps,
                           void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<f16>(
      kLayer, __func__,
      RowArgs{x, R, H, (const f16*)gamma, (const f16*)beta, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps, 1.0 / K},
      (hipStream_t)stream);
}

int dlm_layer_norm_q8_f32(const float* x, int ldx, const float* R, int ldr, float* H, int ldh, const void* gamma,
                          const void* beta, void* q, int ldq, float* scale, int rows, int K, float eps,
                          void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<float>(
      kLayer, __func__,
      RowArgs{x, R, H, (const f16*)gamma, (const f16*)beta, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps, 1.0 / K},
      (hipStream_t)stream);
}

int dlm_dequantize_rows_fp16(const void* q, int ldq, const float* scale, void* y, int ldy, int rows, int K,
                             void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return dequant<f16>(__func__, q, ldq, scale, y, ldy, rows, K, (hipStream_t)stream);
}

int dlm_dequantize_rows_f32(const void* q, int ldq, const float* scale, float* y, int ldy, int rows, int K,
                            void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return dequant<float>(__func__, q, ldq, scale, y, ldy, rows, K, (hipStream_t)stream);
}

}  // extern "C"
