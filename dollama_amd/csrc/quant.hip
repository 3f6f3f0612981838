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
//   LayerNorm   v = (h - mean) / sqrt(var + eps) gamma + beta
//
// Rounding.  127 v / a is formed as v * (127 / a) in fp32, which may fall on
// the wrong side of a half by 2^-17 at most (2^-24 relative error of 127 / a
// on values up to 127).  Quotients within 2^-16 of a half (one in 30,000) are
// decided again by comparing 254 v with (2k + 1) a in fp64, where both
// products are exact.  So q is the quotient's nearest integer whatever the
// launch looks like; for fp16 rows (and fp16 gamma) of the first two kinds,
// where v is exact in fp32, that is the mathematically exact result.
//
// What bounds them: memory, one pass.  A row stays in registers between its
// statistics and its output (up to 64 values a thread); rows of up to 1536
// values take one wave, so a workgroup needs no barrier.
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
};

template <class T>
struct Vec8;  // eight elements as loaded
template <>
struct Vec8<f16> {
  typedef f16x8 type;
};
template <>
struct Vec8<float> {
  typedef float type __attribute__((ext_vector_type(8)));
};
typedef float f32x8 __attribute__((ext_vector_type(8)));

// Eight elements at any element-aligned address: one 16-byte access (two for
// fp32), which the hardware takes at any alignment.
template <class T>
__device__ __forceinline__ f32x8 load8(const T* p) {
  typename Vec8<T>::type v;
  __builtin_memcpy(&v, p, sizeof(v));
  f32x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (float)v[i];
  return r;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const f32x8& x) {
  typename Vec8<T>::type v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
  __builtin_memcpy(p, &v, sizeof(v));
}

// What a row's values are multiplied by on their way to q.
struct RowScale {
  float r;     // 127 / (a m), 0 for rows without a finite positive maximum
  float a;     // a m
  float m;     // fp32 rows: 2^100 where a is so small that 127 / a would overflow; else 1
  float unit;  // a / 127, NaN for a row that holds an infinity or NaN
};
// top: bits of max |v| (of the largest NaN, if there is one).  Values of fp16
// rows are no smaller than 2^-48 where they are not 0 (LayerNorm's 2^-112).
template <class T>
__device__ __forceinline__ RowScale row_scale(unsigned top, bool bad) {
  RowScale s;
  const float a = __uint_as_float(top);
  bad = bad || top >= 0x7f800000u;
  s.m = sizeof(T) == 4 && a < 0x1p-100f ? 0x1p100f : 1.0f;
  s.a = a * s.m;
  s.r = bad || top == 0 ? 0.0f : 127.0f / s.a;
  s.unit = bad ? __uint_as_float(0x7fc00000u) : a / 127.0f;
  return s;
}

// Eight values to eight bytes.  Adding 1.5 * 2^23 rounds to an integer (ties
// to even) and leaves it in the low byte.  A row with an infinity or NaN
// (r = 0) becomes zeros: its values go through a select, as 0 * inf is NaN.
constexpr float kRound = 12582912.0f;
template <class T>
__device__ __forceinline__ u32x2 quant8(const f32x8& v, const RowScale& s) {
  float far = 0.0f;
  unsigned u[8];
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = s.r == 0.0f ? 0.0f : sizeof(T) == 4 ? v[i] * s.m : v[i];
    const float t = __builtin_fmaf(x[i], s.r, kRound);
    u[i] = __float_as_uint(t);
    far = fmaxf(far, fabsf(__builtin_fmaf(x[i], s.r, -(t - kRound))));
  }
  if (far > 0.5f - 0x1p-16f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = __uint_as_float(u[i]) - kRound;
      const float d = __builtin_fmaf(x[i], s.r, -n);
      if (fabsf(d) > 0.5f - 0x1p-16f) {
        const float k = d > 0.0f ? n : n - 1.0f;  // between k and k + 1
        const double e = 254.0 * (double)x[i] - (double)(2.0f * k + 1.0f) * (double)s.a;
        const bool up = e > 0.0 || (e == 0.0 && ((int)k & 1));
        u[i] = __float_as_uint((up ? k + 1.0f : k) + kRound);
      }
    }
  }
  u32x2 o;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const unsigned lo = __builtin_amdgcn_perm(u[4 * j + 1], u[4 * j], 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(u[4 * j + 3], u[4 * j + 2], 0x04000c0cu);
    o[j] = lo | hi;
  }
  return o;
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
  return wave_reduce(v, [](unsigned a, unsigned b) { return a > b ? a : b; });
}

// Reductions over the threads of a row: a wave, or the waves of a workgroup
// through LDS (`slot`: another part of it for each use).
template <int WAVES, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, Op op, V* lds) {
  v = wave_reduce(v, op);
  if constexpr (WAVES > 1) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[w] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v = op(v, lds[i]);
  }
  return v;
}

// A row in the registers of WAVES waves, VPT vectors of eight values a
// thread (K >= 8).  Vector j of a thread starts at 8 (thread + threads j); the
// row's last one starts at K - 8 and repeats values of the one before, which
// sums leave out and whose results are the same bytes.  All loads are issued
// before any is used, at addresses inside the row.
template <class T, RowKind KIND, int WAVES, int VPT>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) row_q8_kernel(RowArgs p) {
  constexpr int TPR = WAVES * 64;
  __shared__ float red[3][WAVES];
  const int t = threadIdx.x & (TPR - 1);
  const int row = WAVES == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (WAVES == 1 && row >= p.rows) return;
  const int K = p.K, S = (K + 7) >> 3;
  const T* x = (const T*)p.x + (size_t)row * p.ldx;
  const T* res = (const T*)p.res + (size_t)row * p.ldr;
  f32x8 v[VPT], g[VPT], b[VPT], r[VPT];
  int at[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    at[j] = min(min(t + TPR * j, S - 1) * 8, K - 8);
    v[j] = load8(x + at[j]);
    if (KIND != kQuant && p.res) r[j] = load8(res + at[j]);
    if (KIND != kQuant && p.gamma) g[j] = load8(p.gamma + at[j]);
    if (KIND == kLayer && p.beta) b[j] = load8(p.beta + at[j]);
  }
  // first new value of vector j (8: the thread has none)
  auto skip = [&](int j) { return t + TPR * j < S ? (t + TPR * j) * 8 - at[j] : 8; };
  if (KIND != kQuant && p.res) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = (float)(T)(v[j][i] + r[j][i]);
  }
  const f32x8* h = v;  // the stream as it is stored
  f32x8 y[KIND == kQuant ? 1 : VPT];
  float rstd = 1.0f;
  bool bad = false;
  if constexpr (KIND == kRms) {
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int s0 = skip(j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss += i >= s0 ? v[j][i] * v[j][i] : 0.0f;
        y[j][i] = p.gamma ? v[j][i] * g[j][i] : v[j][i];
      }
    }
    ss = row_reduce<WAVES>(ss, [](float a, float c) { return a + c; }, red[0]);
    bad = !(ss < INFINITY);
    rstd = 1.0f / sqrtf(ss / (float)K + p.eps);
  } else if constexpr (KIND == kLayer) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int s0 = skip(j);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += i >= s0 ? v[j][i] : 0.0f;
    }
    const float mean = row_reduce<WAVES>(sum, [](float a, float c) { return a + c; }, red[0]) / (float)K;
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int s0 = skip(j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[j][i] - mean;
        sq += i >= s0 ? d * d : 0.0f;
      }
    }
    sq = row_reduce<WAVES>(sq, [](float a, float c) { return a + c; }, red[1]);
    bad = !(sq < INFINITY);
    const float rs = 1.0f / sqrtf(sq / (float)K + p.eps);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = (v[j][i] - mean) * rs;
        y[j][i] = __builtin_fmaf(n, p.gamma ? g[j][i] : 1.0f, p.beta ? b[j][i] : 0.0f);
      }
  }
  const f32x8* out = KIND == kQuant ? v : y;
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(out[j][i]));
  top = row_reduce<WAVES>(top, [](unsigned a, unsigned c) { return a > c ? a : c; }, (unsigned*)red[2]);
  const RowScale s = row_scale<T>(top, bad);
  int8_t* q = p.q + (size_t)row * p.ldq;
  T* ho = (T*)p.h + (size_t)row * p.ldh;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (t + TPR * j >= S) continue;
    if (KIND != kQuant && p.h) store8(ho + at[j], h[j]);
    const u32x2 o = quant8<T>(out[j], s);
    __builtin_memcpy(q + at[j], &o, 8);
  }
  if (t == 0) p.scale[row] = KIND == kRms ? rstd * s.unit : s.unit;
}

// Rows of fewer than 8 values, or of more than the registers of a workgroup
// hold: one workgroup a row, which reads it again for every statistic (from
// the L2).  With a residual the sums are read back from h where the caller
// takes them, from x and the residual otherwise (h may be either of them:
// then h holds what the sum was).
template <class T, RowKind KIND, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) row_q8_long_kernel(RowArgs p) {
  constexpr int NT = WAVES * 64;
  __shared__ float red[3][WAVES];
  const int row = blockIdx.x;
  const int K = p.K;
  const T* x = (const T*)p.x + (size_t)row * p.ldx;
  const T* res = (const T*)p.res + (size_t)row * p.ldr;
  T* ho = (T*)p.h + (size_t)row * p.ldh;
  const bool sum_first = KIND != kQuant && p.res;
  auto first = [&](int k) {
    float v = (float)x[k];
    if (sum_first) {
      v = (float)(T)(v + (float)res[k]);
      if (p.h) ho[k] = (T)v;
    }
    return v;
  };
  auto again = [&](int k) -> float {
    if (sum_first && p.h) return (float)ho[k];
    return sum_first ? (float)(T)((float)x[k] + (float)res[k]) : (float)x[k];
  };
  float rstd = 1.0f, mean = 0.0f, rs = 1.0f;
  bool bad = false;
  auto value = [&](int k, float v) {
    if constexpr (KIND == kRms) return p.gamma ? v * (float)p.gamma[k] : v;
    if constexpr (KIND == kLayer)
      return __builtin_fmaf((v - mean) * rs, p.gamma ? (float)p.gamma[k] : 1.0f, p.beta ? (float)p.beta[k] : 0.0f);
    return v;
  };
  auto add = [](float a, float c) { return a + c; };
  unsigned top = 0;
  if constexpr (KIND == kLayer) {
    float sum = 0.0f;
    for (int k = threadIdx.x; k < K; k += NT) sum += first(k);
    mean = row_reduce<WAVES>(sum, add, red[0]) / (float)K;
    float sq = 0.0f;
    for (int k = threadIdx.x; k < K; k += NT) {
      const float d = again(k) - mean;
      sq += d * d;
    }
    sq = row_reduce<WAVES>(sq, add, red[1]);
    bad = !(sq < INFINITY);
    rs = 1.0f / sqrtf(sq / (float)K + p.eps);
    for (int k = threadIdx.x; k < K; k += NT) top = max(top, abs_bits(value(k, again(k))));
  } else {
    float ss = 0.0f;
    for (int k = threadIdx.x; k < K; k += NT) {
      const float v = first(k);
      ss += v * v;
      top = max(top, abs_bits(value(k, v)));
    }
    if constexpr (KIND == kRms) {
      ss = row_reduce<WAVES>(ss, add, red[0]);
      bad = !(ss < INFINITY);
      rstd = 1.0f / sqrtf(ss / (float)K + p.eps);
    }
  }
  top = row_reduce<WAVES>(top, [](unsigned a, unsigned c) { return a > c ? a : c; }, (unsigned*)red[2]);
  const RowScale s = row_scale<T>(top, bad);
  int8_t* q = p.q + (size_t)row * p.ldq;
  for (int k = threadIdx.x; k < K; k += NT) {
    const float v = value(k, again(k));
    const u32x2 o = quant8<T>(f32x8{v, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, s);
    q[k] = (int8_t)(o[0] & 0xff);
  }
  if (threadIdx.x == 0) p.scale[row] = KIND == kRms ? rstd * s.unit : s.unit;
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
    for (int e = 0; e < V; ++e) o[e] = (T)((float)b[e] * s);
    __builtin_memcpy(y + (size_t)row * ldy + at, o, sizeof(o));
  }
}

template <class T, RowKind KIND, int WAVES, int VPT>
void launch_rows(const RowArgs& a, hipStream_t s) {
  static const std::string name = std::string("row_q8_kernel<") + (sizeof(T) == 2 ? "_Float16" : "float") + ", " +
                                  std::to_string((int)KIND) + ", " + std::to_string(WAVES) + ", " +
                                  std::to_string(VPT) + ">";
  DLM_LAUNCH(name.c_str(), (row_q8_kernel<T, KIND, WAVES, VPT>), dim3(WAVES == 1 ? (a.rows + 3) / 4 : a.rows),
             dim3(WAVES == 1 ? 256 : WAVES * 64), 0, s, a);
}

// A wave holds rows of up to 1536 values (three vectors a lane), a workgroup
// of four or eight waves up to 16384.
template <class T, RowKind KIND>
void row_q8(const RowArgs& a, hipStream_t s) {
  if (a.K < 8)
    DLM_LAUNCH("row_q8_long_kernel<1>", (row_q8_long_kernel<T, KIND, 1>), dim3(a.rows), dim3(64), 0, s, a);
  else if (a.K <= 512)
    launch_rows<T, KIND, 1, 1>(a, s);
  else if (a.K <= 1024)
    launch_rows<T, KIND, 1, 2>(a, s);
  else if (a.K <= 1536)
    launch_rows<T, KIND, 1, 3>(a, s);
  else if (a.K <= 2048)
    launch_rows<T, KIND, 4, 1>(a, s);
  else if (a.K <= 4096)
    launch_rows<T, KIND, 4, 2>(a, s);
  else if (a.K <= 8192)
    launch_rows<T, KIND, 4, 4>(a, s);
  else if (a.K <= 16384)
    launch_rows<T, KIND, 8, 4>(a, s);
  else
    DLM_LAUNCH("row_q8_long_kernel<16>", (row_q8_long_kernel<T, KIND, 16>), dim3(a.rows), dim3(1024), 0, s, a);
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
// Bytes [p, p + n) of two operands: an output may be an input where it is the
// same tensor (same address and row stride, elements of one size), and not
// overlap it otherwise.
struct Span {
  const char* name;
  const void* p;
  long long ld;
  int rows, cols, elem;
  uintptr_t lo() const { return (uintptr_t)p; }
  uintptr_t hi() const { return (uintptr_t)p + ((uintptr_t)(rows - 1) * ld + cols) * elem; }
};
bool overlap(const Span& a, const Span& b) { return a.p && b.p && a.lo() < b.hi() && b.lo() < a.hi(); }
bool same(const Span& a, const Span& b) { return a.p == b.p && a.ld == b.ld && a.elem == b.elem && a.cols == b.cols; }

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
    for (const Span& i : in)
      if (overlap(out[o], i) && !(o == 2 && same(out[o], i)))
        return bad(std::string(out[o].name) + " overlaps " + i.name);
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
                        RowArgs{x, nullptr, nullptr, nullptr, nullptr, (int8_t*)q, scale, ldx, 0, 0, ldq, rows, K, 0.0f},
                        (hipStream_t)stream);
}

int dlm_quantize_rows_f32(const float* x, int ldx, void* q, int ldq, float* scale, int rows, int K, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<float>(
      kQuant, __func__,
      RowArgs{x, nullptr, nullptr, nullptr, nullptr, (int8_t*)q, scale, ldx, 0, 0, ldq, rows, K, 0.0f},
      (hipStream_t)stream);
}

int dlm_rms_norm_q8_fp16(const void* x, int ldx, const void* R, int ldr, void* H, int ldh, const void* gamma, void* q,
                         int ldq, float* scale, int rows, int K, float eps, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<f16>(
      kRms, __func__,
      RowArgs{x, R, H, (const f16*)gamma, nullptr, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps},
      (hipStream_t)stream);
}

int dlm_rms_norm_q8_f32(const float* x, int ldx, const float* R, int ldr, float* H, int ldh, const void* gamma,
                        void* q, int ldq, float* scale, int rows, int K, float eps, void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<float>(
      kRms, __func__,
      RowArgs{x, R, H, (const f16*)gamma, nullptr, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps},
      (hipStream_t)stream);
}

int dlm_layer_norm_q8_fp16(const void* x, int ldx, const void* R, int ldr, void* H, int ldh, const void* gamma,
                           const void* beta, void* q, int ldq, float* scale, int rows, int K, float eps,
                           void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<f16>(
      kLayer, __func__,
      RowArgs{x, R, H, (const f16*)gamma, (const f16*)beta, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps},
      (hipStream_t)stream);
}

int dlm_layer_norm_q8_f32(const float* x, int ldx, const float* R, int ldr, float* H, int ldh, const void* gamma,
                          const void* beta, void* q, int ldq, float* scale, int rows, int K, float eps,
                          void* stream) {
  if (rows <= 0 || K <= 0) return DLM_OK;
  return row_entry<float>(
      kLayer, __func__,
      RowArgs{x, R, H, (const f16*)gamma, (const f16*)beta, (int8_t*)q, scale, ldx, ldr, ldh, ldq, rows, K, eps},
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
