// Linears in 8-bit integers for gfx950:
//   Y[m, n] = act(sx[m] sw[n] sum_k X[m, k] W[n, k] + bias[n]) + beta R[m, n]
// with int8 X (one scale a row: a token) and W (one scale a row: an output
// channel), sums in int32 and the rest in fp32.  No counterpart in the
// reference, whose linears are fp16 (src/infer/unet.cu:517-525).
//
// MFMA: v_mfma_i32_16x16x64_i8 in transposed form (W fragment x X fragment),
// so a lane holds one output row and four consecutive columns.  Products of
// 8-bit values add up exactly, so the order of the sums, and with it the
// split of K, does not show in the result.
#include <algorithm>

#include "common.hpp"

namespace dlm {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// MFMA 16x16x64 i8 -> i32 (gfx950):
//   A (16 rows x 64 k): lane l holds row (l & 15), k = 16*(l >> 4) + [0..15]
//   B (64 k x 16 cols): lane l holds col (l & 15), k = 16*(l >> 4) + [0..15]
//   C/D (16 x 16):      lane l holds col (l & 15), rows 4*(l >> 4) + [0..3]
__device__ __forceinline__ i32x4 mfma16x16x64(i32x4 a, i32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

struct Q8Gemm {
  const int8_t* x;
  const int8_t* w;
  const float* sx;
  const float* sw;
  const f16* bias;  // may be NULL
  const void* res;  // may be NULL
  void* y;
  long long ldx, ldw, ldr, ldy;
  int M, N, K;
  float beta;
  int act;
};

// Keeps the first n bytes of 16 (n <= 0: none, n >= 16: all).
__device__ __forceinline__ i32x4 keep_bytes(i32x4 v, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int b = n - 4 * d;
    v[d] = b >= 4 ? v[d] : b <= 0 ? 0 : v[d] & ((1 << (8 * b)) - 1);
  }
  return v;
}

__device__ __forceinline__ float act_f(float v, int act) {
  if (act == DLM_ACT_SILU) return silu_f(v);
  if (act == DLM_ACT_GELU) return gelu_erf_fast(v);
  return v;
}

// Output row `row`, columns col .. col + 3 of the sums in a.
template <class T>
__device__ __forceinline__ void epi4(const i32x4& a, int row, int col, const Q8Gemm& p) {
  if (row >= p.M) return;
  const float sx = p.sx[row];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int c = col + t;
    if (c >= p.N) continue;
    float v = (float)a[t] * p.sw[c] * sx;
    if (p.bias) v += (float)p.bias[c];
    v = act_f(v, p.act);
    if (p.res) v = __builtin_fmaf(p.beta, (float)((const T*)p.res)[(size_t)row * p.ldr + c], v);
    ((T*)p.y)[(size_t)row * p.ldy + c] = (T)v;
  }
}

// GEGLU: packed columns 8q + [0, 4) are values, 8q + 4 + [0, 4) their gates,
// so values and gates lie in lanes 16 apart; each of the two finishes two
// outputs.  N is a multiple of 16.
template <class T>
__device__ __forceinline__ void epi4_geglu(const i32x4& a, int row, int col, const Q8Gemm& p) {
  const auto s02 = __builtin_amdgcn_permlane16_swap((unsigned)a[0], (unsigned)a[2], false, false);
  const auto s13 = __builtin_amdgcn_permlane16_swap((unsigned)a[1], (unsigned)a[3], false, false);
  if (row >= p.M || col >= p.N) return;
  const float sx = p.sx[row];
  const int vc = col & ~4, t0 = (col & 4) ? 2 : 0;
  const int sv[2] = {(int)s02[0], (int)s13[0]}, sg[2] = {(int)s02[1], (int)s13[1]};
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float v = (float)sv[t] * p.sw[vc + t0 + t] * sx, g = (float)sg[t] * p.sw[vc + 4 + t0 + t] * sx;
    if (p.bias) {
      v += (float)p.bias[vc + t0 + t];
      g += (float)p.bias[vc + 4 + t0 + t];
    }
    v *= gelu_erf_fast(g);
    const size_t o = (vc >> 1) + t0 + t;
    if (p.res) v = __builtin_fmaf(p.beta, (float)((const T*)p.res)[(size_t)row * p.ldr + o], v);
    ((T*)p.y)[(size_t)row * p.ldy + o] = (T)v;
  }
}

// 16 columns and 16 TM rows a workgroup, K dealt to its eight waves in groups
// of 128 bytes; operands go from memory to the MFMA's registers, and the
// waves' sums meet in LDS.
template <class T, int TM>
__global__ void __launch_bounds__(512) q8_rows_kernel(Q8Gemm p) {
  constexpr int NW = 8;
  __shared__ i32x4 red[NW][TM][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * TM;
  const int l15 = lane & 15, kl = 16 * (lane >> 4);
  const int klast = (p.K - 1) & ~15;
  const int8_t* wp = p.w + (size_t)min(n0 + l15, p.N - 1) * p.ldw;
  const int8_t* xp[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) xp[i] = p.x + (size_t)min(m0 + 16 * i + l15, p.M - 1) * p.ldx;
  i32x4 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) acc[i] = i32x4{0, 0, 0, 0};
  const int steps = (p.K + 63) >> 6;
  for (int s0 = 2 * wave; s0 < steps; s0 += 4 * NW) {
    i32x4 fw[4], fx[4][TM];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = min(64 * (s0 + (u >> 1) * 2 * NW + (u & 1)) + kl, klast);
      fw[u] = *reinterpret_cast<const i32x4*>(wp + k);
#pragma unroll
      for (int i = 0; i < TM; ++i) fx[u][i] = *reinterpret_cast<const i32x4*>(xp[i] + k);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + (u >> 1) * 2 * NW + (u & 1);
      if (64 * s + 64 > p.K) {  // uniform: past the end of K, or across it
#pragma unroll
        for (int i = 0; i < TM; ++i) fx[u][i] = keep_bytes(fx[u][i], p.K - 64 * s - kl);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i] = mfma16x16x64(fw[u], fx[u][i], acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= TM) return;
  i32x4 a = red[0][wave][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) a += red[w][wave][lane];
  const int row = m0 + 16 * wave + l15, col = n0 + 4 * (lane >> 4);
  if (p.act == DLM_ACT_GEGLU)
    epi4_geglu<T>(a, row, col, p);
  else
    epi4<T>(a, row, col, p);
}

template <class T, int TM>
void launch_rows(const Q8Gemm& p, hipStream_t s) {
  static const std::string name =
      std::string("q8_rows_kernel<") + (sizeof(T) == 2 ? "_Float16" : "float") + ", " + std::to_string(TM) + ">";
  note_kernel(name.c_str());
  note_dims(p.M, p.N, p.K, (p.res ? 1 : 0) | (p.act << 4));
  launch((q8_rows_kernel<T, TM>), dim3((p.N + 15) / 16, (p.M + 16 * TM - 1) / (16 * TM)), dim3(512), 0, s, p);
}

template <class T>
void q8_gemm(const Q8Gemm& p, hipStream_t s) {
  if (p.M <= 16)
    launch_rows<T, 1>(p, s);
  else if (p.M <= 32)
    launch_rows<T, 2>(p, s);
  else
    launch_rows<T, 4>(p, s);
}

// Largest K: 128 * 128 * K stays below 2^31.
constexpr int kMaxK = 131071;
// Rows of one launch: the grid's y.
constexpr int kMaxRows = 1 << 21;

template <class T>
int linear_q8(const char* fn, Q8Gemm p, hipStream_t s) {
  auto bad = [&](const std::string& m) { return fail(DLM_ERR_INVALID_ARG, std::string(fn) + ": " + m); };
  if (!p.x || !p.w || !p.sx || !p.sw || !p.y) return bad("NULL pointer");
  if (p.act < DLM_ACT_NONE || p.act > DLM_ACT_GELU) return bad("unknown activation");
  if (p.K > kMaxK) return bad("K over " + std::to_string(kMaxK) + " may overflow the 32-bit sums");
  const int k16 = (p.K + 15) & ~15, cols = p.act == DLM_ACT_GEGLU ? p.N / 2 : p.N;
  if (p.act == DLM_ACT_GEGLU && p.N % 16) return bad("GEGLU needs N % 16 == 0");
  if (p.ldx % 16 || p.ldw % 16 || !dlm_aligned16(p.x) || !dlm_aligned16(p.w))
    return bad("X and W need 16-byte aligned rows");
  if (p.ldx < k16 || p.ldw < k16) return bad("row stride of X or W below K rounded up to 16");
  if (p.ldy < cols || (p.res && p.ldr < cols)) return bad("row stride of Y or R below the output columns");
  if ((uintptr_t)p.y % sizeof(T) || (uintptr_t)p.res % sizeof(T) || (uintptr_t)p.bias % 2 || (uintptr_t)p.sx % 4 ||
      (uintptr_t)p.sw % 4)
    return bad("pointer not aligned to its element");
  const uintptr_t y0 = (uintptr_t)p.y, y1 = y0 + ((uintptr_t)(p.M - 1) * p.ldy + cols) * sizeof(T);
  struct {
    const char* name;
    const void* p;
    uintptr_t bytes;
  } in[] = {{"X", p.x, (uintptr_t)(p.M - 1) * p.ldx + k16},
            {"W", p.w, (uintptr_t)(p.N - 1) * p.ldw + k16},
            {"sx", p.sx, (uintptr_t)p.M * 4},
            {"sw", p.sw, (uintptr_t)p.N * 4},
            {"bias", p.bias, (uintptr_t)p.N * 2},
            {"R", p.res, ((uintptr_t)(p.M - 1) * p.ldr + cols) * sizeof(T)}};
  for (const auto& i : in) {
    if (!i.p || (uintptr_t)i.p >= y1 || (uintptr_t)i.p + i.bytes <= y0) continue;
    if (i.p == p.res && p.res == p.y && p.ldr == p.ldy) continue;  // added in place
    return bad(std::string("Y overlaps ") + i.name);
  }
  for (int left = p.M; left > 0; left -= kMaxRows) {
    p.M = std::min(left, kMaxRows);
    q8_gemm<T>(p, s);
    DLM_LAUNCH_CHECK();
    p.x += kMaxRows * p.ldx;
    p.sx += kMaxRows;
    p.y = (T*)p.y + kMaxRows * p.ldy;
    if (p.res) p.res = (const T*)p.res + kMaxRows * p.ldr;
  }
  return DLM_OK;
}

}  // namespace
}  // namespace dlm

using namespace dlm;

extern "C" {

int dlm_linear_q8_fp16(const void* X, int ldx, const float* sx, const void* W, int ldw, const float* sw,
                       const void* bias, const void* R, int ldr, void* Y, int ldy, int M, int N, int K, float beta,
                       int act, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0) return DLM_OK;
  return linear_q8<f16>(__func__,
                        Q8Gemm{(const int8_t*)X, (const int8_t*)W, sx, sw, (const f16*)bias, R, Y, ldx, ldw, ldr, ldy,
                               M, N, K, beta, act},
                        (hipStream_t)stream);
}

int dlm_linear_q8_f32out(const void* X, int ldx, const float* sx, const void* W, int ldw, const float* sw,
                         const void* bias, const float* R, int ldr, float* Y, int ldy, int M, int N, int K, float beta,
                         int act, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0) return DLM_OK;
  return linear_q8<float>(__func__,
                          Q8Gemm{(const int8_t*)X, (const int8_t*)W, sx, sw, (const f16*)bias, R, Y, ldx, ldw, ldr,
                                 ldy, M, N, K, beta, act},
                          (hipStream_t)stream);
}

}  // extern "C"
