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
#include "dlm_tuning.h"
#include "dma.hpp"

namespace dlm {
namespace {

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

// x Phi(x) = max(x, 0) - |x| Q(|x|) with the upper tail Q(z) = erfc(z / sqrt 2) / 2
// by Abramowitz & Stegun 7.1.26 (its coefficients halved, p and the exponent
// scaled by 1 / sqrt 2; |error of Q| <= 7.5e-8, with the roundings 3.1e-7).  Two VALU
// instructions fewer than 0.5 x (1 + erf), where they bound the epilogue (GEGLU
// 2048x10240x1280 39.0 -> 38.4 us), and no cancellation at negative x.  Relative to
// the result that is 6e-7 for |x| < 1 (fp32's erf would give 1.5e-7) and 1.6e-3 at
// -5, where 0.5 x (1 + erf) has lost all but two digits.  Past 16 the tail is 0 in
// fp32, so that infinities keep to their limits; NaN stays NaN.
__device__ __forceinline__ float gelu_tail(float x) {
  const float z = __builtin_elementwise_minimum(fabsf(x), 16.0f);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.231641888f, z, 1.0f));
  float q = __builtin_fmaf(0.5307027145f, t, -0.7265760135f);
  q = __builtin_fmaf(q, t, 0.7107068705f);
  q = __builtin_fmaf(q, t, -0.142248368f);
  q = __builtin_fmaf(q, t, 0.127414796f);
  q *= t * __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  return __builtin_fmaf(-z, q, __builtin_elementwise_maximum(x, 0.0f));
}

__device__ __forceinline__ float act_f(float v, int act) {
  if (act == DLM_ACT_SILU) return silu_f(v);
  if (act == DLM_ACT_GELU) return gelu_tail(v);
  return v;
}

// An fp32 result in the output's type.  The compiler may merge a multiply-add and
// its conversion to fp16 into one instruction that rounds once (v_fma_mixlo_f16),
// and does so in some instantiations: the same sums then differ by a unit in the
// last place between tiles, where they lie close to a tie.  Opaque to it, every
// result is rounded to fp32, then to T.
template <class T>
__device__ __forceinline__ T out_cast(float v) {
  if constexpr (sizeof(T) == 2) asm("" : "+v"(v));
  return (T)v;
}

// ---------------------------------------------------------------------------
// Output tiles of BM x BN, operands through LDS.
// ---------------------------------------------------------------------------
constexpr int kSlice = 128;                // bytes (and values) of K in a slice: one line of a row
constexpr int kOOB = (int)0x80000000;      // any offset past the buffer reads 0
constexpr int kPlain = 0, kPingPong = 1;   // main-loop schedules

// DMA of one operand's tile: the lane's byte offsets, and the slice's.
// K is rounded up to a multiple of 16 here (rows have that room).
template <int I>
struct Q8Rows {
  i32x4 rs;
  int voff[I];
  int soff, kc, K;
  __device__ Q8Rows(const int8_t* base, long long ld, int rows, int K_, int nw, int wave, int lane)
      : rs(dma_rsrc(base, (unsigned)((rows - 1) * (int)ld + K_))), soff(0), K(K_) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int row = dma_row(nw, i, wave, lane);
      voff[i] = row < rows ? row * (int)ld + dma_chunk(row, lane) * 16 : kOOB;
    }
    // nw * 8 rows lie between a wave's DMA instructions, a multiple of 16: a
    // lane's chunk is the same in all of them
    kc = dma_chunk(dma_row(nw, 0, wave, lane), lane) * 16;
  }
  __device__ __forceinline__ void prepare(int kt) {
    soff = kt * kSlice;
    if (kt * kSlice + kSlice > K) {  // uniform: a slice that K ends in or before
#pragma unroll
      for (int i = 0; i < I; ++i) voff[i] = kt * kSlice + kc < K ? voff[i] : kOOB;
    }
  }
};

template <class T>
struct Vec4;
template <>
struct Vec4<f16> {
  typedef f16x4 type;
};
template <>
struct Vec4<float> {
  typedef f32x4 type;
};
// Four elements at any element-aligned address.
template <class T>
__device__ __forceinline__ typename Vec4<T>::type load4(const T* p) {
  typename Vec4<T>::type v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}

// Epilogue of a wave's TM x TN blocks at (m0, n0).  The blocks hold four columns
// of a row a lane; stored from there, an instruction covers 32 bytes of each of
// 16 rows, which makes the stores the longest part of it (8192x1920x640 on
// 128x128 tiles 25.3 us, through LDS 22.1; 2048x1280x128 with a residual 8.6,
// 6.3).  So the scaled sums go through the wave's part of the (now free) operand
// ring, CI blocks' rows at a time, and are finished and stored row by row, 16
// bytes a lane (the hardware takes them at any alignment: off it they cost 1 us
// of 14 at 1975x1283, where 4-byte stores cost 8).
// Every tile forms an output by the same operations in the same order, so that
// it does not depend on the tile that the shape selects:
//   v = fma(float(sum) * sw, sx, bias) on the way in,
//   act(v), fma(beta, R, .), rounding to T on the way out.
// Small wave tiles request scales, bias and residual ahead of the main loop, the
// others once their accumulators are done with.
template <class T, int TM, int TN, int BYTES>
struct Epilogue {
  static constexpr int WN = TN * 16, LD = WN + 4;  // 16 rows' 16-byte writes touch each bank once
  static constexpr int FIT = BYTES / (16 * LD * 4);
  static_assert(FIT >= 1, "a block's rows do not fit");
  static constexpr int CI = TM % 4 == 0 && FIT >= 4 ? 4 : TM % 2 == 0 && FIT >= 2 ? 2 : 1;
  static constexpr int V = 16 / sizeof(T), VR = WN / V, N_IT = (16 * CI * VR + 63) / 64;
  static constexpr bool EARLY = TM * TN <= 8, EARLY_RES = TM * TN <= 4;
  typedef T VecT __attribute__((ext_vector_type(V)));
  const Q8Gemm& p;
  int m0, n0, lane;
  f32x4 cs[TN];
  f16x4 cb[TN];
  float sx[TM];
  // a residual without an activation is requested ahead of the exchange, unless
  // the accumulators leave no room (the 192x128 tile)
  static constexpr bool AHEAD = TM * TN <= 10 || TM == CI;
  VecT rv[AHEAD ? TM / CI : 1][N_IT];

  __device__ Epilogue(const Q8Gemm& p_, int m0_, int n0_, int lane_) : p(p_), m0(m0_), n0(n0_), lane(lane_) {
    if (EARLY) scales();
    if (EARLY_RES) residual();
  }
  __device__ __forceinline__ void scales() {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int col = n0 + 16 * j + 4 * (lane >> 4);
      const int c = p.N >= 4 ? min(col, p.N - 4) : 0;
      cb[j] = f16x4{};
      if (p.N >= 4) {
        cs[j] = load4(p.sw + c);
        if (p.bias) cb[j] = load4(p.bias + c);
      }
      if (col != c || p.N < 4) {  // fewer than four columns are left
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          cs[j][t] = p.sw[min(col + t, p.N - 1)];
          if (p.bias) cb[j][t] = p.bias[min(col + t, p.N - 1)];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] = p.sx[min(m0 + 16 * i + (lane & 15), p.M - 1)];
  }
  // Residual vector of columns col .. col + V - 1.  `whole`: the wave's columns
  // all lie in N, so that no load stands in a branch of lanes (its result
  // would be waited for there).
  __device__ __forceinline__ VecT get_res(int row, int col, int cols, bool whole) const {
    VecT r = {};
    const T* q = (const T*)p.res + (size_t)min(row, p.M - 1) * p.ldr + col;
    if (whole || col + V <= cols) {
      __builtin_memcpy(&r, q, sizeof(r));
    } else {
#pragma unroll
      for (int t = 0; t < V - 1; ++t)
        if (col + t < cols) r[t] = q[t];
    }
    return r;
  }
  __device__ __forceinline__ void residual() {
    if constexpr (AHEAD) {
      if (!p.res || p.act != DLM_ACT_NONE) return;
      const bool whole = n0 + WN <= p.N;
#pragma unroll
      for (int c = 0; c < TM / CI; ++c)
#pragma unroll
        for (int it = 0; it < N_IT; ++it) {
          const int idx = it * 64 + lane;
          rv[c][it] = get_res(m0 + 16 * CI * c + idx / VR, n0 + idx % VR * V, p.N, whole);
        }
    }
  }
  // Stores a finished vector, columns col .. col + V - 1 of a row.
  __device__ __forceinline__ void put(int row, int col, int cols, const VecT& o) const {
    if (row >= p.M || col >= cols) return;
    T* y = (T*)p.y + (size_t)row * p.ldy + col;
    if (col + V <= cols) {
      __builtin_memcpy(y, &o, sizeof(o));
    } else {
#pragma unroll
      for (int t = 0; t < V - 1; ++t)
        if (col + t < cols) y[t] = o[t];
    }
  }
  // fp16 outputs with neither activation nor residual are rounded ahead of the
  // exchange: half the bytes (2048x10240x1280 38.9 -> 36.4 us; GEGLU, whose
  // outputs are half as many, gains nothing by being finished there).
  __device__ __forceinline__ void finish_narrow(const i32x4 (&acc)[TM][TN], f16 DLM_LDS* st) {
    constexpr int LDH = WN + 8, FITH = BYTES / (16 * LDH * 2);
    constexpr int CH = TM % 4 == 0 && FITH >= 4 ? 4 : TM % 3 == 0 && FITH >= 3 ? 3 : TM % 2 == 0 && FITH >= 2 ? 2 : 1;
    constexpr int ITH = (16 * CH * VR + 63) / 64;
#pragma unroll
    for (int c = 0; c < TM / CH; ++c) {
#pragma unroll
      for (int ii = 0; ii < CH; ++ii)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const i32x4& a = acc[c * CH + ii][j];
          f16x4 o;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            o[t] = out_cast<f16>(__builtin_fmaf((float)a[t] * cs[j][t], sx[c * CH + ii], (float)cb[j][t]));
          *reinterpret_cast<f16x4 DLM_LDS*>(st + (ii * 16 + (lane & 15)) * LDH + j * 16 + 4 * (lane >> 4)) = o;
        }
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int it = 0; it < ITH; ++it) {
        const int idx = it * 64 + lane, r = idx / VR, col = idx % VR * V;
        if ((16 * CH * VR) % 64 && idx >= 16 * CH * VR) break;
        const VecT o = *reinterpret_cast<const VecT DLM_LDS*>(st + r * LDH + col);
        put(m0 + 16 * CH * c + r, n0 + col, p.N, o);
      }
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
    }
  }
  __device__ __forceinline__ void finish(const i32x4 (&acc)[TM][TN], float DLM_LDS* st) {
    const int l15 = lane & 15, c4 = 4 * (lane >> 4);
    if (!EARLY_RES) residual();
    if constexpr (sizeof(T) == 2) {
      if (!p.res && p.act == DLM_ACT_NONE) {
        if (!EARLY) scales();
        finish_narrow(acc, (f16 DLM_LDS*)st);
        return;
      }
    }
    if (!EARLY) scales();
#pragma unroll
    for (int c = 0; c < TM / CI; ++c) {
      const int r0 = m0 + 16 * CI * c;
#pragma unroll
      for (int ii = 0; ii < CI; ++ii)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const i32x4& a = acc[c * CI + ii][j];
          f32x4 v;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            v[t] = __builtin_fmaf((float)a[t] * cs[j][t], sx[c * CI + ii], (float)cb[j][t]);
          *reinterpret_cast<f32x4 DLM_LDS*>(st + (ii * 16 + l15) * LD + j * 16 + c4) = v;
        }
      // the LDS takes a wave's accesses in order
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
      if (p.act == DLM_ACT_NONE) {
#pragma unroll
        for (int it = 0; it < N_IT; ++it) {
          const int idx = it * 64 + lane, r = idx / VR, col = idx % VR * V;
          if ((16 * CI * VR) % 64 && idx >= 16 * CI * VR) break;
          VecT o, rg = {};
          if constexpr (AHEAD)
            rg = rv[c][it];
          else if (p.res)
            rg = get_res(r0 + r, n0 + col, p.N, n0 + WN <= p.N);
#pragma unroll
          for (int u = 0; u < V / 4; ++u) {
            const f32x4 v = *reinterpret_cast<const f32x4 DLM_LDS*>(st + r * LD + col + 4 * u);
#pragma unroll
            for (int t = 0; t < 4; ++t)
              o[4 * u + t] = out_cast<T>(p.res ? __builtin_fmaf(p.beta, (float)rg[4 * u + t], v[t]) : v[t]);
          }
          put(r0 + r, n0 + col, p.N, o);
        }
      } else if (p.act == DLM_ACT_GEGLU) {
        // V outputs from V values and V gates, which alternate in groups of four
        constexpr int VG = (WN / 2 + V - 1) / V;
#pragma unroll 1
        for (int idx = lane; idx < 16 * CI * VG; idx += 64) {
          const int r = idx / VG, col = idx % VG * V;
          VecT o, rg = {};
          if (p.res) rg = get_res(r0 + r, (n0 >> 1) + col, p.N >> 1, false);
#pragma unroll
          for (int u = 0; u < V / 4; ++u) {
            const float DLM_LDS* q = st + r * LD + 2 * col + 8 * u;
            const f32x4 v = *reinterpret_cast<const f32x4 DLM_LDS*>(q);
            const f32x4 g = *reinterpret_cast<const f32x4 DLM_LDS*>(q + 4);
#pragma unroll
            for (int t = 0; t < 4; ++t)
              o[4 * u + t] = out_cast<T>(__builtin_fmaf(p.beta, (float)rg[4 * u + t], v[t] * gelu_tail(g[t])));
          }
          put(r0 + r, (n0 >> 1) + col, p.N >> 1, o);
        }
      } else {
#pragma unroll 1
        for (int idx = lane; idx < 16 * CI * VR; idx += 64) {
          const int r = idx / VR, col = idx % VR * V;
          VecT o, rg = {};
          if (p.res) rg = get_res(r0 + r, n0 + col, p.N, false);
#pragma unroll
          for (int u = 0; u < V / 4; ++u) {
            const f32x4 v = *reinterpret_cast<const f32x4 DLM_LDS*>(st + r * LD + col + 4 * u);
#pragma unroll
            for (int t = 0; t < 4; ++t)
              o[4 * u + t] = out_cast<T>(__builtin_fmaf(p.beta, (float)rg[4 * u + t], act_f(v[t], p.act)));
          }
          put(r0 + r, n0 + col, p.N, o);
        }
      }
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
    }
  }
};

// Waves a SIMD is to hold: those of as many workgroups as the LDS takes, two at
// most counted.
constexpr int waves_per_simd(int lds, int waves) { return (lds <= 80 * 1024 ? 2 : 1) * waves / 4; }

// K advances in slices of 128 bytes, copied by DMA into a ring of NS stages
// (LDS rows of 128 bytes, 16-byte chunks XOR-swizzled by (row >> 1) & 7: a
// fragment read touches every bank once).
// SCH kPlain: slice kt + NS - 1 is requested while slice kt is multiplied, the
// next k-step's fragments are read before this one's MFMAs, one barrier a
// slice.
// SCH kPingPong: the second half of the waves runs one barrier behind the
// first, so that between two barriers one half reads fragments and issues DMA
// while the other half, on the same SIMDs, issues nothing but MFMAs.  A
// wave's reads end before the barrier that closes their phase, and the last
// reads of a stage (the late half's) before the phase that refills it; it
// waits for its own part of the next slice a barrier before either half reads
// that.
// KG > 1 (few rows, where a grid of one workgroup a tile would leave most of
// the chip waiting for one workgroup's slices): KG groups of waves take the
// slices in turn, each with a ring of its own, and add their sums up in LDS.
template <class T, int BM, int BN, int WM, int WN, int NS, int SCH, int KG>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * KG * 64,
                                  waves_per_simd(KG* NS* (BM + BN) * kSlice, (BM / WM) * (BN / WN) * KG))
q8_tile_kernel(Q8Gemm p, int tiles_m, int tiles_n) {
  constexpr int WAVES_N = BN / WN, NW = (BM / WM) * WAVES_N;  // waves of a K group
  constexpr int TM = WM / 16, TN = WN / 16;
  constexpr int KS = kSlice / 64;
  constexpr int SA = BM * kSlice, STAGE = (BM + BN) * kSlice;
  constexpr int GA = BM / 8, GB = BN / 8;
  constexpr int IA = (GA + NW - 1) / NW, IB = (GB + NW - 1) / NW;
  static_assert(BM % 8 == 0 && BN % 8 == 0 && WM % 16 == 0 && WN % 16 == 0 && NW % 2 == 0 && NS >= 2, "tile");
  static_assert(KG == 1 || SCH == kPlain, "K groups use the plain loop");
  static_assert(KG * NS * STAGE <= 160 * 1024, "ring larger than the LDS");
  static_assert((KG - 1) * BM * BN * 4 <= KG * NS * STAGE, "the K groups' sums do not fit the ring");
  __shared__ __attribute__((aligned(1024))) unsigned char smem_generic[KG * NS * STAGE];

  const int lane = threadIdx.x & 63, l15 = lane & 15;
  const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave_all / NW, wave = wave_all % NW;
  unsigned char DLM_LDS* all = (unsigned char DLM_LDS*)smem_generic;
  unsigned char DLM_LDS* smem = all + kg * (NS * STAGE);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  int tmi, tni;
  tile_coords(blockIdx.x, tiles_m, tiles_n, tmi, tni);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int K16 = (p.K + 15) & ~15;
  Q8Rows<IA> al(p.x + (size_t)m0 * p.ldx, p.ldx, min(BM, p.M - m0), K16, NW, wave, lane);
  Q8Rows<IB> bl(p.w + (size_t)n0 * p.ldw, p.ldw, min(BN, p.N - n0), K16, NW, wave, lane);
  constexpr int PART = (KG * NS * STAGE - (KG - 1) * BM * BN * 4) / NW & ~15;
  Epilogue<T, TM, TN, PART> ep(p, m0 + wm * WM, n0 + wn * WN, lane);
  // slices of a group: kg, kg + KG, ...; one past the end of K reads zeros
  const int ke = (K16 + KG * kSlice - 1) / (KG * kSlice);

  i32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

  auto dma_a = [&](unsigned char DLM_LDS* st, int i) {
    if (IA * NW == GA || i + 1 < IA || wave < GA - (IA - 1) * NW)
      dma16(al.rs, st + (i * NW + wave) * 1024, al.voff[i], al.soff);
  };
  auto dma_b = [&](unsigned char DLM_LDS* st, int i) {
    if (IB * NW == GB || i + 1 < IB || wave < GB - (IB - 1) * NW)
      dma16(bl.rs, st + SA + (i * NW + wave) * 1024, bl.voff[i], bl.soff);
  };
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) {
    al.prepare(min(s, ke - 1) * KG + kg);
    bl.prepare(min(s, ke - 1) * KG + kg);
#pragma unroll
    for (int i = 0; i < IA; ++i) dma_a(smem + s * STAGE, i);
#pragma unroll
    for (int i = 0; i < IB; ++i) dma_b(smem + s * STAGE, i);
  }
  // The bytes of X past a K that is no multiple of 16 are cleared in LDS, by the
  // lanes whose DMA brought them, between their wait for the last slice and the
  // barrier that publishes it (W's then multiply zeros).
  const int tail = p.K & 15, last = (K16 - 1) / kSlice;
  auto clear_tail = [&](unsigned char DLM_LDS* st, int slice) {
    if (tail == 0 || slice != last) return;  // uniform
    if (al.kc == ((K16 - 16) & (kSlice - 1))) {
#pragma unroll
      for (int i = 0; i < IA; ++i) {
        if (IA * NW == GA || i + 1 < IA || wave < GA - (IA - 1) * NW) {
          i32x4 DLM_LDS* at = (i32x4 DLM_LDS*)(st + (i * NW + wave) * 1024 + lane * 16);
          *at = keep_bytes(*at, tail);
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  };
  // DMA instructions a slice that this wave leaves to others (0..2): its wait
  // for a slice allows P later slices of its own requests
  const int skips = ((IA * NW == GA || wave < GA - (IA - 1) * NW) ? 0 : 1) +
                    ((IB * NW == GB || wave < GB - (IB - 1) * NW) ? 0 : 1);
#define DLM_WAIT_SLICES(P)              \
  do {                                  \
    if (skips == 0) {                   \
      DLM_WAIT_VM((P) * (IA + IB));     \
    } else if (skips == 1) {            \
      DLM_WAIT_VM((P) * (IA + IB - 1)); \
    } else {                            \
      DLM_WAIT_VM((P) * (IA + IB - 2)); \
    }                                   \
  } while (0)
  // byte offset of this lane's first A / B fragment in a stage, k-step 0; the
  // k-step flips bit 6
  const int fc = ((lane >> 4) ^ (l15 >> 1)) * 16;
  const int fa0 = (wm * WM + l15) * kSlice + fc, fb0 = SA + (wn * WN + l15) * kSlice + fc;
  auto rd = [&](const unsigned char DLM_LDS* st, int ks, i32x4 (&fa)[TM], i32x4 (&fb)[TN]) {
    const unsigned char DLM_LDS* pa = st + (fa0 ^ (ks * 64));
    const unsigned char DLM_LDS* pb = st + (fb0 ^ (ks * 64));
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = *reinterpret_cast<const i32x4 DLM_LDS*>(pa + i * 2048);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = *reinterpret_cast<const i32x4 DLM_LDS*>(pb + j * 2048);
  };
  auto mma = [&](const i32x4 (&fa)[TM], const i32x4 (&fb)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mfma16x16x64(fb[j], fa[i], acc[i][j]);
  };
  int slot = 0, nslot = NS - 1;  // stage read, stage refilled
  if constexpr (SCH == kPingPong) {
    const bool late = wave >= NW / 2;
    DLM_WAIT_SLICES(NS - 2);
    clear_tail(smem, 0);
    __builtin_amdgcn_s_barrier();
    if (late) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    for (int kt = 0; kt < ke; ++kt) {
      const unsigned char DLM_LDS* st = smem + slot * STAGE;
      unsigned char DLM_LDS* nst = smem + nslot * STAGE;
      const int nkt = min(kt + NS - 1, ke - 1);
      al.prepare(nkt);
      bl.prepare(nkt);
      i32x4 fa[TM], fb[TN];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        rd(st, ks, fa, fb);
#pragma unroll
        for (int i = 0; i < IA; ++i)
          if (i % KS == ks) dma_a(nst, i);
#pragma unroll
        for (int i = 0; i < IB; ++i)
          if ((IA + i) % KS == ks) dma_b(nst, i);
        if (ks == KS - 1) {
          DLM_WAIT_SLICES(NS - 2);  // slice kt + 1
          clear_tail(smem + (slot + 1 == NS ? 0 : slot + 1) * STAGE, kt + 1);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);         // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        mma(fa, fb);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
      slot = slot + 1 == NS ? 0 : slot + 1;
      nslot = nslot + 1 == NS ? 0 : nslot + 1;
    }
    if (!late) __builtin_amdgcn_s_barrier();
  } else {
    for (int kt = 0; kt < ke; ++kt) {
      DLM_WAIT_SLICES(NS - 2);
      clear_tail(smem + slot * STAGE, kt * KG + kg);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const unsigned char DLM_LDS* st = smem + slot * STAGE;
      unsigned char DLM_LDS* nst = smem + nslot * STAGE;
      const int nkt = min(kt + NS - 1, ke - 1);
      al.prepare(nkt * KG + kg);
      bl.prepare(nkt * KG + kg);
      i32x4 fa[2][TM], fb[2][TN];
      rd(st, 0, fa[0], fb[0]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        __builtin_amdgcn_sched_barrier(0);
        if (ks + 1 < KS) rd(st, ks + 1, fa[(ks + 1) & 1], fb[(ks + 1) & 1]);
#pragma unroll
        for (int i = 0; i < IA; ++i)
          if (i % KS == ks) dma_a(nst, i);
#pragma unroll
        for (int i = 0; i < IB; ++i)
          if ((IA + i) % KS == ks) dma_b(nst, i);
        mma(fa[ks & 1], fb[ks & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      slot = slot + 1 == NS ? 0 : slot + 1;
      nslot = nslot + 1 == NS ? 0 : nslot + 1;
    }
  }
#undef DLM_WAIT_SLICES
  DLM_WAIT_VM(0);  // no DMA may still be writing this workgroup's LDS at exit

  __syncthreads();  // every wave is done with the ring
  if constexpr (KG > 1) {
    i32x4 DLM_LDS* part = (i32x4 DLM_LDS*)all;
    auto at = [&](int g, int i, int j) { return (((g - 1) * NW + wave) * TM * TN + i * TN + j) * 64 + lane; };
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) part[at(kg, i, j)] = acc[i][j];
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int g = 1; g < KG; ++g)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] += part[at(g, i, j)];
    // the first group alone goes on: its waves' parts of the ring, once all
    // of them have read the sums there
    static_assert(KG * NS * STAGE - (KG - 1) * BM * BN * 4 >= NW * 16 * (WN + 4) * 4, "no room beside the sums");
    smem = all + (KG - 1) * BM * BN * 4;
  }
  ep.finish(acc, (float DLM_LDS*)(smem + wave * PART));
}

template <class T, int BM, int BN, int WM, int WN, int NS, int SCH, int KG = 1>
void launch_tile(const Q8Gemm& p, hipStream_t s) {
  static const std::string name = std::string("q8_tile_kernel<") + (sizeof(T) == 2 ? "_Float16" : "float") + ", " +
                                  std::to_string(BM) + ", " + std::to_string(BN) + ", " + std::to_string(WM) + ", " +
                                  std::to_string(WN) + ", " + std::to_string(NS) + ", " + std::to_string(SCH) + ", " +
                                  std::to_string(KG) + ">";
  const int tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  note_kernel(name.c_str());
  note_dims(p.M, p.N, p.K, (p.res ? 1 : 0) | (p.act << 4));
  launch((q8_tile_kernel<T, BM, BN, WM, WN, NS, SCH, KG>), dim3(tm * tn), dim3((BM / WM) * (BN / WN) * KG * 64), 0, s,
         p, tm, tn);
}

// Tile override of dlm_q8_force_tile (0 = the plan below).
thread_local int g_q8_tile = 0;

// A launch's time is modelled as
//   base + (fix + slices * slice) * (1 + more * (n - 1)) + io * words * n   [us]
// n: output tiles a CU, rounded up; slices: of 128 bytes of K; more: what each
// further workgroup on a CU adds, relative to the first (over 1 where it queues
// for the LDS); words: 2-byte words that an output moves beyond the first (fp32,
// a residual).  The constants are fits to 11240 launches of 1165 shapes (1-8192
// rows, 16-14336 columns, K = 64-14336) on 7 to 14 of the tiles each, graph-replayed;
// the modelled choice takes 0.6% longer than the fastest timed in the mean, and up to
// 30% (5517x1155x234 13.7 us against 10.5).  K groups serve few rows and long K (us, without and with them:
// 1x4096x4096 6.8 -> 5.9, 13x1280x5120 9.2 -> 6.2, 48x8192x8192 22.8 -> 17.8,
// 100x4096x14336 31.0 -> 24.3, 256x2048x8192 14.8 -> 12.3), 128x160 the outputs
// that it cuts into one round of 256 (8192x640x2560 22.5 -> 19.1,
// 4096x1280x5120 with a residual 45.7 -> 35.9, 8192x640x640 10.6 -> 9.6).
struct Q8Tile {
  int bm, bn;
  float base, fix, slice, io, more;
};
constexpr Q8Tile kQ8Tiles[] = {
    {16, 32, 1.91f, 1.48f, 0.065f, 0.08f, 1.26f},    // 1: four K groups
    {16, 32, 2.29f, 0.59f, 0.099f, 0.06f, 0.67f},    // 2: two K groups
    {32, 32, 2.17f, 0.66f, 0.149f, 0.05f, 0.64f},    // 3
    {32, 32, 2.13f, 1.14f, 0.101f, 0.07f, 0.87f},    // 4: two K groups
    {64, 32, 2.29f, 0.75f, 0.167f, 0.16f, 0.83f},    // 5
    {64, 64, 2.38f, 1.27f, 0.207f, 0.33f, 0.92f},    // 6
    {64, 128, 1.50f, 2.45f, 0.286f, 0.35f, 1.14f},   // 7
    {128, 128, 1.50f, 3.61f, 0.458f, 0.73f, 1.11f},  // 8: four stages, one workgroup a CU
    {128, 128, 1.50f, 2.81f, 0.799f, 0.74f, 0.64f},  // 9: two stages, two workgroups
    {192, 128, 1.50f, 3.72f, 0.909f, 1.80f, 0.66f},  // 10: the same
    {128, 256, 1.50f, 5.84f, 0.640f, 1.41f, 1.30f},  // 11: ping-pong
    {128, 80, 2.97f, 2.32f, 0.417f, 1.03f, 0.77f},   // 12: four waves, two workgroups
    {128, 160, 2.20f, 4.37f, 0.566f, 1.40f, 1.14f},  // 13: three stages, one workgroup
    {64, 32, 1.96f, 1.64f, 0.133f, 0.17f, 1.30f},    // 14: two K groups
};

template <class T>
int plan_q8(const Q8Gemm& p) {
  const float slices = (float)((p.K + kSlice - 1) / kSlice);
  const float words = (float)(sizeof(T) / 2 * (p.res ? 2 : 1) - 1);
  int best = 1;
  float best_us = 3e38f;
  for (const Q8Tile& t : kQ8Tiles) {
    const long long grid = (long long)((p.M + t.bm - 1) / t.bm) * ((p.N + t.bn - 1) / t.bn);
    const float n = (float)((grid + 255) / 256);
    const float us =
        t.base + (t.fix + slices * t.slice) * (1.0f + t.more * (n - 1.0f)) + t.io * words * n;
    if (us < best_us) {
      best_us = us;
      best = (int)(&t - kQ8Tiles) + 1;
    }
  }
  return best;
}

template <class T>
void q8_gemm(const Q8Gemm& p, hipStream_t s) {
  switch (g_q8_tile > 0 ? g_q8_tile : plan_q8<T>(p)) {
    case 1: return launch_tile<T, 16, 32, 16, 16, 4, kPlain, 4>(p, s);
    case 2: return launch_tile<T, 16, 32, 16, 16, 3, kPlain, 2>(p, s);
    case 3: return launch_tile<T, 32, 32, 16, 16, 4, kPlain>(p, s);
    case 4: return launch_tile<T, 32, 32, 16, 16, 4, kPlain, 2>(p, s);
    case 5: return launch_tile<T, 64, 32, 16, 32, 4, kPlain>(p, s);
    case 6: return launch_tile<T, 64, 64, 32, 32, 4, kPlain>(p, s);
    case 7: return launch_tile<T, 64, 128, 32, 32, 4, kPlain>(p, s);
    case 8: return launch_tile<T, 128, 128, 64, 32, 4, kPlain>(p, s);
    case 9: return launch_tile<T, 128, 128, 64, 32, 2, kPlain>(p, s);
    case 10: return launch_tile<T, 192, 128, 48, 64, 2, kPlain>(p, s);
    case 12: return launch_tile<T, 128, 80, 32, 80, 3, kPlain>(p, s);
    case 13: return launch_tile<T, 128, 160, 32, 80, 3, kPlain>(p, s);
    case 14: return launch_tile<T, 64, 32, 32, 16, 4, kPlain, 2>(p, s);
    default: return launch_tile<T, 128, 256, 64, 64, 3, kPingPong>(p, s);  // 11
  }
}

// Largest K: 128 * 128 * K stays below 2^31.
constexpr int kMaxK = 131071;
// Largest row stride: 256 rows of a tile stay within 32-bit offsets.
constexpr int kMaxLd = 1 << 22;
// Columns a row of workgroups takes: a launch counts threads in 32 bits.
constexpr int kMaxN = 1 << 25;

template <class T>
int linear_q8(const char* fn, Q8Gemm p, hipStream_t s) {
  auto bad = [&](const std::string& m) { return fail(DLM_ERR_INVALID_ARG, std::string(fn) + ": " + m); };
  if (!p.x || !p.w || !p.sx || !p.sw || !p.y) return bad("NULL pointer");
  if (p.act < DLM_ACT_NONE || p.act > DLM_ACT_GELU) return bad("unknown activation");
  if (p.K > kMaxK) return bad("K over " + std::to_string(kMaxK) + " may overflow the 32-bit sums");
  if (p.ldx > kMaxLd || p.ldw > kMaxLd) return bad("row stride of X or W over " + std::to_string(kMaxLd));
  if (p.N > kMaxN) return bad("N over " + std::to_string(kMaxN));
  const int k16 = (p.K + 15) & ~15, cols = p.act == DLM_ACT_GEGLU ? p.N / 2 : p.N;
  if (p.act == DLM_ACT_GEGLU && p.N % 16) return bad("GEGLU needs N % 16 == 0");
  if (p.ldx % 16 || p.ldw % 16 || !dlm_aligned16(p.x) || !dlm_aligned16(p.w))
    return bad("X and W need 16-byte aligned rows");
  if (p.ldx < k16 || p.ldw < k16) return bad("row stride of X or W below K rounded up to 16");
  if (p.ldy < cols || (p.res && p.ldr < cols)) return bad("row stride of Y or R below the output columns");
  if ((uintptr_t)p.y % sizeof(T) || (uintptr_t)p.res % sizeof(T) || (uintptr_t)p.bias % 2 || (uintptr_t)p.sx % 4 ||
      (uintptr_t)p.sw % 4)
    return bad("pointer not aligned to its element");
  if (!p.res) p.beta = 0.0f;  // kernels that add beta times nothing stay clear of infinities
  const int e = (int)sizeof(T);
  const Span y{"Y", p.y, p.ldy, p.M, cols, e};
  for (const Span& in : {Span{"X", p.x, p.ldx, p.M, k16, 1}, Span{"W", p.w, p.ldw, p.N, k16, 1},
                         Span{"sx", p.sx, p.M, 1, p.M, 4}, Span{"sw", p.sw, p.N, 1, p.N, 4},
                         Span{"bias", p.bias, p.N, 1, p.N, 2}})
    if (overlap(y, in)) return bad(std::string("Y overlaps ") + in.name);
  // R alone may be Y: an output's residual is read by the lane that replaces it
  if (!(p.res == p.y && p.ldr == p.ldy) && overlap(y, Span{"R", p.res, p.ldr, p.M, cols, e}))
    return bad("Y overlaps R");
  // rows of one launch: at most 2^31 outputs, of which the smallest tile has one a
  // thread (a launch counts threads in 32 bits), and 64 rows at least, as N <= 2^25
  const int part = (int)std::min(1LL << 24, (1LL << 31) / p.N & ~63LL);
  for (int left = p.M; left > 0; left -= part) {
    p.M = std::min(left, part);
    q8_gemm<T>(p, s);
    DLM_LAUNCH_CHECK();
    p.x += part * p.ldx;
    p.sx += part;
    p.y = (T*)p.y + part * p.ldy;
    if (p.res) p.res = (const T*)p.res + part * p.ldr;
  }
  return DLM_OK;
}

}  // namespace
}  // namespace dlm

using namespace dlm;

extern "C" {

int dlm_q8_force_tile(int tile) {
  DLM_REQUIRE(tile >= 0 && tile <= 14, "tile must be in [0, 14]");
  dlm::g_q8_tile = tile;
  return DLM_OK;
}

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
