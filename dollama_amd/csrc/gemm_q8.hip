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

// 16 columns and 16 TM rows a workgroup, K dealt to its NW waves in groups
// of 128 bytes, G groups of a wave in flight at a time; operands go from
// memory to the MFMA's registers, and the waves' sums meet in LDS.
template <class T, int TM, int NW, int G>
__global__ void __launch_bounds__(NW * 64) q8_rows_kernel(Q8Gemm p) {
  constexpr int U = 2 * G;
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
  auto step = [&](int s0, int u) { return s0 + (u >> 1) * 2 * NW + (u & 1); };
  for (int s0 = 2 * wave; s0 < steps; s0 += U * NW) {
    i32x4 fw[U], fx[U][TM];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(64 * step(s0, u) + kl, klast);
      fw[u] = *reinterpret_cast<const i32x4*>(wp + k);
#pragma unroll
      for (int i = 0; i < TM; ++i) fx[u][i] = *reinterpret_cast<const i32x4*>(xp[i] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = step(s0, u);
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

// ---------------------------------------------------------------------------
// Output tiles of BM x BN, operands through LDS.
// ---------------------------------------------------------------------------
constexpr int kSlice = 128;                // bytes (and values) of K in a slice: one line of a row
constexpr int kOOB = (int)0x80000000;      // any offset past the buffer reads 0
constexpr int kPlain = 0, kPingPong = 1;   // main-loop schedules

// DMA of one operand's tile: the lane's byte offsets, and the slice's.
// K is a multiple of 16 here.
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
    if (kt * kSlice + kSlice > K) {  // uniform: the last slice, where it is not a whole one
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

// A wave's TM x TN blocks: lane holds row row0 + 16 i and columns col0 + 16 j
// + [0, 4) of block (i, j).  Loads go to addresses clamped into the tensors
// and are issued together; the last column group of an N that is no multiple
// of four goes value by value.  N >= 16.
template <class T, int TM, int TN>
__device__ __forceinline__ void epi_tile(const i32x4 (&acc)[TM][TN], int row0, int col0, const Q8Gemm& p) {
  f32x4 cs[TN];
  f16x4 cb[TN];
  float sx[TM];
#pragma unroll
  for (int j = 0; j < TN; ++j) cs[j] = load4(p.sw + min(col0 + 16 * j, p.N - 4));
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < TN; ++j) cb[j] = load4(p.bias + min(col0 + 16 * j, p.N - 4));
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) sx[i] = p.sx[min(row0 + 16 * i, p.M - 1)];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = row0 + 16 * i, r = min(row, p.M - 1);
    typename Vec4<T>::type rv[TN];
    if (p.res) {
      const T* res = (const T*)p.res + (size_t)r * p.ldr;
#pragma unroll
      for (int j = 0; j < TN; ++j) rv[j] = load4(res + min(col0 + 16 * j, p.N - 4));
    }
    T* y = (T*)p.y + (size_t)r * p.ldy;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int col = col0 + 16 * j;
      typename Vec4<T>::type o;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float v = (float)acc[i][j][t] * cs[j][t] * sx[i];
        if (p.bias) v += (float)cb[j][t];
        v = act_f(v, p.act);
        if (p.res) v = __builtin_fmaf(p.beta, (float)rv[j][t], v);
        o[t] = (T)v;
      }
      if (row < p.M) {
        if (col + 4 <= p.N)
          __builtin_memcpy(y + col, &o, sizeof(o));
        else
          epi4<T>(acc[i][j], row, col, p);
      }
    }
  }
}

template <class T, int TM, int TN>
__device__ __forceinline__ void epi_tile_geglu(const i32x4 (&acc)[TM][TN], int row0, int col0, const Q8Gemm& p) {
  const int t0 = (col0 & 4) ? 2 : 0;
  float sv[TN][2], sg[TN][2], bv[TN][2], bg[TN][2], sx[TM];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int vc = min((col0 + 16 * j) & ~4, p.N - 8) + t0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sv[j][t] = p.sw[vc + t];
      sg[j][t] = p.sw[vc + 4 + t];
      bv[j][t] = p.bias ? (float)p.bias[vc + t] : 0.0f;
      bg[j][t] = p.bias ? (float)p.bias[vc + 4 + t] : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) sx[i] = p.sx[min(row0 + 16 * i, p.M - 1)];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = row0 + 16 * i, r = min(row, p.M - 1);
    float rv[TN][2];
    if (p.res) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          rv[j][t] = (float)((const T*)p.res)[(size_t)r * p.ldr + (min((col0 + 16 * j) & ~4, p.N - 8) >> 1) + t0 + t];
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const i32x4& a = acc[i][j];
      const auto s02 = __builtin_amdgcn_permlane16_swap((unsigned)a[0], (unsigned)a[2], false, false);
      const auto s13 = __builtin_amdgcn_permlane16_swap((unsigned)a[1], (unsigned)a[3], false, false);
      const int vc = (col0 + 16 * j) & ~4;
      const int v2[2] = {(int)s02[0], (int)s13[0]}, g2[2] = {(int)s02[1], (int)s13[1]};
      T o[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float v = (float)v2[t] * sv[j][t] * sx[i] + bv[j][t];
        const float g = (float)g2[t] * sg[j][t] * sx[i] + bg[j][t];
        v *= gelu_erf_fast(g);
        if (p.res) v = __builtin_fmaf(p.beta, rv[j][t], v);
        o[t] = (T)v;
      }
      if (row < p.M && vc < p.N) __builtin_memcpy((T*)p.y + (size_t)row * p.ldy + (vc >> 1) + t0, o, sizeof(o));
    }
  }
}

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
// The last 1 to 15 values of a K that is no multiple of 16 follow the loop:
// one MFMA a block on fragments from memory, with what lies past K zeroed.
template <class T, int BM, int BN, int WM, int WN, int NS, int SCH>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64) q8_tile_kernel(Q8Gemm p, int tiles_m, int tiles_n) {
  constexpr int WAVES_N = BN / WN, NW = (BM / WM) * WAVES_N;
  constexpr int TM = WM / 16, TN = WN / 16;
  constexpr int KS = kSlice / 64;
  constexpr int SA = BM * kSlice, STAGE = (BM + BN) * kSlice;
  constexpr int GA = BM / 8, GB = BN / 8;
  constexpr int IA = (GA + NW - 1) / NW, IB = (GB + NW - 1) / NW;
  static_assert(BM % 8 == 0 && BN % 8 == 0 && WM % 16 == 0 && WN % 16 == 0 && NW % 2 == 0 && NS >= 2, "tile");
  static_assert(NS * STAGE <= 160 * 1024, "ring larger than the LDS");
  __shared__ __attribute__((aligned(1024))) unsigned char smem_generic[NS * STAGE];
  unsigned char DLM_LDS* smem = (unsigned char DLM_LDS*)smem_generic;

  const int lane = threadIdx.x & 63, l15 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  int tmi, tni;
  tile_coords(blockIdx.x, tiles_m, tiles_n, tmi, tni);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int K16 = p.K & ~15;
  Q8Rows<IA> al(p.x + (size_t)m0 * p.ldx, p.ldx, min(BM, p.M - m0), K16, NW, wave, lane);
  Q8Rows<IB> bl(p.w + (size_t)n0 * p.ldw, p.ldw, min(BN, p.N - n0), K16, NW, wave, lane);
  const int ke = (K16 + kSlice - 1) / kSlice;

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
    al.prepare(min(s, ke - 1));
    bl.prepare(min(s, ke - 1));
#pragma unroll
    for (int i = 0; i < IA; ++i) dma_a(smem + s * STAGE, i);
#pragma unroll
    for (int i = 0; i < IB; ++i) dma_b(smem + s * STAGE, i);
  }
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
        if (ks == KS - 1) DLM_WAIT_SLICES(NS - 2);  // slice kt + 1
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
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const unsigned char DLM_LDS* st = smem + slot * STAGE;
      unsigned char DLM_LDS* nst = smem + nslot * STAGE;
      const int nkt = min(kt + NS - 1, ke - 1);
      al.prepare(nkt);
      bl.prepare(nkt);
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

  if (p.K & 15) {
    const bool mine = lane < 16;  // the first 16 values of the k-step
    i32x4 fa[TM], fb[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const size_t r = min(m0 + wm * WM + 16 * i + l15, p.M - 1);
      fa[i] = keep_bytes(*reinterpret_cast<const i32x4*>(p.x + r * p.ldx + K16), mine ? p.K & 15 : 0);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const size_t r = min(n0 + wn * WN + 16 * j + l15, p.N - 1);
      fb[j] = *reinterpret_cast<const i32x4*>(p.w + r * p.ldw + K16);
    }
    mma(fa, fb);
  }

  // ------------------------------ epilogue ------------------------------
  const int row0 = m0 + wm * WM + l15, col0 = n0 + wn * WN + 4 * (lane >> 4);
  if (p.act == DLM_ACT_GEGLU)
    epi_tile_geglu<T>(acc, row0, col0, p);
  else
    epi_tile<T>(acc, row0, col0, p);
}

template <class T, int BM, int BN, int WM, int WN, int NS, int SCH>
void launch_tile(const Q8Gemm& p, hipStream_t s) {
  static const std::string name = std::string("q8_tile_kernel<") + (sizeof(T) == 2 ? "_Float16" : "float") + ", " +
                                  std::to_string(BM) + ", " + std::to_string(BN) + ", " + std::to_string(WM) + ", " +
                                  std::to_string(WN) + ", " + std::to_string(NS) + ", " + std::to_string(SCH) + ">";
  const int tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  note_kernel(name.c_str());
  note_dims(p.M, p.N, p.K, (p.res ? 1 : 0) | (p.act << 4));
  launch((q8_tile_kernel<T, BM, BN, WM, WN, NS, SCH>), dim3(tm * tn), dim3((BM / WM) * (BN / WN) * 64), 0, s, p, tm,
         tn);
}

template <class T, int TM, int NW = 8, int G = 2>
void launch_rows(const Q8Gemm& p, hipStream_t s) {
  static const std::string name = std::string("q8_rows_kernel<") + (sizeof(T) == 2 ? "_Float16" : "float") + ", " +
                                  std::to_string(TM) + ", " + std::to_string(NW) + ", " + std::to_string(G) + ">";
  note_kernel(name.c_str());
  note_dims(p.M, p.N, p.K, (p.res ? 1 : 0) | (p.act << 4));
  launch((q8_rows_kernel<T, TM, NW, G>), dim3((p.N + 15) / 16, (p.M + 16 * TM - 1) / (16 * TM)), dim3(NW * 64), 0, s, p);
}

thread_local int g_q8_tile = 0;

template <class T>
void q8_gemm(const Q8Gemm& p, hipStream_t s) {
  switch (g_q8_tile) {
    case 1: return launch_tile<T, 256, 160, 64, 80, 3, kPingPong>(p, s);
    case 3: return launch_tile<T, 128, 160, 32, 80, 4, kPlain>(p, s);
    case 4: return launch_tile<T, 128, 128, 64, 32, 4, kPlain>(p, s);
    case 5: return launch_tile<T, 128, 64, 64, 32, 4, kPlain>(p, s);
    case 6: return launch_tile<T, 128, 80, 16, 80, 4, kPlain>(p, s);
    case 7: return launch_tile<T, 64, 64, 32, 32, 4, kPlain>(p, s);
    case 8: return launch_tile<T, 64, 32, 16, 32, 4, kPlain>(p, s);
    case 10: return launch_tile<T, 256, 128, 64, 64, 3, kPingPong>(p, s);
    case 12: return launch_tile<T, 128, 128, 32, 64, 2, kPlain>(p, s);
    case 13: return launch_rows<T, 1>(p, s);
    case 14: return launch_rows<T, 2>(p, s);
    case 15: return launch_rows<T, 4>(p, s);
    case 16: return launch_tile<T, 64, 128, 32, 32, 4, kPlain>(p, s);
    case 17: return launch_tile<T, 32, 64, 16, 16, 4, kPlain>(p, s);
    case 18: return launch_tile<T, 64, 16, 16, 16, 4, kPlain>(p, s);
    case 19: return launch_tile<T, 128, 256, 64, 64, 3, kPingPong>(p, s);
    case 20: return launch_tile<T, 128, 160, 64, 80, 2, kPlain>(p, s);
    case 21: return launch_tile<T, 128, 128, 64, 64, 2, kPlain>(p, s);
    case 22: return launch_tile<T, 128, 80, 32, 80, 3, kPlain>(p, s);
    case 23: return launch_tile<T, 64, 160, 32, 80, 2, kPlain>(p, s);
    case 24: return launch_tile<T, 32, 32, 16, 16, 4, kPlain>(p, s);
    case 25: return launch_tile<T, 64, 32, 32, 16, 6, kPlain>(p, s);
    case 26: return launch_tile<T, 64, 64, 32, 32, 8, kPlain>(p, s);
    case 27: return launch_tile<T, 64, 64, 32, 16, 8, kPlain>(p, s);
    case 28: return launch_tile<T, 64, 32, 16, 32, 8, kPlain>(p, s);
    case 30: return launch_rows<T, 1, 8, 4>(p, s);
    case 31: return launch_rows<T, 1, 16, 2>(p, s);
    case 32: return launch_rows<T, 1, 16, 1>(p, s);
    case 33: return launch_rows<T, 2, 8, 4>(p, s);
    case 34: return launch_rows<T, 2, 16, 2>(p, s);
    case 35: return launch_rows<T, 4, 16, 2>(p, s);
    case 36: return launch_rows<T, 4, 8, 1>(p, s);
    case 37: return launch_rows<T, 1, 4, 4>(p, s);
    case 38: return launch_rows<T, 4, 16, 1>(p, s);
    default: break;
  }
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

int dlm_q8_force_tile(int tile) {
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
