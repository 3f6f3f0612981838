// Attention with masks, capped scores and biases of distance, for fp16 and bf16,
// grouped heads, from one query to long prompts.  No counterpart in the reference
// (src/kernels/attention.cuh:53-73 has neither masks nor biases).
//
//   s = scale q.k;  s = cap tanh(s / cap);  s += bias(j - p);  o = softmax(s) v
//
// Every mask here is an interval of keys per query (documents, prefixes, lengths,
// causal order, windows), so whole key tiles are left out, whole ones run without
// mask code, and only those an interval ends in compare keys.
//
// Formulation (wave64, v_mfma_f32_32x32x16): a wave owns 32 rows, a row being a query
// of one of the G heads that share a key head (row = query * G + head), so K and V are
// read once for the group.  Scores are computed transposed, S^T = K Q^T, so that a lane
// owns one row and every other four of its keys; exponentiated they are the B operand of O^T = V^T P^T
// as they stand.  V stays [key][d] in LDS: ds_read_b64_tr_b16 hands a lane four keys of
// its d.  K and V tiles come by DMA, 16-byte chunks of a row swizzled so that both kinds
// of read touch every bank once.
//
// The softmax keeps a base m per row and takes no maximum of a tile: p = 2^((s - m) c + SH), and the
// base moves to a tile's maximum only where the tile's sum of p, needed anyway, passes a limit: that
// of fp16's largest value (SH = 7 then leaves weights down to 2^-21 of the base's normal numbers),
// 2^10 times the base's weight in bf16 (SH = -34), so that the accumulators are rescaled rarely.
#pragma once

#include <cfloat>
#include <climits>

#include "dma.hpp"

namespace dlm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Half;
template <> struct Half<f16> {
  typedef f16x8 x8;
  static constexpr float shift = 7.0f;
  static constexpr float limit = 3.0e6f;  // 32 finite values sum to less
  static constexpr unsigned inf = 0x7c00;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return mfma32x32x16(a, b, c); }
  static __device__ __forceinline__ float dot2(f16x2 p, float c) {
    return __builtin_amdgcn_fdot2(p, f16x2{(f16)1.0f, (f16)1.0f}, c, false);
  }
  typedef f16x2 x2;
};
template <> struct Half<__bf16> {
  typedef bf16x8 x8;
  // The sums of p V stay in fp32's range for every finite V: a lane's keys of a tile, 16 or 32, sum to
  // 2^-24 at most and 2^28 keys to 1; weights down to 2^-92 of the base are normal numbers
  static constexpr float shift = -34.0f;
  static constexpr float limit = 0x1p-24f;
  static constexpr unsigned inf = 0x7f80;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float dot2(bf16x2 p, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
  }
  typedef bf16x2 x2;
};

struct AmParams {
  const char* q;
  const char* k;
  const char* v;
  char* o;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh;  // elements
  const int* key_range;
  long long kr_sb;
  const int* q_pos;
  long long qp_sb;
  const float* slopes;
  const float* table;
  int R;
  int Sq, Sk, Hkv, G, Dh, rows;  // rows = Sq * G
  int causal, nrb, heads, splits;  // row blocks, B * Hkv, parts of the keys
  int parts;                       // workgroups that may share a block's rows
  int lpt;                         // row blocks of all heads by their length
  float c;                         // scale, to powers of two
  float ic, cl;                    // scale / cap; the cap, to powers of two
  float small, ct[5];              // q.k up to which the cap is a polynomial; its coefficients times c
  int table_lds;                   // the table's rows of a key head fit LDS
  float* part;                     // [splits][heads][rows][Dh], then [splits][heads][rows][2]
};

#define AM_WAIT_ALL() __builtin_amdgcn_s_waitcnt(0x70)  // vmcnt(0) lgkmcnt(0)
#define AM_WAIT_LGKM() __builtin_amdgcn_s_waitcnt(0xC07F)

__device__ __forceinline__ float am_max_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float am_sum_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ int am_wave_min(int v) {
  return __builtin_amdgcn_readfirstlane(wave_reduce(v, [](int a, int b) { return a < b ? a : b; }));
}
__device__ __forceinline__ int am_wave_max(int v) {
  return __builtin_amdgcn_readfirstlane(wave_reduce(v, [](int a, int b) { return a > b ? a : b; }));
}

enum { AM_PLAIN, AM_CAP, AM_SLOPE, AM_TABLE, AM_BOTH };  // scores: as they are, capped, with a bias, capped with a bias
constexpr int AM_TABLE_MAX = 1024;   // entries of the tables of one key head kept in LDS,
constexpr int AM_TABLE_MARGIN = 96;  // each with its ends repeated behind both: 64 keys and 32 places beyond
constexpr float AM_LOG2E = 1.4426950408889634f;

// tanh(t) / t in u = t^2 on [0, 1/4]: Chebyshev fit of degree 4, relative error 1.4e-8
constexpr double AM_TANH[5] = {0.9999999870693153, -0.3333307189419686, 0.13324828997687793, -0.052989241174895264,
                               0.017141319047070502};
__device__ __forceinline__ float capped_small(const AmParams& p, float x) {
  const float t = x * p.ic, u = t * t;
  float r = __builtin_fmaf(p.ct[4], u, p.ct[3]);
  r = __builtin_fmaf(r, u, p.ct[2]);
  r = __builtin_fmaf(r, u, p.ct[1]);
  r = __builtin_fmaf(r, u, p.ct[0]);
  return x * r;
}
// ... else tanh(t) = 1 - 2 / (1 + e^2t), whose error, of 1's last bits, would outgrow a small score.
// The form goes by x alone, so that no score depends on another row's or on masked keys.
__device__ __forceinline__ float capped(const AmParams& p, float x) {
  const float e = __builtin_amdgcn_exp2f(x * (p.ic * (2.0f * AM_LOG2E)));
  const float far = __builtin_fmaf(-2.0f * p.cl, __builtin_amdgcn_rcpf(1.0f + e), p.cl);
  return fabsf(x) <= p.small ? capped_small(p, x) : far;
}

// A bias to powers of two; the lowest values stay finite, infinities and NaN what they are.
__device__ __forceinline__ float am_log2(float b) {
  return __builtin_isfinite(b) ? fmaxf(-FLT_MAX, fminf(FLT_MAX, b * AM_LOG2E)) : b;
}

// A slope to powers of two, held where its product with any distance (below 2^31) is finite
__device__ __forceinline__ float am_slope(float x) {
  const float y = x * AM_LOG2E;
  return y != y ? y : fmaxf(-0x1p96f, fminf(0x1p96f, y));
}

// What a wave's rows see: keys from the first to behind the last that one of them sees, the
// keys that all of them see, and their places.
struct KeySpan {
  int tlo, thi, flo, fhi, pmin, pmax;
  __device__ __forceinline__ bool any(int k0, int n) const { return k0 < thi && k0 + n > tlo; }
  __device__ __forceinline__ bool whole(int k0, int n) const { return k0 >= flo && k0 + n <= fhi; }
};

// A row's place and what it sees, in LDS (an array of 64 per field and wave): the loop needs
// little of it and rarely, and registers spilled to memory would be read back behind the copies
// in flight.
struct Row {
  enum { LO, HI, FLAGS, P, HEAD, SUB, SLOPE, LEFT = SLOPE, RIGHT, N };  // SUB: the head among its key head's
  static constexpr int fields(int mode) { return mode == AM_PLAIN || mode == AM_CAP ? P : N; }
  enum { LIVE = 1, EMPTY = 2 };  // a row that is stored; one that sees no key
  int DLM_LDS* at;
  const float DLM_LDS* table;  // the tables of the key head's heads, where they fit
  __device__ __forceinline__ int get(int f) const { return at[f * 64]; }
  __device__ __forceinline__ float num(int f) const { return __int_as_float(at[f * 64]); }
  __device__ __forceinline__ void set(int f, int v) const { at[f * 64] = v; }
};

struct RowInit {
  int i, h;  // query, head
  bool live, empty;
  int lo, hi, p;
};

__device__ __forceinline__ RowInit am_row(const AmParams& p, int b, int hk, int r) {
  RowInit w;
  w.live = r < p.rows;
  const int rc = w.live ? r : p.rows - 1;
  w.i = rc / p.G;
  w.h = hk * p.G + rc - w.i * p.G;
  w.lo = 0;
  w.hi = p.Sk;
  if (p.key_range) {
    const int2 x = *reinterpret_cast<const int2*>(p.key_range + b * p.kr_sb + 2LL * w.i);
    w.lo = max(x.x, 0);
    w.hi = min(x.y, p.Sk);
  }
  w.p = w.i + p.Sk - p.Sq;
  if (p.q_pos) w.p = max(-(1 << 30), min(1 << 30, p.q_pos[b * p.qp_sb + w.i]));
  if (p.causal && w.p < p.Sk) w.hi = min(w.hi, w.p + 1);
  w.empty = w.lo >= w.hi;
  return w;
}

// Rows that see nothing, and those that are not this workgroup's, run along unmasked: what
// they compute is never stored.
__device__ __forceinline__ void am_span(const RowInit& w, KeySpan& s) {
  const bool on = w.live && !w.empty;
  s.tlo = am_wave_min(on ? w.lo : INT_MAX);
  s.thi = am_wave_max(on ? w.hi : 0);
  s.flo = am_wave_max(on ? w.lo : 0);
  s.fhi = am_wave_min(on ? w.hi : INT_MAX);
}

// The table's entry for a row and a key, from memory
__device__ __forceinline__ float am_table(const AmParams& p, const Row& row, int key) {
  const int d = max(-p.R, min(p.R, key - row.get(Row::P)));
  return am_log2(p.table[(long long)row.get(Row::HEAD) * (2 * p.R + 1) + p.R + d]);
}

template <int MODE>
__device__ __forceinline__ void am_keep(const AmParams& p, const RowInit& w, KeySpan& s, const Row& row) {
  const bool on = w.live && !w.empty;
  row.set(Row::LO, on ? w.lo : INT_MIN);
  row.set(Row::HI, on ? w.hi : INT_MAX);
  row.set(Row::FLAGS, (w.live ? Row::LIVE : 0) | (w.empty ? Row::EMPTY : 0));
  if constexpr (Row::fields(MODE) == Row::N) {
    s.pmin = am_wave_min(w.p);
    s.pmax = am_wave_max(w.p);
    row.set(Row::P, w.p);
    row.set(Row::HEAD, w.h);
    row.set(Row::SUB, w.h % p.G);
    if (p.slopes) row.set(Row::SLOPE, __float_as_int(am_slope(p.slopes[w.h])));
    if (p.table) {
      const float* tab = p.table + (long long)w.h * (2 * p.R + 1);
      row.set(Row::LEFT, __float_as_int(am_log2(tab[0])));
      row.set(Row::RIGHT, __float_as_int(am_log2(tab[2 * p.R])));
    }
  }
}

// The tables of a key head go to LDS where they fit, and are looked through for -infinity (others
// count as having some): true where there is one.
template <int MODE>
__device__ __forceinline__ bool am_tables(const AmParams& p, int hk, int tid, int threads, float* lds) {
  bool none = !p.table || p.table_lds;
  if (p.table && p.table_lds) {
    const int n = 2 * p.R + 1, pitch = n + 2 * AM_TABLE_MARGIN;
    const float* tab = p.table + (long long)hk * p.G * n;
    for (int i = tid; i < pitch * p.G; i += threads) {
      const int h = i / pitch, j = i - h * pitch - AM_TABLE_MARGIN;
      const float x = am_log2(tab[h * n + max(0, min(n - 1, j))]);
      none &= x != -INFINITY;
      if (MODE == AM_TABLE) lds[i] = x;
    }
  }
  return !none;
}

// What a wave does with tiles of KB * 32 keys.  PB: bytes of a key's row in LDS, DK:
// steps of 16 dims, DV: blocks of 32 dims; NW: waves that fill a tile together.
template <typename T, int PB, int DK, int DV, int MODE, int KB, int NW>
struct Core {
  using Hf = Half<T>;
  using x8 = typename Hf::x8;
  static constexpr int BK = KB * 32;
  static constexpr int TILE = BK * PB;       // bytes of the K (or V) tile
  static constexpr int RPI = 1024 / PB;      // rows of one DMA instruction
  static constexpr int NI = BK / RPI / NW;   // instructions of a wave and operand
  static constexpr int CH = PB / 16;
  // distinct swizzles among a wave's instructions
  static constexpr int NKV = std::max(1, 16 / (NW * RPI));
  static constexpr int NVV = std::max(1, 4 / (NW * RPI));
  static_assert(NI * RPI * NW == BK && NI % NKV == 0 && NI % NVV == 0, "whole instructions");

  const int lane, g, wave;
  // the next tile of either operand that is copied: its first row, and the keys from it on
  const char* kptr;
  const char* vptr;
  int kleft, vleft, kss, vss, dh;
  unsigned koff[NKV], voff[NVV];
  x8 qf[DK];
  f32x16 o[DV];
  float m, l, mref, lim;  // base, sum, base less shift, the sum that moves it
  bool special = false;  // some tile's V was not finite where a row does not see it

  static __device__ __forceinline__ int kswz(int r) { return PB == 128 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int vswz(int r) { return PB == 128 ? (r & 2) << 1 : (r & 3) << 2; }

  __device__ __forceinline__ Core(const AmParams& p, int lane_, int wave_) : lane(lane_), g(lane_ >> 5), wave(wave_) {
    kss = (int)p.k_ss * 2;
    vss = (int)p.v_ss * 2;
    dh = p.Dh * 2;
    const int r0 = wave * RPI + lane / CH, phys = lane % CH;
#pragma unroll
    for (int i = 0; i < NKV; ++i) {
      const int r = i * NW * RPI + r0, ch = phys ^ kswz(r);
      koff[i] = ch * 16 < dh ? (unsigned)(r * kss + ch * 16) : 0x80000000u;
    }
#pragma unroll
    for (int i = 0; i < NVV; ++i) {
      const int r = i * NW * RPI + r0, ch = phys ^ vswz(r);
      voff[i] = ch * 16 < dh ? (unsigned)(r * vss + ch * 16) : 0x80000000u;
    }
  }

  // The next tile is t; `step` tiles lie between one copy and the next
  __device__ __forceinline__ void start(const AmParams& p, int b, int hk, int t) {
    kptr = p.k + (b * p.k_sb + hk * p.k_sh) * 2 + (long long)t * BK * kss;
    vptr = p.v + (b * p.v_sb + hk * p.v_sh) * 2 + (long long)t * BK * vss;
    kleft = vleft = p.Sk - t * BK;
  }

  __device__ __forceinline__ void load_q(const AmParams& p, const RowInit& row, int b) {
    const T* qp = (const T*)p.q + b * p.q_sb + row.i * p.q_ss + row.h * p.q_sh + g * 8;
#pragma unroll
    for (int ds = 0; ds < DK; ++ds) {
      const bool in = ds * 16 + g * 8 < p.Dh;
      const x8 v = *reinterpret_cast<const x8*>(in ? qp + ds * 16 : qp - g * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[ds][e] = in ? v[e] : (T)0.0f;
    }
#pragma unroll
    for (int dt = 0; dt < DV; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    m = -INFINITY;
    mref = 0.0f;
    l = 0.0f;
    lim = -1.0f;  // no key seen: the first tile's sum moves the base
  }

  // A value that the compiler cannot follow: what is made of it is made where it is used (kept
  // for all of the kernel, addresses take registers that the main loop needs, and come back from memory
  // behind the copies in flight)
  static __device__ __forceinline__ unsigned here(unsigned x) {
    asm volatile("" : "+v"(x));
    return x;
  }

  // Copies the next tile of an operand into LDS: a buffer that starts at the tile's first row, so
  // offsets stay small however long the cache, and ends with the last key's row (what lies
  // past it, and dims past Dh, are zeros).
  __device__ __forceinline__ void issue_k(unsigned char DLM_LDS* st, int step = 1) {
    const i32x4 r = dma_rsrc(kptr, (unsigned)((min(BK, kleft) - 1) * kss + dh));
#pragma unroll
    for (int i = 0; i < NI; ++i)
      dma16(r, st + (i * NW + wave) * 1024, (int)(here(koff[i % NKV]) + (unsigned)(i / NKV * NKV * NW * RPI * kss)), 0);
    kptr += (long long)step * BK * kss;
    kleft -= step * BK;
  }
  __device__ __forceinline__ void issue_v(unsigned char DLM_LDS* st, int step = 1) {
    const i32x4 r = dma_rsrc(vptr, (unsigned)((min(BK, vleft) - 1) * vss + dh));
#pragma unroll
    for (int i = 0; i < NI; ++i)
      dma16(r, st + (i * NW + wave) * 1024, (int)(here(voff[i % NVV]) + (unsigned)(i / NVV * NVV * NW * RPI * vss)), 0);
    vptr += (long long)step * BK * vss;
    vleft -= step * BK;
  }

  __device__ __forceinline__ void scores(const unsigned char DLM_LDS* st, f32x16 (&s)[KB], int lane) const {
    const int base = (lane & 31) * PB + (((lane >> 5) ^ kswz(lane & 31)) * 16);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
#pragma unroll
    for (int ds = 0; ds < DK; ++ds)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const x8 kf = *reinterpret_cast<const x8 DLM_LDS*>(st + (base ^ (32 * ds)) + kb * 32 * PB);
        s[kb] = Hf::mfma(kf, qf[ds], s[kb]);
      }
  }

  // key of element e of block kb, against the tile's first key and without the lane's 4 g
  static constexpr __device__ int key_of(int kb, int e) { return kb * 32 + 8 * (e >> 2) + (e & 3); }

  static __device__ __forceinline__ bool near(const KeySpan& span) {
    return (unsigned)span.pmax - (unsigned)span.pmin < 32;
  }

  // Calls f(z): z(x, kb, e) is the score of element e of block kb in powers of two, made of
  // its q.k x.  (Plain scores stay q.k: their scale goes into the exponent's one operation.)  WHOLE: of a
  // tile that every row sees whole.
  template <bool WHOLE = false, typename F>
  __device__ __forceinline__ void with_scores(const AmParams& p, const KeySpan& span, const Row& row,
                                              const f32x16 (&s)[KB], int k0, int g, F f) const {
    if constexpr (MODE == AM_PLAIN) f([](float x, int, int) { return x; });
    if constexpr (MODE == AM_CAP) {
      // a wave with no score past half the cap leaves the second form out
      float top = 0.0f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(s[kb][e]));
      if (__builtin_amdgcn_ballot_w64(!(top <= p.small)) == 0)
        f([&](float x, int, int) { return capped_small(p, x); });
      else
        f([&](float x, int, int) { return capped(p, x); });
    }
    if constexpr (MODE == AM_SLOPE) {
      // slopes are in powers of two.  A row that has every key of the tile on one side takes the bias as
      // linear in the key, with an operation less; so does a row among others that have not, since the two
      // are rounded apart
      const int first = k0 - row.get(Row::P);
      const float c = p.c, f0 = (float)(first + 4 * g), slope = row.num(Row::SLOPE);
      const bool before = k0 + BK - 1 <= span.pmin;
      if (PB < 512 && (before || k0 >= span.pmax)) {  // (wide heads: one copy of the loop's body, for registers)
        const float d = before ? slope : -slope;
        f([&](float x, int kb, int e) {
          return __builtin_fmaf(x, c, __builtin_fmaf(d, (float)key_of(kb, e), d * f0));
        });
      } else {
        const bool side = first + BK - 1 <= 0 || first >= 0;
        const float d = first < 0 ? slope : -slope;
        f([&](float x, int kb, int e) {
          const float linear = __builtin_fmaf(x, c, __builtin_fmaf(d, (float)key_of(kb, e), d * f0));
          return side ? linear : __builtin_fmaf(-slope, fabsf(f0 + (float)key_of(kb, e)), x * c);
        });
      }
    }
    if constexpr (MODE == AM_TABLE) {
      const float c = p.c;
      if (k0 + BK - 1 - span.pmin <= -p.R || k0 - span.pmax >= p.R) {
        const float t = row.num(k0 - span.pmax >= p.R ? Row::RIGHT : Row::LEFT);
        f([&](float x, int, int) { return __builtin_fmaf(x, c, t); });
      } else if ((WHOLE && PB == 512) || (p.table_lds && near(span))) {
        // (places this near: no distance of the tile passes the margin behind the ends)
        const int d0 = k0 + 4 * g - row.get(Row::P), pitch = 2 * (p.R + AM_TABLE_MARGIN) + 1;
        const float DLM_LDS* tab = row.table + row.get(Row::SUB) * pitch + p.R + AM_TABLE_MARGIN + d0;
        f([&](float x, int kb, int e) { return __builtin_fmaf(x, c, tab[key_of(kb, e)]); });
      } else {
        f([&](float x, int kb, int e) {
          return __builtin_fmaf(x, c, am_table(p, row, k0 + 4 * g + key_of(kb, e)));
        });
      }
    }
    if constexpr (MODE == AM_BOTH) {
      const float f0 = (float)(k0 + 4 * g - row.get(Row::P)), slope = p.slopes ? row.num(Row::SLOPE) : 0.0f;
      if (p.slopes)
        f([&](float x, int kb, int e) {
          return __builtin_fmaf(-slope, fabsf(f0 + (float)key_of(kb, e)), capped(p, x));
        });
      else
        f([&](float x, int kb, int e) {
          return capped(p, x) + am_table(p, row, k0 + 4 * g + key_of(kb, e));
        });
    }
  }

  static __device__ __forceinline__ x8 vfrag(const unsigned char DLM_LDS* st, int j, int dt, int lane) {
    const int r4 = (lane & 15) >> 2;
    const int base = (4 * (lane >> 5) + r4) * PB + vswz(r4) * 16 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    const unsigned char DLM_LDS* a = st + (base ^ (64 * dt)) + 16 * j * PB;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 DLM_LDS*)a);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 DLM_LDS*)(a + 8 * PB));
    return __builtin_bit_cast(x8, i16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }

  // 2^(score - base)
  __device__ __forceinline__ T weight(const AmParams& p, float s) const {
    return (T)__builtin_amdgcn_exp2f(MODE == AM_PLAIN ? __builtin_fmaf(s, p.c, -mref) : s - mref);
  }
  // The sum that moves a base of m: from 2^26 on every sum does, so that `settle` makes the weights again
  static __device__ __forceinline__ float limit_at(float m) {
    if (MODE == AM_PLAIN && !(fabsf(m) < 0x1p26f)) return -1.0f;
    return Hf::shift < 0.0f && !(fabsf(m) < 0x1p30f) ? 0x1p10f : Hf::limit;  // (no shift is left from 2^30 on)
  }
  // ... of a tile, and this lane's sum of them, pairs added in the order of `look_ahead`: which of the
  // two makes a row's sum goes by the other rows of its wave, and must not show in a bit of it
  // ... LARGE: also of plain scores so large that the base's own rounding, which the fused product has
  // not, is whole powers of two.  Those are rounded as the base was (one of `first` and `then` is 1)
  template <bool LARGE = false>
  __device__ __forceinline__ float weights(const AmParams& p, const f32x16 (&s)[KB], x8 (&pf)[2 * KB]) const {
    float sum[2] = {0.0f, 0.0f};
    const float first = lim < 0.0f ? p.c : 1.0f, then = lim < 0.0f ? 1.0f : p.c;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        pf[2 * kb + (e >> 3)][e & 7] = LARGE && MODE == AM_PLAIN
                                           ? (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e] * first, then, -mref))
                                           : weight(p, s[kb][e]);
#pragma unroll
    for (int i = 0; i < 8 * KB; ++i) {
      const int j = i >> 2, e = 2 * (i & 3);
      sum[i & 1] = Hf::dot2(typename Hf::x2{pf[j][e], pf[j][e + 1]}, sum[i & 1]);
    }
    return sum[0] + sum[1];
  }

  // The base from a first tile that is seen whole, ahead of its exponentials
  __device__ __forceinline__ void begin(const AmParams& p, const f32x16 (&s)[KB]) {
    float mt = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[kb][e]);
    m = am_max_halves(mt * p.c);
    if (m != -INFINITY) {
      mref = m - Hf::shift;
      lim = limit_at(m);
    }
  }

  // What this wave's sums are in powers of two of: -infinity before the first key
  __device__ __forceinline__ float unit() const { return m == -INFINITY ? m : mref; }

  // A tile's weights against the row's base, given their sum.  No maximum is taken: the sum, which is
  // needed anyway, tells when some weight came near the end of its type; only then (and at a row's first
  // keys) the base moves to the tile's maximum and the weights are made again.  That a row moves goes
  // by its own values, so its result depends on no other row.
  __device__ __forceinline__ void settle(const AmParams& p, const f32x16 (&s)[KB], x8 (&pf)[2 * KB], float sum) {
    const bool past = !(sum <= lim);
    if (__builtin_amdgcn_ballot_w64(past) != 0) {
      asm volatile("" ::: "memory");  // a real branch
      float mt = s[0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[kb][e]);
      mt = am_max_halves(MODE == AM_PLAIN ? mt * p.c : mt);
      const bool move = am_max_halves(past ? 1.0f : 0.0f) > 0.0f && mt > m;
      // (from one base less shift to the next, not from base to base: near 2^24 and beyond the shift is
      // rounded off them, to more or less)
      const float next = mt - Hf::shift;
      const float alpha = !move ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mref - next);
      m = move ? mt : m;
      lim = move ? limit_at(m) : lim;
      mref = move ? next : mref;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DV; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
      sum = weights<true>(p, s, pf);
    }
    l += sum;
  }

  // The weights of a tile (s: q.k, then scores) while the next tile's sn are made of K at st: step by
  // step of 16 dims two products, a share of the exponentials, and the next step's fragments.  The
  // steps are kept apart, or all fragments would be read ahead, into registers there are not.
  template <typename Z>
  __device__ __forceinline__ float look_ahead(const AmParams& p, const unsigned char DLM_LDS* st, f32x16 (&sn)[KB],
                                              f32x16 (&s)[KB], x8 (&pf)[2 * KB], Z z, int lane) const {
    const int base = (lane & 31) * PB + (((lane >> 5) ^ kswz(lane & 31)) * 16);
    auto frag = [&](int ds, int kb) {
      return *reinterpret_cast<const x8 DLM_LDS*>(st + (base ^ (32 * ds)) + kb * 32 * PB);
    };
    x8 k[2][KB];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      k[0][kb] = frag(0, kb);
#pragma unroll
      for (int e = 0; e < 16; ++e) sn[kb][e] = 0.0f;
    }
#pragma unroll
    for (int ds = 0; ds < DK; ++ds) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        if (ds + 1 < DK) k[(ds + 1) & 1][kb] = frag(ds + 1, kb);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) sn[kb] = Hf::mfma(k[ds & 1][kb], qf[ds], sn[kb]);
#pragma unroll
      for (int i = 8 * KB * ds / DK; i < 8 * KB * (ds + 1) / DK; ++i) {  // pairs of elements
        const int kb = i >> 3, e = 2 * (i & 7);
        typename Hf::x2 w;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[kb][e + u] = z(s[kb][e + u], kb, e + u);
          w[u] = weight(p, s[kb][e + u]);
        }
        pf[2 * kb + (e >> 3)][e & 7] = w[0];
        pf[2 * kb + (e >> 3)][(e & 7) + 1] = w[1];
        sum[i & 1] = Hf::dot2(w, sum[i & 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return sum[0] + sum[1];
  }

  // O^T += V^T P^T
  __device__ __forceinline__ void pv(const unsigned char DLM_LDS* st, const x8 (&pf)[2 * KB], int lane) {
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
      for (int dt = 0; dt < DV; ++dt) o[dt] = Hf::mfma(vfrag(st, j, dt, lane), pf[j], o[dt]);
  }

  // The same of a tile whose V holds infinities or NaN, where 0 * V would spoil rows that
  // do not see them: the finite values alone.
  __device__ __forceinline__ void pv_finite(const unsigned char DLM_LDS* st, const x8 (&pf)[2 * KB], int lane) {
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
      for (int dt = 0; dt < DV; ++dt) {
        u16x8 v = __builtin_bit_cast(u16x8, vfrag(st, j, dt, lane));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (v[e] & Hf::inf) == Hf::inf ? 0 : v[e];
        o[dt] = Hf::mfma(__builtin_bit_cast(x8, v), pf[j], o[dt]);
        __builtin_amdgcn_sched_barrier(0);
      }
  }

  // ... and behind the loop over tiles (first, first + step, ... below last) the others, read from
  // memory again: a second product counts those that a row sees, 1 for infinity, 128 for
  // -infinity, both for NaN (whole numbers up to 64 * 129, exact in either type and in the sums).
  __device__ __forceinline__ void add_special(const AmParams& p, const KeySpan& span, const Row& row, int b, int hk,
                                              int first, int last, int step) {
    const T* v = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    const int lo = row.get(Row::LO), hi = row.get(Row::HI);
    for (int t = first; t < last; t += step) {
      const int k0 = t * BK;
      if (!span.any(k0, BK) || (span.whole(k0, BK) && !p.table)) continue;
#pragma unroll
      for (int dt = 0; dt < DV; ++dt) {
        const int d = dt * 32 + (lane & 31);
        f32x16 n;
#pragma unroll
        for (int e = 0; e < 16; ++e) n[e] = 0.0f;
#pragma unroll 1
        for (int j = 0; j < 2 * KB; ++j) {
          x8 kind, one;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = k0 + 16 * j + 4 * g + (e & 3) + 8 * (e >> 2);
            unsigned short x = 0;
            if (key < p.Sk && d < p.Dh) x = __builtin_bit_cast(unsigned short, v[key * p.v_ss + d]);
            const bool odd = (x & Hf::inf) == Hf::inf, nan = (x & 0x7fff) != Hf::inf;
            bool sees = key >= lo && key < hi;
            if (MODE >= AM_TABLE && p.table) sees = sees && am_table(p, row, key) != -INFINITY;
            kind[e] = (T)(!odd ? 0.0f : nan ? 129.0f : x & 0x8000 ? 128.0f : 1.0f);
            one[e] = (T)(sees ? 1.0f : 0.0f);
          }
          n = Hf::mfma(kind, one, n);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int count = (int)n[e];
          const float all = o[dt][e] + (count & 127 ? INFINITY : 0.0f) - (count >> 7 ? INFINITY : 0.0f);
          o[dt][e] = count ? all : o[dt][e];  // (without branches, of which 128 and more kept their masks)
        }
      }
    }
  }

  // Softmax and product of tile t, whose scores are in s and whose V is in LDS at st; any mask
  __device__ __forceinline__ void finish(const AmParams& p, const KeySpan& span, const Row& row, f32x16 (&s)[KB],
                                         const unsigned char DLM_LDS* st, int t) {
    const int k0 = t * BK, lane = (int)here(this->lane), g = lane >> 5;
    // (a cap takes even -infinity, which masks a key below, to a number)
    if constexpr (MODE != AM_PLAIN)
      with_scores(p, span, row, s, k0, g, [&](auto z) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = z(s[kb][e], kb, e);
      });
    bool guard = false;
    if (!span.whole(k0, BK)) {
      guard = true;
      // in 32 bits whatever the bounds: lo and hi against the tile's first key
      if (k0 < span.flo) {
        const int lo = max(row.get(Row::LO), k0) - k0 - 4 * g;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = key_of(kb, e) < lo ? -INFINITY : s[kb][e];
      }
      if (k0 + BK > span.fhi) {
        const int hi = min(row.get(Row::HI), k0 + BK) - k0 - 4 * g;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = key_of(kb, e) >= hi ? -INFINITY : s[kb][e];
      }
    }
    if constexpr (MODE >= AM_TABLE) {
      if (p.table) {  // an entry of -infinity masks its distance
        float low = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) low = __builtin_elementwise_minimum(low, s[kb][e]);
        guard |= __builtin_amdgcn_ballot_w64(!(low > -INFINITY)) != 0;
        // ... whatever its key holds: added to infinity or NaN it gave NaN
        if (__builtin_amdgcn_ballot_w64(low != low) != 0) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (s[kb][e] != s[kb][e] && am_table(p, row, k0 + 4 * g + key_of(kb, e)) == -INFINITY) s[kb][e] = -INFINITY;
        }
      }
    }
    x8 pf[2 * KB];
    bool finite = true;
    if (guard) {
      // V times zeros: NaN where V is not finite (the matrix pipe has room here, the vector pipe
      // has not)
      f32x16 n;
      x8 zero;
#pragma unroll
      for (int e = 0; e < 16; ++e) n[e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) zero[e] = (T)0.0f;
#pragma unroll
      for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
        for (int dt = 0; dt < DV; ++dt) n = Hf::mfma(vfrag(st, j, dt, lane), zero, n);
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) sum += n[e];
      finite = __builtin_amdgcn_ballot_w64(sum != 0.0f) == 0;
    }
    settle(p, s, pf, weights(p, s, pf));
    if (finite) {
      pv(st, pf, lane);
    } else {
      special = true;
      pv_finite(st, pf, lane);
    }
  }
};

// d of element e of output block dt, without the lane's 4 g
__device__ __forceinline__ int am_dim(int dt, int e4) { return dt * 32 + 8 * e4; }

__device__ __forceinline__ float* am_part_o(const AmParams& p, int split, int head, int r) {
  return p.part + (((long long)split * p.heads + head) * p.rows + r) * p.Dh;
}
__device__ __forceinline__ float* am_part_ml(const AmParams& p, int split, int head, int r) {
  return p.part + (long long)p.splits * p.heads * p.rows * p.Dh +
         (((long long)split * p.heads + head) * p.rows + r) * 2;
}

template <typename T>
__device__ __forceinline__ void am_store4(const AmParams& p, int b, int i, int h, int d, float x0, float x1, float x2,
                                          float x3) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<t4*>((T*)p.o + b * p.o_sb + i * p.o_ss + h * p.o_sh + d) = t4{(T)x0, (T)x1, (T)x2, (T)x3};
}

// Tiles of part `split` of the keys [lo, hi).
__device__ __forceinline__ void am_tiles(int lo, int hi, int bk, int splits, int split, int& t0, int& t1) {
  if (lo >= hi) {
    t0 = t1 = 0;
    return;
  }
  const int a = lo / bk, b = (hi - 1) / bk + 1;
  const int per = (b - a + splits - 1) / splits;
  t0 = min(b, a + split * per);
  t1 = min(b, t0 + per);
}

// The order in which an XCD's n blocks, from `first` on in the order of heads and, in each, of row blocks
// from the last to the first, are started where masks make the last row blocks the longest: by row
// block, those of all heads next to one another, and in rounds of one for each of its 32 CUs, the second
// round from the shortest up, so that a CU's first two take about as long as any other's.
__device__ __forceinline__ int am_by_weight(int slot, int first, int n, int nrb) {
  if (slot >= 32 && slot < 64) slot = 32 + min(32, n - 32) - 1 - (slot - 32);
  // positions c in a head's order: the first head lacks those below a, the last one those from z on
  const int a = first % nrb, z = (first + n - 1) % nrb + 1, heads = (a + n + nrb - 1) / nrb;
  const int lo = min(a, z), hi = max(a, z);
  const int m1 = heads - (a > 0), m2 = a < z ? heads : heads - 2, m3 = heads - 1;
  // of n blocks: lo positions of m1 heads each, hi - lo of m2, the rest of m3 (a head that lacks
  // nothing counts as complete: a = 0, or z = nrb)
  int c, k;
  if (slot < lo * m1) {
    c = slot / m1;
    k = slot - c * m1;
  } else if (slot < lo * m1 + (hi - lo) * m2) {
    const int s = slot - lo * m1;
    c = s / m2;
    k = s - c * m2;
    c += lo;
  } else {
    const int s = slot - lo * m1 - (hi - lo) * m2;
    c = s / m3;
    k = s - c * m3;
    c += hi;
  }
  return (k + (c < a)) * nrb + c - a;
}

// ---------------------------------------------------------------------------
// Many rows: 4 waves of 32 rows share tiles of 64 keys.  The scores of tile t + 1 are
// issued ahead of tile t's softmax, so a wave's matrix and vector instructions overlap;
// K therefore runs a tile ahead of V, and two buffers of each suffice: the barrier that
// shows K of t + 1 and V of t to all also proves K of t and V of t - 1 read.  (A third buffer of
// each changed nothing: 2x4096x10x64 130 us either way.)
// ---------------------------------------------------------------------------
template <typename T, int PB, int DK, int DV, int MODE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PB == 512 ? 1 : PB == 128 && MODE == AM_PLAIN ? 3 : 2)))
attn_masked_kernel(AmParams p) {
  using C = Core<T, PB, DK, DV, MODE, 2, 4>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem_g[4 * C::TILE];
  __shared__ int shared[32];
  __shared__ int rows[4 * Row::fields(MODE) * 64];
  __shared__ float table[MODE == AM_TABLE ? AM_TABLE_MAX : 1];
  unsigned char DLM_LDS* smem = (unsigned char DLM_LDS*)smem_g;
  // consecutive blocks (the row blocks of one key head, then the next head) on one XCD,
  // whose L2 then holds the K and V of its own heads; the last row blocks, which see the most
  // keys where the mask is causal, first
  int split, head, rb, part;
  {
    const int total = p.nrb * p.heads * p.splits;
    int at = blockIdx.x;
    part = 0;
    if (p.parts > 1) {  // the second parts, most of which have nothing to do, start first
      part = at < total;
      at -= part ? 0 : total;
    }
    const int q8 = total >> 3, r8 = total & 7;
    const int x = at & 7, slot = at >> 3;
    const int first = x * q8 + (x < r8 ? x : r8), n = q8 + (x < r8);
    const int logical = first + (p.lpt ? am_by_weight(slot, first, n, p.nrb) : slot);
    const int u = logical / p.splits;
    split = logical - u * p.splits;
    head = u / p.nrb;
    rb = p.nrb - 1 - (u - head * p.nrb);
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = rb * 128 + wave * 32 + (lane & 31);
  const Row row{(int DLM_LDS*)rows + wave * Row::fields(MODE) * 64 + lane, (const float DLM_LDS*)table};
  KeySpan span{};
  int hidden = 0;
  C c(p, lane, wave);
  RowInit init;
  {
    const int b = head / p.Hkv, hk = head - b * p.Hkv;
    init = am_row(p, b, hk, r);
    c.load_q(p, init, b);
    if constexpr (MODE >= AM_TABLE) hidden = __syncthreads_or(am_tables<MODE>(p, hk, tid, 256, table));
  }
  // Tiles [t0, t1) hold the block's keys; [f0, f1) of them, an even number, are seen whole by
  // every row
  int t0, t1, f0, f1;
  {
    auto least = [](int x, int y) { return x < y ? x : y; };
    auto most = [](int x, int y) { return x > y ? x : y; };
    auto share = [&](int longest) {
      am_span(init, span);
      if (lane == 0) {
        int DLM_LDS* s = (int DLM_LDS*)shared + 8 * wave;
        s[0] = span.tlo;
        s[1] = span.thi;
        s[2] = span.flo;
        s[3] = span.fhi;
        s[4] = longest;
      }
      AM_WAIT_LGKM();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    auto all = [&](int i, auto op) {
      return __builtin_amdgcn_readfirstlane(op(op(shared[i], shared[8 + i]), op(shared[16 + i], shared[24 + i])));
    };
    share(p.parts > 1 ? am_wave_max(init.live && !init.empty ? init.hi - init.lo : 0) : 0);
    if (p.parts > 1) {
      // Rows of two documents see the keys of both between them: then one workgroup takes the
      // rows that see the first half of those keys and a second one the others (documents of 2112 and
      // 1984 tokens, x10x64: 104 -> 66 us).  Where the rows see much the same (less than four tiles and
      // an eighth more than one of them) the second one has nothing to do.
      const int lo = all(0, least), hi = all(1, most), longest = all(4, most);
      const bool apart = hi - lo - longest >= max(4 * C::BK, longest / 8);
      if (part == 1 && !apart) return;
      if (apart) {
        const bool second = !init.empty && (init.lo >> 1) + (init.hi >> 1) >= (lo >> 1) + (hi >> 1);
        init.live = init.live && second == (part == 1);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        share(0);
      }
    }
    am_keep<MODE>(p, init, span, row);
    am_tiles(all(0, least), all(1, most), C::BK, p.splits, split, t0, t1);
    const int flo = all(2, most), fhi = all(3, least);
    f0 = max(t0, (flo + C::BK - 1) / C::BK);
    f1 = min(t1, fhi / C::BK);
    f1 -= (f1 - f0) & 1;
    // (wide heads have no registers for a third form of the bias in that loop; f1 may differ among the waves,
    // which meet once a tile either way)
    if (hidden || (PB == 512 && MODE == AM_TABLE && !C::near(span))) f1 = f0;
  }
  if (t0 < t1) {
    unsigned char DLM_LDS* const vmem = smem + 2 * C::TILE;
    // K of t + 1 and V of t have arrived (this wave's part, then everyone's), and all are done with K
    // of t and V of t - 1
    auto arrive = [&] {
      AM_WAIT_ALL();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    // ... whose places the next copies take (tile t is in the buffers `par`)
    auto copy = [&](int t, int par) {
      if (t + 2 < t1) c.issue_k(smem + par * C::TILE);
      if (t + 1 < t1) c.issue_v(vmem + (par ^ 1) * C::TILE);
    };
    {
      const int b = head / p.Hkv;
      c.start(p, b, head - b * p.Hkv, t0);
    }
    f32x16 sa[2], sb[2];
    // tile t is in the buffers of t - f0's parity, so that the loop over whole tiles knows its own
    const int even = f0 & 1;
    c.issue_k(smem + ((t0 ^ even) & 1) * C::TILE);
    c.issue_v(vmem + ((t0 ^ even) & 1) * C::TILE);
    if (t0 + 1 < t1) c.issue_k(smem + ((t0 ^ even ^ 1) & 1) * C::TILE);
    arrive();
    c.scores(smem + ((t0 ^ even) & 1) * C::TILE, sa, (int)C::here(lane));
    if (MODE == AM_PLAIN && t0 == f0 && f0 < f1) c.begin(p, sa);
    // a tile that every row sees whole, its scores in sc; the next tile's go to sn (behind the
    // last tile they are made of whatever the buffer holds and not used)
    auto whole = [&](int t, int par, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
      arrive();
      copy(t, par);
      typename C::x8 pf[4];
      float sum = 0.0f;
      c.template with_scores<true>(p, span, row, sc, t * C::BK, c.g, [&](auto z) {
        sum = c.look_ahead(p, smem + (par ^ 1) * C::TILE, sn, sc, pf, z, lane);
      });
      c.settle(p, sc, pf, sum);
      c.pv(vmem + par * C::TILE, pf, lane);
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
      for (int i = 0; i < 4 * DV; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    int t = t0;
    while (t < t1) {
      if (t == f0) {
        for (; t < f1; t += 2) {
          whole(t, 0, sa, sb);
          whole(t + 1, 1, sb, sa);
        }
        f0 = -1;
        if (t >= t1) break;
      }
      // a tile that some row does not see, or not whole: its scores are not needed any more when the next
      // tile's are made, which leaves registers for the masks
      const int par = (t ^ even) & 1;
      arrive();
      copy(t, par);
      const int k0 = t * C::BK;
      if (span.any(k0, C::BK)) c.finish(p, span, row, sa, vmem + par * C::TILE, t);
      if (span.any(k0 + C::BK, C::BK)) c.scores(smem + (par ^ 1) * C::TILE, sa, (int)C::here(lane));
      __builtin_amdgcn_sched_barrier(0);
      ++t;
    }
    if (c.special) {
      const int b = head / p.Hkv;
      c.add_special(p, span, row, b, head - b * p.Hkv, t0, t1, 1);
    }
  }
  const float l = am_sum_halves(c.l);
  const int flags = row.get(Row::FLAGS);
  const bool empty = flags & Row::EMPTY;
  if (!(flags & Row::LIVE)) return;
  // the arguments are read again here rather than kept in scalar registers through the loop
  const AmParams __attribute__((address_space(4)))* q =
      (const AmParams __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(q));
  const int Dh = q->Dh;
  if (q->splits > 1) {
    const long long at = ((long long)split * q->heads + head) * q->rows + r;
    float* po = q->part + at * Dh;
#pragma unroll
    for (int dt = 0; dt < DV; ++dt)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int d = am_dim(dt, e4) + 4 * c.g;
        if (d < Dh)
          *reinterpret_cast<f32x4*>(po + d) =
              f32x4{c.o[dt][4 * e4], c.o[dt][4 * e4 + 1], c.o[dt][4 * e4 + 2], c.o[dt][4 * e4 + 3]};
      }
    if (c.g == 0) {
      float* ml = q->part + (long long)q->splits * q->heads * q->rows * Dh + at * 2;
      ml[0] = empty ? -INFINITY : c.unit();
      ml[1] = empty ? 0.0f : l;
    }
    return;
  }
  const bool none = empty || l == 0.0f;
  const float inv = 1.0f / l;
  const int query = r / q->G, sub = r - query * q->G;
  typedef T t4 __attribute__((ext_vector_type(4)));
  const int batch = head / q->Hkv;
  T* po = (T*)q->o + batch * q->o_sb + query * q->o_ss + ((head - batch * q->Hkv) * q->G + sub) * q->o_sh;
#pragma unroll
  for (int dt = 0; dt < DV; ++dt)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int d = am_dim(dt, e4) + 4 * c.g;
      t4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (T)(none ? 0.0f : c.o[dt][4 * e4 + e] * inv);
      if (d < Dh) *reinterpret_cast<t4*>(po + d) = x;
    }
}

// ---------------------------------------------------------------------------
// Few rows: every wave of a workgroup holds the same 32 rows and takes every NW-th tile of
// 32 keys through a ring of its own, without barriers; the waves' parts meet in LDS.  Bound
// by K and V from memory, two tiles a wave in flight.
// ---------------------------------------------------------------------------
template <typename T, int PB, int DK, int DV, int MODE>
__global__ void __launch_bounds__(PB == 512 ? 128 : 256) __attribute__((amdgpu_waves_per_eu(1)))
attn_masked_rows_kernel(AmParams p) {
  constexpr int NW = PB == 512 ? 2 : 4;
  using C = Core<T, PB, DK, DV, MODE, 1, 1>;
  constexpr int STAGE = 2 * C::TILE, RING = 2 * STAGE;
  constexpr int D = DV * 32;
  static_assert(NW * 32 * D * 4 <= NW * RING, "the waves' parts fit the rings");
  __shared__ __attribute__((aligned(1024))) unsigned char smem_g[NW * RING];
  __shared__ float ml[NW][32][2];
  const int rb = blockIdx.x, head = blockIdx.y, split = blockIdx.z;
  const int b = head / p.Hkv, hk = head - b * p.Hkv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned char DLM_LDS* smem = (unsigned char DLM_LDS*)smem_g + wave * RING;
  __shared__ int rows[NW * Row::fields(MODE) * 64];
  __shared__ float table[MODE == AM_TABLE ? AM_TABLE_MAX : 1];
  const Row row{(int DLM_LDS*)rows + wave * Row::fields(MODE) * 64 + lane, (const float DLM_LDS*)table};
  if constexpr (MODE == AM_TABLE) {
    am_tables<MODE>(p, hk, tid, NW * 64, table);
    __syncthreads();
  }
  const RowInit init = am_row(p, b, hk, rb * 32 + (lane & 31));
  KeySpan span{};
  am_span(init, span);
  C c(p, lane, 0);
  int t0, t1;
  am_tiles(span.tlo, span.thi, C::BK, p.splits, split, t0, t1);
  int t = t0 + wave;
  c.start(p, b, hk, t);
  auto issue = [&](unsigned char DLM_LDS* st) {
    c.issue_k(st, NW);
    c.issue_v(st + C::TILE, NW);
  };
  if (t < t1) issue(smem);
  if (t + NW < t1) issue(smem + STAGE);
  c.load_q(p, init, b);
  am_keep<MODE>(p, init, span, row);
  int buf = 0;
  for (; t < t1; t += NW) {
    if (t + NW < t1) {
      DLM_WAIT_VM(2 * C::NI);  // the next tile's requests may be in flight
    } else {
      DLM_WAIT_VM(0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    f32x16 s[1];
    c.scores(smem + buf * STAGE, s, lane);
    c.finish(p, span, row, s, smem + buf * STAGE + C::TILE, t);
    __builtin_amdgcn_sched_barrier(0);
    AM_WAIT_LGKM();  // this tile's fragments are read
    asm volatile("" ::: "memory");
    if (t + 2 * NW < t1) issue(smem + buf * STAGE);
    buf ^= 1;
  }
  if (c.special) c.add_special(p, span, row, b, hk, t0 + wave, t1, NW);
  const float l = am_sum_halves(c.l);
  if (lane < 32) {
    ml[wave][lane][0] = c.unit();
    ml[wave][lane][1] = l;
  }
  __syncthreads();
  // this wave's sums in the largest unit, then all waves' together
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w][lane & 31][0]);
  auto weight = [&](float m) { return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top); };
#pragma unroll
  for (int w = 0; w < NW; ++w) sum += ml[w][lane & 31][1] * weight(ml[w][lane & 31][0]);
  const float mine = weight(c.unit());
  float DLM_LDS* part = (float DLM_LDS*)smem_g;  // [wave][d][row]
#pragma unroll
  for (int dt = 0; dt < DV; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      part[(wave * D + am_dim(dt, e >> 2) + 4 * c.g + (e & 3)) * 32 + (lane & 31)] =
          c.m == -INFINITY ? 0.0f : c.o[dt][e] * mine;
  __syncthreads();
  if (!init.live) return;
  const int r = rb * 32 + (lane & 31);
  const bool none = init.empty || sum == 0.0f;
  const float inv = 1.0f / sum;
  for (int d = (tid >> 5) * 4; d < p.Dh; d += NW * 8) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) a += part[(w * D + d + e) * 32 + (lane & 31)];
      x[e] = a;
    }
    if (p.splits > 1) {
      *reinterpret_cast<f32x4*>(am_part_o(p, split, head, r) + d) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = none ? 0.0f : x[e] * inv;
      am_store4<T>(p, b, init.i, init.h, d, x[0], x[1], x[2], x[3]);
    }
  }
  if (p.splits > 1 && tid < 32) {
    float* q = am_part_ml(p, split, head, r);
    q[0] = init.empty ? -INFINITY : top;
    q[1] = init.empty ? 0.0f : sum;
  }
}

// Joins the parts of a row, a wave each.  A lane knows the weight of one part; groups of
// DL lanes (four dims a lane) take every 64 / DL-th part, eight requested at a time (one after the other
// they took half a microsecond each).
template <typename T, int DL>
__global__ void __launch_bounds__(256) attn_masked_join_kernel(AmParams p) {
  constexpr int NG = 64 / DL;
  const int lane = threadIdx.x & 63, group = lane / DL, d = (lane % DL) * 4;
  const long long hr = blockIdx.x * 4LL + (threadIdx.x >> 6);
  if (hr >= (long long)p.heads * p.rows) return;
  const long long step = (long long)p.heads * p.rows;  // rows between one part and the next
  const float* po = p.part + hr * p.Dh + d;
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (lane < p.splits) ml = *reinterpret_cast<const float2*>(p.part + (p.splits * step) * p.Dh + (lane * step + hr) * 2);
  const float top = wave_max(ml.x);
  const bool saw = !(ml.x == -INFINITY && ml.y == 0.0f);
  const float w = saw ? __builtin_amdgcn_exp2f(ml.x - top) : 0.0f;
  const float sum = wave_sum(saw ? ml.y * w : 0.0f);
  f32x4 a{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < p.splits; s0 += 8 * NG) {
    f32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + i * NG + group;
      x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (s < p.splits && d < p.Dh) x[i] = *reinterpret_cast<const f32x4*>(po + s * step * p.Dh);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + i * NG + group;
      const float ws = __shfl(w, min(s, 63), 64);
      const bool on = __shfl((int)saw, min(s, 63), 64) != 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = on ? __builtin_fmaf(x[i][e], ws, a[e]) : a[e];
    }
  }
#pragma unroll
  for (int o = DL; o < 64; o *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += __shfl_xor(a[e], o, 64);
  const float inv = 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = sum == 0.0f ? 0.0f : a[e] * inv;
  const int head = (int)(hr / p.rows), r = (int)(hr - (long long)head * p.rows);
  const int b = head / p.Hkv, hk = head - b * p.Hkv, i = r / p.G;
  if (group == 0 && d < p.Dh) am_store4<T>(p, b, i, hk * p.G + r - i * p.G, d, a[0], a[1], a[2], a[3]);
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// Which kernel, and over how many parts of the keys: by the sizes alone, since what the
// masks leave is known on the device only.
struct AmPlan {
  bool few;
  int nrb, splits;
};
template <typename T, int PB, int DK, int DV, int MODE>
static int am_launch(const AmParams& p, const AmPlan& pl, hipStream_t s) {
  if (pl.few)
    DLM_LAUNCH("attn_masked_rows_kernel", (attn_masked_rows_kernel<T, PB, DK, DV, MODE>),
               dim3(pl.nrb, p.heads, pl.splits), dim3(PB == 512 ? 128 : 256), 0, s, p);
  else
    DLM_LAUNCH("attn_masked_kernel", (attn_masked_kernel<T, PB, DK, DV, MODE>), dim3(pl.nrb * p.heads * pl.splits * p.parts),
               dim3(256), 0, s, p);
  DLM_LAUNCH_CHECK();
  if (pl.splits > 1) {
    const dim3 grid((unsigned)(((long long)p.heads * p.rows + 3) / 4));
    auto join = [&](auto kernel) { DLM_LAUNCH("attn_masked_join_kernel", kernel, grid, dim3(256), 0, s, p); };
    p.Dh <= 64 ? join(attn_masked_join_kernel<T, 16>)
               : p.Dh <= 128 ? join(attn_masked_join_kernel<T, 32>) : join(attn_masked_join_kernel<T, 64>);
    DLM_LAUNCH_CHECK();
  }
  return DLM_OK;
}

template <typename T, int MODE>
static int am_by_head(const AmParams& p, const AmPlan& pl, hipStream_t s) {
  if (p.Dh <= 64) return am_launch<T, 128, 4, 2, MODE>(p, pl, s);
  if (p.Dh <= 96) return am_launch<T, 256, 6, 3, MODE>(p, pl, s);
  if (p.Dh <= 128) return am_launch<T, 256, 8, 4, MODE>(p, pl, s);
  // (These fill all 512 registers.  Accumulators that are spilled to AGPRs in part and to scratch memory in part
  // come back incomplete, by the assembly; so none of these kernels may use scratch memory.)
  return am_launch<T, 512, 16, 8, MODE>(p, pl, s);
}

template <typename T>
static int am_run(const AmParams& p, const AmPlan& pl, bool cap, hipStream_t s) {
  const bool bias = p.slopes || p.table;
  if (cap && bias) return am_by_head<T, AM_BOTH>(p, pl, s);
  if (cap) return am_by_head<T, AM_CAP>(p, pl, s);
  if (p.slopes) return am_by_head<T, AM_SLOPE>(p, pl, s);
  if (p.table) return am_by_head<T, AM_TABLE>(p, pl, s);
  return am_by_head<T, AM_PLAIN>(p, pl, s);
}

int am_run_f16(const AmParams& p, const AmPlan& pl, bool cap, hipStream_t s);
int am_run_bf16(const AmParams& p, const AmPlan& pl, bool cap, hipStream_t s);

}  // namespace dlm
