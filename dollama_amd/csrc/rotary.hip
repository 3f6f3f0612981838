// Rotary positions with several axes, and the RMS norm of every query and key
// head in the same pass.  No counterpart in the reference, whose transformer has
// neither (src/infer/unet.cu:677-802).
//
//   n = x / sqrt(mean(x^2) + eps) * gamma          over a head's Dh values
//   (y1, y2) = (n1 cos a - n2 sin a, n2 cos a + n1 sin a),  a = pos[axis(i)] * freq[i]
//
// for the P pairs i of a head, elements (i, i + P) or (2i, 2i + 1); what lies past
// 2P stays as it is.  Everything is fp32 between the load and one rounding at the
// store, but for the angle: its turns pos * freq / 2 pi are an fp64 product, of
// which only the fraction matters (in fp32 a position of 10^6 would leave errors of
// 0.06 rad).  v_sin_f32 and v_cos_f32 take turns.
#include <cfloat>

#include "common.hpp"
#include "views.hpp"

namespace dlm {

struct RotaryParams {
  const char* x[2];   // queries, keys
  char* y[2];
  const char* gamma[2];
  long long xb[2], xs[2], xh[2];  // strides in elements: batch, token, head
  long long yb[2], ys[2], yh[2];
  int heads[2], blocks[2], hpg[2];  // heads, and blocks of `hpg` heads along the grid's y
  const void* pos;
  long long pb, ps;
  int pos_type, axes;
  int ends[4];                    // pairs up to and with each axis
  const double* freqs;
  int P, Dh, norm;
  int tokens, S;
  float eps, inv_dh;
};

// The sum over a group of W consecutive lanes (W a power of two), the same bits in
// each of them.
template <int W>
__device__ __forceinline__ float group_sum(float v) {
  auto dpp = [&](auto c) { v += __uint_as_float(dpp_u32<decltype(c)::value>(__float_as_uint(v))); };
  if constexpr (W >= 2) dpp(std::integral_constant<int, kDppXor1>{});
  if constexpr (W >= 4) dpp(std::integral_constant<int, kDppXor2>{});
  if constexpr (W >= 8) dpp(std::integral_constant<int, kDppHalfMirror>{});
  if constexpr (W >= 16) dpp(std::integral_constant<int, kDppMirror>{});
  if constexpr (W >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  if constexpr (W >= 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return v;
}

// A group of W lanes takes one token and some heads of it: the angles are computed once for
// all of them.  Groups side by side take tokens side by side (heads side by side, which makes a wave's
// accesses longer, took 41 instead of 31 us for 8192x(32+8)x128 in place).  A lane holds two vectors of V elements of a head (C chunks
// of them where a head has more lanes than a wave):
//   halves:      V pairs (i, i + P) as V elements at i and V at P + i; behind 2P, any two vectors
//   interleaved: V at i and V at Dh / 2 + i, V / 2 pairs in each (V = 1: elements 2i
//                and 2i + 1)
// Memory bounds it: U heads are requested at a time, the first ones ahead of the angles.  A few heads
// of a few tokens (U = 1) are bound by the instructions' way to the CUs instead: 32 heads of one token 5.2 us with
// the code for four heads at a time, the norm's among it, 3.3 us without.
template <typename T, int V, int W, int C, bool IL, bool NORM, int U>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4)))
rotary_kernel(RotaryParams p) {
  typedef T TV __attribute__((ext_vector_type(V)));
  const int lane = threadIdx.x & (W - 1);
  const int token = (int)blockIdx.x * (256 / W) + threadIdx.x / W;
  const bool live = token < p.tokens;
  const unsigned tok = live ? token : p.tokens - 1;  // dead groups follow along: the sums need whole waves
  const int kv = (int)blockIdx.y >= p.blocks[0];
  const int h0 = ((int)blockIdx.y - (kv ? p.blocks[0] : 0)) * p.hpg[kv];
  const int h1 = min(p.heads[kv], h0 + p.hpg[kv]);
  const unsigned b = tok / (unsigned)p.S, s = tok - b * (unsigned)p.S;

  // where this lane's two vectors start, and whether they are in the head
  int at[C][2];
  bool in[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (c * W + lane) * V;
    in[c] = 2 * i < p.Dh;
    at[c][0] = IL ? (V == 1 ? 2 * i : i) : i < p.P ? i : 2 * i;
    at[c][1] = IL ? (V == 1 ? 2 * i + 1 : p.Dh / 2 + i) : i < p.P ? p.P + i : 2 * i + V;
  }
  const T* src = (const T*)p.x[kv] + (long long)b * p.xb[kv] + (long long)s * p.xs[kv];
  T* dst = (T*)p.y[kv] + (long long)b * p.yb[kv] + (long long)s * p.ys[kv];
  TV r[U][C][2];
  auto request = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          r[u][c][w] = TV{};
          if (in[c] && h + u < h1)
            r[u][c][w] = *reinterpret_cast<const TV*>(src + (h + u) * p.xh[kv] + at[c][w]);
        }
  };
  int h = h0;
  request(h);

  // the token's places, the pairs' angles, gamma
  double place[4] = {0.0, 0.0, 0.0, 0.0};
  if (p.P > 0) {
    const long long at0 = (long long)b * p.pb + (long long)s * p.ps;
    auto places = [&](auto* q) {
#pragma unroll
      for (int a = 0; a < 4; ++a)
        if (a < p.axes) place[a] = (double)q[at0 + a];
    };
    if (p.pos_type == DLM_POS_I32)
      places((const int*)p.pos);
    else if (p.pos_type == DLM_POS_I64)
      places((const long long*)p.pos);
    else
      places((const float*)p.pos);
  }
  float cs[C][V], sn[C][V];
  float gam[C][2][V];
  unsigned plain[C];  // pairs that stay as they are
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = (c * W + lane) * V;
    plain[c] = (1u << V) - 1;
    if (p.P > 0) {
      plain[c] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int pair = IL && V > 1 ? (e < V / 2 ? i / 2 + e : p.Dh / 4 + i / 2 + (e - V / 2)) : i + e;
        const bool turns = pair < p.P;
        double x = place[0];
#pragma unroll
        for (int a = 0; a < 3; ++a) x = pair >= p.ends[a] ? place[a + 1] : x;
        x *= p.freqs[turns ? pair : 0] * 0.15915494309189533577;
        const float f = (float)(x - __builtin_floor(x));
        cs[c][e] = __builtin_amdgcn_cosf(f);
        sn[c][e] = __builtin_amdgcn_sinf(f);
        plain[c] |= turns ? 0 : 1u << e;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        cs[c][e] = 1.0f;
        sn[c][e] = 0.0f;
      }
    }
    if constexpr (NORM) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        TV g;
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = (T)1.0f;
        if (in[c] && p.gamma[kv]) g = *reinterpret_cast<const TV*>((const T*)p.gamma[kv] + at[c][w]);
#pragma unroll
        for (int e = 0; e < V; ++e) gam[c][w][e] = (float)g[e];
      }
    }
  }

  for (;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[C][2][V];
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int e = 0; e < V; ++e) x[c][w][e] = (float)r[u][c][w][e];
      if constexpr (NORM) {
        auto squares = [&] {
          float q = 0.0f;
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
              for (int e = 0; e < V; ++e) q = __builtin_fmaf(x[c][w][e], x[c][w][e], q);
          return group_sum<W>(q);
        };
        float q = squares(), eps = p.eps;
        if constexpr (std::is_same_v<T, __bf16>) {
          // squares at the ends of fp32's range: the head in units of 2^80 or 2^-80
          // (an eps from 1e-30 on outweighs what small squares lose)
          const bool big = !(q < 3.0e38f), small = q < 1e-30f && eps < 1e-30f;
          if (__builtin_amdgcn_ballot_w64(big || small)) {
            const float unit = big ? 0x1p-80f : small ? 0x1p80f : 1.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
              for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int e = 0; e < V; ++e) x[c][w][e] *= unit;
            q = squares();
            eps = eps * unit * unit;
          }
        }
        const float rs = __builtin_amdgcn_rsqf(__builtin_fmaf(q, p.inv_dh, eps));
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int e = 0; e < V; ++e) x[c][w][e] = x[c][w][e] * rs * gam[c][w][e];
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        TV o[2];
        if constexpr (IL && V > 1) {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float co = cs[c][w * (V / 2) + e / 2], si = sn[c][w * (V / 2) + e / 2];
              const float a = x[c][w][e], d = x[c][w][e + 1];
              o[w][e] = (T)__builtin_fmaf(a, co, -(d * si));
              o[w][e + 1] = (T)__builtin_fmaf(d, co, a * si);
            }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float a = x[c][0][e], d = x[c][1][e];
            o[0][e] = (T)__builtin_fmaf(a, cs[c][e], -(d * sn[c][e]));
            o[1][e] = (T)__builtin_fmaf(d, cs[c][e], a * sn[c][e]);
          }
        }
        if (plain[c]) {  // an infinity there is its own alone
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const int k = IL && V > 1 ? w * (V / 2) + e / 2 : e;
              o[w][e] = plain[c] >> k & 1 ? (T)x[c][w][e] : o[w][e];
            }
        }
        if (in[c] && live && h + u < h1) {
          *reinterpret_cast<TV*>(dst + (h + u) * p.yh[kv] + at[c][0]) = o[0];
          *reinterpret_cast<TV*>(dst + (h + u) * p.yh[kv] + at[c][1]) = o[1];
        }
      }
    }
    h += U;
    if (h >= h1) break;
    request(h);
  }
}

template <typename T, int V, int W, int C, bool IL>
static int rotary_go(RotaryParams& p, hipStream_t s) {
  // Heads of one group: as many as leave the card 4096 waves (16 a CU), alike in all groups
  const int tiles = (p.tokens + 256 / W - 1) / (256 / W);
  const int want = std::max(1, (1024 + tiles - 1) / tiles), total = p.heads[0] + p.heads[1];
  for (int i = 0; i < 2; ++i) {
    const int parts = (int)std::min<long long>(p.heads[i], ((long long)want * p.heads[i] + total - 1) / total);
    p.hpg[i] = parts ? (p.heads[i] + parts - 1) / parts : 1;
    p.blocks[i] = (p.heads[i] + p.hpg[i] - 1) / p.hpg[i];
  }
  const dim3 grid(tiles, p.blocks[0] + p.blocks[1]);
  const bool many = V > 1 && std::max(p.hpg[0], p.hpg[1]) > 2;
  auto go = [&](auto kernel) { DLM_LAUNCH("rotary_kernel", kernel, grid, dim3(256), 0, s, p); };
  constexpr int U = V > 1 ? 4 : 1;
  if (p.norm)
    many ? go(rotary_kernel<T, V, W, C, IL, true, U>) : go(rotary_kernel<T, V, W, C, IL, true, 1>);
  else
    many ? go(rotary_kernel<T, V, W, C, IL, false, U>) : go(rotary_kernel<T, V, W, C, IL, false, 1>);
  DLM_LAUNCH_CHECK();
  return DLM_OK;
}

template <typename T, bool IL>
static int rotary_by_width(RotaryParams& p, int V, hipStream_t s) {
  const int lanes = p.Dh / (2 * V);  // of one head
  if (V == 8) {
    if (lanes <= 4) return rotary_go<T, 8, 4, 1, IL>(p, s);
    if (lanes <= 8) return rotary_go<T, 8, 8, 1, IL>(p, s);
    return rotary_go<T, 8, 16, 1, IL>(p, s);
  }
  if (V == 4) return lanes <= 16 ? rotary_go<T, 4, 16, 1, IL>(p, s) : rotary_go<T, 4, 32, 1, IL>(p, s);
  return lanes <= 64 ? rotary_go<T, 1, 64, 1, IL>(p, s) : rotary_go<T, 1, 64, 2, IL>(p, s);
}

// Elements of a vector that every head, pair section and address of the call keeps
// whole: 8, 4 or 1.
static int rotary_vector(const dlm_rotary_args* a, int P) {
  for (const int V : {8, 4}) {
    auto whole = [&](const void* p, long long b, long long s, long long h) {
      return p == nullptr || ((uintptr_t)p % (2 * V) == 0 && b % V == 0 && s % V == 0 && h % V == 0);
    };
    const bool pairs = a->interleaved ? a->Dh % (2 * V) == 0 : P % V == 0 && a->Dh % (2 * V) == 0;
    if (pairs && whole(a->q, a->q_sb, a->q_ss, a->q_sh) && whole(a->k, a->k_sb, a->k_ss, a->k_sh) &&
        whole(a->q_out, a->qo_sb, a->qo_ss, a->qo_sh) && whole(a->k_out, a->ko_sb, a->ko_ss, a->ko_sh) &&
        whole(a->q_gamma, 0, 0, 0) && whole(a->k_gamma, 0, 0, 0))
      return V;
  }
  return 1;
}

static int rotary_check(const char* fn, const dlm_rotary_args* a, int& P) {
  auto bad = [&](const std::string& m) { return fail(DLM_ERR_INVALID_ARG, std::string(fn) + ": " + m); };
  if (!a->q || !a->q_out) return bad("NULL operand");
  if ((a->k == nullptr) != (a->k_out == nullptr)) return bad("k and k_out come together");
  if (a->k && a->Hkv <= 0) return bad("keys of no heads");
  if (a->dtype != DLM_DTYPE_F16 && a->dtype != DLM_DTYPE_BF16) return bad("unknown dtype");
  if (a->Dh % 2 != 0 || a->Dh > 256) return bad("Dh must be even and at most 256");
  if (a->axes < 0 || a->axes > 4) return bad("axes must be 0 to 4");
  long long pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0) return bad("a section has a negative number of pairs");
    pairs += a->sections[i];
  }
  if (2 * pairs > a->Dh) return bad("the sections hold more pairs than a head");
  P = (int)pairs;
  if (P > 0 && (!a->pos || !a->freqs)) return bad("positions and frequencies are needed for the sections");
  if (P > 0 && a->pos_type != DLM_POS_I32 && a->pos_type != DLM_POS_I64 && a->pos_type != DLM_POS_F32)
    return bad("unknown type of positions");
  if (P > 0 && ((uintptr_t)a->pos % (a->pos_type == DLM_POS_I64 ? 8 : 4) != 0 || (uintptr_t)a->freqs % 8 != 0))
    return bad("positions and frequencies must be aligned to their elements");
  if (P > 0 && (a->pos_sb < 0 || a->pos_ss < 0)) return bad("negative stride of the positions");
  if (P > 0 && (double)(a->B - 1) * (double)a->pos_sb + (double)(a->S - 1) * (double)a->pos_ss > 0x1p46)
    return bad("the positions span more than 2^46 elements");
  if (a->norm && !(a->eps >= 0.0f && a->eps < INFINITY)) return bad("eps must be finite and not negative");
  if (!a->norm && (a->q_gamma || a->k_gamma)) return bad("gamma without the norm");
  for (const void* p : {a->q, (const void*)a->q_out, a->k, (const void*)a->k_out, a->q_gamma, a->k_gamma})
    if ((uintptr_t)p % 2 != 0) return bad("operands must be aligned to their elements");
  // (a grid has fewer than 2^32 threads: 64 a token where heads are wide or unaligned, in whole blocks of
  // four tokens)
  if ((long long)a->B * a->S > (1LL << 26) - 4) return bad("more than 2^26 - 4 tokens");
  if ((long long)a->H + (a->k ? a->Hkv : 0) > 65535) return bad("more than 65535 heads");
  const View v[4] = {{"q", a->q, a->q_sb, a->q_ss, a->q_sh, a->S, a->H},
                     {"k", a->k, a->k_sb, a->k_ss, a->k_sh, a->S, a->Hkv},
                     {"q_out", a->q_out, a->qo_sb, a->qo_ss, a->qo_sh, a->S, a->H},
                     {"k_out", a->k_out, a->ko_sb, a->ko_ss, a->ko_sh, a->S, a->Hkv}};
  for (const View& x : v) {
    if (!x.p) continue;
    if (x.sb < 0 || x.ss < 0 || x.sh < 0) return bad(std::string(x.name) + ": negative stride");
    if ((double)(a->B - 1) * (double)x.sb + (double)(a->S - 1) * (double)x.ss + (double)(x.H - 1) * (double)x.sh > 0x1p46)
      return bad(std::string(x.name) + " spans more than 2^46 elements");
  }
  for (int i = 2; i < 4; ++i) {
    if (!v[i].p) continue;
    // an output's own elements have to lie apart (a stride of 0 would write one twice)
    long long st[3], in[3];
    int n = 0;
    auto add = [&](long long stride, int count) {
      if (count > 1) st[n] = stride, in[n++] = count;
    };
    add(v[i].sb, a->B), add(v[i].ss, a->S), add(v[i].sh, v[i].H);
    long long inner = a->Dh;
    for (int done = 0; done < n; ++done) {
      int k = -1;
      for (int j = 0; j < n; ++j)
        if (in[j] > 0 && (k < 0 || st[j] < st[k])) k = j;
      if (st[k] < inner) return bad(std::string(v[i].name) + " overlaps itself");
      inner += (in[k] - 1) * st[k];
      in[k] = 0;
    }
    for (int j = 0; j < i; ++j) {
      // in place: the very view (a stride of a dimension of one says nothing)
      const bool same = j == i - 2 && v[i].p == v[j].p && (a->B == 1 || v[i].sb == v[j].sb) &&
                        (a->S == 1 || v[i].ss == v[j].ss) && (v[i].H == 1 || v[i].sh == v[j].sh);
      if (!same && views_overlap(v[i], v[j], a->B, a->Dh, 2))
        return bad(std::string(v[i].name) + " overlaps " + v[j].name);
    }
    // nor may it lie on what every head reads
    const long long vec = 2LL * a->Dh, places = a->pos_type == DLM_POS_I64 ? 8 : 4;
    const struct {
      const char* name;
      const void* p;
      long long bytes;
    } shared[4] = {{"q_gamma", a->q_gamma, vec},
                   {"k_gamma", a->k_gamma, vec},
                   {"pos", P > 0 ? a->pos : nullptr,
                    ((a->B - 1) * a->pos_sb + (a->S - 1) * a->pos_ss + a->axes) * places},
                   {"freqs", P > 0 ? a->freqs : nullptr, 8LL * P}};
    for (const auto& x : shared)
      if (view_meets(v[i], a->B, a->Dh, 2, x.p, x.bytes))
        return bad(std::string(v[i].name) + " overlaps " + x.name);
  }
  return DLM_OK;
}

static int rotary_run(const char* fn, const dlm_rotary_args* a, hipStream_t s) {
  int P = 0;
  if (const int st = rotary_check(fn, a, P)) return st;
  RotaryParams p{};
  p.x[0] = (const char*)a->q, p.x[1] = (const char*)a->k;
  p.y[0] = (char*)a->q_out, p.y[1] = (char*)a->k_out;
  p.gamma[0] = (const char*)a->q_gamma, p.gamma[1] = (const char*)a->k_gamma;
  p.xb[0] = a->q_sb, p.xs[0] = a->q_ss, p.xh[0] = a->q_sh;
  p.xb[1] = a->k_sb, p.xs[1] = a->k_ss, p.xh[1] = a->k_sh;
  p.yb[0] = a->qo_sb, p.ys[0] = a->qo_ss, p.yh[0] = a->qo_sh;
  p.yb[1] = a->ko_sb, p.ys[1] = a->ko_ss, p.yh[1] = a->ko_sh;
  p.heads[0] = a->H, p.heads[1] = a->k ? a->Hkv : 0;
  p.pos = a->pos, p.pb = a->pos_sb, p.ps = a->pos_ss;
  p.pos_type = a->pos_type, p.axes = a->axes;
  int end = 0;
  for (int i = 0; i < 4; ++i) {
    end += i < a->axes ? a->sections[i] : 0;
    p.ends[i] = i < a->axes - 1 ? end : P;  // the last axis ends the pairs
  }
  p.freqs = a->freqs;
  p.P = P, p.Dh = a->Dh, p.norm = a->norm != 0;
  p.tokens = a->B * a->S, p.S = a->S;
  // (v_rsq_f32 takes a subnormal number as 0.  A mean of fp16 squares is 2^-56 at least or 0; bf16 heads are
  // brought into range)
  p.eps = a->dtype == DLM_DTYPE_F16 && a->eps > 0.0f ? std::max(a->eps, FLT_MIN) : a->eps;
  p.inv_dh = 1.0f / (float)a->Dh;
  const int V = rotary_vector(a, P);
  if (a->dtype == DLM_DTYPE_F16)
    return a->interleaved ? rotary_by_width<f16, true>(p, V, s) : rotary_by_width<f16, false>(p, V, s);
  return a->interleaved ? rotary_by_width<__bf16, true>(p, V, s) : rotary_by_width<__bf16, false>(p, V, s);
}

}  // namespace dlm

using namespace dlm;

extern "C" {

int dlm_rotary_axes(const dlm_rotary_args* a, void* stream) {
  DLM_REQUIRE(a != nullptr, "args is NULL");
  if (a->B <= 0 || a->S <= 0 || a->H <= 0 || a->Dh <= 0) return DLM_OK;
  DLM_REQUIRE(!a->norm, "the norm is dlm_qk_norm_rotary's");
  return rotary_run(__func__, a, (hipStream_t)stream);
}

int dlm_qk_norm_rotary(const dlm_rotary_args* a, void* stream) {
  DLM_REQUIRE(a != nullptr, "args is NULL");
  if (a->B <= 0 || a->S <= 0 || a->H <= 0 || a->Dh <= 0) return DLM_OK;
  DLM_REQUIRE(a->norm, "the rotation alone is dlm_rotary_axes's");
  return rotary_run(__func__, a, (hipStream_t)stream);
}

}  // extern "C"
