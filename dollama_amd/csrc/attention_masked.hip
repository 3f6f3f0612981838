// Masked attention: the entry points, the choice of a kernel, and the kernels for fp16 (those for bf16
// are the same in a file of their own, so that the two compile side by side).
#include "attention_masked.hpp"
#include "views.hpp"

namespace dlm {

int am_run_f16(const AmParams& p, const AmPlan& pl, bool cap, hipStream_t s) { return am_run<f16>(p, pl, cap, s); }

static AmPlan am_plan(const dlm_attention_masked_args* a) {
  const long long heads = (long long)a->B * a->Hkv, rows = (long long)a->Sq * (a->H / a->Hkv);
  AmPlan pl;
  pl.few = rows <= 32;
  pl.nrb = (int)((rows + (pl.few ? 31 : 127)) / (pl.few ? 32 : 128));
  // Parts of 256 keys at least, as many as cost least by a model in us: the keys' time in one part (a
  // tile of 64 in 1.2, as of heads of 128; or 55 kB of few rows' K and V a us), the rounds of workgroups over 256 CUs, and the
  // parts' way through memory.  (us with 1 / 4 / 8 / 16 / 32 parts, 32/8 heads of 128: one token over 4096 keys
  // 38 / 19 / 14 / 12 / 12, over 65536 485 / 132 / 72 / 51 / 50; 64 tokens over 30001
  // 420 / 117 / 67 / 45 / 53; 256 over 4096 68 / 39 / 38 / 50 / 78.)  Few rows, whose
  // workgroups have a CU to themselves, stay whole past eight rounds, where the last one's share is small;
  // many rows where there is a workgroup for every CU: a CU runs two or three of them at once, masks leave
  // less than the model's time, and the parts are large (documents of 426 to 1439 in 8192 tokens x10x64, 640
  // workgroups: 50 us whole, 102 in two parts, 56 of them to join).
  const long long blocks = heads * pl.nrb;
  const double whole = pl.few ? a->Sk * (double)a->Dh * 4 / 55e3 : a->Sk / 64 * 1.2;
  const double part = (double)heads * rows * (a->Dh + 2) * 8 / 4e6;
  double best = 0.0;
  pl.splits = 1;
  for (int s = 1; s <= (blocks <= (pl.few ? 8 * 256 : 255) ? std::min(64, std::max(1, a->Sk / 256)) : 1); ++s) {
    const double t = whole * (double)((blocks * s + 255) / 256) / s + (s > 1 ? 3.0 + part * s : 0.0);
    if (s == 1 || t < best) best = t, pl.splits = s;
  }
  return pl;
}

static size_t am_workspace(const dlm_attention_masked_args* a, const AmPlan& pl) {
  if (pl.splits == 1) return 0;
  return (size_t)pl.splits * a->B * a->H * a->Sq * (a->Dh + 2) * 4;
}

// Every check of a call; its plan where they pass
static int am_check(const char* fn, const dlm_attention_masked_args* a, const void* workspace, size_t workspace_bytes,
                    AmPlan& pl) {
  auto bad = [&](const std::string& m) { return fail(DLM_ERR_INVALID_ARG, std::string(fn) + ": " + m); };
  if (!a->q || !a->o || (a->Sk > 0 && (!a->k || !a->v))) return bad("NULL operand");
  if (a->dtype != DLM_DTYPE_F16 && a->dtype != DLM_DTYPE_BF16) return bad("unknown dtype");
  if (a->Sk < 0) return bad("negative number of keys");
  if (a->Dh % 8 != 0 || a->Dh > 256) return bad("Dh must be a multiple of 8 and at most 256");
  if (a->Hkv <= 0 || a->H % a->Hkv != 0) return bad("H must be a multiple of Hkv");
  if (!(a->scale > 0.0f && a->scale <= 0x1p127f)) return bad("scale must be positive and at most 2^127");
  if (!(a->cap >= 0.0f && a->cap < INFINITY)) return bad("cap must be finite and not negative");
  if (a->cap > 0.0f && a->scale / a->cap > 1e30f) return bad("cap is too small for the scale");
  if (a->slopes && a->rel_bias) return bad("one bias of distance, slopes or a table");
  if (a->rel_bias && (a->R < 0 || a->R > (1 << 24))) return bad("R must be 0 to 2^24");
  if (a->Sq > (1 << 28) || a->Sk > (1 << 28)) return bad("more than 2^28 queries or keys");
  const long long G = a->H / a->Hkv;
  if (a->Sq * G >= (1LL << 29) || (long long)a->B * a->Hkv > 65535) return bad("more rows or heads than a grid takes");
  if ((long long)a->B * a->Hkv * ((a->Sq * G + 31) / 32) >= (1LL << 23)) return bad("more rows than a grid takes");
  View ops[4] = {{"q", a->q, a->q_sb, a->q_ss, a->q_sh, a->Sq, a->H},
                 {"k", a->k, a->k_sb, a->k_ss, a->k_sh, a->Sk, a->Hkv},
                 {"v", a->v, a->v_sb, a->v_ss, a->v_sh, a->Sk, a->Hkv},
                 {"o", a->o, a->o_sb, a->o_ss, a->o_sh, a->Sq, a->H}};
  for (int i = 0; i < 4; ++i) {
    View& x = ops[i];
    const int unit = i < 3 ? 8 : 4, align = 2 * unit;
    if (a->B == 1) x.sb = 0;  // a dimension of one has no stride
    if (x.S <= 1) x.ss = 0;
    if (x.H == 1) x.sh = 0;
    if (x.sb < 0 || x.ss < 0 || x.sh < 0) return bad(std::string(x.name) + ": negative stride");
    if ((uintptr_t)x.p % align != 0 || x.sb % unit != 0 || x.ss % unit != 0 || x.sh % unit != 0)
      return bad(std::string(x.name) + (i < 3 ? ": address and strides must keep 16-byte alignment"
                                              : ": address and strides must keep 8-byte alignment"));
    const double last = (double)(a->B - 1) * (double)x.sb + (double)(std::max(x.S, 1) - 1) * (double)x.ss +
                        (double)(x.H - 1) * (double)x.sh + a->Dh;
    if (last > 0x1p46) return bad(std::string(x.name) + " spans more than 2^46 elements");
    if ((i == 1 || i == 2) && x.S > 1 && (x.ss < a->Dh || x.ss >= (1 << 23)))
      return bad(std::string(x.name) + ": a key row's stride must be Dh to 2^23");
  }
  // an output's own elements have to lie apart
  {
    struct Dim {
      long long st;
      int n;
    } d[3] = {{ops[3].sb, a->B}, {ops[3].ss, a->Sq}, {ops[3].sh, a->H}};
    std::sort(d, d + 3, [](const Dim& x, const Dim& y) { return x.st < y.st; });
    long long inner = a->Dh;
    for (const Dim& x : d) {
      if (x.n <= 1) continue;
      if (x.st < inner) return bad("o overlaps itself");
      inner += (x.n - 1) * x.st;
    }
  }
  for (int i = 0; i < 3; ++i)
    if (views_overlap(ops[3], ops[i], a->B, a->Dh, 2)) return bad(std::string("o overlaps ") + ops[i].name);
  if ((uintptr_t)a->key_range % 8 != 0 || (uintptr_t)a->q_pos % 4 != 0 || (uintptr_t)a->slopes % 4 != 0 ||
      (uintptr_t)a->rel_bias % 4 != 0)
    return bad("key_range must be 8-byte, q_pos, slopes and rel_bias 4-byte aligned");
  if (a->kr_sb < 0 || a->kr_sb % 2 != 0 || a->qp_sb < 0) return bad("batch strides of the masks must be whole and not negative");
  if ((double)(a->B - 1) * (double)std::max(a->kr_sb, a->qp_sb) > 0x1p46) return bad("the masks span more than 2^46 elements");
  pl = am_plan(a);
  const size_t need = am_workspace(a, pl);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return bad("the workspace is too small");
  if (need > 0 && !dlm_aligned16(workspace)) return bad("the workspace must be 16-byte aligned");
  // the output may not lie on what every row reads, nor the parts of the keys on anything
  const struct {
    const char* name;
    const void* p;
    long long bytes;
  } flat[4] = {{"key_range", a->key_range, ((a->B - 1) * a->kr_sb + 2LL * a->Sq) * 4},
               {"q_pos", a->q_pos, ((a->B - 1) * a->qp_sb + a->Sq) * 4},
               {"slopes", a->slopes, 4LL * a->H},
               {"rel_bias", a->rel_bias, (2LL * a->R + 1) * a->H * 4}};
  auto meets = [&](const View& x, const void* p, long long bytes) { return view_meets(x, a->B, a->Dh, 2, p, bytes); };
  for (const auto& x : flat)
    if (meets(ops[3], x.p, x.bytes)) return bad(std::string("o overlaps ") + x.name);
  if (need > 0) {
    const uintptr_t at = (uintptr_t)workspace;
    for (const View& x : ops)
      if (meets(x, workspace, (long long)need)) return bad(std::string("the workspace overlaps ") + x.name);
    for (const auto& x : flat)
      if (x.p && at < (uintptr_t)x.p + x.bytes && (uintptr_t)x.p < at + need)
        return bad(std::string("the workspace overlaps ") + x.name);
  }
  return DLM_OK;
}

}  // namespace dlm

using namespace dlm;

extern "C" {

size_t dlm_attention_masked_workspace_bytes(const dlm_attention_masked_args* a) {
  if (!a || a->B <= 0 || a->Sq <= 0 || a->H <= 0 || a->Dh <= 0 || a->Hkv <= 0 || a->H % a->Hkv != 0) return 0;
  return am_workspace(a, am_plan(a));
}

int dlm_attention_masked(const dlm_attention_masked_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  DLM_REQUIRE(a != nullptr, "args is NULL");
  if (a->B <= 0 || a->Sq <= 0 || a->H <= 0 || a->Dh <= 0) return DLM_OK;
  AmPlan pl;
  if (const int st = am_check(__func__, a, workspace, workspace_bytes, pl)) return st;
  AmParams p{};
  p.q = (const char*)a->q, p.k = (const char*)a->k, p.v = (const char*)a->v, p.o = (char*)a->o;
  p.q_sb = a->q_sb, p.q_ss = a->q_ss, p.q_sh = a->q_sh;
  p.k_sb = a->k_sb, p.k_ss = a->Sk > 1 ? a->k_ss : a->Dh, p.k_sh = a->k_sh;
  p.v_sb = a->v_sb, p.v_ss = a->Sk > 1 ? a->v_ss : a->Dh, p.v_sh = a->v_sh;
  p.o_sb = a->o_sb, p.o_ss = a->o_ss, p.o_sh = a->o_sh;
  p.key_range = a->key_range, p.kr_sb = a->kr_sb;
  p.q_pos = a->q_pos, p.qp_sb = a->qp_sb;
  p.slopes = a->slopes, p.table = a->rel_bias, p.R = a->R;
  p.Sq = a->Sq, p.Sk = a->Sk, p.Hkv = a->Hkv, p.G = a->H / a->Hkv, p.Dh = a->Dh;
  p.rows = a->Sq * p.G;
  p.causal = a->causal != 0, p.nrb = pl.nrb, p.heads = a->B * a->Hkv, p.splits = pl.splits;
  p.parts = a->key_range ? 2 : 1;
  // (more blocks than these even out by themselves, and a head's next to one another share its K and V)
  const long long blocks = (long long)pl.nrb * p.heads;
  p.lpt = (a->causal || a->key_range) && pl.splits == 1 && pl.nrb > 1 && blocks <= 8 * 256;
  p.part = (float*)workspace;
  p.c = a->scale * AM_LOG2E;
  // A cap from 2^126 on changes no softmax: scores up to 2^113 it leaves as they are in fp32, and larger
  // ones are so far apart that one weight alone is not 0, before it and behind.  Its own terms would pass
  // fp32's range.
  const bool cap = a->cap > 0.0f && a->cap < 0x1p126f;
  if (cap) {
    p.ic = a->scale / a->cap;
    p.cl = a->cap * AM_LOG2E;
    const double ic = (double)a->scale / a->cap;
    p.small = (float)std::min(0.5 / ic, (double)FLT_MAX);
    for (int i = 0; i < 5; ++i) p.ct[i] = (float)(AM_TANH[i] * a->scale * 1.4426950408889634);
  }
  p.table_lds = a->rel_bias && (2LL * (a->R + AM_TABLE_MARGIN) + 1) * p.G <= AM_TABLE_MAX;
  return a->dtype == DLM_DTYPE_F16 ? am_run_f16(p, pl, cap, (hipStream_t)stream)
                                   : am_run_bf16(p, pl, cap, (hipStream_t)stream);
}

}  // extern "C"
