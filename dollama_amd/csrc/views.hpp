// Which operands of a call lie on one another: [batch, token, head, Dh] views with strides.
#pragma once

#include <algorithm>
#include <cstdint>

namespace dlm {

struct View {
  const char* name;
  const void* p;
  long long sb, ss, sh;
  int S, H;
};

// Whether two views of B x S x H x Dh elements share one.  Of views with the same
// strides, each longer than what lies inside it (slices of one tensor), the places
// are compared; any others count by their whole extents.
inline bool views_overlap(const View& a, const View& b, int B, int Dh, int elem) {
  if (!a.p || !b.p || a.S <= 0 || b.S <= 0) return false;
  auto extent = [&](const View& v) {
    return ((B - 1) * v.sb + (v.S - 1) * v.ss + (v.H - 1) * v.sh + Dh) * (long long)elem;
  };
  const long long delta = (long long)((intptr_t)b.p - (intptr_t)a.p);
  if (delta >= extent(a) || -delta >= extent(b)) return false;
  struct Dim {
    long long stride;
    int na, nb;
  } d[3];
  int n = 0;
  bool alike = delta % elem == 0;
  auto add = [&](long long sa, int na, long long sb, int nb) {
    if (na > 1 || nb > 1) d[n++] = {na > 1 ? sa : sb, na, nb};
    alike = alike && (na <= 1 || nb <= 1 || sa == sb);
  };
  add(a.sb, B, b.sb, B);
  add(a.ss, a.S, b.ss, b.S);
  add(a.sh, a.H, b.sh, b.H);
  if (!alike) return true;
  std::sort(d, d + n, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  long long inner = Dh;  // extents of what lies inside a dimension
  for (int i = n - 1; i >= 0; --i) {
    if (d[i].stride < inner) return true;
    inner += (std::max(d[i].na, d[i].nb) - 1) * d[i].stride;
  }
  // does some index pair bring b's element box onto a's?
  auto meet = [&](auto& self, int i, long long off) -> bool {
    if (i == n) return off < Dh && -off < Dh;
    const long long st = d[i].stride;
    const long long k = off >= 0 ? off / st : -((-off + st - 1) / st);
    // a's index minus b's: only these two leave less than a stride
    for (const long long t : {k, k + 1})
      if (t <= d[i].na - 1 && -t <= d[i].nb - 1 && self(self, i + 1, off - t * st)) return true;
    return false;
  };
  return meet(meet, 0, delta / elem);
}

// Whether one of a view's elements lies in the `bytes` bytes from q on.
inline bool view_meets(const View& v, int B, int Dh, int elem, const void* q, long long bytes) {
  if (!v.p || !q || v.S <= 0 || bytes <= 0) return false;
  struct Dim {
    long long stride;
    int n;
  } d[3];
  int n = 0;
  auto add = [&](long long st, int count) {
    if (count > 1) d[n++] = {st * elem, count};
  };
  add(v.sb, B);
  add(v.ss, v.S);
  add(v.sh, v.H);
  std::sort(d, d + n, [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
  long long extent[4];  // of what lies inside a dimension, and of all
  extent[n] = (long long)Dh * elem;
  for (int i = n - 1; i >= 0; --i) extent[i] = extent[i + 1] + (d[i].n - 1) * d[i].stride;
  const long long lo = (long long)((intptr_t)q - (intptr_t)v.p);
  auto meet = [&](auto& self, int i, long long lo, long long hi) -> bool {
    if (lo >= extent[i] || hi <= 0) return false;
    if (i == n || d[i].stride < extent[i + 1]) return true;
    // the indices whose part [k stride, k stride + inner) the bytes reach; those between the first and the
    // last lie in them whole
    const long long st = d[i].stride, inner = extent[i + 1];
    const long long first = lo < inner ? 0 : (lo - inner) / st + 1, last = std::min<long long>(d[i].n - 1, (hi - 1) / st);
    if (last - first > 1) return true;
    for (long long k = first; k <= last; ++k)
      if (self(self, i + 1, lo - k * st, hi - k * st)) return true;
    return false;
  };
  return meet(meet, 0, lo, lo + bytes);
}

}  // namespace dlm
