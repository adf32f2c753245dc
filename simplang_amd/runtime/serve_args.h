// serve_args.h -- operand checks shared by the entry points that serve a batch of
// sequences (attention.hip, kv8.hip).
#pragma once

#include <cfloat>
#include <cmath>

#include "rt_internal.h"

namespace simp {

// A rank-3 descriptor as the entry points take it, and its element extent.
template <class T>
struct Desc3 {
  T *p;
  int64_t off, s[3], st[3], span;
  // A dimension of one element may have any stride: it gets the span of those inside it.
  int check(const char *name) {
    uint64_t inner = 1;  // (what overflows is refused below)
    for (int i = 2; i >= 0; i--) {
      if (s[i] == 1) st[i] = (int64_t)inner;
      inner += (uint64_t)(s[i] - 1) * (uint64_t)st[i];
    }
    return check_descn(name, p, off, 3, s, st, &span);
  }
  bool is(int64_t a, int64_t b, int64_t c) const { return s[0] == a && s[1] == b && s[2] == c; }
  T *data() const { return p + off; }
  size_t bytes() const { return (size_t)span * sizeof(T); }
};

// The kernels take the scale in fp32, times log2(e) for powers of two.
inline bool scale_fits(double scale) { return std::fabs(scale) * 1.4426950408889634 <= FLT_MAX; }

// Device memory of another GPU than the one that the call launches on is refused.
inline int check_here(const Operand &o, int dev, const char *name) {
  if (o.device() >= 0 && o.device() != dev)
    return set_error(SIMP_RT_EINVAL, "%s: lies on device %d, the call is on device %d", name,
                     o.device(), dev);
  return SIMP_RT_OK;
}

inline int bind_here(Operand &o, const void *p, size_t bytes, Operand::Dir dir, int dev,
                     const char *name, bool stage = true) {
  const int rc = o.bind(p, bytes, dir, name, stage);
  return rc ? rc : check_here(o, dev, name);
}

// Whether two byte ranges share any.
inline bool overlap(const void *a, size_t an, const void *b, size_t bn) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return an && bn && x < y + bn && y < x + an;
}

// Dimensions of an array, the outer ones first, each with a stride of at least the span of
// those inside it.  One of size 1 has any stride.
struct Level {
  int64_t n, stride;
};

// Whether two arrays with these dimensions share an element, the second's first one
// `delta` elements behind the first's: sum (i - j) stride = delta has a solution.  What the
// inner dimensions add is less than a stride, so only two differences come into question.
inline bool meet(const Level *level, int levels, int64_t delta) {
  if (levels == 0) return delta == 0;
  const Level &l = *level;
  if (l.n <= 1) return l.n == 1 && meet(level + 1, levels - 1, delta);
  int64_t d = delta / l.stride;
  if (delta % l.stride < 0) d--;  // rounded down
  for (int i = 0; i < 2; i++, d++)
    if (d > -l.n && d < l.n && meet(level + 1, levels - 1, delta - d * l.stride)) return true;
  return false;
}

// Whether two arrays of one shape share elements.  One may lie between the rows or the
// heads of the other, as the parts of a fused product do.
template <class T>
bool share(const Desc3<T> &a, const Desc3<T> &b) {
  if (!overlap(a.data(), a.bytes(), b.data(), b.bytes())) return false;
  const int64_t bytes = (int64_t)((uintptr_t)b.data() - (uintptr_t)a.data());
  if (bytes % (int64_t)sizeof(T) || a.st[0] != b.st[0] || a.st[1] != b.st[1]) return true;
  const Level l[] = {{a.s[0], a.st[0]}, {a.s[1], a.st[1]}, {a.s[2], 1}};
  return meet(l, 3, bytes / (int64_t)sizeof(T));
}

}  // namespace simp
