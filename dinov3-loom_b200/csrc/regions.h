// regions.h - whether two strided tensors share memory. Plain C++, for the host's argument checks.
#pragma once

#include <stdint.h>

#include <utility>

namespace dv3 {

// n_outer x n_inner vectors of `bytes` contiguous bytes, the given strides (in bytes) apart.
struct Region {
  const void *base;
  int64_t outer, inner;
  uint32_t n_outer, n_inner;
  int64_t bytes;
};

// Whether no byte of `a` is a byte of `b`. Exact where their ranges do not meet, and for views that
// lie side by side in one buffer (columns of fused rows, keys and values of one pool). Where ranges meet
// under strides that differ the answer is no.
inline bool apart(Region a, Region b) {
  using wide = __int128;
  for (Region *r : {&a, &b}) {
    if (!r->base || r->n_outer == 0 || r->n_inner == 0 || r->bytes == 0) return true;
    if (r->n_outer == 1 || (r->n_inner > 1 && r->inner > r->outer)) {  // the longer stride outside
      std::swap(r->outer, r->inner);
      std::swap(r->n_outer, r->n_inner);
    }
  }
  const auto row = [](const Region &r) { return static_cast<wide>(r.n_inner - 1) * r.inner + r.bytes; };
  const wide at = static_cast<wide>(reinterpret_cast<uintptr_t>(b.base)) -
                  static_cast<wide>(reinterpret_cast<uintptr_t>(a.base));
  if (at >= static_cast<wide>(a.n_outer - 1) * a.outer + row(a)) return true;
  if (-at >= static_cast<wide>(b.n_outer - 1) * b.outer + row(b)) return true;
  // Disjoint in one period of a stride that both repeat with. A single row repeats with any.
  const auto beside = [](wide at, wide a, wide b, wide period) {
    if (period <= 0) return false;
    at %= period;
    if (at < 0) at += period;
    return at >= a && at + b <= period;
  };
  if (a.n_outer > 1 && b.n_outer > 1 && a.outer != b.outer) return false;
  const wide outer = a.n_outer > 1 ? a.outer : b.outer;
  if ((a.n_outer > 1 || b.n_outer > 1) && beside(at, row(a), row(b), outer)) return true;
  if (a.n_inner > 1 && b.n_inner > 1 && a.inner != b.inner) return false;
  const wide inner = a.n_inner > 1 ? a.inner : b.inner;
  if ((a.n_outer > 1 || b.n_outer > 1) && (inner <= 0 || outer % inner != 0)) return false;
  return (a.n_inner > 1 || b.n_inner > 1) && beside(at, a.bytes, b.bytes, inner);
}

}  // namespace dv3
