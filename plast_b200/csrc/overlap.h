// Do two strided tensors share an element? Host code, without the CUDA headers.
#pragma once

#include "plast_b200.h"

#include <stdint.h>

namespace pb {

// A sum of strides with integer factors, each in its range, equals `target`? Strides descend, so that in views of
// ordinary arrays at most a few factors of each come into question; a search that gets long counts as a yes.
struct StrideTerm {
  __int128 stride, low, high;
};
struct StrideSum {
  StrideTerm term[2 * MAX_NDIM];
  int n = 0;
  void add(long long stride, __int128 low, __int128 high) { // equal strides are one term
    if (stride == 0 || low == high) return; // (a range of one is 0 to 0)
    if (stride < 0) add_positive(-(__int128)stride, -high, -low);
    else add_positive(stride, low, high);
  }
  bool reaches(__int128 target) {
    int budget = 4096;
    return reaches(0, target, budget);
  }
  // 0 by factors that are not all 0 (the ranges are symmetric: the first of them is positive)
  bool returns() const {
    int budget = 4096;
    for (int k = 0; k < n; ++k) {
      __int128 high = 0; // of the terms behind
      for (int i = k + 1; i < n; ++i) high += term[i].stride * term[i].high;
      for (__int128 v = 1; v <= term[k].high && term[k].stride * v <= high; ++v)
        if (reaches(k + 1, -term[k].stride * v, budget)) return true;
    }
    return false;
  }

private:
  void add_positive(__int128 stride, __int128 low, __int128 high) {
    int k = 0;
    while (k < n && term[k].stride > stride) ++k;
    if (k < n && term[k].stride == stride) {
      term[k].low += low;
      term[k].high += high;
      return;
    }
    for (int i = n; i > k; --i) term[i] = term[i - 1];
    term[k] = StrideTerm{stride, low, high};
    ++n;
  }
  bool reaches(int k, __int128 target, int &budget) const {
    if (k == n) return target == 0;
    if (--budget < 0) return true;
    __int128 low = 0, high = 0; // what the terms behind this one can add
    for (int i = k + 1; i < n; ++i) {
      low += term[i].stride * term[i].low;
      high += term[i].stride * term[i].high;
    }
    const __int128 s = term[k].stride;
    auto down = [&](__int128 v) { return v >= 0 ? v / s : -((-v + s - 1) / s); };
    __int128 first = -down(high - target), last = down(target - low); // ceil((target - high) / s), floor((target - low) / s)
    if (first < term[k].low) first = term[k].low;
    if (last > term[k].high) last = term[k].high;
    for (__int128 v = first; v <= last; ++v)
      if (reaches(k + 1, target - s * v, budget)) return true;
    return false;
  }
};

// A tensor's elements lie in [begin, end) (bytes; empty: begin == end).
struct Extent {
  const Tensor *t;
  __int128 begin, end;
};
inline Extent extent_of(const Tensor *t) {
  Extent e = {t, 0, 0};
  if (!t) return e;
  __int128 low = 0, high = 0;
  for (u64 d = 0; d < t->ndim; ++d) {
    if (t->shape[d] == 0) return e;
    const __int128 reach = (__int128)(t->shape[d] - 1) * (long long)t->strides[d];
    if (reach < 0) low += reach; else high += reach;
  }
  e.begin = (__int128)(uintptr_t)t->data + 4 * low;
  e.end = (__int128)(uintptr_t)t->data + 4 * (high + 1);
  return e;
}
inline bool share_an_element(const Extent &a, const Extent &b) {
  if (a.begin >= b.end || b.begin >= a.end) return false;
  const __int128 apart = (__int128)(uintptr_t)b.t->data - (__int128)(uintptr_t)a.t->data;
  if (apart % 4) return true; // parts of elements
  StrideSum sum;
  for (u64 d = 0; d < a.t->ndim; ++d) sum.add((long long)a.t->strides[d], 0, (__int128)a.t->shape[d] - 1);
  for (u64 d = 0; d < b.t->ndim; ++d) sum.add((long long)b.t->strides[d], 1 - (__int128)b.t->shape[d], 0);
  return sum.reaches(apart / 4);
}
// A tensor that is written element by element must not hold one element at two indices (an expanded view, or strides
// that let rows run into each other).
inline bool has_repeated_elements(const Tensor *t) {
  StrideSum sum;
  for (u64 d = 0; d < t->ndim; ++d)
    if (t->shape[d] == 0) return false;
  for (u64 d = 0; d < t->ndim; ++d) {
    if (t->shape[d] == 1) continue;
    if (t->strides[d] == 0) return true;
    for (u64 e = 0; e < d; ++e)
      if (t->shape[e] > 1 && (t->strides[e] == t->strides[d] || t->strides[e] == 0 - t->strides[d])) return true;
    sum.add((long long)t->strides[d], 1 - (__int128)t->shape[d], (__int128)t->shape[d] - 1);
  }
  return sum.returns();
}

// The same elements at the same indices.
inline bool same_elements(const Tensor *a, const Tensor *b) {
  if (a->data != b->data || a->ndim != b->ndim) return false;
  for (u64 d = 0; d < a->ndim; ++d)
    if (a->shape[d] != b->shape[d] || (a->shape[d] > 1 && a->strides[d] != b->strides[d])) return false;
  return true;
}

} // namespace pb
