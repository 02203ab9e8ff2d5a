// Rows of a strided tensor and the checks that the row operators (token log probabilities, rotary
// positions, head norms) share.
#pragma once

#include "common.cuh"
#include "overlap.h"

namespace pb {

// Element offset of row r of up to three tensors whose leading dims have one shape. Metadata travels
// by value; a contiguous tensor has one dim and costs no division.
struct RowMap {
  int nd;
  unsigned size[MAX_NDIM];
  u64 stride[3][MAX_NDIM];
};

__device__ __forceinline__ void row_offsets(const RowMap &m, unsigned r, u64 off[3]) {
  off[0] = off[1] = off[2] = 0;
  for (int d = m.nd - 1; d > 0; --d) {
    const unsigned q = r / m.size[d], at = r - q * m.size[d];
    r = q;
#pragma unroll
    for (int a = 0; a < 3; ++a) off[a] += at * m.stride[a][d];
  }
#pragma unroll
  for (int a = 0; a < 3; ++a) off[a] += r * m.stride[a][0];
}

// Builds the map over the first `nd` dims of the given tensors' strides (size-1 dims dropped,
// neighbours merged where every tensor walks them as one run).
inline void make_row_map(RowMap *m, const u64 *shape, u64 nd, const u64 *s0, const u64 *s1, const u64 *s2) {
  static const u64 none[MAX_NDIM] = {};
  const u64 *s[3] = {s0 ? s0 : none, s1 ? s1 : none, s2 ? s2 : none};
  m->nd = 0;
  for (u64 d = 0; d < nd; ++d) {
    if (shape[d] == 1) continue;
    const int k = m->nd;
    bool merge = k > 0;
    for (int a = 0; a < 3 && merge; ++a) merge = m->stride[a][k - 1] == s[a][d] * shape[d];
    if (merge) {
      m->size[k - 1] *= (unsigned)shape[d];
      for (int a = 0; a < 3; ++a) m->stride[a][k - 1] = s[a][d];
    } else {
      m->size[k] = (unsigned)shape[d];
      for (int a = 0; a < 3; ++a) m->stride[a][k] = s[a][d];
      m->nd = k + 1;
    }
  }
  if (m->nd == 0) {
    m->nd = 1;
    m->size[0] = 1;
    for (int a = 0; a < 3; ++a) m->stride[a][0] = 0;
  }
}

// Row-major without gaps (dims of size 1 may carry any stride).
inline bool is_packed(const Tensor *t) {
  u64 expect = 1;
  for (u64 d = t->ndim; d-- > 0;) {
    if (t->shape[d] != 1 && t->strides[d] != expect) return false;
    expect *= t->shape[d];
  }
  return true;
}

// A tensor that is written may lie over `own` (may be NULL) element by element, and over none of the others.
inline bool check_apart(const char *name, const char *what, const Extent &written, const Extent &own, const Extent *others, int n) {
  bool ok = !own.t || !share_an_element(written, own) || same_elements(written.t, own.t);
  for (int i = 0; ok && i < n; ++i) ok = !share_an_element(written, others[i]);
  if (!ok) set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: %s overlaps another tensor of the call", name, what);
  return ok;
}

inline bool same_shape(const Tensor *a, const Tensor *b) {
  if (a->ndim != b->ndim) return false;
  for (u64 d = 0; d < a->ndim; ++d)
    if (a->shape[d] != b->shape[d]) return false;
  return true;
}

// Checks one tensor: present, at most MAX_NDIM dims, of the dtype, with data.
inline bool check_typed(const Tensor *t, DTYPE dtype, const char *what) {
  if (!check_tensor(t, what)) return false;
  if (t->dtype != dtype) {
    set_error(PLAST_B200_ERR_DTYPE, "%s: dtype must be %s", what, dtype == INT32 ? "INT32" : "FLOAT32");
    return false;
  }
  return true;
}

// The gradient buffer of `t`, which backward adds to: FLOAT32, t's shape, every element its own.
inline bool check_grad(const Tensor *t, const char *what) {
  if (!t->grad || (!t->grad->data && numel(t) > 0)) {
    set_error(PLAST_B200_ERR_NULL, "%s: requires grad but has no grad buffer", what);
    return false;
  }
  if (t->grad->dtype != FLOAT32) {
    set_error(PLAST_B200_ERR_DTYPE, "%s: the gradient must be FLOAT32", what);
    return false;
  }
  if (!same_shape(t, t->grad)) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: the gradient's shape differs", what);
    return false;
  }
  if (has_repeated_elements(t->grad)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: the gradient holds an element at two indices", what);
    return false;
  }
  return true;
}

} // namespace pb
