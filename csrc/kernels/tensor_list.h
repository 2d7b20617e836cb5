// Operands' memory: ranges, and lists of tensors as clip.cu and adamw.cu take them (host arithmetic only).
#pragma once
#include <stdint.h>

#include "nn_ops.h"

struct MemoryRange { const void* at; long long bytes; };
// Does one of the first `written` ranges share memory with another of all?  Absent ones have no bytes.
inline bool ranges_overlap(const MemoryRange* r, int written, int all) {
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < all; ++j)
      if (r[i].bytes > 0 && r[j].bytes > 0 && (uintptr_t)r[i].at < (uintptr_t)r[j].at + r[j].bytes && (uintptr_t)r[j].at < (uintptr_t)r[i].at + r[i].bytes) return true;
  return false;
}

struct TensorRange { uintptr_t from, to; };
inline TensorRange tensor_range(const GeepsTensors& t, long long i) {
  const uintptr_t p = (uintptr_t)t.ptr[i];
  return {p, p + (uintptr_t)t.count[i] * (t.fp32[i] ? 4 : 2)};
}
// Is there a tensor that begins between two values?
inline bool tensors_between(const GeepsTensors& t) {
  for (long long i = 0; i < t.n; ++i)
    if (t.count[i] && ((uintptr_t)t.ptr[i] & (t.fp32[i] ? 3 : 1))) return true;
  return false;
}
// Is there a tensor of `a` that shares memory with one of `b` (a itself: with another of its own)?  Both are sorted by address
// and each without overlaps, so one merge finds it.  b[i] may be a[i].
inline bool tensors_overlap(const GeepsTensors& t) {
  uintptr_t end = 0;
  for (long long k = 0; k < t.n; ++k) {
    const TensorRange r = tensor_range(t, t.order[k]);
    if (r.from == r.to) continue;
    if (r.from < end) return true;
    end = r.to;
  }
  return false;
}
inline bool tensors_overlap(const GeepsTensors& a, const GeepsTensors& b) {
  long long i = 0, j = 0;
  while (i < a.n && j < b.n) {
    const long long x = a.order[i], y = b.order[j];
    const TensorRange p = tensor_range(a, x), q = tensor_range(b, y);
    const bool same = x == y && p.from == q.from && a.fp32[x] == b.fp32[y];
    if (p.from < q.to && q.from < p.to && p.from != p.to && q.from != q.to && !same) return true;
    if (p.to < q.to) ++i; else ++j;
  }
  return false;
}
// Does a tensor of the (sorted, disjoint) list share memory with [from, to)?
inline bool tensors_meet(const GeepsTensors& t, const void* at, unsigned long long bytes) {
  if (at == nullptr || bytes == 0) return false;
  const uintptr_t from = (uintptr_t)at, to = from + bytes;
  for (long long lo = 0, hi = t.n; lo < hi;) {
    const long long mid = (lo + hi) >> 1;
    const TensorRange r = tensor_range(t, t.order[mid]);
    if (r.from == r.to) {          // an empty one says nothing about its neighbours: all of the rest, one by one
      for (long long i = lo; i < hi; ++i) {
        const TensorRange q = tensor_range(t, t.order[i]);
        if (q.from != q.to && q.from < to && from < q.to) return true;
      }
      return false;
    }
    if (r.to <= from) lo = mid + 1;
    else if (r.from >= to) hi = mid;
    else return true;
  }
  return false;
}
