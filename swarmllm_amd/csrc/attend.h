// attend.h — what the kernels and the entry point of the paged attention
// share: the arguments, a sequence's bounds and the page of a position.
#pragma once

#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

// The bounds of sequence b, whatever the device arrays hold: its first row
// q0, its rows nq (at most max_q, inside the q rows) and its cached positions
// kv (inside its table).
__device__ __forceinline__ void sequence(const AttendArgs& a, int b, int64_t& q0, int& nq, int& kv) {
  const int64_t s = a.q_starts[b], e = a.q_starts[b + 1];
  q0 = s < 0 ? 0 : (s > a.tokens ? a.tokens : s);
  const int64_t q1 = e < q0 ? q0 : (e > a.tokens ? a.tokens : e);
  nq = q1 - q0 > a.max_q ? a.max_q : (int)(q1 - q0);
  const int n = a.kv_lens[b];
  kv = n < 0 ? 0 : (n > a.max_kv ? a.max_kv : n);
}

// The page that holds position j of sequence b, -1 for one outside the cache.
__device__ __forceinline__ int64_t page_of(const AttendArgs& a, int b, int64_t j) {
  const int p = a.tables[(int64_t)b * a.table_stride + j / a.c.page];
  return p < 0 || p >= a.c.pages ? -1 : p;
}

}  // namespace qmm
