// attend.h — what the attention kernels (attend_few.hip, attend_chunk.hip)
// share: a sequence's bounds, the page of a position, the cache's codes as
// f16, and the partial results that a context cut into parts leaves.
#pragma once

#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;  // positions a step of either kernel takes
// Weights may reach 2^kSlack (lifted, f16 holds 2^15) before the running maximum that
// they are relative to is moved and what is summed so far rescaled.
constexpr float kSlack = 8.0f;
// Weights are lifted by 2^kLift, which leaves again with the division by their
// sum: f16 holds them down to 2^-31 of the largest and not to 2^-24 only (a
// million positions of 2^-25.5 beside one of 1 are 2 % of a row's output).
constexpr float kLift = 7.0f;
// Weights are 2^(s sc - m sc + kLift), m the maximum they are relative to. Up to this
// size m sc is rounded by 2^-17 at most and one fused multiply-add a weight
// does it; where some row's is larger the scores are taken as s - m first, for
// the rounding grows with m sc (from 2^28 on by 16 and more: weights past f16,
// or all of them zero) and ends in an infinity.
constexpr float kFar = 256.0f;

// The bounds of sequence b, whatever the device arrays hold: its first row
// q0, its rows nq (at most max_q, inside the q rows), its cached positions kv
// (inside its table) and the first row's position pos0 (negative where it
// stands before the cache).
__device__ __forceinline__ void sequence(const AttendArgs& a, int b, int64_t& q0, int& nq, int& kv, int& pos0) {
  const int64_t s = a.q_starts[b], e = a.q_starts[b + 1];
  q0 = s < 0 ? 0 : (s > a.tokens ? a.tokens : s);
  const int64_t q1 = e < q0 ? q0 : (e > a.tokens ? a.tokens : e);
  nq = q1 - q0 > a.max_q ? a.max_q : (int)(q1 - q0);
  const int n = a.kv_lens[b];
  kv = n < 0 ? 0 : (n > a.max_kv ? a.max_kv : n);
  pos0 = kv - (int)(q1 - q0);  // rows past max_q count
}

// The first position that a row standing at `pos` sees.
__device__ __forceinline__ int first_seen(const AttendArgs& a, int pos) {
  return a.window > 0 && a.window <= pos ? pos - (int)a.window + 1 : 0;
}

// The page that holds position j < kv of sequence b; -1 where j is past kv or
// the table names no page there.
__device__ __forceinline__ int page_of(const AttendArgs& a, int b, int j, int kv) {
  if (j >= kv) return -1;
  const int p = a.tables[(int64_t)b * a.table_stride + (j >> a.page_bits)];
  return p < 0 || p >= a.c.pages ? -1 : p;
}

// 4 codes as f16, exactly: a byte b = code + 128 under 0x64 is the f16 1024 + b.
__device__ __forceinline__ void codes_f16(uint32_t c, h2v& lo, h2v& hi) {
  const uint32_t x = c ^ 0x80808080u;
  const h2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
  lo = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off;
  hi = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off;
}

union H8 {
  h8v v;
  h2v h[4];
  uint4 u;
};

// 8 codes times their scales, each product rounded once to f16: a key's 8
// share one scale, a value's 8 positions have one each.
__device__ __forceinline__ h8v key8(uint32_t a, uint32_t b, h2v s) {
  H8 r;
  codes_f16(a, r.h[0], r.h[1]);
  codes_f16(b, r.h[2], r.h[3]);
#pragma unroll
  for (int i = 0; i < 4; i++) r.h[i] = r.h[i] * s;
  return r.v;
}
__device__ __forceinline__ h8v value8(uint32_t a, uint32_t b, const uint4& s) {
  H8 r, d;
  d.u = s;
  codes_f16(a, r.h[0], r.h[1]);
  codes_f16(b, r.h[2], r.h[3]);
#pragma unroll
  for (int i = 0; i < 4; i++) r.h[i] = r.h[i] * d.h[i];
  return r.v;
}
__device__ __forceinline__ h2v both(uint32_t f16bits) {
  return __builtin_bit_cast(h2v, (f16bits & 0xFFFFu) * 0x10001u);
}

// Query row r of a kv head as (new token, head of the group): r / group by a
// multiplication (rows times group stay below 2^32).
__device__ __forceinline__ int token_of(const AttendArgs& a, int r) {
  return a.group_inv ? (int)__umulhi((uint32_t)r, a.group_inv) : r;
}

// N pieces of 8 of a query's values as f16, piece s from element at(s) on: exact
// for an f16 query and for a bf16 one of ordinary size; an f32 query rounds
// once. Past f16's range they saturate. The scale's sign goes with them, its
// size into the softmax.
__device__ __forceinline__ _Float16 query_f16(const AttendArgs& a, float x) {
  x *= a.q_sign;
  return (_Float16)(x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x);
}
template <int N, typename At>
__device__ __forceinline__ void load_query(const AttendArgs& a, bool on, At at, h8v* q) {
#pragma unroll
  for (int s = 0; s < N; s++) q[s] = h8v{};
  if (!on) return;
  if (!a.q_vec) {
#pragma unroll
    for (int s = 0; s < N; s++)
      for (int i = 0; i < 8; i++) {
        const int64_t e = at(s) + i;
        q[s][i] = query_f16(a, a.qdt == QMM_X_F32 ? load1<QMM_X_F32>(a.q, e)
                                                  : a.qdt == QMM_X_F16 ? load1<QMM_X_F16>(a.q, e) : load1<QMM_X_BF16>(a.q, e));
      }
  } else if (a.qdt == QMM_X_F32) {
#pragma unroll
    for (int s = 0; s < N; s++) {
      float x[8];
      load4<QMM_X_F32, true>(a.q, at(s), x);
      load4<QMM_X_F32, true>(a.q, at(s) + 4, x + 4);
#pragma unroll
      for (int i = 0; i < 8; i++) q[s][i] = query_f16(a, x[i]);
    }
  } else {
    H8 r[N];
#pragma unroll
    for (int s = 0; s < N; s++) r[s].u = *(const uint4*)((const uint16_t*)a.q + at(s));
    if (a.qdt == QMM_X_F16) {
#pragma unroll
      for (int s = 0; s < N; s++)
#pragma unroll
        for (int i = 0; i < 8; i++) q[s][i] = query_f16(a, (float)r[s].v[i]);
    } else {
#pragma unroll
      for (int s = 0; s < N; s++) {
        const uint32_t w[4] = {r[s].u.x, r[s].u.y, r[s].u.z, r[s].u.w};
#pragma unroll
        for (int i = 0; i < 8; i++) q[s][i] = query_f16(a, widen<QMM_X_BF16>(w[i >> 1] >> (16 * (i & 1))));
      }
    }
  }
}

// The steps [begin, end) of a part of a row block whose rows see positions
// [lo, hi): parts of equal length, the last ones shorter or empty.
__device__ __forceinline__ void part_steps(int lo, int hi, int part, int parts, int& begin, int& end) {
  const int t0 = lo / kTile, tiles = hi > 0 ? (hi + kTile - 1) / kTile - t0 : 0;
  const int each = parts > 1 ? (int)(((uint32_t)tiles + parts - 1) / (uint32_t)parts) : tiles;
  const int first = part * each;
  begin = t0 + (first < tiles ? first : tiles);
  end = t0 + (first + each < tiles ? first + each : tiles);
}

// Scales of 8 positions j0 .. j0 + 7 with those outside [lo, hi) zeroed: what
// lies there need not be finite, and a weight of zero would not hide it.
__device__ __forceinline__ uint4 cut_scales(uint4 s, int j0, int lo, int hi) {
  uint32_t w[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int j = j0 + 2 * i;
    if (j < lo || j >= hi) w[i] &= 0xFFFF0000u;
    if (j + 1 < lo || j + 1 >= hi) w[i] &= 0x0000FFFFu;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Partial results: rows of a block (kv head of a sequence, `rows` query rows)
// for each part of its context: sums of weights times values [cut_index][part][row][hd],
// then (the score that they are relative to, as the product gives it, and the
// sum of weights) [part][row][2]; that score is -inf in a part that a row sees
// nothing of.
struct AttendParts {
  float* o;
  float* ml;
  int parts, rows;  // query rows of a block
  int blocks, cut;  // row blocks of a kv head of a sequence; blocks that are in parts
  int cut_rows, cut_more;  // those: every head's first cut_rows, and the next of the last cut_more heads
  int4* split;      // shares (attend_chunk.hip): the block that each leaves unfinished
  int shares;       // 0: none
};
// The place of a block among those in parts (every head's first cut_rows, then
// the last heads' next); -1: it is whole.
__device__ __forceinline__ int cut_index(const AttendArgs& a, const AttendParts& p, int head_of_seq, int block) {
  const int heads = a.seqs * a.c.heads, x = head_of_seq - (heads - p.cut_more);
  return block < p.cut_rows ? head_of_seq * p.cut_rows + block : block == p.cut_rows && x >= 0 ? heads * p.cut_rows + x : -1;
}
__device__ __forceinline__ int64_t part_row(const AttendParts& p, int cut_index, int part, int row) {
  return ((int64_t)cut_index * p.parts + part) * p.rows + row;
}

// What sums relative to score m count for beside ones relative to `base`
// (finite). The scores meet before the scale, whose product with either may
// pass f32's range.
__device__ __forceinline__ float weight_of(const AttendArgs& a, float m, float base) {
  return exp2_fast((m - base) * a.sc);
}

// A row's outputs from its sums of weights times values (relative to score
// `top`) and of weights, the head's sink joined.
template <int N>
__device__ __forceinline__ void finish_row(const AttendArgs& a, int head, float top, float sum, const float* acc,
                                           float* out) {
  float f = 1.0f;
  if (a.sinks && sum != 0.0f) {
    const float at = fminf(fmaxf(top * a.sc, -3e38f), 3e38f);  // finite
    const float sink = a.sinks[head] * kLog2e, mx = fmaxf(at, sink);
    f = exp2_fast(at - mx);
    sum = sum * f + exp2_fast(sink == mx ? kLift : sink - mx + kLift);  // (an infinite sink less itself is NaN)
  }
  const float inv = sum == 0.0f ? 0.0f : f / sum;
#pragma unroll
  for (int i = 0; i < N; i++) out[i] = sum == 0.0f ? 0.0f : acc[i] * inv;
}

// 4 outputs at element e.
__device__ __forceinline__ void store_out4(const AttendArgs& a, int64_t e, const float v[4]) {
  if (a.out_vec)
    store4<true>(a.out, a.odt, e, v);
  else
    store4<false>(a.out, a.odt, e, v);
}

constexpr int kShareRows = 256;  // query rows of a block that shares may split
// Partial results of share w: slot 2 w for a block that a share before it
// began, 2 w + 1 for one that it leaves to the next.
__device__ __forceinline__ int64_t share_row(int slot, int row) { return (int64_t)slot * kShareRows + row; }

// The launches of either kernel over the sequences with lo < rows <= hi query
// rows a kv head (tokens times group); parts > 1: into `p`.
hipError_t launch_attend_few(const AttendArgs& a, int lo, int hi, const AttendParts& p, hipStream_t st);
hipError_t launch_attend_chunk(const AttendArgs& a, int lo, const AttendParts& p, hipStream_t st);

constexpr int kFewWaves = 4;     // waves of a few-row workgroup
constexpr int kFewRows = 32;     // the most query rows of the few-row kernel

}  // namespace qmm
