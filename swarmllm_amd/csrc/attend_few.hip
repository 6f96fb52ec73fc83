// attend_few.hip — attention of a sequence's few new tokens (at most 32 query
// rows a kv head: decode, drafts) over its pages of the cache.
//
// What bounds it is the cache's bytes: every key and value is read once for
// all the query rows of its kv head, straight from the planes into the
// matrix instructions' operands. A wave takes 64 positions at a time:
//   S^T = K q^T   (16x16x32: rows positions, columns query rows)
//   O^T += V^T P^T (rows dims, columns query rows)
// The order of the positions within a step is free. K row r of tile t is
// position 16 (r / 4) + 4 t + r % 4, so that lane (column, g) holds the scores
// of positions 16 g .. 16 g + 15: as they stand they are the second product's
// operand, and a lane's V operand is 16 consecutive bytes of a V row. No
// score, key or value passes through LDS; the running maximum, the sum and
// the rescaling of O all belong to the lane's own column. The waves of a
// workgroup take steps in turn, joined at the end through LDS; a long context
// is cut into parts of the same kind, joined by attend_join_kernel.
//
// 64 sequences of 4000 tokens (64 query heads on 8 of 128 dims) take 88 us, 420 MB
// at 4.8 TB/s, a copy's rate; 16 of 8000, ragged, 47 and 4.7 us of join. Few
// short sequences are bound by the chain of one step (bounds, page, planes, some
// 850 vector instructions, join): one of 500 tokens takes 11 us. The loads of a
// step's keys and values are all issued before its first product: with the
// values' loaded behind the scores the 16 sequences took 71 us.
#include "attend.h"

namespace qmm {

namespace {

template <int HD>
struct FewSizes {
  static constexpr int kWide = HD / 64;        // 64-dim groups of a key, 16 dims a lane
  static constexpr int kTail = HD % 64 ? 1 : 0;  // a 32-dim group behind them, 8 dims a lane
  static constexpr int kSteps = HD / 32;       // matrix products of a score
  static constexpr int kDims = HD / 16;        // 16-dim tiles of the output
};

// NT tiles of 16 query rows.
template <int HD, int NT>
__global__ __launch_bounds__(64 * kFewWaves) void attend_few_kernel(AttendArgs a, int lo_rows, int hi_rows, AttendParts parts) {
  using Z = FewSizes<HD>;
  constexpr int W = kFewWaves;
  constexpr int kJoin = HD < 128 ? HD : 128;  // dims that go through LDS at a time when the waves join
  static_assert(kJoin % 16 == 0 && HD % kJoin == 0, "whole tiles of 16 dims");
  constexpr int kJoinRow = kJoin + 4;  // padded off the banks of the next row
  __shared__ float s_o[W][16][kJoinRow];
  __shared__ float s_m[W][16 * NT], s_l[W][16 * NT];
  const CachePlanes& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x, part = blockIdx.y, b = blockIdx.z;
  int64_t q0;
  int nq, kv, pos0;
  sequence(a, b, q0, nq, kv, pos0);
  const int rows = nq * a.group;
  if (rows <= lo_rows || rows > hi_rows) return;  // another launch's (or none)

  // this workgroup's steps: its part of [first position any row sees, kv)
  const int lo = first_seen(a, pos0 < 0 ? 0 : pos0);
  int begin, end;
  part_steps(lo, kv, part, parts.parts, begin, end);

  // queries: lane (column, g) holds the dims its keys' lanes hold
  h8v q[NT][Z::kSteps];
  int pos[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const int r = 16 * n + col, i = token_of(a, r);
    pos[n] = pos0 + i;
    const int64_t e = (q0 + i) * a.qs + (int64_t)(kvh * a.group + r - i * a.group) * a.qhs;
    load_query<Z::kSteps>(a, r < rows, [&](int s) {
      return e + (s < 2 * Z::kWide ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 64 * Z::kWide + 8 * g);
    }, q[n]);
  }

  f4v o[NT][Z::kDims];
  float m[NT], l[NT], bs[NT];  // bs: m sc - kLift, what the weights' exponents are less (far: m is taken off before)
  bool far[NT];  // some row's maximum is past kFar (the same for the wave)
#pragma unroll
  for (int n = 0; n < NT; n++) {
    far[n] = false;
    m[n] = -INFINITY;
    l[n] = bs[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < Z::kDims; d++) o[n][d] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int ka = col >> 2;  // the 16-position chunk of the lane's K rows; its V chunk is g
  int kp = begin + wave < end ? page_of(a, b, (begin + wave) * kTile + 16 * ka, kv) : -1;
  int vp = begin + wave < end ? page_of(a, b, (begin + wave) * kTile + 16 * g, kv) : -1;
  for (int tile = begin + wave; tile < end; tile += W) {
    const int j0 = tile * kTile;
    const bool k_there = kp >= 0, v_there = vp >= 0;
    const int64_t kph = (int64_t)(k_there ? kp : 0) * c.heads + kvh, vph = (int64_t)(v_there ? vp : 0) * c.heads + kvh;
    const int kat = ((j0 + 16 * ka) & (c.page - 1)) + (col & 3), vat = (j0 + 16 * g) & (c.page - 1);
    const int8_t* kc = c.k_codes + (kph * c.page + kat) * HD;
    const uint16_t* ks = c.k_scales + (kph * c.page + kat) * (HD / 32);
    const int8_t* vc = c.v_codes + (vph * HD + col) * c.page + vat;
    const uint16_t* vs = c.v_scales + vph * (HD / 32) * c.page + vat;
    if (tile + W < end) {
      kp = page_of(a, b, j0 + W * kTile + 16 * ka, kv);
      vp = page_of(a, b, j0 + W * kTile + 16 * g, kv);
    }
    // whether some position of the step is hidden from some row (the same for the wave)
    const bool partial = j0 + kTile - 1 > pos0 || (a.window > 0 && j0 <= (int64_t)kv - 1 - a.window) ||
                         __ballot(!k_there) != 0;

    // the step's planes, all of them in flight at once
    uint4 wide[4][Z::kWide ? Z::kWide : 1];
    uint2 tail[4];
    uint32_t sc[4][Z::kWide + Z::kTail];
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
      for (int u = 0; u < Z::kWide; u++) wide[t][u] = *(const uint4*)(kc + 4 * t * HD + 64 * u + 16 * g);
      const uint16_t* kst = ks + 4 * t * (HD / 32);
      if constexpr (Z::kTail) {
        tail[t] = *(const uint2*)(kc + 4 * t * HD + 64 * Z::kWide + 8 * g);
#pragma unroll
        for (int u = 0; u < Z::kWide; u++) sc[t][u] = kst[2 * u + (g >> 1)];
        sc[t][Z::kWide] = kst[2 * Z::kWide];
      } else if constexpr (Z::kWide == 1) {
        sc[t][0] = *(const uint32_t*)kst >> (16 * (g >> 1));
      } else if constexpr (Z::kWide == 2) {
        const uint2 w = *(const uint2*)kst;
        sc[t][0] = w.x >> (16 * (g >> 1));
        sc[t][1] = w.y >> (16 * (g >> 1));
      } else {
        const uint4 w = *(const uint4*)kst;
        sc[t][0] = w.x >> (16 * (g >> 1));
        sc[t][1] = w.y >> (16 * (g >> 1));
        sc[t][2] = w.z >> (16 * (g >> 1));
        sc[t][3] = w.w >> (16 * (g >> 1));
      }
    }
    // (the scales of 256 dims would not fit the registers beside their codes)
    constexpr bool kScalesToo = HD <= 128;
    uint4 vw[Z::kDims], vd[kScalesToo ? Z::kDims : 1];
#pragma unroll
    for (int d = 0; d < Z::kDims; d++) {
      vw[d] = *(const uint4*)(vc + 16 * d * c.page);
      if constexpr (kScalesToo) vd[d] = *(const uint4*)(vs + (d >> 1) * c.page + 8 * (d & 1));
    }

    f4v s[NT][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
      for (int n = 0; n < NT; n++) s[n][t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < Z::kWide; u++) {
        const h2v d = both(sc[t][u]);
        const h8v k0 = key8(wide[t][u].x, wide[t][u].y, d), k1 = key8(wide[t][u].z, wide[t][u].w, d);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[n][2 * u], s[n][t], 0, 0, 0);
          s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[n][2 * u + 1], s[n][t], 0, 0, 0);
        }
      }
      if constexpr (Z::kTail) {
        const h8v k0 = key8(tail[t].x, tail[t].y, both(sc[t][Z::kWide]));
#pragma unroll
        for (int n = 0; n < NT; n++)
          s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[n][Z::kSteps - 1], s[n][t], 0, 0, 0);
      }
    }

    // weights: lane (column, g) has positions j0 + 16 g + 4 t + i
    h8v p[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      if (partial) {
        const int first = first_seen(a, pos[n]);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int j = j0 + 16 * g + 4 * t + i;
            if (j > pos[n] || j < first || !v_there) s[n][t][i] = -INFINITY;
          }
      }
      float mt = s[n][0][0];
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) mt = fmaxf(mt, s[n][t][i]);
      if (__ballot((mt - m[n]) * a.sc > kSlack) != 0 || far[n]) {
        mt = fmaxf(mt, __shfl_xor(mt, 16, kWave));
        mt = fmaxf(mt, __shfl_xor(mt, 32, kWave));
        const float mn = fmaxf(m[n], mt), to = mn == -INFINITY ? 0.0f : mn, f = weight_of(a, m[n], to);
        far[n] = __ballot(fabsf(to) * a.sc > kFar) != 0;
        m[n] = mn;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < Z::kDims; d++) o[n][d] *= f;
        bs[n] = far[n] ? -kLift : __builtin_fmaf(to, a.sc, -kLift);
        if (far[n])
#pragma unroll
          for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][t][i] -= to;
      }
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float w = exp2_fast(__builtin_fmaf(s[n][t][i], a.sc, -bs[n]));
          sum += w;
          p[n][t >> 1][4 * (t & 1) + i] = (_Float16)w;
        }
      l[n] += sum;
    }

    // values
    uint4 d0 = make_uint4(0, 0, 0, 0), d1 = d0;
#pragma unroll
    for (int d = 0; d < Z::kDims; d++) {
      const uint4 w = vw[d];
      if ((d & 1) == 0) {
        if constexpr (kScalesToo) {
          d0 = vd[d];
          d1 = vd[d + 1];
        } else {
          d0 = *(const uint4*)(vs + (d >> 1) * c.page);
          d1 = *(const uint4*)(vs + (d >> 1) * c.page + 8);
        }
        if (partial) {
          const int hi = v_there ? kv : 0;
          d0 = cut_scales(d0, j0 + 16 * g, lo, hi);
          d1 = cut_scales(d1, j0 + 16 * g + 8, lo, hi);
        }
      }
      const h8v v0 = value8(w.x, w.y, d0), v1 = value8(w.z, w.w, d1);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[n][0], o[n][d], 0, 0, 0);
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[n][1], o[n][d], 0, 0, 0);
      }
    }
  }

  // the waves' results joined: O of 16 rows and kJoin dims at a time
#pragma unroll
  for (int n = 0; n < NT; n++) {
    l[n] += __shfl_xor(l[n], 16, kWave);
    l[n] += __shfl_xor(l[n], 32, kWave);
    if (g == 0) {
      s_m[wave][16 * n + col] = m[n];
      s_l[wave][16 * n + col] = l[n];
    }
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int h = 0; h < HD; h += kJoin) {
      __syncthreads();
#pragma unroll
      for (int d = 0; d < kJoin / 16; d++) *(f4v*)&s_o[wave][col][16 * d + 4 * g] = o[n][h / 16 + d];
      __syncthreads();
      // 4 dims a thread
      for (int x = threadIdx.x; x < 16 * (kJoin / 4); x += 64 * W) {
        const int r16 = x / (kJoin / 4), e = 4 * (x - r16 * (kJoin / 4)), r = 16 * n + r16;
        if (r >= rows) continue;
        float mw[W], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
          mw[w] = s_m[w][r];
          top = fmaxf(top, mw[w]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; w++) {
          const float f = weight_of(a, mw[w], base);
          sum += s_l[w][r] * f;
          acc += *(const f4v*)&s_o[w][r16][e] * f;
        }
        if (parts.parts > 1) {
          const int64_t pr = part_row(parts, b * c.heads + kvh, part, r);
          *(f4v*)(parts.o + pr * HD + h + e) = acc;
          if (h + e == 0) {
            parts.ml[2 * pr] = top;
            parts.ml[2 * pr + 1] = sum;
          }
        } else {
          const int i = token_of(a, r), head = kvh * a.group + r - i * a.group;
          float out[4];
          finish_row<4>(a, head, top, sum, (const float*)&acc, out);
          store_out4(a, (q0 + i) * a.os + (int64_t)head * HD + h + e, out);
        }
      }
    }
}

template <int HD>
hipError_t launch_hd(const AttendArgs& a, int lo, int hi, const AttendParts& p, hipStream_t st) {
  const dim3 grid((unsigned)a.c.heads, (unsigned)p.parts, (unsigned)a.seqs);
  if (hi <= 16)
    attend_few_kernel<HD, 1><<<grid, 64 * kFewWaves, 0, st>>>(a, lo, hi, p);
  else
    attend_few_kernel<HD, 2><<<grid, 64 * kFewWaves, 0, st>>>(a, lo, hi, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attend_few(const AttendArgs& a, int lo, int hi, const AttendParts& p, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  switch (a.c.hd) {
    case 64: return launch_hd<64>(a, lo, hi, p, st);
    case 96: return launch_hd<96>(a, lo, hi, p, st);
    case 128: return launch_hd<128>(a, lo, hi, p, st);
    case 256: return launch_hd<256>(a, lo, hi, p, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace qmm
