// attend_chunk.hip — attention of a prompt's chunk of new tokens over its
// pages of the cache.
//
// What bounds it is the matrix cores and the vector work beside them. A
// workgroup takes 128 or 256 query rows of a kv head (the heads that share it
// side by side, token after token), 32 a wave, against steps of 64 positions:
// the step's keys and values are read once for all the rows, turned into f16
// (codes times scales, one rounding) and laid into LDS, the next step's planes
// in flight meanwhile. Per step a wave computes
//   S^T = K q^T   (32x32x16: rows positions, columns query rows)
//   O^T += V^T P^T (rows dims, columns query rows)
// K row r of a tile is the position whose index has bits 2 and 3 of r
// exchanged: so a lane's 8 scores of a 16-position step are consecutive
// positions, and the weights made of them are the second product's operand as
// they stand. The running maximum, the sum and O's rescaling belong to the
// lane's own column.
//
// Two prompts' chunks of 2000 tokens over 7777 (64 query heads on 8 of 128 dims)
// take 866-888 us, 0.76 PFLOP/s; a library product of 8192^3 reaches 1.15. The
// products (matrix cores busy 43% of the CUs' cycles), the softmax's and the conversions' vector instructions (about 290 a
// wave and step with 128 rows a workgroup, 230 with 256) and the LDS reads (32
// operands of 1 KiB a wave and step) each take a third to a half of a step and
// overlap only between the two waves of a SIMD. Tried and slower: a step's
// scores beside the weights of the one before (the second set of scores spills
// at 256 registers), steps of 32 positions, 64 rows a wave (accumulators past 256
// registers are copied back and forth each step), and products and vector
// instructions interleaved by hand.
#include "attend.h"
#include "mv_common.h"

namespace qmm {

namespace {

// Instruction classes of __builtin_amdgcn_sched_group_barrier.
constexpr int kMfma = 0x008, kDsRead = 0x100;
constexpr int kAhead = 4;  // LDS reads of operands in flight ahead of their products

template <int HD, int W>
struct ChunkSizes {
  // a step's keys (and values) in items of 32: the 32 dims of a block for one
  // position, 16 positions of two dims of a block; one scale, 16 scales
  static constexpr int kItems = kTile * HD / 32;
  static constexpr int kThreads = 64 * W;
  static constexpr bool kHalves = kItems * 2 <= kThreads;   // half the threads take keys, half values
  static constexpr int kEach = (kItems + kThreads - 1) / kThreads;  // a thread's of either
  static constexpr int kRow = HD + 8;                       // f16s of a K row in LDS, padded off the next row's banks
  static constexpr int kVRow = kTile + 8;                   // and of a V row
  static constexpr int kHalfs = kTile * kRow + HD * kVRow;  // one buffer
  static constexpr size_t kLds = 2 * kHalfs * sizeof(uint16_t);
};

// One step's planes in a thread's registers.
template <int HD, int W>
struct Staged {
  static constexpr int kEach = ChunkSizes<HD, W>::kEach;
  uint4 k[kEach][2], v[kEach][2], d0[kEach], d1[kEach];
  uint32_t ks[kEach];
};

// A thread's i-th item of keys, or of values; on: whether it has one.
template <int HD, int W>
__device__ __forceinline__ int k_item(int i, bool& on) {
  const int x = (int)threadIdx.x + ChunkSizes<HD, W>::kThreads * i;
  on = ChunkSizes<HD, W>::kItems % ChunkSizes<HD, W>::kThreads == 0 || x < ChunkSizes<HD, W>::kItems;
  return x;
}
template <int HD, int W>
__device__ __forceinline__ int v_item(int i, bool& on) {
  if (!ChunkSizes<HD, W>::kHalves) return k_item<HD, W>(i, on);
  const int x = (int)threadIdx.x - ChunkSizes<HD, W>::kThreads / 2;
  on = x >= 0 && x < ChunkSizes<HD, W>::kItems;
  return x;
}

// The lower dim of item x of values: 16 dims of a block, then the next block's.
__device__ __forceinline__ int v_dim(int x) { return (x >> 6) * 32 + ((x >> 2) & 15); }

// A step's pages. ONE: pages of 64 positions and more, so a step has one, the
// same for the wave; otherwise lane x < 4 of every wave holds that of the step's
// x-th 16 positions. -1: none.
template <bool ONE>
__device__ __forceinline__ int step_page(const AttendArgs& a, int b, int tile, int end, int kv) {
  if (tile >= end) return -1;
  return page_of(a, b, tile * kTile + (ONE ? 0 : 16 * (int)(threadIdx.x & 3)), kv);
}
// ONE: into a scalar register, once the load has surely landed.
template <bool ONE>
__device__ __forceinline__ int settled(int page) {
  return ONE ? __builtin_amdgcn_readfirstlane(page) : page;
}

template <int HD, int W, bool ONE>
__device__ __forceinline__ void fetch(const AttendArgs& a, int kvh, int j0, int pages, Staged<HD, W>& s) {
  using Z = ChunkSizes<HD, W>;
  const CachePlanes& c = a.c;
  const int8_t* k1 = nullptr;
  const int8_t* v1 = nullptr;
  const uint16_t *ks1 = nullptr, *vs1 = nullptr;
  if constexpr (ONE) {
    // a step's keys lie side by side, its values in rows of a page
    const int64_t ph = (int64_t)(pages < 0 ? 0 : pages) * c.heads + kvh;
    const int at = j0 & (c.page - 1);
    k1 = c.k_codes + (ph * c.page + at) * HD;
    ks1 = c.k_scales + (ph * c.page + at) * (HD / 32);
    v1 = c.v_codes + ph * HD * c.page + at;
    vs1 = c.v_scales + ph * (HD / 32) * c.page + at;
  }
#pragma unroll
  for (int i = 0; i < Z::kEach; i++) {
    bool k_on, v_on;
    const int xk = k_item<HD, W>(i, k_on), xv = v_item<HD, W>(i, v_on);
    const int vc = xv & 3, d = v_dim(xv);  // 16 positions from 16 vc on, dims d and d + 16
    if constexpr (ONE) {
      if (k_on) {
        s.k[i][0] = *(const uint4*)(k1 + 32 * (uint32_t)xk);
        s.k[i][1] = *(const uint4*)(k1 + 32 * (uint32_t)xk + 16);
        s.ks[i] = ks1[(uint32_t)xk];
      }
      if (v_on) {
        s.v[i][0] = *(const uint4*)(v1 + (uint32_t)d * (uint32_t)c.page + 16 * vc);
        s.v[i][1] = *(const uint4*)(v1 + (uint32_t)(d + 16) * (uint32_t)c.page + 16 * vc);
        const uint16_t* vs = vs1 + (uint32_t)(d >> 5) * (uint32_t)c.page + 16 * vc;
        s.d0[i] = *(const uint4*)vs;
        s.d1[i] = *(const uint4*)(vs + 8);
      }
    } else {
      const int row = xk / (HD / 32), e = 32 * (xk - row * (HD / 32));
      const int kp = __shfl(pages, (row >> 4) & 3, kWave), vp = __shfl(pages, vc, kWave);
      if (k_on) {
        const int64_t kr = ((int64_t)(kp < 0 ? 0 : kp) * c.heads + kvh) * c.page + ((j0 + row) & (c.page - 1));
        s.k[i][0] = *(const uint4*)(c.k_codes + kr * HD + e);
        s.k[i][1] = *(const uint4*)(c.k_codes + kr * HD + e + 16);
        s.ks[i] = c.k_scales[kr * (HD / 32) + (e >> 5)];
      }
      if (v_on) {
        const int64_t vph = (int64_t)(vp < 0 ? 0 : vp) * c.heads + kvh;
        const int at = (j0 + 16 * vc) & (c.page - 1);
        const int8_t* v = c.v_codes + (vph * HD + d) * c.page + at;
        s.v[i][0] = *(const uint4*)v;
        s.v[i][1] = *(const uint4*)(v + 16 * c.page);
        const uint16_t* vs = c.v_scales + (vph * (HD / 32) + (d >> 5)) * c.page + at;
        s.d0[i] = *(const uint4*)vs;
        s.d1[i] = *(const uint4*)(vs + 8);
      }
    }
  }
}

// The step's keys and values as f16 into an LDS buffer. CUT: the values of
// positions outside [lo, hi), or on no page, are laid as zeros.
template <int HD, int W, bool ONE, bool CUT>
__device__ __forceinline__ void lay(const Staged<HD, W>& s, int j0, int pages, int lo, int hi, uint16_t* buf) {
  using Z = ChunkSizes<HD, W>;
#pragma unroll
  for (int i = 0; i < Z::kEach; i++) {
    bool k_on, v_on;
    const int xk = k_item<HD, W>(i, k_on), xv = v_item<HD, W>(i, v_on);
    const int vc = xv & 3, d = v_dim(xv);
    const int vp = !CUT ? 0 : ONE ? pages : __shfl(pages, vc, kWave);
    H8 h;
    if (k_on) {
      const int row = xk / (HD / 32), e = 32 * (xk - row * (HD / 32));
      const h2v ks = both(s.ks[i]);
      uint16_t* kb = buf + row * Z::kRow + e;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        h.v = key8(s.k[i][u].x, s.k[i][u].y, ks);
        *(uint4*)(kb + 16 * u) = h.u;
        h.v = key8(s.k[i][u].z, s.k[i][u].w, ks);
        *(uint4*)(kb + 16 * u + 8) = h.u;
      }
    }
    if (v_on) {
      uint4 d0 = s.d0[i], d1 = s.d1[i];
      if constexpr (CUT) {
        const int j = j0 + 16 * vc;
        d0 = cut_scales(d0, j, lo, vp < 0 ? 0 : hi);
        d1 = cut_scales(d1, j + 8, lo, vp < 0 ? 0 : hi);
      }
      uint16_t* vb = buf + kTile * Z::kRow + d * Z::kVRow + 16 * vc;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        h.v = value8(s.v[i][u].x, s.v[i][u].y, d0);
        *(uint4*)(vb + 16 * u * Z::kVRow) = h.u;
        h.v = value8(s.v[i][u].z, s.v[i][u].w, d1);
        *(uint4*)(vb + 16 * u * Z::kVRow + 8) = h.u;
      }
    }
  }
}

template <int HD, int W, bool ONE>
__global__ __launch_bounds__(64 * W, HD > 128 || W > 4 ? 1 : 2) void attend_chunk_kernel(AttendArgs a, int lo_rows,
                                                                                         AttendParts parts) {
  using Z = ChunkSizes<HD, W>;
  constexpr int kRows = 32 * W;
  extern __shared__ __attribute__((aligned(16))) uint16_t s_buf[];
  const CachePlanes& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, hi = lane >> 5;
  const int b = (int)((uint32_t)blockIdx.x / (uint32_t)c.heads), kvh = blockIdx.x - b * c.heads;
  // the rows that see most first; behind the whole blocks the parts of those cut
  const int z = blockIdx.z, cut_z = z - (parts.blocks - parts.cut);
  const bool whole = cut_z < 0;
  const int nparts = whole ? 1 : parts.parts;
  const int down = whole ? 0 : (int)((uint32_t)cut_z / (uint32_t)nparts);
  const int block = whole ? parts.blocks - 1 - z : parts.cut - 1 - down;
  const int part = whole ? 0 : cut_z - down * nparts;
  int64_t q0;
  int nq, kv, pos0;
  sequence(a, b, q0, nq, kv, pos0);
  const int rows = nq * a.group;
  const int r0 = block * kRows;
  if (rows <= lo_rows || r0 >= rows) return;

  const int last_row = rows - 1 < r0 + kRows - 1 ? rows - 1 : r0 + kRows - 1;
  const int low_pos = pos0 + token_of(a, r0), high_pos = pos0 + token_of(a, last_row);
  const int lo = first_seen(a, low_pos < 0 ? 0 : low_pos), seen = high_pos + 1;  // [lo, seen): what the rows see
  int begin, end;
  part_steps(lo, seen, part, nparts, begin, end);

  // this wave's rows
  const int r = r0 + 32 * wave + col, qi = token_of(a, r);
  const int pos = pos0 + qi;
  const int wave_low = pos0 + token_of(a, r0 + 32 * wave);
  const int wave_last = r0 + 32 * wave + 31 < rows - 1 ? r0 + 32 * wave + 31 : rows - 1;
  const int wave_high = r0 + 32 * wave < rows ? pos0 + token_of(a, wave_last) : -1;  // no rows: sees nothing
  const int wave_first = first_seen(a, wave_low < 0 ? 0 : wave_low);
  const int first = first_seen(a, pos);
  const bool row_on = r < rows;
  const int64_t row_q = q0 + qi;
  const int head = kvh * a.group + r - qi * a.group;

  h8v q[HD / 16];
  load_query<HD / 16>(a, row_on, [&](int s) { return row_q * a.qs + (int64_t)head * a.qhs + 16 * s + 8 * hi; }, q);

  f16v o[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  auto lay_step = [&](const Staged<HD, W>& s, int tile, int pages, int buf) {
    const int j0 = tile * kTile;
    uint16_t* to = s_buf + buf * Z::kHalfs;
    if (j0 < lo || j0 + kTile > kv || __ballot(pages < 0) != 0)
      lay<HD, W, ONE, true>(s, j0, pages, lo, kv, to);
    else
      lay<HD, W, ONE, false>(s, j0, pages, lo, kv, to);
  };

  Staged<HD, W> st;
  int pages = settled<ONE>(step_page<ONE>(a, b, begin, end, kv));
  int next_pages = settled<ONE>(step_page<ONE>(a, b, begin + 1, end, kv));
  if (begin < end) {
    fetch<HD, W, ONE>(a, kvh, begin * kTile, pages, st);
    lay_step(st, begin, pages, 0);
  }
  __syncthreads();
  // K's LDS row of this lane: bits 2 and 3 exchanged
  const int krow = (col & 19) | ((col & 4) << 1) | ((col & 8) >> 1);
  for (int tile = begin, cur = 0; tile < end; tile++, cur ^= 1) {
    const int j0 = tile * kTile;
    const int after_pages = step_page<ONE>(a, b, tile + 2, end, kv);
    if (tile + 1 < end) fetch<HD, W, ONE>(a, kvh, j0 + kTile, next_pages, st);

    if (j0 <= wave_high && j0 + kTile > wave_first) {
      const uint16_t* kb = s_buf + cur * Z::kHalfs + krow * Z::kRow + 8 * hi;
      f16v s[2];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 16; d++)
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const h8v k = *(const h8v*)(kb + 32 * t * Z::kRow + 16 * d);
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[d], s[t], 0, 0, 0);
        }
      // kAhead reads in flight before the first product, then one a product
      __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
      for (int x = 0; x < HD / 8 - kAhead; x++) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kMfma, kAhead, 0);
      const uint64_t absent = ONE ? (pages < 0 ? 15 : 0) : __ballot(pages < 0) & 15;
      if (j0 + kTile - 1 > wave_low || (a.window > 0 && j0 <= (int64_t)wave_high - a.window) || absent) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int x = 32 * t + 16 * (i >> 3) + 8 * hi + (i & 7), j = j0 + x;
            if (j > pos || j < first || ((absent >> (x >> 4)) & 1)) s[t][i] = -INFINITY;
          }
      }
      float mt = s[0][0];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) mt = fmaxf(mt, s[t][i]);
      // the weights are relative to a maximum that follows the scores only once
      // one has outgrown it by 2^kSlack (exact in f16 and f32 alike)
      if (__ballot((mt - m) * a.sc > kSlack) != 0) {
        mt = fmaxf(mt, __shfl_xor(mt, 32, kWave));
        const float mn = fmaxf(m, mt), f = exp2_fast((m - (mn == -INFINITY ? 0.0f : mn)) * a.sc);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) o[d] *= f;
      }
      const float bs = m == -INFINITY ? 0.0f : m * a.sc;
      h8v p[4];
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float w = exp2_fast(__builtin_fmaf(s[t][i], a.sc, -bs));
          sum += w;
          p[2 * t + (i >> 3)][i & 7] = (_Float16)w;
        }
      l += sum;
      const uint16_t* vb = s_buf + cur * Z::kHalfs + kTile * Z::kRow + col * Z::kVRow + 8 * hi;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int d = 0; d < HD / 32; d++) {
          const h8v v = *(const h8v*)(vb + 32 * d * Z::kVRow + 16 * t);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[t], o[d], 0, 0, 0);
        }
      __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 1);
#pragma unroll
      for (int x = 0; x < HD / 8 - kAhead; x++) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 1);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 1);
      }
      __builtin_amdgcn_sched_group_barrier(kMfma, kAhead, 1);
    }
    if (tile + 1 < end) lay_step(st, tile + 1, next_pages, cur ^ 1);
    pages = next_pages;
    next_pages = settled<ONE>(after_pages);
    __syncthreads();
  }

  l += __shfl_xor(l, 32, kWave);
  if (!row_on) return;
  if (nparts > 1) {
    const int64_t pr = part_row(parts, (int64_t)blockIdx.x, block, part, r - r0);
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(f4v*)(parts.o + pr * HD + 32 * d + 2 * i + 4 * hi) = f4v{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
    if (hi == 0) {
      parts.ml[2 * pr] = m * a.sc;
      parts.ml[2 * pr + 1] = l;
    }
    return;
  }
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float acc[4] = {o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
      float out[4];
      finish_row<4>(a, head, m * a.sc, l, acc, out);
      store_out4(a, row_q * a.os + (int64_t)head * HD + 32 * d + 2 * i + 4 * hi, out);
    }
}

template <int HD, int W, bool ONE>
hipError_t launch_pages(const AttendArgs& a, int lo, const AttendParts& p, hipStream_t st) {
  if constexpr (ChunkSizes<HD, W>::kLds > 64 * 1024) {
    const hipError_t e = set_max_dynamic_lds<attend_chunk_kernel<HD, W, ONE>>();
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)(a.seqs * a.c.heads), 1, (unsigned)(p.blocks + p.cut * (p.parts - 1)));
  attend_chunk_kernel<HD, W, ONE><<<grid, 64 * W, ChunkSizes<HD, W>::kLds, st>>>(a, lo, p);
  return hipGetLastError();
}

template <int HD>
hipError_t launch_hd(const AttendArgs& a, int lo, const AttendParts& p, hipStream_t st) {
  if constexpr (HD <= 128)
    if (p.rows > 128)
      return a.c.page >= kTile ? launch_pages<HD, 8, true>(a, lo, p, st) : launch_pages<HD, 8, false>(a, lo, p, st);
  return a.c.page >= kTile ? launch_pages<HD, 4, true>(a, lo, p, st) : launch_pages<HD, 4, false>(a, lo, p, st);
}

}  // namespace

hipError_t launch_attend_chunk(const AttendArgs& a, int lo, const AttendParts& p, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  switch (a.c.hd) {
    case 64: return launch_hd<64>(a, lo, p, st);
    case 96: return launch_hd<96>(a, lo, p, st);
    case 128: return launch_hd<128>(a, lo, p, st);
    case 256: return launch_hd<256>(a, lo, p, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace qmm
