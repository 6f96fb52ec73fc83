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
// Chunks of 2000 and 1333 tokens over 7777 and 5832 (64 query heads on 8 of 128
// dims) take 741-781 us from card to card, 0.86-0.90 PFLOP/s; a library product of 8192^3
// reaches 1.15.
// The products, the softmax's and the conversions' vector instructions (about
// 290 a wave and step with 128 rows a workgroup, 235 with 256) and the LDS reads
// (32 operands of 1 KiB a wave and step) each take a third to a half of a step
// and overlap only between the two waves of a SIMD. Tried and slower: a step's
// scores beside the weights of the one before (the second set of scores spills
// at 256 registers), steps of 32 positions, 64 rows a wave (accumulators past 256
// registers are copied back and forth each step), and products and vector
// instructions interleaved by hand.
#include "attend.h"
#include "mv_common.h"

namespace qmm {

namespace {

// A kernel's arguments, all of them.
struct ChunkCall {
  AttendArgs a;
  AttendParts parts;
  int lo_rows;
};

// Read afresh where they are wanted: 60 registers of arguments that live through
// a block's steps would push what a step needs out of the scalar registers
// (into lanes of vector registers and back, 136 moves a step).
__device__ __forceinline__ ChunkCall call_args() {
  auto p = (const __attribute__((address_space(4))) ChunkCall*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  ChunkCall c;
  __builtin_memcpy(&c, (const ChunkCall*)p, sizeof c);
  return c;
}

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
__device__ __forceinline__ int k_item(int tid, int i, bool& on) {
  const int x = tid + ChunkSizes<HD, W>::kThreads * i;
  on = ChunkSizes<HD, W>::kItems % ChunkSizes<HD, W>::kThreads == 0 || x < ChunkSizes<HD, W>::kItems;
  return x;
}
template <int HD, int W>
__device__ __forceinline__ int v_item(int tid, int i, bool& on) {
  if (!ChunkSizes<HD, W>::kHalves) return k_item<HD, W>(tid, i, on);
  const int x = tid - ChunkSizes<HD, W>::kThreads / 2;
  on = x >= 0 && x < ChunkSizes<HD, W>::kItems;
  return x;
}

// The lower dim of item x of values: 16 dims of a block, then the next block's.
__device__ __forceinline__ int v_dim(int x) { return (x >> 6) * 32 + ((x >> 2) & 15); }

// A step's pages. ONE: pages of 64 positions and more, so a step has one, the
// same for the wave; otherwise lane x < 4 of every wave holds that of the step's
// x-th 16 positions. -1: none.
// The table's entry (-1 behind the last), looked at only in settled() so
// that nothing waits for it meanwhile.
template <bool ONE>
__device__ __forceinline__ int step_page(const AttendArgs& a, int tid, int b, int tile, int end, int kv) {
  const int j = tile * kTile + (ONE ? 0 : 16 * (tid & 3));
  return tile < end && j < kv ? a.tables[(int64_t)b * a.table_stride + (j >> a.page_bits)] : -1;
}
// ONE: into a scalar register.
template <bool ONE>
__device__ __forceinline__ int settled(const AttendArgs& a, int page) {
  if (page >= a.c.pages) page = -1;
  return ONE ? __builtin_amdgcn_readfirstlane(page) : page;
}

template <int HD, int W, bool ONE>
__device__ __forceinline__ void fetch(const AttendArgs& a, int tid, int kvh, int j0, int pages, Staged<HD, W>& s) {
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
    const int xk = k_item<HD, W>(tid, i, k_on), xv = v_item<HD, W>(tid, i, v_on);
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
__device__ __forceinline__ void lay(const Staged<HD, W>& s, int tid, int j0, int pages, int lo, int hi, uint16_t* buf) {
  using Z = ChunkSizes<HD, W>;
#pragma unroll
  for (int i = 0; i < Z::kEach; i++) {
    bool k_on, v_on;
    const int xk = k_item<HD, W>(tid, i, k_on), xv = v_item<HD, W>(tid, i, v_on);
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

// The steps of one block of 32 W query rows of kv head kvh of sequence b: its
// rows from r0 on, steps [begin, end) of those that its rows see. Partial rows
// from part_at on, or (-1) the outputs themselves. Ends with the workgroup's
// waves past their last use of LDS.
template <int HD, int W, bool ONE>
__device__ __forceinline__ void attend_block(int tid, int b, int kvh, int64_t q0, int rows, int kv, int pos0, int r0,
                                             int lo, int begin, int end, int64_t part_at, uint16_t* s_buf) {
  using Z = ChunkSizes<HD, W>;
  const ChunkCall call = call_args();
  const AttendArgs& a0 = call.a;
  const int lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, hi = lane >> 5;

  // this wave's rows
  const int r = r0 + 32 * wave + col, qi = token_of(a0, r);
  const int pos = pos0 + qi;
  const int wave_low = pos0 + token_of(a0, r0 + 32 * wave);
  const int wave_last = r0 + 32 * wave + 31 < rows - 1 ? r0 + 32 * wave + 31 : rows - 1;
  const int wave_high = r0 + 32 * wave < rows ? pos0 + token_of(a0, wave_last) : -1;  // no rows: sees nothing
  const int wave_first = first_seen(a0, wave_low < 0 ? 0 : wave_low);
  const int first = first_seen(a0, pos);
  const bool row_on = r < rows;
  const int64_t row_q = q0 + qi;
  const int head = kvh * a0.group + r - qi * a0.group;

  h8v q[HD / 16];
  load_query<HD / 16>(a0, row_on, [&](int s) { return row_q * a0.qs + (int64_t)head * a0.qhs + 16 * s + 8 * hi; }, q);

  f16v o[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
  float m = -INFINITY, l = 0.0f, bs = 0.0f;  // bs: m sc - kLift, what the weights' exponents are less (far: m is taken off before)
  bool far = false;  // some row's maximum is past kFar (the same for the wave)
  const ChunkCall in_steps = call_args();
  const AttendArgs& a = in_steps.a;

  auto lay_step = [&](const Staged<HD, W>& s, int tile, int pages, int buf) {
    const int j0 = tile * kTile;
    uint16_t* to = s_buf + buf * Z::kHalfs;
    if (j0 < lo || j0 + kTile > kv || __ballot(pages < 0) != 0)
      lay<HD, W, ONE, true>(s, tid, j0, pages, lo, kv, to);
    else
      lay<HD, W, ONE, false>(s, tid, j0, pages, lo, kv, to);
  };

  Staged<HD, W> st;
  int pages = settled<ONE>(a, step_page<ONE>(a, tid, b, begin, end, kv));
  int next_pages = settled<ONE>(a, step_page<ONE>(a, tid, b, begin + 1, end, kv));
  if (begin < end) {
    fetch<HD, W, ONE>(a, tid, kvh, begin * kTile, pages, st);
    lay_step(st, begin, pages, 0);
  }
  __syncthreads();
  // K's LDS row of this lane: bits 2 and 3 exchanged
  const int krow = (col & 19) | ((col & 4) << 1) | ((col & 8) >> 1);
  for (int tile = begin, cur = 0; tile < end; tile++, cur ^= 1) {
    const int j0 = tile * kTile;
    const int after_pages = step_page<ONE>(a, tid, b, tile + 2, end, kv);
    if (tile + 1 < end) fetch<HD, W, ONE>(a, tid, kvh, j0 + kTile, next_pages, st);

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
      if (__ballot((mt - m) * a.sc > kSlack) != 0 || far) {
        mt = fmaxf(mt, __shfl_xor(mt, 32, kWave));
        const float mn = fmaxf(m, mt), to = mn == -INFINITY ? 0.0f : mn, f = weight_of(a, m, to);
        far = __ballot(fabsf(to) * a.sc > kFar) != 0;
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) o[d] *= f;
        bs = far ? -kLift : __builtin_fmaf(to, a.sc, -kLift);
        if (far)
#pragma unroll
          for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[t][i] -= to;
      }
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
    next_pages = settled<ONE>(a, after_pages);
    __syncthreads();
  }

  l += __shfl_xor(l, 32, kWave);
  if (!row_on) return;
  const ChunkCall after = call_args();
  if (part_at >= 0) {
    const AttendParts& parts = after.parts;
    const int64_t pr = part_at + r - r0;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(f4v*)(parts.o + pr * HD + 32 * d + 2 * i + 4 * hi) = f4v{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
    if (hi == 0) {
      parts.ml[2 * pr] = m;
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
      finish_row<4>(after.a, head, m, l, acc, out);
      store_out4(after.a, row_q * after.a.os + (int64_t)head * HD + 32 * d + 2 * i + 4 * hi, out);
    }
}

// What the rows of a block see: positions [lo, seen).
__device__ __forceinline__ void block_sees(const AttendArgs& a, int rows, int pos0, int r0, int block_rows, int& lo,
                                           int& seen) {
  const int last_row = rows - 1 < r0 + block_rows - 1 ? rows - 1 : r0 + block_rows - 1;
  const int low = pos0 + token_of(a, r0);
  lo = first_seen(a, low < 0 ? 0 : low);
  seen = pos0 + token_of(a, last_row) + 1;
}

// A workgroup a block of 32 W rows, or a part of one.
template <int HD, int W, bool ONE>
__global__ __launch_bounds__(64 * W, HD > 128 || W > 4 ? 1 : 2) void attend_chunk_kernel(ChunkCall call) {
  constexpr int kRows = 32 * W;
  const AttendArgs& a = call.a;
  const AttendParts& parts = call.parts;
  extern __shared__ __attribute__((aligned(16))) uint16_t s_buf[];
  // the rows that see most first, every head's block in a row of the grid; then
  // the parts of the rows of blocks that are cut, and last what a row cut for its
  // last heads only has more than the first parts, which stand in that row
  const int heads = gridDim.x, z = blockIdx.z, top = parts.blocks - parts.cut_rows;
  int hs = blockIdx.x, block = parts.blocks - 1 - z, part = 0, nparts = 1;
  if (z < top) {
    if (z == top - 1 && hs >= heads - parts.cut_more) nparts = parts.parts;
  } else {
    nparts = parts.parts;
    const int row = z - top, down = (int)((uint32_t)row / (uint32_t)nparts);
    part = row - down * nparts;
    block = parts.cut_rows - 1 - down;
    if (block < 0) {
      const uint32_t at = (uint32_t)(row - parts.cut_rows * nparts) * heads + hs, more = parts.cut_more;
      if (at >= more * (nparts - 1)) return;  // the grid's last row
      const uint32_t n = at / more;
      part = 1 + (int)n;
      block = parts.cut_rows;
      hs = heads - (int)(more - (at - n * more));
    }
  }
  const int b = (int)((uint32_t)hs / (uint32_t)a.c.heads), kvh = hs - b * a.c.heads;
  int64_t q0;
  int nq, kv, pos0;
  sequence(a, b, q0, nq, kv, pos0);
  const int rows = nq * a.group, r0 = block * kRows;
  if (rows <= call.lo_rows || r0 >= rows) return;
  int lo, seen, begin, end;
  block_sees(a, rows, pos0, r0, kRows, lo, seen);
  part_steps(lo, seen, part, nparts, begin, end);
  attend_block<HD, W, ONE>(threadIdx.x, b, kvh, q0, rows, kv, pos0, r0, lo, begin, end,
                           nparts > 1 ? part_row(parts, cut_index(a, parts, hs, block), part, 0) : -1, s_buf);
}

// The blocks of 256 rows of a sequence's kv head as lengths of work: block j's
// is first + more * j (the positions that its rows see, times the group, and
// four steps more for its beginning and end). An estimate: all that the shares
// ask of it is that every workgroup finds the same.
struct BlockWork {
  int64_t first;
  int more, blocks;
  __device__ __forceinline__ int64_t before(int j) const { return first * j + (int64_t)more * j * (j - 1) / 2; }
};
__device__ __forceinline__ BlockWork block_work(const AttendArgs& a, int nq, int kv, int pos0, int lo_rows) {
  const int rows = nq * a.group;
  BlockWork w;
  w.blocks = rows <= lo_rows ? 0 : (rows + kShareRows - 1) / kShareRows;
  const bool cut = a.window > 0 && a.window < kv;
  w.more = cut ? 0 : kShareRows;
  w.first = (int64_t)((cut ? (int)a.window : pos0 < 0 ? 0 : pos0) + 4 * kTile) * a.group + kShareRows;
  return w;
}

// Where a share stands: in LDS, for a step wants the scalar registers itself.
struct ShareAt {
  int64_t wave[8];
  int64_t each, u, end;  // a share's length, the place of the piece at hand, the share's end
  int64_t base;          // the work before sequence b
  int b, kvh, block;     // the piece's (b: -1 behind a sequence's last block)
};

// The sequence whose work place u falls into (s.b) and the work before it
// (s.base). START: u is that of share w of n, found with the share's length and
// end. Every thread of the workgroup calls; ends with a barrier.
template <bool START>
__device__ __forceinline__ void find_sequence(const ChunkCall& c, int tid, int w, ShareAt& s) {
  const AttendArgs& a = c.a;
  const int lane = tid & 63, wv = tid >> 6;
  int64_t u = START ? -1 : s.u, all = 0;
  // the work of all sequences, then (START) the place among them: in one pass where 512 threads have one each
  for (int pass = START && a.seqs > 512 ? 0 : 1; pass < 2; pass++) {
    all = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 512) {
      int64_t mine = 0;
      if (b0 + tid < a.seqs) {
        int64_t q0;
        int nq, kv, pos0;
        sequence(a, b0 + tid, q0, nq, kv, pos0);
        const BlockWork bw = block_work(a, nq, kv, pos0, c.lo_rows);
        mine = bw.before(bw.blocks) * a.c.heads;
      }
      int64_t upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t t = __shfl_up(upto, d, kWave);
        if (lane >= d) upto += t;
      }
      __syncthreads();
      if (lane == 63) s.wave[wv] = upto;
      __syncthreads();
      int64_t before = all;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (i < wv) before += s.wave[i];
        all += s.wave[i];
      }
      before += upto - mine;
      if (START && pass == 1 && u < 0) {
        // 8 steps of a block at least
        const int64_t least = (int64_t)8 * kTile * a.group, even = (all + c.parts.shares - 1) / c.parts.shares;
        const int64_t each = even < least ? least : even;
        u = w * each;
        if (tid == 0) {
          s.each = each;
          s.u = u;
          s.end = u + each < all ? u + each : all;
        }
      }
      if (u >= before && u < before + mine) {
        s.b = b0 + tid;
        s.base = before;
      }
    }
    if (START && pass == 0) {
      const int64_t least = (int64_t)8 * kTile * a.group, even = (all + c.parts.shares - 1) / c.parts.shares;
      const int64_t each = even < least ? least : even;
      u = w * each;
      if (tid == 0) {
        s.each = each;
        s.u = u;
        s.end = u + each < all ? u + each : all;
      }
    }
  }
  __syncthreads();
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
  return ((int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// A place x of a block's work (its length `work`) as one of its steps, at least 3
// steps from either end of the block or on it.
__device__ __forceinline__ int step_at(int64_t x, int64_t work, int steps) {
  const int s = (int)((double)x * steps / (double)work);
  return s < 3 ? 0 : steps - s < 3 ? steps : s;
}

// The blocks of 256 rows of all sequences and kv heads in a row, dealt to the
// workgroups in equal lengths of work: a share begins and ends inside a block
// as it falls, and what it leaves of one is joined by attend_join_shares_kernel
// (attend.hip). Ragged batches so keep all CUs busy to the end: chunks of 2000
// and 1333 tokens over 7777 and 5832, 840 blocks of 71 to 122 steps, took 887 us
// a block a workgroup.
template <int HD, bool ONE>
__global__ __launch_bounds__(512, 1) void attend_shares_kernel(ChunkCall) {
  extern __shared__ __attribute__((aligned(16))) uint16_t s_buf[];
  ShareAt& s = *(ShareAt*)(s_buf + 2 * ChunkSizes<HD, 8>::kHalfs);  // behind the two buffers
  for (bool start = true;; start = false) {
    const ChunkCall call = call_args();
    const AttendArgs& a = call.a;
    // (anew each time: what follows from it would live through the steps from outside the loop, 38 registers)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    // neighbours in the row on one XCD (workgroups go to the 8 in turn): they share keys and values
    const int n = call.parts.shares, id = blockIdx.x, w = n % 8 == 0 ? (id & 7) * (n / 8) + (id >> 3) : id;
    bool found = start;
    if (start) {
      if (tid == 0) call.parts.split[w] = make_int4(0, 0, 0, -1);
      find_sequence<true>(call, tid, w, s);
    } else {
      __syncthreads();
    }
    const int64_t u = uniform(s.u), u1 = uniform(s.end), each = uniform(s.each);
    if (u >= u1) return;
    if (!start && __builtin_amdgcn_readfirstlane(s.b) < 0) {
      find_sequence<false>(call, tid, w, s);
      found = true;
    }
    const int b = __builtin_amdgcn_readfirstlane(s.b);
    int64_t q0;
    int nq, kv, pos0;
    sequence(a, b, q0, nq, kv, pos0);
    q0 = uniform(q0);  // (read through vector registers: what a block's steps take from these is scalar)
    nq = __builtin_amdgcn_readfirstlane(nq);
    kv = __builtin_amdgcn_readfirstlane(kv);
    pos0 = __builtin_amdgcn_readfirstlane(pos0);
    const BlockWork bw = block_work(a, nq, kv, pos0, call.lo_rows);
    int kvh, block;
    int64_t from = u;
    if (found) {
      const int64_t per_head = bw.before(bw.blocks), in = u - uniform(s.base);
      kvh = (int)(in / per_head);
      const int64_t at = in - kvh * per_head;
      block = 0;
      for (int d = 1 << (31 - __builtin_clz(bw.blocks)); d; d >>= 1)
        if (block + d < bw.blocks && bw.before(block + d) <= at) block += d;
      from = u - at + bw.before(block);
    } else {
      kvh = s.kvh;
      block = s.block;
    }
    kvh = __builtin_amdgcn_readfirstlane(kvh);
    block = __builtin_amdgcn_readfirstlane(block);
    const int64_t work = bw.first + (int64_t)bw.more * block, to = from + work;
    const int rows = nq * a.group, r0 = block * kShareRows;
    int lo, seen, t0, t1;
    block_sees(a, rows, pos0, r0, kShareRows, lo, seen);
    part_steps(lo, seen, 0, 1, t0, t1);
    const int steps = t1 - t0;
    const int begin = __builtin_amdgcn_readfirstlane(start ? step_at(u - from, work, steps) : 0);
    const int end = __builtin_amdgcn_readfirstlane(to <= u1 ? steps : step_at(u1 - from, work, steps));
    __syncthreads();
    if (tid == 0) {
      const bool head_left = block + 1 < bw.blocks, left = head_left || kvh + 1 < a.c.heads;
      s.u = to;
      s.block = head_left ? block + 1 : 0;
      s.kvh = head_left ? kvh : kvh + 1;
      if (!left) s.b = -1;
      if (begin == 0 && end > 0 && end < steps) {
        int64_t last = (to - 1) / each;  // the share that takes the block's last steps
        while (step_at(last * each - from, work, steps) == steps) last--;
        call.parts.split[w] = make_int4(b, kvh, block, (int)last);
      }
    }
    // (a boundary moved to the block's first or last step leaves a share nothing of it)
    if (steps > 0 && (begin == steps || (begin == 0 && end == 0))) continue;
    const int64_t part_at = begin == 0 && end == steps ? -1 : share_row(begin > 0 ? 2 * w : 2 * w + 1, 0);
    attend_block<HD, 8, ONE>(tid, b, kvh, q0, rows, kv, pos0, r0, lo, t0 + begin, t0 + end, part_at, s_buf);
  }
}

template <int HD, int W, size_t kMore, auto Kernel>
hipError_t launch_pages(const dim3& grid, const AttendArgs& a, int lo, const AttendParts& p, hipStream_t st) {
  constexpr size_t kLds = ChunkSizes<HD, W>::kLds + kMore;
  static_assert(ChunkSizes<HD, W>::kLds % alignof(ShareAt) == 0, "where the search's place lies");
  if constexpr (kLds > 64 * 1024) {
    const hipError_t e = set_max_dynamic_lds<Kernel>();
    if (e != hipSuccess) return e;
  }
  Kernel<<<grid, 64 * W, kLds, st>>>(ChunkCall{a, p, lo});
  return hipGetLastError();
}

template <int HD>
hipError_t launch_hd(const AttendArgs& a, int lo, const AttendParts& p, hipStream_t st) {
  const bool one = a.c.page >= kTile;
  const int64_t heads = (int64_t)a.seqs * a.c.heads, more = (int64_t)p.cut_more * (p.parts - 1);
  const dim3 grid((unsigned)heads, 1, (unsigned)(p.blocks + p.cut_rows * (p.parts - 1) + (more + heads - 1) / heads));
  if constexpr (HD <= 128) {
    const dim3 shares((unsigned)p.shares);
    if (p.shares)
      return one ? launch_pages<HD, 8, sizeof(ShareAt), attend_shares_kernel<HD, true>>(shares, a, lo, p, st)
                 : launch_pages<HD, 8, sizeof(ShareAt), attend_shares_kernel<HD, false>>(shares, a, lo, p, st);
    if (p.rows > 128)
      return one ? launch_pages<HD, 8, 0, attend_chunk_kernel<HD, 8, true>>(grid, a, lo, p, st)
                 : launch_pages<HD, 8, 0, attend_chunk_kernel<HD, 8, false>>(grid, a, lo, p, st);
  }
  return one ? launch_pages<HD, 4, 0, attend_chunk_kernel<HD, 4, true>>(grid, a, lo, p, st)
             : launch_pages<HD, 4, 0, attend_chunk_kernel<HD, 4, false>>(grid, a, lo, p, st);
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
