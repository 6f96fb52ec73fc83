// lora.hip — low-rank adapters of many requests beside a shared projection:
//   out[r] = y[r] + scales[i] * (x[r] A_i^T) B_i^T,  i = ids[r]
// for A [slots][rank][k] and B [slots][n][rank] of up to four projections of
// one activation; a row whose id names no slot keeps its y.
//
// Both products are bound by memory: of a row, A and B are read once and y goes in
// and out, 2 operations a byte of adapter for a row alone; many rows of one adapter
// share its A and B. So few rows are taken one by one on the vector units, and
// many are sorted by their adapters into tiles of 32, whose products run on the
// matrix cores (form_of, below). All sums are f32.
#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));

constexpr int kMostRank = 128;

// 8 values as they lie in memory, on their way to registers.
template <int T>
struct Raw {
  uint4 u[T == QMM_X_F32 ? 2 : 1];
  template <bool VEC>
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if (VEC) {
      const uint4* q = (const uint4*)((const char*)p + i * (T == QMM_X_F32 ? 4 : 2));
      u[0] = q[0];
      if (T == QMM_X_F32) u[sizeof(u) / 16 - 1] = q[1];
    } else if (T == QMM_X_F32) {
      const uint32_t* q = (const uint32_t*)p + i;
      u[0] = make_uint4(q[0], q[1], q[2], q[3]);
      u[sizeof(u) / 16 - 1] = make_uint4(q[4], q[5], q[6], q[7]);
    } else {
      const uint16_t* q = (const uint16_t*)p + i;
      u[0] = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16,
                        q[6] | (uint32_t)q[7] << 16);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(u) / 16); i++) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(float* v) const {
    const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (T == QMM_X_F32) {
        const uint4 h = u[sizeof(u) / 16 - 1];
        const uint32_t z[4] = {h.x, h.y, h.z, h.w};
        v[e] = __uint_as_float(w[e]);
        v[4 + e] = __uint_as_float(z[e]);
      } else {
        v[2 * e] = widen<T>(w[e] & 0xFFFFu);
        v[2 * e + 1] = widen<T>(w[e] >> 16);
      }
    }
  }
};

// A value as a sum of bf16 ones, and nothing left: 1 for a bf16 value, 2 for f16, 3
// for f32. The first is the nearest, so that what it leaves has no sign of its
// own: of a value of 2^e at least and under 2^(e+1) 2^(e-8) at most, of which the second leaves
// the third under 2^(e-16). (With the first cut off, the products that are left out reach
// 2^-21 of a product, all of one sign.) The second of three is cut off, not rounded:
// it cannot carry a sum of the two past the value, f32's largest among them.
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));
template <int T>
constexpr int kPieces = T == QMM_X_BF16 ? 1 : T == QMM_X_F16 ? 2 : 3;
// the nearest of a and b, side by side (one instruction)
__device__ __forceinline__ uint32_t nearest(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v{a, b}), b2v));
}
// their upper halves
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
template <int N>
__device__ __forceinline__ void pieces_of(float v[8], b8v out[N]) {
  constexpr float kMost = 0x1.fep127f;  // the largest bf16 value: f32 ones past it would round to infinity
#pragma unroll
  for (int p = 0; p < N; p++) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float a = v[2 * e], b = v[2 * e + 1];
      if (N == 3 && p == 0) {
        a = __builtin_amdgcn_fmed3f(a, -kMost, kMost);
        b = __builtin_amdgcn_fmed3f(b, -kMost, kMost);
      }
      w[e] = N == 3 && p == 1 ? upper_halves(a, b) : nearest(a, b);
    }
    out[p] = __builtin_bit_cast(b8v, make_uint4(w[0], w[1], w[2], w[3]));
    if (p + 1 < N) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[2 * e] -= __uint_as_float(w[e] << 16);
        v[2 * e + 1] -= __uint_as_float(w[e] & 0xFFFF0000u);
      }
    }
  }
}
template <int T>
__device__ __forceinline__ void pieces_of(const Raw<T>& r, b8v out[kPieces<T>]) {
  if constexpr (T == QMM_X_BF16) {
    out[0] = __builtin_bit_cast(b8v, r.u[0]);
  } else {
    float v[8];
    r.values(v);
    pieces_of<kPieces<T>>(v, out);
  }
}

// 8 values from i on. VEC: at an address that is a multiple of 16 bytes;
// otherwise a value at a time.
template <int T, bool VEC>
__device__ __forceinline__ void load_values(const void* p, int64_t i, float* v) {
  Raw<T> r;
  r.template load<VEC>(p, i);
  r.values(v);
}

// The adapter of row r, -1 without one.
__device__ __forceinline__ int id_of(const LoraArgs& a, int64_t r) {
  const int id = r < a.rows ? a.ids[r] : -1;
  return id >= 0 && id < a.slots ? id : -1;
}

// ---- rows one by one (decode batches: few rows of one adapter) --------------

// The products of a row of x with `J` rows of A, rows `lda` apart, over the
// 8-value units first, first + step, ... of k; lanes take units in turn.
template <int XT, int WT, bool VEC, int J>
__device__ __forceinline__ void dots(const void* x, int64_t xi, const void* w, int64_t wi, int64_t lda, int first, int step,
                                     int units, float* sum) {
#pragma unroll
  for (int j = 0; j < J; j++) sum[j] = 0.0f;
#pragma unroll 4
  for (int u = first; u < units; u += step) {
    float v[8];
    load_values<XT, VEC>(x, xi + 8 * u, v);
#pragma unroll
    for (int j = 0; j < J; j++) {
      float a[8];
      load_values<WT, true>(w, wi + j * lda + 8 * u, a);
#pragma unroll
      for (int e = 0; e < 8; e++) sum[j] = fmaf(a[e], v[e], sum[j]);
    }
  }
}

constexpr int kRowThreads = 512, kRowOut = 1024;

// A row's 1 + rank / 2 times k values of A and x at most, and 1024 outputs' B: bound
// by the latency of its loads (1 row of 4096 to 4096 by rank 16, FUSED, 6.1 us of
// which an empty launch is 2.6; 21 rows of it beside 2 x 1024 more outputs 10.4).
//
// kRowOut outputs of one row. FUSED: with the row's products with A, which each
// workgroup of the row makes for itself; otherwise they come from mid.
template <int XT, int WT, bool VEC, bool FUSED>
__global__ __launch_bounds__(kRowThreads) void lora_row_kernel(LoraArgs a) {
  __shared__ float s_mid[kMostRank];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const LoraTarget& t = a.t[blockIdx.z];
  const int64_t n0 = (int64_t)blockIdx.x * kRowOut, row = blockIdx.y;
  if (n0 >= t.n) return;
  const int id = id_of(a, row);
  if (id >= 0) {
    const float scale = t.scales ? t.scales[id] : 1.0f;
    if (FUSED) {
      constexpr int J = 2;  // of a multiple of 8
      for (int j = J * wave; j < t.rank; j += J * (kRowThreads / 64)) {
        float sum[J];
        dots<XT, WT, VEC, J>(a.x, row * a.xs, t.a, ((int64_t)id * t.rank + j) * a.k, a.k, lane, 64, (int)(a.k / 8), sum);
#pragma unroll
        for (int i = 0; i < J; i++) {
          const float v = wave_sum(sum[i]);
          if (lane == 0) s_mid[j + i] = v * scale;
        }
      }
    } else {
      for (int j = tid; j < t.rank; j += kRowThreads) s_mid[j] = t.mid[row * t.rank + j] * scale;
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kRowOut / kRowThreads; i++) {
    const int64_t n = n0 + i * kRowThreads + tid;
    if (n >= t.n) break;
    float v = t.y[row * t.ldy + n];
    if (id >= 0) {
      const int64_t at = ((int64_t)id * t.n + n) * t.rank;
      float sum = 0.0f;
#pragma unroll 2
      for (int j = 0; j < t.rank; j += 8) {
        float b[8];
        load_values<WT, true>(t.b, at + j, b);
#pragma unroll
        for (int e = 0; e < 8; e++) sum = fmaf(b[e], s_mid[j + e], sum);
      }
      v += sum;
    } else if (t.y == t.out) {
      return;
    }
    t.out[row * t.ldo + n] = v;
  }
}

// A row's products with 4 rows of A (more workgroups where rows are few, x read
// rank / 4 times from the caches: with the launch after it 64 rows of 8192 to 8192 by rank 64, each
// with an adapter of its own, 36 us, of 134 MB 3.7 TB/s), k dealt to the workgroup's waves.
template <int XT, int WT, bool VEC>
__global__ __launch_bounds__(256) void lora_row_down_kernel(LoraArgs a) {
  constexpr int J = 4;
  __shared__ float s_part[4][J];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const LoraTarget& t = a.t[blockIdx.z];
  const int64_t row = blockIdx.y;
  const int j0 = J * blockIdx.x, id = id_of(a, row);
  if (j0 >= t.rank || id < 0) return;
  float sum[J];
  dots<XT, WT, VEC, J>(a.x, row * a.xs, t.a, ((int64_t)id * t.rank + j0) * a.k, a.k, threadIdx.x, 256, (int)(a.k / 8), sum);
#pragma unroll
  for (int j = 0; j < J; j++) {
    const float v = wave_sum(sum[j]);
    if (lane == 0) s_part[wave][j] = v;
  }
  __syncthreads();
  if (threadIdx.x < J)
    t.mid[row * t.rank + j0 + threadIdx.x] =
        (s_part[0][threadIdx.x] + s_part[1][threadIdx.x]) + (s_part[2][threadIdx.x] + s_part[3][threadIdx.x]);
}

// ---- tiles of rows on the matrix cores (prompts) ----------------------------

constexpr int kTile = 32, kMostSlots = 4096;
// Waves of a down workgroup: few where registers leave a CU 12 waves or fewer (two
// workgroups of 8 would not fit, three of 4 do), and as 64 KiB of LDS allow.
constexpr int down_waves(int rt, int wt) { return rt > 4 && wt == QMM_X_F32 ? 2 : rt > 1 ? 4 : 8; }

// One workgroup, bound by its passes over the ids one after another (512 rows 4.7 us,
// 2000 6.7).
//
// Rows with one adapter together, in tiles of kTile: a tile's adapter in whose
// (-1: rows without one; kNoTile: past the last tile), its rows in order (-1:
// none). Which place a row has in its adapter's tiles does not matter: a row's
// results come from its own column of the matrix products.
constexpr int kNoTile = -2, kEarly = 4;

// A place among the rows of adapter id (-1: none is wanted), one addition for
// each adapter that a wave's rows have.
__device__ __forceinline__ int take_places(int id, int32_t* count) {
  const int lane = threadIdx.x & 63;
  int place = -1;
  uint64_t left = __ballot(id >= 0);
  while (left) {
    const int lead = __builtin_ctzll(left), who = __builtin_amdgcn_readlane(id, lead);
    const uint64_t same = __ballot(id == who);
    int first = 0;
    if (lane == lead) first = atomicAdd(&count[who], __popcll(same));
    first = __builtin_amdgcn_readlane(first, lead);
    if (id == who) place = first + __popcll(same & (((uint64_t)1 << lane) - 1));
    left &= ~same;
  }
  return place;
}

__global__ __launch_bounds__(1024) void lora_tiles_kernel(LoraArgs a, int tiles, int with_none) {
  extern __shared__ int32_t s_count[];  // [slots + 1] rows of an adapter, then the places given out
  int32_t* const s_first = s_count + a.slots + 1;  // [slots + 1] its first tile
  __shared__ int32_t s_waves[16];
  const int n = a.slots + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < n; i += 1024) s_count[i] = 0;
  __syncthreads();
  auto id_at = [&](int64_t r) {
    const int id = id_of(a, r);
    return id < 0 && with_none && r < a.rows ? a.slots : id;
  };
  int early[kEarly];  // the ids of the first rows, read once
#pragma unroll
  for (int e = 0; e < kEarly; e++) early[e] = id_at(e * 1024 + tid);
#pragma unroll
  for (int e = 0; e < kEarly; e++) (void)take_places(early[e], s_count);
  for (int64_t r = kEarly * 1024; r < a.rows; r += 1024) (void)take_places(id_at(r + tid), s_count);
  __syncthreads();
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + tid, count = i < n ? s_count[i] : 0, mine = (count + kTile - 1) / kTile;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d, 64);
      if (lane >= d) sum += up;
    }
    if (lane == 63) s_waves[wave] = sum;
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < 16; w++) {
      if (w < wave) before += s_waves[w];
      all += s_waves[w];
    }
    const int first = before + sum - mine;
    if (i < n) {
      s_first[i] = first;
      s_count[i] = 0;
      for (int t = 0; t < mine; t++) a.whose[first + t] = i < a.slots ? i : -1;
      for (int r = count; r < mine * kTile; r++) a.order[first * kTile + r] = -1;
    }
    base += all;
    __syncthreads();
  }
  for (int t = base + tid; t < tiles; t += 1024) a.whose[t] = kNoTile;
  auto put = [&](int64_t r, int id) {
    const int place = take_places(id, s_count);
    if (place >= 0) a.order[s_first[id] * kTile + place] = (int32_t)r;
  };
#pragma unroll
  for (int e = 0; e < kEarly; e++) put(e * 1024 + tid, early[e]);
  for (int64_t r = kEarly * 1024; r < a.rows; r += 1024) put(r + tid, id_at(r + tid));
}

// 16 bytes of a row.
template <int T, bool VEC>
__device__ __forceinline__ uint4 load16(const void* p, int64_t i) {
  if (VEC) return *(const uint4*)((const char*)p + i * (T == QMM_X_F32 ? 4 : 2));
  if (T == QMM_X_F32) {
    const uint32_t* q = (const uint32_t*)p + i;
    return make_uint4(q[0], q[1], q[2], q[3]);
  }
  const uint16_t* q = (const uint16_t*)p + i;
  return make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16,
                    q[6] | (uint32_t)q[7] << 16);
}

// A tile's rows x all ranks over one part of k, its steps of 32 dealt to the
// waves: lane (row, g) holds ranks 4 g .. 4 g + 3 of each 16 for rows `col` and
// 16 + col. x and A come in whole lines (consecutive lanes in one row) and change
// lanes in LDS of the wave's own: loaded as the products take them, a lane a row,
// every 16 bytes were a line looked up. Bound by x's bytes where rows are many (2000 rows
// of 28672 f32 by rank 64, f16: 62 us for 240 MB, 3.85 TB/s; a copy runs at 4.76), by
// the chain of its steps where they are few (512 rows of 4096 bf16, rank 32, two projections: 6.4).
template <int XT, int WT, int RT, bool VEC>
__global__ __launch_bounds__(64 * down_waves(RT, WT)) void lora_down_kernel(LoraArgs a, int tiles) {
  constexpr int R = 16 * RT, W = down_waves(RT, WT);
  // 16-byte chunks of a row's step, and loads a lane
  constexpr int C = XT == QMM_X_F32 ? 8 : 4, I = kTile * C / 64, WC = WT == QMM_X_F32 ? 8 : 4, WI = R * WC / 64;
  constexpr int kWaveBytes = 16 * (kTile * (C + 1) + R * (WC + 1)), kPartBytes = 16 * (R + 4) * 4;
  __shared__ __attribute__((aligned(16))) char s_mem[W * (kWaveBytes > kPartBytes ? kWaveBytes : kPartBytes)];
  uint4 (*const s_x)[C + 1] = (uint4 (*)[C + 1])(s_mem + kWaveBytes * (threadIdx.x >> 6));
  uint4 (*const s_w)[WC + 1] = (uint4 (*)[WC + 1])(s_x + kTile);
  float (*const s_part)[16][R + 4] = (float (*)[16][R + 4]) s_mem;
  // parts of k in eights: a part's tiles one after another on one XCD, whose L2 then holds the part's A
  const int turn = blockIdx.x >> 3;
  const int tile = a.splits % 8 ? (int)blockIdx.x % tiles : turn % tiles;
  const int part = a.splits % 8 ? (int)blockIdx.x / tiles : (int)(blockIdx.x & 7) + 8 * (turn / tiles);
  const int who = a.whose[tile];
  if (who < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const LoraTarget& t = a.t[blockIdx.y];
  const int32_t* rows = a.order + (int64_t)tile * kTile;
  const int64_t steps = a.k / 32;
  const int64_t begin = steps * part / a.splits, end = steps * (part + 1) / a.splits;
  int64_t xrow[I], arow[WI];
#pragma unroll
  for (int i = 0; i < I; i++)
    xrow[i] = (int64_t)max(0, rows[64 / C * i + lane / C]) * a.xs + 32 / C * (lane % C);
#pragma unroll
  for (int i = 0; i < WI; i++) {
    const int j = 64 / WC * i + lane / WC;
    arow[i] = ((int64_t)who * t.rank + (j < t.rank ? j : t.rank - 1)) * a.k + 32 / WC * (lane % WC);
  }
  f4v acc[2][RT];
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int i = 0; i < RT; i++) acc[h][i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  // two steps in flight; past the last one it is loaded again
  uint4 x[2][I];
  uint4 w[2][WI];
  auto load = [&](int b, int64_t s) {
    s = s < end ? s : end - 1;
#pragma unroll
    for (int i = 0; i < I; i++) x[b][i] = load16<XT, VEC>(a.x, xrow[i] + 32 * s);
#pragma unroll
    for (int i = 0; i < WI; i++) w[b][i] = load16<WT, true>(t.a, arow[i] + 32 * s);
  };
  // products of pieces down to 2^-16 of the first; of the next ones two f32 values have two,
  // f16 and f32 one, under 2^-24 of the product each. The larger ones first: in an
  // instruction a product's low bits are lost where larger ones stand beside it
  auto multiply = [&](int b) {
#pragma unroll
    for (int i = 0; i < I; i++) s_x[64 / C * i + lane / C][lane % C] = x[b][i];
#pragma unroll
    for (int i = 0; i < WI; i++) s_w[64 / WC * i + lane / WC][lane % WC] = w[b][i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    b8v xp[2][kPieces<XT>];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      Raw<XT> r;
#pragma unroll
      for (int u = 0; u < C / 4; u++) r.u[u] = s_x[16 * h + col][C / 4 * g + u];
      pieces_of<XT>(r, xp[h]);
    }
#pragma unroll
    for (int i = 0; i < RT; i++) {
      Raw<WT> r;
#pragma unroll
      for (int u = 0; u < WC / 4; u++) r.u[u] = s_w[16 * i + col][WC / 4 * g + u];
      b8v wp[kPieces<WT>];
      pieces_of<WT>(r, wp);
#pragma unroll
      for (int d = 0; d < 3; d++)
#pragma unroll
        for (int p = 0; p < kPieces<WT>; p++) {
          const int q = d - p;
          if (q >= 0 && q < kPieces<XT>) {
#pragma unroll
            for (int h = 0; h < 2; h++)
              acc[h][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wp[p], xp[h][q], acc[h][i], 0, 0, 0);
          }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  const int64_t mine = begin + wave;
  if (mine < end) load(0, mine);
  for (int64_t s = mine; s < end; s += 2 * W) {
    load(1, s + W);
    multiply(0);
    load(0, s + 2 * W);
    if (s + W < end) multiply(1);
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; i++) *(f4v*)&s_part[wave][col][16 * i + 4 * g] = acc[h][i];
    __syncthreads();
    for (int at = threadIdx.x; at < 16 * R; at += 64 * W) {
      const int r = at / R, j = at - r * R, row = rows[16 * h + r];
      if (row >= 0 && j < t.rank) {
        float v = s_part[0][r][j];
#pragma unroll
        for (int q = 1; q < W; q++) v += s_part[q][r][j];
        t.mid[(part * a.rows + row) * t.rank + j] = v;
      }
    }
  }
}

// The parts of k added, in the first one's place (512 rows, 24 parts, 3.5 us;
// 2000 rows by rank 64, 4.8).
__global__ __launch_bounds__(256) void lora_join_kernel(LoraArgs a) {
  const LoraTarget& t = a.t[blockIdx.y];
  const int64_t n = a.rows * t.rank, i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (i >= n) return;
  f4v v = *(const f4v*)(t.mid + i);
#pragma unroll 4
  for (int s = 1; s < a.splits; s++) v += *(const f4v*)(t.mid + s * n + i);
  *(f4v*)(t.mid + i) = v;
}

constexpr int kUpWaves = 4, kUpTiles = 4, kUpOut = 16 * kUpTiles * kUpWaves;

__device__ __forceinline__ f4v load_row4(const LoraTarget& t, const float* p, int64_t n) {
  if (t.vec && n + 4 <= t.n) return __builtin_nontemporal_load((const f4v*)(p + n));
  f4v y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int v = 0; v < 4; v++)
    if (n + v < t.n) y[v] = p[n + v];
  return y;
}
__device__ __forceinline__ void store_row4(const LoraTarget& t, float* p, int64_t n, f4v y) {
  if (t.vec && n + 4 <= t.n) {
    __builtin_nontemporal_store(y, (f4v*)(p + n));
    return;
  }
#pragma unroll
  for (int v = 0; v < 4; v++)
    if (n + v < t.n) p[n + v] = y[v];
}

// A tile's rows x 256 outputs, 64 a wave: lane (row, g) holds outputs 4 g .. 4 g + 3
// of each 16 for rows `col` and 16 + col, and takes the ranks 8 g .. 8 g + 7 of
// each of S runs of 32. They pass through LDS, so that y and out are read and
// written a row's 1 KiB at a time, past the caches. The workgroups of one
// range of outputs follow each other on one XCD (tiles fastest, ranges dealt to
// the XCDs), whose L2 then holds the range's B.
// Bound by y in and out: 512 rows of 2 x 14336 by rank 32 32 us for 117 MB, 3.6 TB/s;
// by rank 64 the pieces' products stand beside it (2000 rows of 8192, f16: 47 us
// for 131 MB; three products of a bf16 adapter for the five of an f16 one).
template <int WT, int S>
__global__ __launch_bounds__(64 * kUpWaves) void lora_up_kernel(LoraArgs a, int tiles) {
  constexpr int P = kTile / kUpWaves, MP = kPieces<QMM_X_F32>;
  // at ranks past 32 y comes after the products, whose registers it then takes: four workgroups a CU
  // for three (2000 rows of 8192 to 28672 by rank 64 166 us, 189 with y first; rank
  // 32 47 and 44, rank 128, which two fill either way, 173 and 169)
  constexpr bool LATE = S == 2;
  __shared__ float s_sum[kTile][kUpOut + 4];
  const LoraTarget& t = a.t[blockIdx.z];
  const int turn = blockIdx.x >> 3, tile = turn % tiles;
  const int64_t n0 = (int64_t)kUpOut * ((blockIdx.x & 7) + 8 * (turn / tiles));
  const int who = a.whose[tile];
  if (who == kNoTile || (who < 0 && t.y == t.out) || n0 >= t.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int32_t* rows = a.order + (int64_t)tile * kTile;
  f4v y[P];
  auto load_y = [&]() {
#pragma unroll
    for (int i = 0; i < P; i++) {
      const int64_t row = rows[kUpWaves * i + wave];
      y[i] = row >= 0 ? load_row4(t, t.y + row * t.ldy, n0 + 4 * lane) : f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
  };
  if (!LATE || who < 0) load_y();
  if (who >= 0) {
    Raw<WT> w[kUpTiles][S];
#pragma unroll
    for (int c = 0; c < kUpTiles; c++) {
      const int64_t n = n0 + 16 * (kUpTiles * wave + c) + col;
      const int64_t at = ((int64_t)who * t.n + (n < t.n ? n : t.n - 1)) * t.rank;
#pragma unroll
      for (int s = 0; s < S; s++) {
        const int j = 32 * s + 8 * g;
        w[c][s].zero();
        if (j < t.rank) w[c][s].template load<true>(t.b, at + j);
      }
    }
    const float scale = t.scales ? t.scales[who] : 1.0f;
    b8v m[2][S][MP];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t row = max(0, rows[16 * h + col]);
#pragma unroll
      for (int s = 0; s < S; s++) {
        const int j = 32 * s + 8 * g;
        float v[8];
        load_values<QMM_X_F32, true>(t.mid, row * t.rank + (j < t.rank ? j : 0), v);
#pragma unroll
        for (int q = 0; q < 8; q++) v[q] = j < t.rank ? v[q] * scale : 0.0f;
        pieces_of<MP>(v, m[h][s]);
      }
    }
#pragma unroll
    for (int c = 0; c < kUpTiles; c++) {
      f4v acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int s = 0; s < S; s++) {
        b8v wp[kPieces<WT>];
        pieces_of<WT>(w[c][s], wp);
#pragma unroll
        for (int d = 0; d < 3; d++)
#pragma unroll
          for (int p = 0; p < kPieces<WT>; p++) {
            const int q = d - p;
            if (q >= 0 && q < MP) {
#pragma unroll
              for (int h = 0; h < 2; h++)
                acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wp[p], m[h][s][q], acc[h], 0, 0, 0);
            }
          }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) *(f4v*)&s_sum[16 * h + col][16 * (kUpTiles * wave + c) + 4 * g] = acc[h];
    }
    if (LATE) load_y();
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int r = kUpWaves * i + wave;
    const int64_t row = rows[r];
    if (row < 0) continue;
    if (who >= 0) y[i] += *(const f4v*)&s_sum[r][4 * lane];
    store_row4(t, t.out + row * t.ldo, n0 + 4 * lane, y[i]);
  }
}

// Tiles that the rows can make: whole ones, and one begun for each adapter and for none.
int64_t tiles_of(const LoraArgs& a) {
  return (a.rows + kTile - 1) / kTile + (a.slots + 1 < a.rows ? a.slots + 1 : a.rows);
}

// How a call runs, all times of calls in a replayed graph (bf16 adapters, f32 x).
//
// Rows one by one read their A and B once a row, tiles once for 32 rows of one
// adapter, but a tile is as dear for one row as for 32, and the rows have to be sorted
// first. So rows one by one while all of them together read at most 3 * 2^25 values
// of A and B (and up to 1024 rows; us one by one / in tiles, a row's place by n and k; all rows
// with 1 adapter, or each with one of 64 in turn):
//     64 rows, rank 16, 4096 to 2 x 14336    38M values   14 / 23     20 / 48
//     32 rows, rank 64, 4096 to 2 x 14336    75M          28 / 26     48 / 53
//     128 rows, rank 32, 14336 to 4096       75M          20 / 26     29 / 43
//     16 rows, rank 128, 4096 to 2 x 14336   75M          28 / 30     50 / 67
//     128 rows, rank 64, 8192 to 8192        134M         34 / 27     55 / 67
//     256 rows, rank 16, 4096 to 2 x 14336   151M         31 / 28     50 / 76
//     64 rows, rank 64, 4096 to 2 x 14336    151M         44 / 28     80 / 81
//     128 rows, rank 64, 4096 to 2 x 14336   302M         77 / 32     144 / 106
//     512 rows, rank 64, 8192 to 8192        537M         110 / 36    165 / 80
// Where the line lies is a choice between the two columns: with many adapters it
// would lie higher (256 rows of 64 adapters lose some 25 us past it), with one lower. The
// table is of bf16 adapters, and so are its bytes: f32 ones read twice as many.
//
// Of rows one by one, the small ones in one launch: every workgroup of a row makes
// the row's products with A for itself, which a second launch would hand it. That
// is for an A of 2^16 values and while all workgroups together read at most 2^23
// of them: then the one launch takes 1.5 to 2 us less or at most 3 more (one
// launch / two: 1 row, rank 8, 896 to 896 4.7 / 6.7; 8 rows, rank 16, 4096 to
// 4096 7.3 / 7.5; 16 rows, rank 16, 4096 to 6144 10.5 / 9.0), and a call that no
// graph replays saves the host 4 us (8.4 / 12.3). Past it: 16 rows, rank 32, 4096
// to 2 x 14336 19.9 / 12.6.
enum Form { kFused, kRows, kTiles };

Form form_of(const LoraArgs& a) {
  int rank = 0;
  int64_t groups = 0, values = 0;
  for (int i = 0; i < a.count; i++) {
    rank = rank > a.t[i].rank ? rank : a.t[i].rank;
    groups += a.rows * ((a.t[i].n + kRowOut - 1) / kRowOut);
    values += a.rows * a.t[i].rank * (a.k + a.t[i].n);
  }
  if (a.rows > 1024 || values > (int64_t)3 << 25) return kTiles;
  return rank * a.k <= 1 << 16 && groups * rank * a.k <= 1 << 23 ? kFused : kRows;
}

// Parts of k: until the CUs have the 12 waves each that registers leave, of 4 steps
// a wave at least (us in parts / with k whole: 300 rows of 14336 by rank 32 29 / 69,
// 2000 by rank 64 79 / 132, 2000 of 4096 by rank 16 42 / 42; with twice the parts 29, 84, 42).
int splits_of(const LoraArgs& a, int cus) {
  if (form_of(a) != kTiles) return 1;
  int rank = 0;
  for (int i = 0; i < a.count; i++) rank = rank > a.t[i].rank ? rank : a.t[i].rank;
  const int waves = down_waves((rank + 15) / 16, QMM_X_BF16);
  const int64_t groups = (a.rows + kTile - 1) / kTile * a.count, most = a.k / (128 * waves);
  int64_t s = 12 / waves * cus / groups;
  s = s < most ? s : most;
  if (s > 8) s -= s % 8;  // parts that the XCDs share evenly
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}

template <int XT, int WT, int RT, bool VEC>
hipError_t launch_tiles(const LoraArgs& a, int64_t widest, int64_t rank, hipStream_t st) {
  const int64_t tiles = tiles_of(a), ranges = (widest + kUpOut - 1) / kUpOut;
  int with_none = 0;
  for (int i = 0; i < a.count; i++) with_none |= a.t[i].y != a.t[i].out;
  lora_tiles_kernel<<<1, 1024, 2 * (a.slots + 1) * sizeof(int32_t), st>>>(a, (int)tiles, with_none);
  lora_down_kernel<XT, WT, RT, VEC><<<dim3((unsigned)(tiles * a.splits), (unsigned)a.count), 64 * down_waves(RT, WT), 0, st>>>(a, (int)tiles);
  if (a.splits > 1)
    lora_join_kernel<<<dim3((unsigned)((a.rows * rank + 1023) / 1024), (unsigned)a.count), 256, 0, st>>>(a);
  lora_up_kernel<WT, (RT + 1) / 2><<<dim3((unsigned)((ranges + 7) / 8 * 8 * tiles), 1, (unsigned)a.count), 64 * kUpWaves, 0,
                                     st>>>(a, (int)tiles);
  return hipGetLastError();
}

template <int XT, int WT, bool VEC>
hipError_t launch_form(const LoraArgs& a, hipStream_t st) {
  int64_t widest = 0, rank = 0;
  for (int i = 0; i < a.count; i++) {
    widest = widest > a.t[i].n ? widest : a.t[i].n;
    rank = rank > a.t[i].rank ? rank : a.t[i].rank;
  }
  const Form form = form_of(a);
  if (form == kTiles) {
    if (rank <= 16) return launch_tiles<XT, WT, 1, VEC>(a, widest, rank, st);
    if (rank <= 32) return launch_tiles<XT, WT, 2, VEC>(a, widest, rank, st);
    if (rank <= 64) return launch_tiles<XT, WT, 4, VEC>(a, widest, rank, st);
    return launch_tiles<XT, WT, 8, VEC>(a, widest, rank, st);
  }
  const dim3 grid((unsigned)((widest + kRowOut - 1) / kRowOut), (unsigned)a.rows, (unsigned)a.count);
  if (form == kFused) {
    lora_row_kernel<XT, WT, VEC, true><<<grid, kRowThreads, 0, st>>>(a);
  } else {
    lora_row_down_kernel<XT, WT, VEC><<<dim3((unsigned)(rank / 4), (unsigned)a.rows, (unsigned)a.count), 256, 0, st>>>(a);
    lora_row_kernel<XT, WT, VEC, false><<<grid, kRowThreads, 0, st>>>(a);
  }
  return hipGetLastError();
}

template <int XT, int WT>
hipError_t launch_types(const LoraArgs& a, hipStream_t st) {
  return a.x_vec ? launch_form<XT, WT, true>(a, st) : launch_form<XT, WT, false>(a, st);
}

template <int XT>
hipError_t launch_x(const LoraArgs& a, int wdt, hipStream_t st) {
  switch (wdt) {
    case QMM_X_F16: return launch_types<XT, QMM_X_F16>(a, st);
    case QMM_X_BF16: return launch_types<XT, QMM_X_BF16>(a, st);
    default: return launch_types<XT, QMM_X_F32>(a, st);
  }
}

}  // namespace

int lora_most_rank() { return kMostRank; }
int lora_most_slots() { return kMostSlots; }

// A launch's threads in x stay below 2^32.
bool lora_fits(const LoraArgs& a) {
  if (form_of(a) != kTiles) return true;
  int64_t widest = 0;
  for (int i = 0; i < a.count; i++) widest = widest > a.t[i].n ? widest : a.t[i].n;
  return (widest / kUpOut + 8) * tiles_of(a) < ((int64_t)1 << 32) / (64 * kUpWaves);
}

size_t lora_plan(LoraArgs& a, void* ws, int cus) {
  a.splits = splits_of(a, cus);
  if (form_of(a) == kFused) return 0;
  size_t at = 0;
  for (int i = 0; i < a.count; i++) {
    a.t[i].mid = (float*)((uintptr_t)ws + at);
    at += align_up((size_t)a.splits * a.rows * a.t[i].rank * sizeof(float), 16);
  }
  if (form_of(a) == kTiles) {
    a.order = (int32_t*)((uintptr_t)ws + at);
    at += tiles_of(a) * kTile * sizeof(int32_t);
    a.whose = (int32_t*)((uintptr_t)ws + at);
    at += align_up(tiles_of(a) * sizeof(int32_t), 16);
  }
  return at;
}

hipError_t launch_lora(const LoraArgs& a, int xdt, int wdt, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  switch (xdt) {
    case QMM_X_F16: return launch_x<QMM_X_F16>(a, wdt, st);
    case QMM_X_BF16: return launch_x<QMM_X_BF16>(a, wdt, st);
    default: return launch_x<QMM_X_F32>(a, wdt, st);
  }
}

}  // namespace qmm
