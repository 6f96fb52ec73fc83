// lora.hip — low-rank adapters of many requests beside a shared projection:
//   out[r] = y[r] + scales[i] * (x[r] A_i^T) B_i^T,  i = ids[r]
// for A [slots][rank][k] and B [slots][n][rank] of up to four projections of
// one activation; a row whose id names no slot keeps its y.
//
// Two launches: x against A into partial results in f32 (k in parts where the
// rows alone do not fill the CUs), and those against B, y added.
#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));

// Values [i, i + N) of an array of type T, N * its size a multiple of 8 bytes.
// VEC: at 8 * that size's alignment; otherwise a value at a time.
template <int T, int N, bool VEC>
__device__ __forceinline__ void load_values(const void* p, int64_t i, float* v) {
#pragma unroll
  for (int e = 0; e < N; e += 4) load4<T, VEC>(p, i + e, v + e);
}

// The rows of a tile that `id` holds: lanes whose row is of the adapter next in
// turn. `left` has a bit for each of the tile's 16 rows still to be served.
struct Turn {
  uint32_t left;
  __device__ __forceinline__ explicit Turn(int id) { left = (uint32_t)__ballot(id >= 0) & 0xFFFFu; }
  // the next adapter (the same for the wave), its rows taken off
  __device__ __forceinline__ int next(int id) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    left &= ~(uint32_t)__ballot(id == a);
    return a;
  }
};

// The adapter of row r, -1 without one.
__device__ __forceinline__ int id_of(const LoraArgs& a, int64_t r) {
  const int id = r < a.rows ? a.ids[r] : -1;
  return id >= 0 && id < a.slots ? id : -1;
}

constexpr int kDownWaves = 4;

// 16 rows x all ranks over one part of k: lane (row, g) holds ranks 4 g .. 4 g + 3 of each 16.
template <int XT, int WT, int RT, bool VEC>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(LoraArgs a) {
  constexpr int R = 16 * RT;
  __shared__ float s_part[kDownWaves][16][R + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const LoraTarget& t = a.t[blockIdx.z];
  const int64_t row = (int64_t)blockIdx.x * 16 + col;
  const int id = id_of(a, row);
  const int64_t steps = a.k / 32;
  const int64_t begin = steps * blockIdx.y / a.splits, end = steps * (blockIdx.y + 1) / a.splits;
  const int64_t xrow = (row < a.rows ? row : a.rows - 1) * a.xs;
  for (Turn turn(id); turn.left;) {
    const int who = turn.next(id);
    f4v acc[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) acc[i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t s = begin + wave; s < end; s += kDownWaves) {
      const int64_t e = 32 * s + 8 * g;
      float x[8];
      load_values<XT, 8, VEC>(a.x, xrow + e, x);
#pragma unroll
      for (int i = 0; i < RT; i++) {
        float w[8];
        const int j = 16 * i + col;
        load_values<WT, 8, true>(t.a, ((int64_t)who * t.rank + (j < t.rank ? j : t.rank - 1)) * a.k + e, w);
#pragma unroll
        for (int q = 0; q < 8; q++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[q], x[q], acc[i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < RT; i++) *(f4v*)&s_part[wave][col][16 * i + 4 * g] = acc[i];
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * R; x += 64 * kDownWaves) {
      const int r = x / R, j = x - r * R;
      const int64_t at = (int64_t)blockIdx.x * 16 + r;
      if (j < t.rank && id_of(a, at) == who) {
        float v = s_part[0][r][j];
#pragma unroll
        for (int w = 1; w < kDownWaves; w++) v += s_part[w][r][j];
        t.mid[(blockIdx.y * a.rows + at) * t.rank + j] = v;
      }
    }
    __syncthreads();
  }
}

constexpr int kUpWaves = 4, kUpTiles = 4;

// 16 rows x 64 outputs a wave: lane (row, g) holds outputs 4 g .. 4 g + 3 of each 16.
template <int WT, int RT>
__global__ __launch_bounds__(64 * kUpWaves) void lora_up_kernel(LoraArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const LoraTarget& t = a.t[blockIdx.z];
  const int64_t n0 = ((int64_t)blockIdx.x * kUpWaves + wave) * 16 * kUpTiles;
  if (n0 >= t.n) return;
  const int64_t row = (int64_t)blockIdx.y * 16 + col;
  const int id = id_of(a, row);
  const bool in = row < a.rows;
  f4v y[kUpTiles];
#pragma unroll
  for (int i = 0; i < kUpTiles; i++) {
    const int64_t n = n0 + 16 * i + 4 * g;
    y[i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    if (!in) continue;
    if (t.vec && n + 4 <= t.n) {
      y[i] = *(const f4v*)(t.y + row * t.ldy + n);
    } else {
#pragma unroll
      for (int v = 0; v < 4; v++)
        if (n + v < t.n) y[i][v] = t.y[row * t.ldy + n + v];
    }
  }
  for (Turn turn(id); turn.left;) {
    const int who = turn.next(id);
    const float scale = t.scales ? t.scales[who] : 1.0f;
    f4v acc[kUpTiles];
#pragma unroll
    for (int i = 0; i < kUpTiles; i++) acc[i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const int j = 16 * i + 4 * g;
      if (16 * i >= t.rank) break;
      f4v m = {0.0f, 0.0f, 0.0f, 0.0f};
      if (id == who && j < t.rank) {
        for (int s = 0; s < a.splits; s++) m += *(const f4v*)(t.mid + (s * a.rows + row) * t.rank + j);
        m *= scale;
      }
#pragma unroll
      for (int c = 0; c < kUpTiles; c++) {
        const int64_t n = n0 + 16 * c + col;
        float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (j < t.rank && n < t.n) load4<WT, true>(t.b, ((int64_t)who * t.n + n) * t.rank + j, w);
#pragma unroll
        for (int q = 0; q < 4; q++) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[q], m[q], acc[c], 0, 0, 0);
      }
    }
    // an adapter's values reach its own rows only
    if (id == who) {
#pragma unroll
      for (int i = 0; i < kUpTiles; i++) y[i] += acc[i];
    }
  }
  if (!in || (id < 0 && t.y == t.out)) return;
#pragma unroll
  for (int i = 0; i < kUpTiles; i++) {
    const int64_t n = n0 + 16 * i + 4 * g;
    if (t.vec && n + 4 <= t.n) {
      *(f4v*)(t.out + row * t.ldo + n) = y[i];
    } else {
#pragma unroll
      for (int v = 0; v < 4; v++)
        if (n + v < t.n) t.out[row * t.ldo + n + v] = y[i][v];
    }
  }
}

int64_t tiles_of(int64_t rows) { return (rows + 15) / 16; }

int splits_of(const LoraArgs& a, int cus) {
  const int64_t groups = tiles_of(a.rows) * a.count, most = a.k / 512;
  int64_t s = 2 * cus / groups;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}

template <int XT, int WT, int RT>
hipError_t launch_ranks(const LoraArgs& a, hipStream_t st) {
  int64_t widest = 0;
  for (int i = 0; i < a.count; i++) widest = widest > a.t[i].n ? widest : a.t[i].n;
  const int64_t tiles = tiles_of(a.rows), wide = 16 * kUpTiles * kUpWaves;
  const dim3 down((unsigned)tiles, (unsigned)a.splits, (unsigned)a.count);
  if (a.x_vec)
    lora_down_kernel<XT, WT, RT, true><<<down, 64 * kDownWaves, 0, st>>>(a);
  else
    lora_down_kernel<XT, WT, RT, false><<<down, 64 * kDownWaves, 0, st>>>(a);
  const dim3 up((unsigned)((widest + wide - 1) / wide), (unsigned)tiles, (unsigned)a.count);
  lora_up_kernel<WT, RT><<<up, 64 * kUpWaves, 0, st>>>(a);
  return hipGetLastError();
}

template <int XT, int WT>
hipError_t launch_types(const LoraArgs& a, hipStream_t st) {
  int rank = 0;
  for (int i = 0; i < a.count; i++) rank = rank > a.t[i].rank ? rank : a.t[i].rank;
  if (rank <= 16) return launch_ranks<XT, WT, 1>(a, st);
  if (rank <= 32) return launch_ranks<XT, WT, 2>(a, st);
  if (rank <= 64) return launch_ranks<XT, WT, 4>(a, st);
  return launch_ranks<XT, WT, 8>(a, st);
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

int lora_most_rank() { return 128; }

size_t lora_plan(LoraArgs& a, void* ws, int cus) {
  a.splits = splits_of(a, cus);
  size_t at = 0;
  for (int i = 0; i < a.count; i++) {
    a.t[i].mid = (float*)((uintptr_t)ws + at);
    at += align_up((size_t)a.splits * a.rows * a.t[i].rank * sizeof(float), 16);
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
