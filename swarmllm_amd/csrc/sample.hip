// sample.hip — a token for each row of logits, from a given uniform number.
//
//   w_i = exp((x_i - max x) / T)
// (64-bit weights and sums, of the logits as they are: the steps of w are far under
// those of u). The values are ordered by x (equal ones by index, the lowest first). Of them
// the first top_k are kept; of those the shortest run whose weight reaches
// top_p of theirs (the first always); of those the ones with w >= min_p. The
// token is the first, by index, of the kept ones at which their running sum
// passes u times their total.
//
// The first launch reads the logits once: of every 1024 values (a wave's, a chunk)
// the weight relative to the chunk's own largest, in 64 bits and one order, and
// the largest of each 256 (16 lanes' values, a group). Rows without settings then
// draw a chunk by the chunks' weights and read that one again (sample_pick_kernel).
//
// Settings need the values past a bound only: top_k the groups whose largest is
// among the k largest of the groups (the k-th of them bounds the k-th value from
// below), min_p those past its own line, top_p those past (1 - top_p) Z / n, which
// no value that ends the run can be under (n values of at most that weight
// follow it). Up to 1024 values are sorted in LDS, or 64 in a wave, and every
// setting cut there (sample_select_kernel, a workgroup a row).
// A run by weight (or the k largest of very many) is narrowed down first: the row's
// slices make histograms of counts or weights over the bound's range (a bucket's
// weights are within 3% of each other and have 24 bits each, so that 64 bits add
// up to 2^19 of them exactly, in any order); sample_finish_kernel adds the slices', finds the bucket in which the run ends,
// sums the weights above it chunk by chunk and lists the bucket's own values,
// which the row's last workgroup sorts, cuts and draws from. More than 1024 values
// at a border (equal logits) are narrowed down further by one workgroup, by their
// bits and then by index.
#include <cfloat>

#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"
#include "wave_sums.h"

namespace qmm {

namespace {

constexpr int kChunk = 1024, kGroups = 4;  // values a wave holds; groups in them
constexpr int kMostVocab = 1 << 19;
constexpr int kMostChunks = kMostVocab / kChunk;
constexpr int kThreads = 1024;
constexpr int kMostRows = 2048;  // of a launch: what the workspace holds
enum { kHistogram = 1, kLine = 2 };  // what a row leaves to sample_finish_kernel
constexpr int kList = 1024;     // values that are sorted
constexpr int kBuckets = 2048;  // two a thread
constexpr double kLog2e = 1.4426950408889634;

// 16 values of chunk c at a lane's places 256 q + 4 lane + e; what is past the
// row is -inf.
template <int T, bool VEC>
__device__ __forceinline__ void load_chunk(const SampleArgs& a, int64_t row, int c, int lane, float v[16]) {
  const int64_t at = row * a.stride + c * kChunk + 4 * lane;
  if ((c + 1) * kChunk <= a.vocab) {
#pragma unroll
    for (int q = 0; q < 4; q++) load4<T, VEC>(a.logits, at + 256 * q, v + 4 * q);
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int i = 256 * (e >> 2) + (e & 3);
      v[e] = c * kChunk + 4 * lane + i < a.vocab ? load1<T>(a.logits, at + i) : -INFINITY;
    }
  }
}
__device__ __forceinline__ int index_of(int c, int lane, int e) { return c * kChunk + 256 * (e >> 2) + 4 * lane + (e & 3); }

// 2^y by the nearest 64th below or above it, whose power is looked up (one of 64
// in LDS, by its low six bits), and the Taylor polynomial of 2^r over what is
// left: |r ln 2| <= 0.0055, whose sixth power over 6! is 2^-55. y in [-1000, 0];
// under it 0 (power; near takes none such).
struct Powers {
  double p[64];
  // by the first 64 threads; a barrier follows
  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 64) p[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
  }
  __device__ __forceinline__ double near(double y) const {
    constexpr double kShift = 105553116266496.0;  // 1.5 * 2^46: its half step is 2^-7
    const double t = y + kShift;
    const uint32_t n = (uint32_t)__double2loint(t);  // 64 y, rounded
    const double r = y - (t - kShift);
    const double q = r * fma(r, fma(r, fma(r, fma(r, 1.3333558146428443e-3, 9.6181291076284772e-3), 5.5504108664821580e-2),
                                    2.4022650695910071e-1),
                             6.9314718055994531e-1);
    const double b = p[n & 63];
    const double s = __hiloint2double(__double2hiint(b) + (int)((n & ~63u) << 14), __double2loint(b));
    return fma(s, q, s);
  }
  // for any y <= 0: what is under 2^-1000 (-inf too) is 0
  __device__ __forceinline__ double power(double y) const {
    const double w = near(y);
    return y >= -1000.0 ? w : 0.0;
  }
};

// A row's weights: exp((x - top) / T), scale = log2(e) / T; 0 for -inf. Where that
// is no number (top or scale infinite) the largest values alone count.
struct Weights {
  const Powers* powers;
  float top;
  double scale;
  __device__ __forceinline__ double operator()(float x) const {
    if (top == INFINITY || scale == (double)INFINITY) return x == top ? 1.0 : 0.0;
    return powers->power(((double)x - (double)top) * scale);
  }
};

__device__ __forceinline__ double scale_of(const SampleArgs& a, int64_t row, bool& greedy) {
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  greedy = !(t > 0.0f);
  return greedy ? 1.0 : kLog2e / (double)t;
}

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// Bound by the logits' bytes and by the 64-bit arithmetic of a weight, 17 instructions:
// 512 rows of 128256 f32 values in 65 us, 263 MB at 4.0 TB/s; 1 row 3.9 us.
template <int T, bool VEC>
__global__ __launch_bounds__(256) void sample_chunks_kernel(SampleArgs a, int chunks) {
  __shared__ Powers powers;
  const int lane = threadIdx.x & 63, c = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = blockIdx.y;
  powers.fill();
  __syncthreads();
  if (c >= chunks) return;
  float v[16];
  load_chunk<T, VEC>(a, row, c, lane, v);
#pragma unroll
  for (int e = 0; e < 16; e++) v[e] = v[e] == v[e] ? v[e] : -INFINITY;
  bool greedy;
  const double scale = scale_of(a, row, greedy);
  float m = v[0];
#pragma unroll
  for (int e = 1; e < 16; e++) m = fmaxf(m, v[e]);
  // over 16 lanes, then over the four groups (the same for the wave)
  m = fmaxf(m, __uint_as_float(dpp_u<0xB1>(__float_as_uint(m))));
  m = fmaxf(m, __uint_as_float(dpp_u<0x4E>(__float_as_uint(m))));
  m = fmaxf(m, __uint_as_float(dpp_u<0x141>(__float_as_uint(m))));
  m = fmaxf(m, __uint_as_float(dpp_u<0x140>(__float_as_uint(m))));
  if ((lane & 15) == 0) a.maxima[(row * chunks + c) * kGroups + (lane >> 4)] = m;
  m = fmaxf(fmaxf(lane_value(m, 0), lane_value(m, 16)), fmaxf(lane_value(m, 32), lane_value(m, 48)));
  double s = 0.0;
  if (!greedy && m != -INFINITY) {
    const Weights weight{&powers, m, scale};
    if (m < INFINITY && scale < INFINITY) {
      // (2^-1000 for what is under it: beside the largest's 1 no sum sees it)
#pragma unroll
      for (int e = 0; e < 16; e++) s += powers.near(fmax(((double)v[e] - (double)m) * scale, -1000.0));
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) s += weight(v[e]);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
  }
  if (lane == 0) a.masses[row * chunks + c] = s;
  if (c == 0 && lane == 0 && a.states) a.states[row] = SampleState{};
}

// A weight as a whole number of units, 2^-bits of the largest weight each (bits at
// most 62): the bits past them are cut off.
struct Units {
  int bits;
  // Of a row whose weights add up to total (1 at least): 2^62 to 2^63 of them, a unit at most 2^-62 of it.
  static __device__ __forceinline__ Units of(double total) { return Units{62 - ((__double2hiint(total) >> 20) - 1023)}; }
  __device__ __forceinline__ uint64_t operator()(double w) const {
    const uint64_t b = (uint64_t)__double_as_longlong(w);
    const int shift = min(63, 1023 + 62 - bits - (int)(b >> 52));  // (0 and what is under a unit: all of them)
    return ((b << 10 & 0x3FFFFFFFFFFFFC00ull) | 0x4000000000000000ull) >> shift;
  }
  __device__ __forceinline__ double size() const { return __hiloint2double((1023 + bits) << 20, 0); }
};

// Values in the order of their keys: key(x) < key(y) where x < y.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// A value and its place as one number: larger values first, of equal ones the lower index.
__device__ __forceinline__ uint64_t rank_of(float x, int i) { return (uint64_t)key_of(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float ranked_value(uint64_t r) { return value_of((uint32_t)(r >> 32)); }

struct Shared {
  Powers powers;
  float maxima[kMostChunks * kGroups];
  uint16_t active[kMostChunks * kGroups];
  union {
    struct {
      uint64_t mass[kBuckets];
      uint32_t count[kBuckets];
    } h;
    double group_mass[kMostChunks * kGroups];
    double part[kBuckets];
  };
  uint64_t list[kList];
  double sums[16];
  uint64_t sums64[16];
  uint32_t sums32[16];
  int n_active, n_list, found, found2;  // (the last two one after the other)
};

// The value of lane ^ M of the wave, on the vector unit (a shuffle goes through LDS: a
// stage of a sort took 125 ns with it).
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  const int lane = threadIdx.x & 63;
  if constexpr (M == 1) return dpp_u<0xB1>(v);             // quad 1,0,3,2
  if constexpr (M == 2) return dpp_u<0x4E>(v);             // quad 2,3,0,1
  if constexpr (M == 4) return dpp_u<0x1B>(dpp_u<0x141>(v));  // 8 mirrored, each quad mirrored
  if constexpr (M == 8) return dpp_u<0x128>(v);            // 16 turned by 8
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int M>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return (uint64_t)lane_xor<M>((uint32_t)(v >> 32)) << 32 | lane_xor<M>((uint32_t)v);
}

// Of a workgroup of NT threads (NT / 64 waves).
template <int NT>
__device__ __forceinline__ float block_max(float v, double* waves) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  float* const w = (float*)waves;
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = w[0];
#pragma unroll
  for (int i = 1; i < NT / 64; i++) v = fmaxf(v, w[i]);
  __syncthreads();
  return v;
}

// The sum of the values of this thread and the ones before it, and all of them;
// in one order, whatever the values.
template <int NT, typename T>
__device__ __forceinline__ T block_sums(T v, T* waves, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_sums(v);
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; w++) {
    if (w == wave) before = total;
    total += waves[w];
  }
  __syncthreads();
  return before + v;
}

// The least of the threads' numbers.
__device__ __forceinline__ int block_least(int v, int* found) {
  if (threadIdx.x == 0) *found = INT32_MAX;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = min(v, __shfl_xor(v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0 && v != INT32_MAX) atomicMin(found, v);
  __syncthreads();
  v = *found;
  __syncthreads();
  return v;
}

// The lesser of two lanes' numbers to the lower lane (up) or to the upper one.
template <int M>
__device__ __forceinline__ uint64_t sort_step(uint64_t v, bool up) {
  const uint64_t o = lane_xor<M>(v);
  return (((threadIdx.x & M) == 0) == up) == (o < v) ? o : v;
}

// The least of the threads' numbers a, and of b.
__device__ __forceinline__ int2 block_least2(int a, int b, int* found) {
  if (threadIdx.x < 2) found[threadIdx.x] = INT32_MAX;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    a = min(a, __shfl_xor(a, d, 64));
    b = min(b, __shfl_xor(b, d, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    if (a != INT32_MAX) atomicMin(found, a);
    if (b != INT32_MAX) atomicMin(found + 1, b);
  }
  __syncthreads();
  const int2 r = make_int2(found[0], found[1]);
  __syncthreads();
  return r;
}

// One number a thread, sorted over the first n2 threads (a power of two, 64 at
// least), the least first. The waves past them only meet the barriers.
__device__ __forceinline__ uint64_t block_sort(uint64_t v, int n2, uint64_t* buf) {
  const int tid = threadIdx.x;
  const bool in = tid < n2;  // the same for a wave
  for (int size = 2; size <= n2; size <<= 1) {
    const bool up = (tid & size) == 0;
    int stride = size >> 1;
    for (; stride >= 64; stride >>= 1) {
      __syncthreads();
      if (in) buf[tid] = v;
      __syncthreads();
      if (!in) continue;
      const uint64_t o = buf[tid ^ stride];
      if (((tid & stride) == 0) == up ? o < v : o > v) v = o;
    }
    if (!in) continue;
    switch (stride) {
      case 32: v = sort_step<32>(v, up); [[fallthrough]];
      case 16: v = sort_step<16>(v, up); [[fallthrough]];
      case 8: v = sort_step<8>(v, up); [[fallthrough]];
      case 4: v = sort_step<4>(v, up); [[fallthrough]];
      case 2: v = sort_step<2>(v, up); [[fallthrough]];
      default: v = sort_step<1>(v, up);
    }
  }
  return v;
}

__device__ __forceinline__ int sort_size(int n) {
  int s = 64;
  while (s < n) s <<= 1;
  return s;
}

// f(x, i) for the values of the groups that are active, 16 lanes a group.
template <int T, bool VEC, typename F>
__device__ __forceinline__ void each_value(const SampleArgs& a, int64_t row, const Shared& s, F f) {
  const int n = s.n_active;
  for (int k = threadIdx.x >> 4; k < n; k += kThreads / 16) {
    const int g = s.active[k], lane = (g & 3) * 16 + (threadIdx.x & 15);
    float v[16];
    load_chunk<T, VEC>(a, row, g >> 2, lane, v);
#pragma unroll
    for (int e = 0; e < 16; e++) f(v[e], index_of(g >> 2, lane, e));
  }
}

// The groups from g0 to g1 whose largest value `in` takes.
template <typename In>
__device__ __forceinline__ void activate(Shared& s, int g0, int g1, In in) {
  __syncthreads();
  if (threadIdx.x == 0) s.n_active = 0;
  __syncthreads();
  for (int g = g0 + (int)threadIdx.x; g < g1; g += kThreads)
    if (s.maxima[g] != -INFINITY && in(s.maxima[g])) s.active[atomicAdd(&s.n_active, 1)] = (uint16_t)g;
  __syncthreads();
}

// The values from lo on that `in` takes into the list (the first kList that
// come), and how many there are. lo is a number: NaN and -inf are not there.
template <int T, bool VEC, typename In>
__device__ __forceinline__ int collect(const SampleArgs& a, int64_t row, Shared& s, In in) {
  constexpr int kUnits = kThreads / 16;
  if (threadIdx.x == 0) s.n_list = 0;
  __syncthreads();
  const int n = s.n_active;
  // two groups on their way at once; over once the list is
  for (int k = threadIdx.x >> 4; k < n && *(volatile int*)&s.n_list <= kList; k += 2 * kUnits) {
    float v[2][16];
    int g[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      g[h] = s.active[min(k + h * kUnits, n - 1)];
      load_chunk<T, VEC>(a, row, g[h] >> 2, (g[h] & 3) * 16 + (threadIdx.x & 15), v[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if (k + h * kUnits >= n) break;
      int those = 0;
#pragma unroll
      for (int e = 0; e < 16; e++) those += in(v[h][e]) ? 1 : 0;
      if (those == 0) continue;
      int at = atomicAdd(&s.n_list, those);  // one addition a lane
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (in(v[h][e])) {
          if (at < kList) s.list[at] = rank_of(v[h][e], index_of(g[h] >> 2, (g[h] & 3) * 16 + (threadIdx.x & 15), e));
          at++;
        }
    }
  }
  __syncthreads();
  return s.n_list;
}

// What a row's settings ask of a prefix of the ordered values: `want` of them
// at most, or their weight.
struct Goal {
  bool by_count;
  uint64_t want;
};

// A histogram over the values that `bucket` gives a bucket (the larger the
// value, the lower; -1: none).
template <int T, bool VEC, typename B>
__device__ __forceinline__ void histogram(const SampleArgs& a, int64_t row, Shared& s, const Weights& weight, const Units& unit,
                                          bool weights, B bucket) {
  for (int b = threadIdx.x; b < kBuckets; b += kThreads) {
    s.h.mass[b] = 0;
    s.h.count[b] = 0;
  }
  __syncthreads();
  each_value<T, VEC>(a, row, s, [&](float x, int i) {
    const int b = x > -INFINITY ? bucket(x, i) : -1;
    if (b < 0) return;
    atomicAdd(&s.h.count[b], 1u);
    if (weights) atomicAdd((unsigned long long*)&s.h.mass[b], (unsigned long long)unit(weight(x)));
  });
  __syncthreads();
}

// The first bucket at which the goal is met (kBuckets: none), from the counts and
// weights of a thread's two buckets. Those of the buckets before it are added to
// above_*, `inside` is the bucket's own count.
__device__ __forceinline__ int first_met(Shared& s, const Goal& goal, const uint32_t c[2], const uint64_t m[2],
                                         uint64_t& above_count, uint64_t& above_mass, uint32_t& inside) {
  const int tid = threadIdx.x;
  uint32_t all_count;
  uint64_t all_mass;
  const uint64_t count = above_count + block_sums<kThreads, uint32_t>(c[0] + c[1], s.sums32, all_count);
  const uint64_t mass = above_mass + block_sums<kThreads, uint64_t>(m[0] + m[1], s.sums64, all_mass);
  auto met = [&](uint64_t n, uint64_t w) { return n > 0 && (goal.by_count ? n : w) >= goal.want; };
  int b = INT32_MAX;
  if (met(count, mass)) b = met(count - c[1], mass - m[1]) ? 2 * tid : 2 * tid + 1;
  b = block_least(b, &s.found);
  if (b >= kBuckets) return kBuckets;
  // the sums before it are its thread's
  if (tid == b / 2) {
    s.sums64[0] = count - c[1] - (b & 1 ? 0 : c[0]);
    s.sums64[1] = mass - m[1] - (b & 1 ? 0 : m[0]);
    s.sums32[0] = c[b & 1];
  }
  __syncthreads();
  above_count = s.sums64[0];
  above_mass = s.sums64[1];
  inside = s.sums32[0];
  __syncthreads();
  return b;
}

template <int T, bool VEC, typename B>
__device__ __forceinline__ int narrow(const SampleArgs& a, int64_t row, Shared& s, const Goal& goal, bool both,
                                      const Weights& weight, const Units& unit, uint64_t& above_count, uint64_t& above_mass,
                                      uint32_t& inside, B bucket) {
  histogram<T, VEC>(a, row, s, weight, unit, both, bucket);
  const uint32_t c[2] = {s.h.count[2 * threadIdx.x], s.h.count[2 * threadIdx.x + 1]};
  const uint64_t m[2] = {s.h.mass[2 * threadIdx.x], s.h.mass[2 * threadIdx.x + 1]};
  return first_met(s, goal, c, m, above_count, above_mass, inside);
}

// Buckets of equal width from a row's largest value down to its bound.
struct Buckets {
  float top, lo, inv;
  __device__ __forceinline__ Buckets(float top, float lo) : top(top), lo(lo) {
    const float width = top - lo;
    inv = width > 0.0f && width < INFINITY ? (float)(kBuckets - 1) / width : 0.0f;
  }
  __device__ __forceinline__ int operator()(float x, int) const {
    return x < lo ? -1 : x == top ? 0 : min(kBuckets - 1, (int)((top - x) * inv));
  }
};

// The list's n values (all that lie in one bucket), sorted: the rank of the last
// one of the prefix that meets the goal, and the prefix's weight.
__device__ __forceinline__ uint64_t last_in_list(Shared& s, const Goal& goal, const Weights& weight, const Units& unit, int n,
                                                 uint64_t above_count, uint64_t above_mass, uint64_t& mass) {
  const int tid = threadIdx.x;
  const uint64_t mine = ~block_sort(tid < n ? ~s.list[tid] : ~0ull, sort_size(n), s.list);
  const uint64_t w = tid < n ? unit(weight(ranked_value(mine))) : 0;
  uint64_t total;
  const uint64_t m = above_mass + block_sums<kThreads, uint64_t>(w, s.sums64, total);
  const bool met = (goal.by_count ? above_count + tid + 1 : m) >= goal.want;
  const int at = min(block_least(tid < n && met ? tid : INT32_MAX, &s.found), n - 1);
  if (tid == at) {
    s.sums64[0] = mine;
    s.sums64[1] = m;
  }
  __syncthreads();
  const uint64_t last = s.sums64[0];
  mass = s.sums64[1];
  __syncthreads();
  return last;
}

// The same for a bucket of any number of values, over the active groups: by one workgroup.
template <int T, bool VEC>
__device__ __forceinline__ uint64_t last_of_prefix(const SampleArgs& a, int64_t row, Shared& s, const Goal& goal,
                                                   const Weights& weight, const Units& unit, uint64_t& mass,
                                                   const Buckets& bucket, int first, uint64_t above_count,
                                                   uint64_t above_mass, uint32_t inside) {
  // the keys of the bucket, which falls as they rise: between the first with
  // bucket <= `first` and the last with bucket >= it
  uint32_t lo, hi = key_of(bucket.top);
  {
    uint32_t l = key_of(-FLT_MAX), h = hi;
    while (l < h) {
      const uint32_t m = l + (h - l) / 2;
      const int b = bucket(value_of(m), 0);
      if (b <= first && b >= 0) h = m; else l = m + 1;
    }
    lo = l;
    h = hi;
    while (l < h) {
      const uint32_t m = l + (h - l + 1) / 2;
      if (bucket(value_of(m), 0) >= first) l = m; else h = m - 1;
    }
    hi = l;
  }
  while (inside > kList && lo < hi) {
    const uint32_t span = hi - lo, l = lo, h = hi;
    const int shift = span < (uint32_t)kBuckets ? 0 : 32 - __builtin_clz(span) - 11;
    const int b = narrow<T, VEC>(a, row, s, goal, true, weight, unit, above_count, above_mass, inside, [=](float x, int) {
      const uint32_t k = key_of(x);
      return k >= l && k <= h ? (int)((h - k) >> shift) : -1;
    });
    if (b >= kBuckets) break;  // (the bucket above met the goal: this is not reached)
    hi = h - ((uint32_t)b << shift);
    const uint32_t width = (1u << shift) - 1;
    lo = hi - l > width ? hi - width : l;
  }
  const uint32_t l = lo, h = hi;
  if (inside <= kList) {
    const int n = min(kList, collect<T, VEC>(a, row, s, [=](float x) {
                         const uint32_t k = key_of(x);
                         return x == x && k >= l && k <= h;
                       }));
    return last_in_list(s, goal, weight, unit, n, above_count, above_mass, mass);
  }
  // more equal values than the list holds: the first of them by index
  const uint64_t w = unit(weight(value_of(h)));
  uint64_t n = goal.by_count ? goal.want - above_count : w ? (goal.want - above_mass + w - 1) / w : inside;
  if (n < 1 || (!goal.by_count && goal.want <= above_mass)) n = 1;
  if (n > inside) n = inside;
  mass = above_mass + n * w;
  const Goal nth{true, n};
  uint64_t before = 0, unused = 0;
  uint32_t within = 0;
  int from = 0;
  for (int shift = 8; shift >= 0; shift -= 8) {  // 2^11 ranges of 2^8 places, then the place
    const int base = from, width = kBuckets << shift;
    const int b = narrow<T, VEC>(a, row, s, nth, false, weight, unit, before, unused, within, [=](float x, int i) {
      return key_of(x) == h && i >= base && i - base < (shift ? width : 256) ? (i - base) >> shift : -1;
    });
    from = base + (min(b, kBuckets - 1) << shift);
  }
  return (uint64_t)h << 32 | (uint32_t)~from;
}

__device__ __forceinline__ void answer(const SampleArgs& a, int64_t row, int id, double p) {
  a.ids[row] = id;
  if (a.probs) a.probs[row] = (float)p;
}

// Which values stay, of a row whose prefix is known: those of rank `last` or more
// (and of `lo` or more), of weight `floor` or more.
struct Stay {
  float lo;
  uint64_t last;
  double floor;
  __device__ __forceinline__ double operator()(const Weights& weight, float x, int i) const {
    if (!(x >= lo && x > -INFINITY && (last == 0 || rank_of(x, i) >= last))) return 0.0;
    const double w = weight(x);
    return w >= floor ? w : 0.0;
  }
};

// The first by index of the values that stay at which their sum passes u of the
// total: the chunk from the chunks' weights (thread c's of chunk c), the value
// from the chunk.
template <int NT, int T>
__device__ __forceinline__ void draw(const SampleArgs& a, int64_t row, const Weights& weight, const Stay& stay, double mass,
                                     double u, int chunks, double* sums, int* found) {
  const int tid = threadIdx.x;
  double total;
  const double upto = block_sums<NT, double>(mass, sums, total), r = u * total;
  const bool some = tid < chunks && mass > 0.0;
  int c = block_least(some && upto > r ? tid : INT32_MAX, found);
  if (c == INT32_MAX) c = -block_least(some ? -tid : INT32_MAX, found);
  if (tid == c) sums[0] = upto - mass;
  __syncthreads();
  const double sum = sums[0];
  __syncthreads();
  constexpr int E = kChunk / NT;
  double w[E], mine = 0.0, unused;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int i = c * kChunk + E * tid + e;
    w[e] = i < a.vocab ? stay(weight, load1<T>(a.logits, row * a.stride + i), i) : 0.0;
    mine += w[e];
  }
  double before = sum + (block_sums<NT, double>(mine, sums, unused) - mine);
  int place = INT32_MAX, end = -1;
#pragma unroll
  for (int e = 0; e < E; e++) {
    before += w[e];
    if (w[e] > 0.0) {
      end = E * tid + e;
      if (place == INT32_MAX && before > r) place = end;
    }
  }
  int at = block_least(place, found);
  // (the sums of the chunk, in another order, can end below r: the last value with a weight)
  if (at == INT32_MAX) at = -block_least(end >= 0 ? -end : INT32_MAX, found);
#pragma unroll
  for (int e = 0; e < E; e++)
    if (at == E * tid + e) answer(a, row, c * kChunk + at, w[e] / total);
}

// The weights of the values that stay, a thread each, added to their chunks:
// thread c's of chunk c. As whole numbers, so in any order (of 2^-52 at least, of which
// a chunk's 1024 values add up to 2^62).
__device__ __forceinline__ double to_chunks(Shared& s, const Units& row_unit, int chunks, bool stays, uint64_t rank, double w) {
  const Units unit{max(52, row_unit.bits)};
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid < chunks) s.list[tid] = 0;
  __syncthreads();
  if (stays) atomicAdd((unsigned long long*)&s.list[(uint32_t)~rank >> 10], (unsigned long long)unit(w));
  __syncthreads();
  return tid < chunks ? (double)s.list[tid] / unit.size() : 0.0;
}

__device__ __forceinline__ double number_of(const SampleArgs& a, int64_t row) {
  return fmin(fmax((double)a.u[row], 0.0), 1.0);
}

// The first value, by index, of the row's largest ones.
template <int T, bool VEC>
__device__ __forceinline__ int first_largest(const SampleArgs& a, int64_t row, const float* maxima, int chunks, float top,
                                             int* found) {
  int mine = INT32_MAX;
  for (int c = threadIdx.x >> 6; c < chunks; c += blockDim.x >> 6) {
    const float* m = maxima + kGroups * c;
    if (fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) != top) continue;
    float v[16];
    load_chunk<T, VEC>(a, row, c, threadIdx.x & 63, v);
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (v[e] == top) mine = min(mine, index_of(c, threadIdx.x & 63, e));
    break;  // (a wave's later chunks come behind it)
  }
  return block_least(mine, found);
}

// The weights of the chunks relative to the row's largest value, thread c's of chunk c.
__device__ __forceinline__ double chunk_weight(const SampleArgs& a, int64_t row, const float* maxima, int chunks,
                                               const Weights& weight) {
  const int c = threadIdx.x;
  if (c >= chunks) return 0.0;
  const float* m = maxima + kGroups * c;
  const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  return top != -INFINITY ? a.masses[row * chunks + c] * weight(top) : 0.0;
}

// Rows without settings but the temperature: one chunk of each read again (512 rows 6.6 us).
template <int T, bool VEC>
__global__ __launch_bounds__(kMostChunks) void sample_pick_kernel(SampleArgs a, int chunks) {
  constexpr int NT = kMostChunks;
  __shared__ Powers powers;
  __shared__ float maxima[kMostChunks * kGroups];
  __shared__ double sums[NT / 64];
  __shared__ int found;
  const int64_t row = blockIdx.x;
  bool greedy;
  const double scale = scale_of(a, row, greedy);
  powers.fill();
  float m = -INFINITY;
  for (int g = threadIdx.x; g < chunks * kGroups; g += NT) {
    const float v = a.maxima[row * chunks * kGroups + g];
    maxima[g] = v;
    m = fmaxf(m, v);
  }
  const float top = block_max<NT>(m, sums);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) answer(a, row, -1, 0.0);
  } else if (greedy) {
    const int first = first_largest<T, VEC>(a, row, maxima, chunks, top, &found);
    if (threadIdx.x == 0) answer(a, row, first, 1.0);
  } else {
    const Weights weight{&powers, top, scale};
    draw<NT, T>(a, row, weight, Stay{-INFINITY, 0, 0.0}, chunk_weight(a, row, maxima, chunks, weight), number_of(a, row),
                     chunks, sums, &found);
  }
}

// What the settings leave of at most 64 values (top_p only beside top_k), the largest first, a lane each: a wave's.
__device__ __forceinline__ void finish_wave(const SampleArgs& a, int64_t row, const Weights& weight, uint64_t r, int n, int k,
                                            double p, double floor, double u) {
  const int lane = threadIdx.x;
  r = ~block_sort(lane < n ? ~r : ~0ull, 64, nullptr);
  double w = lane < n && lane < k ? weight(ranked_value(r)) : 0.0;
  const double sum = wave_sums(w);
  const double goal = fmax(p, 0.0) * __shfl(sum, 63, 64);
  const bool stays = lane < n && lane < k && (p >= 1.0 || lane == 0 || sum - w < goal) && w >= floor;
  if (!stays) w = 0.0;
  const uint64_t those = __ballot(stays);
  // the sums by index, each in the order of the ranks
  const int i = (int)(uint32_t)~r, m = 64 - __builtin_clzll(those);
  double upto = 0.0, all = 0.0;
  for (int j = 0; j < m; j++) {
    const int ij = __builtin_amdgcn_readlane(i, j);
    const double wj = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(w), j),
                                       __builtin_amdgcn_readlane(__double2loint(w), j));
    upto += ij <= i ? wj : 0.0;
    all += wj;
  }
  // the least index whose sum passes the number (or the last one: u of 1)
  const bool hit = stays && upto > u * all;
  int best = hit ? i : INT32_MAX;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) best = min(best, __shfl_xor(best, d, 64));
  if (best == INT32_MAX) {
    best = stays ? i : -1;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) best = max(best, __shfl_xor(best, d, 64));
  }
  if (stays && i == best) answer(a, row, best, w / all);
}

// The part of the row's chunks that a slice takes.
__device__ __forceinline__ int slice_begin(int chunks, int slice, int slices) { return chunks * slice / slices; }

// A row, or a slice of one, is a chain of short passes over what the CU holds (maxima,
// a scan, the groups past the bound, a sort), each waiting for the one before:
// 1 row of 128256 by top_k 40 and top_p 9 us, 64 rows of mixed settings 22.
//
// Whether the k-th largest of the groups' maxima leaves few values (`few`) past it to
// sort: of values in any order, n over `groups` groups leave k of them with one when
// k = groups (1 - exp(-n / groups)).
__device__ __forceinline__ bool few_past(int k, int groups, float few) {
  return k < groups && -(float)groups * __logf(1.0f - (float)k / (float)groups) <= few;
}

template <int T, bool VEC>
__global__ __launch_bounds__(kThreads) void sample_select_kernel(SampleArgs a, int chunks) {
  __shared__ Shared s;
  const int tid = threadIdx.x, groups = chunks * kGroups, slice = blockIdx.x;
  const int64_t row = blockIdx.y;
  const int k_set = a.top_k ? a.top_k[row] : 0, merged = min(groups, kThreads);
  const bool k_on = k_set > 0 && k_set < a.vocab;
  const int k = k_on ? k_set : a.vocab;
  const double p_set = a.top_p ? (double)a.top_p[row] : 1.0, p = p_set < 1.0 ? p_set : 1.0;  // (NaN too is off)
  const bool p_on = p < 1.0;
  bool greedy;
  const double scale = scale_of(a, row, greedy);
  // rows that every slice makes a histogram of; the others are the first one's. (By
  // count, us with the border sorted by one workgroup / narrowed down by all: 4 rows of
  // 128256 f32 by top_k 100 22 / 30, 320 34 / 31, 400 37 / 31, 450, whose bound
  // leaves more than the list holds, 76 / 31; 64 rows 33 / 50, 44 / 51, 48 / 51, 88 / 52.
  // Beside rows by top_p, which wait for all slices anyway, sooner: 21 rows of mixed
  // settings with top_k to 320 55 / 45, 64 70 / 64; 8 of which none is by top_p alone 33 / 40)
  const float few = (a.top_p ? 0.4f : 0.75f) * kList;
  const bool wide = !greedy && (k_on ? !p_on && !few_past(k, merged, few) : p_on);
  if (!wide && slice > 0) return;
  s.powers.fill();
  float m = -INFINITY;
  for (int g = tid; g < groups; g += kThreads) {
    const float v = a.maxima[row * groups + g];
    s.maxima[g] = v;
    m = fmaxf(m, v);
  }
  const float top = block_max<kThreads>(m, s.sums);
  if (top == -INFINITY) {  // no value left
    if (tid == 0 && slice == 0) answer(a, row, -1, 0.0);
    return;
  }
  if (greedy) {
    const int first = first_largest<T, VEC>(a, row, s.maxima, chunks, top, &s.found);
    if (tid == 0) answer(a, row, first, 1.0);
    return;
  }
  const Weights weight{&s.powers, top, scale};
  const double mass = chunk_weight(a, row, s.maxima, chunks, weight);
  const double floor = a.min_p && a.min_p[row] > 0.0f ? fmin((double)a.min_p[row], 1.0) : 0.0;
  const double u = number_of(a, row);
  if (!k_on && !p_on && floor == 0.0) {
    draw<kThreads, T>(a, row, weight, Stay{-INFINITY, 0, 0.0}, mass, u, chunks, s.sums, &s.found);
    return;
  }
  double total;
  (void)block_sums<kThreads, double>(mass, s.sums, total);
  const Units unit = Units::of(total);

  // no value under `line` is kept (in units of log2 w), nor counts for another's place: under 2^-60 none does
  double line = -60.0;
  if (p_on && !k_on) line = fmax(line, log2(fmin((1.0 - p) * total / a.vocab, 1.0)) - 1e-6);
  if (floor > 0.0 && !(k_on && p_on)) line = fmax(line, log2(floor) - 1e-6);
  const double at = (double)top + line / scale;
  float lo = at >= (double)top ? top : (float)at;
  if ((double)lo > at) lo = value_of(key_of(lo) - 1);
  if (top == INFINITY) lo = top;
  lo = fmaxf(lo, -FLT_MAX);  // -inf is never drawn

  if (wide) {
    // the slice's part of the histogram: counts, or weights in 32 bits (they say where
    // to look; the sums that decide are the next launch's)
    activate(s, kGroups * slice_begin(chunks, slice, a.slices), kGroups * slice_begin(chunks, slice + 1, a.slices),
             [=](float x) { return x >= lo; });
    for (int b = tid; b < kBuckets; b += kThreads) s.part[b] = 0.0;
    __syncthreads();
    const Buckets bucket(top, lo);
    const float scale32 = (float)scale;
    each_value<T, VEC>(a, row, s, [&](float x, int i) {
      if (!(x >= lo)) return;
      // (no NaN: of an infinite scale, or of a difference past f32's range)
      const float w = x == top ? 1.0f : __builtin_amdgcn_exp2f(fmaxf((x - top) * scale32, -200.0f));
      atomicAdd(&s.part[bucket(x, i)], k_on ? 1.0 : (double)w);
    });
    __syncthreads();
    float* const part = a.parts + (row * a.slices + slice) * kBuckets;  // (counts are whole in 32 bits too)
    for (int b = tid; b < kBuckets; b += kThreads) part[b] = (float)s.part[b];
    if (tid == 0 && slice == 0)
      a.states[row] = SampleState{kHistogram, top, lo, 0, 0, k_on, 0, unit.bits, k_on ? (double)k : fmax(p, 0.0) * total, 0, scale, floor};
    return;
  }

  const Buckets bucket(top, lo);
  int deepest = kBuckets;  // the bucket past which no value of the k largest lies
  if (k_on && k <= merged) {
    // that of the k-th largest of the groups' maxima
    for (int b = tid; b < kBuckets; b += kThreads) s.h.count[b] = 0;
    __syncthreads();
    float v = tid < groups ? s.maxima[tid] : -INFINITY;
    if (tid + kThreads < groups) v = fmaxf(v, s.maxima[tid + kThreads]);
    const int mine = v != -INFINITY ? bucket(v, 0) : -1;
    if (mine >= 0) atomicAdd(&s.h.count[mine], 1u);
    __syncthreads();
    const uint32_t c1 = s.h.count[2 * tid + 1];
    uint32_t all_count;
    const uint32_t upto = block_sums<kThreads, uint32_t>(s.h.count[2 * tid] + c1, s.sums32, all_count);
    const int b = block_least(upto >= (uint32_t)k ? 2 * tid + (upto - c1 < (uint32_t)k) : INT32_MAX, &s.found);
    deepest = min(b, kBuckets);
  }
  // (its lower border, a bucket lower for the roundings)
  if (deepest < kBuckets && bucket.inv > 0.0f) lo = fmaxf(lo, top - (float)(deepest + 2) / bucket.inv);
  activate(s, 0, groups, [=](float x) { return x >= lo; });
  // min_p alone, and most groups hold some of its values: more than the list does, as
  // a rule, and to see that by listing costs more than it finds (16 rows by min_p 1e-5
  // 28 us with this, 39 without; by 0.05 27, and 34 with a quarter for the three)
  const bool overfull = !k_on && s.n_active > 3 * groups / 4 && groups >= 256;
  int n = overfull ? kList + 1 : collect<T, VEC>(a, row, s, [=](float x) { return x >= lo; });
  uint64_t last = 0;  // the rank of the last value of the prefix
  if (n > kList) {
    if (!k_on) {  // min_p alone: all the values past its line, which every slice then sums
      if (tid == 0) a.states[row] = SampleState{kLine, top, lo, 0, 0, 0, 0, unit.bits, 0.0, 0, scale, floor};
      return;
    }
    // very many values, or equal ones: narrowed down by this workgroup
    const Buckets bucket(top, lo);
    const Goal goal{true, (uint64_t)k};
    uint64_t above_count = 0, above_mass = 0, kept_mass = 0;
    uint32_t inside = 0;
    int b = narrow<T, VEC>(a, row, s, goal, true, weight, unit, above_count, above_mass, inside, bucket);
    if (b < kBuckets && above_count + inside <= kList) {
      const int edge = b;
      n = collect<T, VEC>(a, row, s, [=](float x) { return x >= lo && bucket(x, 0) <= edge; });
    } else {
      if (b < kBuckets)
        last = last_of_prefix<T, VEC>(a, row, s, goal, weight, unit, kept_mass, bucket, b, above_count, above_mass, inside);
      else
        kept_mass = (uint64_t)(total * unit.size());  // fewer than k values have any weight
      if (p_on) {
        const Goal run{false, (uint64_t)(fmax(p, 0.0) * (double)kept_mass)};
        above_count = above_mass = 0;
        b = narrow<T, VEC>(a, row, s, run, true, weight, unit, above_count, above_mass, inside, bucket);
        if (b < kBuckets)
          last = max(last, last_of_prefix<T, VEC>(a, row, s, run, weight, unit, kept_mass, bucket, b, above_count,
                                                  above_mass, inside));
      }
      if (tid == 0) a.states[row] = SampleState{kLine, top, lo, 0, 0, 0, 0, unit.bits, 0.0, last, scale, floor};
      return;
    }
  }
  // every value that can stay (by top_p beside top_k only: the others by it are wide)
  if (n <= 64) {
    if (tid < 64) finish_wave(a, row, weight, tid < n ? s.list[tid] : 0, n, k, p, floor, u);
    return;
  }
  const uint64_t r = ~block_sort(tid < n ? ~s.list[tid] : ~0ull, sort_size(n), s.list);
  const double w = tid < n && tid < k ? weight(ranked_value(r)) : 0.0;
  double all;
  const double sum = block_sums<kThreads, double>(w, s.sums, all);
  const double run = fmax(p, 0.0) * all;
  const bool stays = tid < n && tid < k && (!p_on || tid == 0 || sum - w < run) && w >= floor;
  const int staying = min(block_least(stays ? INT32_MAX : tid, &s.found), n);  // (they come first)
  if (tid == staying - 1) s.sums64[0] = r;
  const double kept = to_chunks(s, unit, chunks, stays, r, w);
  draw<kThreads, T>(a, row, weight, Stay{lo, s.sums64[0], floor}, kept, u, chunks, s.sums, &s.found);
}

// Rows of which many values stay: sums by chunk, and the border's values sorted
// by the last of the row's workgroups: again a chain of passes, and the 64-bit weights of
// the values that stay (64 rows of mixed settings 29 us).
template <int T, bool VEC>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a, int chunks) {
  __shared__ Shared s;
  const int tid = threadIdx.x, groups = chunks * kGroups, slice = blockIdx.x;
  const int64_t row = blockIdx.y;
  SampleState* const state = a.states + row;
  const int mode = state->mode;
  if (mode == 0) return;
  s.powers.fill();
  for (int g = tid; g < groups; g += kThreads) s.maxima[g] = a.maxima[row * groups + g];
  const float top = state->top, lo = state->lo;
  const double floor = state->floor, goal = state->goal;
  const bool by_count = state->by_count != 0;
  const Weights weight{&s.powers, top, state->scale};
  const Buckets bucket(top, lo);
  const Units unit{state->bits};
  uint64_t last = state->last;
  int from = kBuckets, to = kBuckets - 1;  // the buckets that hold the border
  if (mode == kHistogram) {
    double m[2] = {0.0, 0.0};
#pragma unroll 8
    for (int i = 0; i < a.slices; i++) {
      const float2 p = *(const float2*)(a.parts + (row * a.slices + i) * kBuckets + 2 * tid);
      m[0] += (double)p.x;
      m[1] += (double)p.y;
    }
    double all;
    const double upto = block_sums<kThreads, double>(m[0] + m[1], s.sums, all);
    // the exponents of 32-bit weights are off by three half steps, 2^-22.4 of theirs; over
    // the weights' sum they are 20 in the mean at most (2^19 values): 2.5e-6 of it, and
    // 1e-7 of exp2 (a wider range has the border's many small values in it: top_p 0.999 of
    // 16 rows 158 us with 1e-4 here, 48 with this). Where it does not hold the exact sums show it.
    const double off = by_count ? 0.0 : 4e-6 * goal;
    auto first = [&](double want) {
      const bool met = upto > 0.0 && upto >= want, sooner = upto - m[1] > 0.0 && upto - m[1] >= want;
      return met ? 2 * tid + !sooner : INT32_MAX;
    };
    const int2 both = block_least2(first(goal - off), first(goal + off), &s.found);
    from = min(both.x, kBuckets);
    to = min(both.y, kBuckets - 1);
  }
  // the border's range of values: what is above it stays, what is in it is listed
  const float least = last ? fmaxf(lo, ranked_value(last)) : lo;
  float hi = least, low = least;
  if (from < kBuckets) {
    // (the step above the bucket's upper edge: what lies on it is listed)
    hi = bucket.inv > 0.0f && from > 0 ? value_of(key_of(top - (float)from / bucket.inv) + 1) : INFINITY;
    low = bucket.inv > 0.0f && to < kBuckets - 1 ? fmaxf(lo, top - (float)(to + 1) / bucket.inv) : lo;
  }
  const int slices = gridDim.x, c0 = slice_begin(chunks, slice, slices), c1 = slice_begin(chunks, slice + 1, slices);
  activate(s, kGroups * c0, kGroups * c1, [=](float x) { return x >= low; });
  for (int g = kGroups * c0 + tid; g < kGroups * c1; g += kThreads) s.group_mass[g] = 0.0;
  __syncthreads();
  const int n_active = s.n_active;
  int count = 0;
  for (int j = tid >> 4; j < n_active; j += kThreads / 16) {
    const int g = s.active[j], lane = (g & 3) * 16 + (tid & 15);
    float v[16];
    load_chunk<T, VEC>(a, row, g >> 2, lane, v);
    double sum = 0.0;
    int border = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      if (v[e] >= hi && (last == 0 || rank_of(v[e], index_of(g >> 2, lane, e)) >= last)) {
        const double w = weight(v[e]);
        sum += w >= floor ? w : 0.0;
        count++;
      }
      border += v[e] >= low && v[e] < hi ? 1 : 0;
    }
    if (border) {
      int at = atomicAdd(&state->listed, border);
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (v[e] >= low && v[e] < hi) {
          if (at < kList) a.lists[row * kList + at] = rank_of(v[e], index_of(g >> 2, lane, e));
          at++;
        }
    }
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if ((tid & 15) == 0) s.group_mass[g] = sum;
  }
  if (by_count) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) count += __shfl_xor(count, d, 64);
    if ((tid & 63) == 0 && count) atomicAdd(&state->above, count);
  }
  __syncthreads();
  for (int c = c0 + tid; c < c1; c += kThreads) {
    double sum = 0.0;
#pragma unroll
    for (int g = 0; g < kGroups; g++) sum += s.group_mass[kGroups * c + g];
    a.kept[row * chunks + c] = sum;
  }
  // The row's last workgroup goes on. What the others wrote has to be there for it, on
  // another XCD as a rule: each wave waits until its own stores and additions have
  // reached its L2 (a barrier does not), and the first thread then has the L2
  // written back and takes the workgroup's ticket. (A release by every wave writes back
  // sixteen times: 64 rows by top_p 88 us with it, 47 with this.)
  if (slices > 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) s.found = __hip_atomic_fetch_add(&state->ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool final = s.found == slices - 1;
    __syncthreads();
    if (!final) return;
  } else {
    __threadfence_block();
    __syncthreads();
  }
  double mass = tid < chunks ? ((const volatile double*)a.kept)[row * chunks + tid] : 0.0;
  if (from < kBuckets) {
    const int n = ((const volatile SampleState*)state)->listed;
    bool sure = n <= kList;
    if (sure) {
      double all, above = (double)((const volatile SampleState*)state)->above;
      // (without what is under the floor: where some of it lies above the border, all of the border's values are under it)
      if (!by_count) (void)block_sums<kThreads, double>(mass, s.sums, above);
      if (tid < n) s.list[tid] = ((const volatile uint64_t*)a.lists)[row * kList + tid];
      __syncthreads();
      const uint64_t r = ~block_sort(tid < n ? ~s.list[tid] : ~0ull, sort_size(n), s.list);
      const double w = tid < n ? weight(ranked_value(r)) : 0.0;
      const double upto = block_sums<kThreads, double>(w, s.sums, all);
      // the border's prefix: its first value too where nothing lies above it
      const bool in = tid < n && (by_count ? above + tid < goal : (tid == 0 && above == 0.0) || above + (upto - w) < goal);
      const int m = min(block_least(in ? INT32_MAX : tid, &s.found), n);
      // whether the border is where the histogram said
      sure = (above < goal || above == 0.0) && (above + (by_count ? n : all) >= goal || low <= lo);
      if (sure) {
        if (tid == m - 1) s.sums64[0] = r;
        mass += to_chunks(s, unit, chunks, in && w >= floor, r, w);
        last = m ? s.sums64[0] : 0;
        __syncthreads();
      }
    }
    if (!sure) {
      // more values than the list holds (equal ones, as a rule): narrowed down by this workgroup
      const Goal exact{by_count, by_count ? (uint64_t)goal : (uint64_t)(goal * unit.size())};
      uint64_t above_count = 0, above_mass = 0, unused = 0;
      uint32_t inside = 0;
      activate(s, 0, groups, [=](float x) { return x >= lo; });
      const int b = narrow<T, VEC>(a, row, s, exact, true, weight, unit, above_count, above_mass, inside, bucket);
      last = b < kBuckets ? last_of_prefix<T, VEC>(a, row, s, exact, weight, unit, unused, bucket, b, above_count, above_mass,
                                                   inside)
                          : 0;
      __syncthreads();
      for (int g = tid; g < groups; g += kThreads) s.group_mass[g] = 0.0;
      __syncthreads();
      for (int j = tid >> 4; j < s.n_active; j += kThreads / 16) {
        const int g = s.active[j], lane = (g & 3) * 16 + (tid & 15);
        float v[16];
        load_chunk<T, VEC>(a, row, g >> 2, lane, v);
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 16; e++) sum += Stay{lo, last, floor}(weight, v[e], index_of(g >> 2, lane, e));
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if ((tid & 15) == 0) s.group_mass[g] = sum;
      }
      __syncthreads();
      mass = 0.0;
      if (tid < chunks)
        for (int g = 0; g < kGroups; g++) mass += s.group_mass[kGroups * tid + g];
      __syncthreads();
    }
  }
  draw<kThreads, T>(a, row, weight, Stay{lo, last, floor}, mass, number_of(a, row), chunks, s.sums, &s.found);
}

// Slices of a row until each CU has a workgroup (its registers hold one of 1024
// threads), of 8 chunks at least, 8 at most (the finish reads all their parts). us by
// top_p 0.9 of 128256 f32 values in 1, 2, 4 or 8 slices: 1 row 80, 54, 41, 34; 16 rows 85, 59,
// 45, 41; 64 rows 92, 68, 59, and 90 in 8, twice what the CUs hold.
int slices_of(int64_t rows, int chunks, int cus) {
  const int64_t want = cus / rows, most = chunks / 8;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}

template <int T, bool VEC>
hipError_t launch_rows(const SampleArgs& a, hipStream_t st) {
  const int chunks = (a.vocab + kChunk - 1) / kChunk;
  sample_chunks_kernel<T, VEC><<<dim3((unsigned)((chunks + 3) / 4), (unsigned)a.rows), 256, 0, st>>>(a, chunks);
  if (!a.states) {
    sample_pick_kernel<T, VEC><<<(unsigned)a.rows, kMostChunks, 0, st>>>(a, chunks);
  } else {
    sample_select_kernel<T, VEC><<<dim3((unsigned)a.slices, (unsigned)a.rows), kThreads, 0, st>>>(a, chunks);
    sample_finish_kernel<T, VEC><<<dim3((unsigned)a.slices, (unsigned)a.rows), kThreads, 0, st>>>(a, chunks);
  }
  return hipGetLastError();
}

template <int T>
hipError_t launch_type(const SampleArgs& a, hipStream_t st) {
  return a.vec ? launch_rows<T, true>(a, st) : launch_rows<T, false>(a, st);
}

}  // namespace

int64_t sample_most_vocab() { return kMostVocab; }

size_t sample_plan(SampleArgs& a, void* ws, int cus) {
  const int chunks = (a.vocab + kChunk - 1) / kChunk;
  const size_t rows = a.rows < kMostRows ? a.rows : kMostRows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const uintptr_t p = (uintptr_t)ws + at;  // (integers: a plan has no workspace)
    at += align_up(bytes, 16);
    return (void*)p;
  };
  a.masses = (double*)take(rows * chunks * sizeof(double));
  a.maxima = (float*)take(rows * chunks * kGroups * sizeof(float));
  if (a.top_k || a.top_p || a.min_p) {
    a.slices = slices_of(rows, chunks, cus);
    a.kept = (double*)take(rows * chunks * sizeof(double));
    a.parts = (float*)take(rows * a.slices * kBuckets * sizeof(float));
    a.lists = (uint64_t*)take(rows * kList * sizeof(uint64_t));
    a.states = (SampleState*)take(rows * sizeof(SampleState));
  }
  return at;
}

hipError_t launch_sample(const SampleArgs& all, int dtype, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  hipError_t e = hipSuccess;
  for (int64_t r = 0; r < all.rows && e == hipSuccess; r += kMostRows) {
    SampleArgs a = all;
    a.rows = (int)(all.rows - r < kMostRows ? all.rows - r : kMostRows);
    a.logits = (const char*)all.logits + r * all.stride * value_bytes(dtype);
    a.u += r;
    a.ids += r;
    if (a.temperature) a.temperature += r;
    if (a.top_k) a.top_k += r;
    if (a.top_p) a.top_p += r;
    if (a.min_p) a.min_p += r;
    if (a.probs) a.probs += r;
    switch (dtype) {
      case QMM_X_F16: e = launch_type<QMM_X_F16>(a, st); break;
      case QMM_X_BF16: e = launch_type<QMM_X_BF16>(a, st); break;
      default: e = launch_type<QMM_X_F32>(a, st);
    }
  }
  return e;
}

}  // namespace qmm
