// sample.hip — a token for each row of logits, from a given uniform number.
//
//   w_i = exp((x_i - max x) / T)
// The values are ordered by x (equal ones by index, the lowest first). Of them
// the first top_k are kept; of those the shortest run whose weight reaches
// top_p of theirs (the first always); of those the ones with w >= min_p. The
// token is the first, by index, of the kept ones at which their running sum
// passes u times their total.
//
// Two launches. The first reads the logits once: of every 1024 values (a wave's,
// a chunk) the weight relative to the chunk's own largest, in 64 bits and one
// order, and the largest of each 256 (16 lanes' values, a group). The second, a
// workgroup a row, works from those: a row without settings draws a chunk by
// the chunks' weights and reads that one again. Settings need the values past
// a bound only: top_k the groups whose largest is among the k largest of the
// groups (the k-th of them bounds the k-th value from below), min_p those past
// its own line, top_p those past (1 - top_p) Z / n, which no value that ends
// the run can be under (n values of at most that weight follow it). Up to 1024
// values are sorted in LDS and every setting cut there; more are narrowed
// down first by histograms of counts and weights, the weights as whole numbers
// (2^S to the largest), so that no order of additions shows in them.
#include <cfloat>

#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

constexpr int kChunk = 1024, kGroups = 4;  // values a wave holds; groups in them
constexpr int kMostVocab = 1 << 19;
constexpr int kMostChunks = kMostVocab / kChunk;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kList = 1024;     // values that are sorted
constexpr int kBuckets = 2048;  // two a thread
constexpr double kLog2e = 1.4426950408889634;

// 16 values of chunk c at a lane's places 256 q + 4 lane + e; what is past the
// row, or NaN, is -inf.
template <int T, bool VEC>
__device__ __forceinline__ void load_chunk(const SampleArgs& a, int64_t row, int c, int lane, float v[16]) {
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int i = c * kChunk + 256 * q + 4 * lane;
    float* const o = v + 4 * q;
    if (i + 4 <= a.vocab) {
      load4<T, VEC>(a.logits, row * a.stride + i, o);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = i + e < a.vocab ? load1<T>(a.logits, row * a.stride + i + e) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = o[e] == o[e] ? o[e] : -INFINITY;
  }
}
__device__ __forceinline__ int index_of(int c, int lane, int e) { return c * kChunk + 256 * (e >> 2) + 4 * lane + (e & 3); }

// exp((x - top) / T), scale = log2(e) / T; 0 for -inf. (x == top: 1, also where both are inf.)
__device__ __forceinline__ double weight(float x, float top, double scale) {
  if (x == top) return 1.0;
  const double y = ((double)x - (double)top) * scale;
  return y > -1074.0 ? exp2(y) : 0.0;
}

__device__ __forceinline__ double scale_of(const SampleArgs& a, int64_t row, bool& greedy) {
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  greedy = !(t > 0.0f);
  return greedy ? 1.0 : kLog2e / (double)t;
}

template <int T, bool VEC>
__global__ __launch_bounds__(256) void sample_chunks_kernel(SampleArgs a, int chunks) {
  const int lane = threadIdx.x & 63, c = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = blockIdx.y;
  if (c >= chunks) return;
  float v[16];
  load_chunk<T, VEC>(a, row, c, lane, v);
  bool greedy;
  const double scale = scale_of(a, row, greedy);
  float m = v[0];
#pragma unroll
  for (int e = 1; e < 16; e++) m = fmaxf(m, v[e]);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if ((lane & 15) == 0) a.maxima[(row * chunks + c) * kGroups + (lane >> 4)] = m;
  m = fmaxf(m, __shfl_xor(m, 16, 64));
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  double s = 0.0;
  if (!greedy && m != -INFINITY) {
#pragma unroll
    for (int e = 0; e < 16; e++) s += weight(v[e], m, scale);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
  }
  if (lane == 0) a.masses[row * chunks + c] = s;
}

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
  float maxima[kMostChunks * kGroups];
  uint16_t active[kMostChunks * kGroups];
  union {
    struct {
      uint64_t mass[kBuckets];
      uint32_t count[kBuckets];
    } h;
    double group_mass[kMostChunks * kGroups];
  };
  uint64_t list[kList];
  double sums[kWaves];
  uint64_t sums64[kWaves];
  uint32_t sums32[kWaves];
  float tops[kWaves];
  int n_active, n_list, found;
};

__device__ __forceinline__ float block_max(float v, Shared& s) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.tops[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.tops[0];
  for (int w = 1; w < kWaves; w++) v = fmaxf(v, s.tops[w]);
  return v;
}

// The sum of the values of this thread and the ones before it, and all of them;
// in one order, whatever the values.
template <typename T>
__device__ __forceinline__ T block_sums(T v, T* waves, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T up = __shfl_up(v, d, 64);
    if (lane >= d) v += up;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  T before = 0;
  total = 0;
  for (int w = 0; w < kWaves; w++) {
    if (w == wave) before = total;
    total += waves[w];
  }
  return before + v;
}

// The least of the threads' numbers.
__device__ __forceinline__ int block_least(int v, Shared& s) {
  if (threadIdx.x == 0) s.found = INT32_MAX;
  __syncthreads();
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = min(v, __shfl_xor(v, d, 64));
  if ((threadIdx.x & 63) == 0) atomicMin(&s.found, v);
  __syncthreads();
  v = s.found;
  __syncthreads();
  return v;
}

// One number a thread, sorted over the first n2 threads (a power of two, 64 at least), the least first.
__device__ __forceinline__ uint64_t block_sort(uint64_t v, int n2, uint64_t* buf) {
  const int tid = threadIdx.x;
  for (int size = 2; size <= n2; size <<= 1) {
    for (int stride = size >> 1; stride >= 1; stride >>= 1) {
      uint64_t o;
      if (stride >= 64) {
        __syncthreads();
        buf[tid] = v;
        __syncthreads();
        o = buf[tid ^ stride];
      } else {
        o = __shfl_xor((unsigned long long)v, stride, 64);
      }
      const bool low = (tid & stride) == 0, up = (tid & size) == 0;
      if ((low == up) == (o < v)) v = o;
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

// The groups that hold a value of `lo` or more.
__device__ __forceinline__ void activate(Shared& s, int groups, float lo) {
  __syncthreads();
  if (threadIdx.x == 0) s.n_active = 0;
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kThreads)
    if (s.maxima[g] >= lo && s.maxima[g] != -INFINITY) s.active[atomicAdd(&s.n_active, 1)] = (uint16_t)g;
  __syncthreads();
}

// The values that `in` takes into the list (the first kList that come), and how many there are.
template <int T, bool VEC, typename In>
__device__ __forceinline__ int collect(const SampleArgs& a, int64_t row, Shared& s, In in) {
  __syncthreads();
  if (threadIdx.x == 0) s.n_list = 0;
  __syncthreads();
  each_value<T, VEC>(a, row, s, [&](float x, int i) {
    if (x != -INFINITY && in(x, i)) {
      const int at = atomicAdd(&s.n_list, 1);
      if (at < kList) s.list[at] = rank_of(x, i);
    }
  });
  __syncthreads();
  return s.n_list;
}

// What a row's settings ask of a prefix of the ordered values: `k` of them at
// most, or their weight.
struct Goal {
  bool by_count;
  uint64_t want;
};

// A histogram over the values that `bucket` gives a bucket (the larger the
// value, the lower), and the first bucket at which the goal is met: kBuckets
// if none. Counts and weights of the buckets before it are added to above_*,
// `inside` the bucket's own count.
template <int T, bool VEC, typename B>
__device__ __forceinline__ int narrow(const SampleArgs& a, int64_t row, Shared& s, const Goal& goal, float top,
                                      double scale, double unit, uint64_t& above_count, uint64_t& above_mass,
                                      uint32_t& inside, B bucket) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int b = tid; b < kBuckets; b += kThreads) {
    s.h.mass[b] = 0;
    s.h.count[b] = 0;
  }
  __syncthreads();
  each_value<T, VEC>(a, row, s, [&](float x, int i) {
    const int b = x != -INFINITY ? bucket(x, i) : -1;
    if (b < 0) return;
    atomicAdd(&s.h.count[b], 1u);
    atomicAdd((unsigned long long*)&s.h.mass[b], (unsigned long long)(weight(x, top, scale) * unit + 0.5));
  });
  __syncthreads();
  const uint32_t c0 = s.h.count[2 * tid], c1 = s.h.count[2 * tid + 1];
  const uint64_t m0 = s.h.mass[2 * tid], m1 = s.h.mass[2 * tid + 1];
  uint32_t all_count;
  uint64_t all_mass;
  const uint64_t count = above_count + block_sums<uint32_t>(c0 + c1, s.sums32, all_count);
  const uint64_t mass = above_mass + block_sums<uint64_t>(m0 + m1, s.sums64, all_mass);
  auto met = [&](uint64_t n, uint64_t m) { return n > 0 && (goal.by_count ? n : m) >= goal.want; };
  int b = INT32_MAX;
  if (met(count, mass)) b = met(count - c1, mass - m1) ? 2 * tid : 2 * tid + 1;
  b = block_least(b, s);
  if (b >= kBuckets) return kBuckets;
  // the sums before it are its thread's
  if (tid == b / 2) {
    s.sums64[0] = (b & 1 ? count - c1 : count - c1 - c0);
    s.sums64[1] = (b & 1 ? mass - m1 : mass - m1 - m0);
    s.sums32[0] = b & 1 ? c1 : c0;
  }
  __syncthreads();
  above_count = s.sums64[0];
  above_mass = s.sums64[1];
  inside = s.sums32[0];
  __syncthreads();
  return b;
}

// The rank of the last value of the prefix that meets the goal (0: all values
// meet it together or not at all), `mass` the prefix's weight.
template <int T, bool VEC, typename B>
__device__ __forceinline__ uint64_t last_of_prefix(const SampleArgs& a, int64_t row, Shared& s, const Goal& goal,
                                                   float top, double scale, double unit, uint64_t& mass, B bucket,
                                                   int first, uint64_t above_count, uint64_t above_mass, uint32_t inside) {
  // the keys of the bucket, which falls as they rise: between the first with
  // bucket <= `first` and the last with bucket >= it
  uint32_t lo = key_of(-FLT_MAX), hi = key_of(top);
  {
    uint32_t l = lo, h = hi;
    while (l < h) {
      const uint32_t m = l + (h - l) / 2;
      if (bucket(value_of(m), 0) <= first && bucket(value_of(m), 0) >= 0) h = m; else l = m + 1;
    }
    const uint32_t from = l;
    h = hi;
    while (l < h) {
      const uint32_t m = l + (h - l + 1) / 2;
      if (bucket(value_of(m), 0) >= first) l = m; else h = m - 1;
    }
    lo = from;
    hi = l;
  }
  while (inside > kList && lo < hi) {
    const uint32_t span = hi - lo, l = lo, h = hi;
    const int shift = span < (uint32_t)kBuckets ? 0 : 32 - __builtin_clz(span) - 11;
    const int b = narrow<T, VEC>(a, row, s, goal, top, scale, unit, above_count, above_mass, inside,
                                 [=](float x, int) {
                                   const uint32_t k = key_of(x);
                                   return k >= l && k <= h ? (int)((h - k) >> shift) : -1;
                                 });
    if (b >= kBuckets) break;  // (the bucket above met the goal: this is not reached)
    hi = h - ((uint32_t)b << shift);
    const uint32_t width = (1u << shift) - 1;
    lo = hi - l > width ? hi - width : l;
  }
  uint64_t last;
  const uint32_t l = lo, h = hi;
  if (inside <= kList) {
    const int n = min(kList, collect<T, VEC>(a, row, s, [=](float x, int) {
                         const uint32_t k = key_of(x);
                         return k >= l && k <= h;
                       }));
    const uint64_t r = ~block_sort(threadIdx.x < n ? ~s.list[threadIdx.x] : ~0ull, sort_size(n), s.list);
    const uint64_t w = threadIdx.x < n ? (uint64_t)(weight(ranked_value(r), top, scale) * unit + 0.5) : 0;
    uint64_t total;
    const uint64_t m = above_mass + block_sums<uint64_t>(w, s.sums64, total);
    const bool met = (goal.by_count ? above_count + threadIdx.x + 1 : m) >= goal.want;
    int at = block_least(threadIdx.x < n && met ? (int)threadIdx.x : INT32_MAX, s);
    at = min(at, n - 1);
    if (threadIdx.x == at) {
      s.sums64[0] = r;
      s.sums64[1] = m;
    }
    __syncthreads();
    last = s.sums64[0];
    mass = s.sums64[1];
    __syncthreads();
    return last;
  }
  // more equal values than the list holds: the first of them by index
  const uint64_t w = (uint64_t)(weight(value_of(h), top, scale) * unit + 0.5);
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
    const int b = narrow<T, VEC>(a, row, s, nth, top, scale, 0.0, before, unused, within, [=](float x, int i) {
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

template <int T, bool VEC>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a, int chunks, int bits) {
  __shared__ Shared s;
  const int tid = threadIdx.x, groups = chunks * kGroups;
  const int64_t row = blockIdx.x;
  bool greedy;
  const double scale = scale_of(a, row, greedy);
  float m = -INFINITY;
  for (int g = tid; g < groups; g += kThreads) {
    const float v = a.maxima[row * groups + g];
    s.maxima[g] = v;
    m = fmaxf(m, v);
  }
  const float top = block_max(m, s);
  if (top == -INFINITY) {  // no value left
    if (tid == 0) answer(a, row, -1, 0.0);
    return;
  }
  if (greedy) {
    activate(s, groups, top);
    int first = INT32_MAX;
    each_value<T, VEC>(a, row, s, [&](float x, int i) {
      if (x == top) first = min(first, i);
    });
    first = block_least(first, s);
    if (tid == 0) answer(a, row, first, 1.0);
    return;
  }

  // the chunks' weights relative to the row's largest value
  double mass = 0.0, total;
  if (tid < chunks) {
    float c = s.maxima[kGroups * tid];
#pragma unroll
    for (int g = 1; g < kGroups; g++) c = fmaxf(c, s.maxima[kGroups * tid + g]);
    if (c != -INFINITY) mass = a.masses[row * chunks + tid] * weight(c, top, scale);
  }
  double upto = block_sums<double>(mass, s.sums, total);

  const int k = a.top_k ? a.top_k[row] : 0;
  const bool k_on = k > 0 && k < a.vocab;
  const double p = a.top_p ? (double)a.top_p[row] : 1.0;
  const bool p_on = p < 1.0;
  const double floor = a.min_p && a.min_p[row] > 0.0f ? fmin((double)a.min_p[row], 1.0) : 0.0;
  const double unit = exp2((double)(63 - bits)), r_u = fmin(fmax((double)a.u[row], 0.0), 1.0);

  uint64_t last = 0;  // the rank of the last value kept
  const bool cut = k_on || p_on || floor > 0.0;
  if (cut) {
    // no value under `line` is kept (in units of log2 w), nor counts for another's place: under 2^-60 none does
    double line = -60.0;
    if (p_on && !k_on) line = fmax(line, log2(fmin((1.0 - p) * total / a.vocab, 1.0)) - 1e-6);
    if (floor > 0.0 && !(k_on && p_on)) line = fmax(line, log2(floor) - 1e-6);
    const double at = (double)top + line / scale;
    float lo = at >= (double)top ? top : (float)at;
    if ((double)lo > at) lo = value_of(key_of(lo) - 1);
    if (top == INFINITY) lo = top;
    const int merged = min(groups, kThreads);
    if (k_on && k <= merged) {
      float g = tid < groups ? s.maxima[tid] : -INFINITY;
      for (int j = tid + kThreads; j < groups; j += kThreads) g = fmaxf(g, s.maxima[j]);
      const uint64_t sorted = ~block_sort(tid < merged ? ~((uint64_t)key_of(g) << 32) : ~0ull, sort_size(merged), s.list);
      if (tid == k - 1) s.tops[0] = ranked_value(sorted);
      __syncthreads();
      lo = fmaxf(lo, s.tops[0]);
    }
    activate(s, groups, lo);
    // a run by weight alone asks for more values than it ends up with
    const bool narrow_first = p_on && !k_on;
    int n = narrow_first ? kList + 1 : collect<T, VEC>(a, row, s, [=](float x, int) { return x >= lo; });
    if (n > kList) {
      // narrowed down along the values first
      const float width = top - lo, inv = width > 0.0f && width < INFINITY ? (float)(kBuckets - 1) / width : 0.0f;
      auto bucket = [=](float x, int) {
        return x < lo ? -1 : x == top ? 0 : min(kBuckets - 1, (int)((top - x) * inv));
      };
      Goal goal{k_on, k_on ? (uint64_t)k : p_on ? (uint64_t)(fmax(p, 0.0) * total * unit) : ~0ull};
      uint64_t above_count = 0, above_mass = 0, kept_mass = 0;
      uint32_t inside = 0;
      int b = narrow<T, VEC>(a, row, s, goal, top, scale, unit, above_count, above_mass, inside, bucket);
      if (b < kBuckets && above_count + inside <= kList) {
        const int edge = b;
        n = collect<T, VEC>(a, row, s, [=](float x, int i) { return x >= lo && bucket(x, i) <= edge; });
      } else {
        if (b < kBuckets)
          last = last_of_prefix<T, VEC>(a, row, s, goal, top, scale, unit, kept_mass, bucket, b, above_count, above_mass,
                                        inside);
        else if (k_on && p_on)
          kept_mass = (uint64_t)(total * unit);  // fewer than k values have any weight
        if (k_on && p_on) {
          const Goal run{false, (uint64_t)(fmax(p, 0.0) * (double)kept_mass)};
          above_count = above_mass = 0;
          b = narrow<T, VEC>(a, row, s, run, top, scale, unit, above_count, above_mass, inside, bucket);
          if (b < kBuckets) {
            const uint64_t end = last_of_prefix<T, VEC>(a, row, s, run, top, scale, unit, kept_mass, bucket, b,
                                                        above_count, above_mass, inside);
            last = max(last, end);
          }
        }
        n = kList + 1;
      }
    }
    if (n <= kList) {
      // every value that can stay, the largest first
      uint64_t r = ~block_sort(tid < n ? ~s.list[tid] : ~0ull, sort_size(n), s.list);
      double w = tid < n && (!k_on || tid < k) ? weight(ranked_value(r), top, scale) : 0.0;
      double all;
      const double sum = block_sums<double>(w, s.sums, all);
      const double goal = fmax(p, 0.0) * (k_on ? all : total);
      const bool stays = tid < n && (!k_on || tid < k) && (!p_on || tid == 0 || sum - w < goal) && w >= floor;
      // and those that stay, by index
      __syncthreads();
      r = block_sort(stays ? (uint64_t)(uint32_t)~r << 32 | r >> 32 : ~0ull, sort_size(n), s.list);
      const bool there = r != ~0ull;
      const float x = value_of((uint32_t)r);
      w = there ? weight(x, top, scale) : 0.0;
      const double upto_here = block_sums<double>(w, s.sums, all);
      int hit = block_least(w > 0.0 && upto_here > r_u * all ? tid : INT32_MAX, s);
      if (hit == INT32_MAX) hit = -block_least(w > 0.0 ? -tid : INT32_MAX, s);  // u of 1
      if (tid == hit) answer(a, row, (int)(r >> 32), w / all);
      return;
    }
    // many values stay: their weight chunk by chunk
    if (last) activate(s, groups, fmaxf(lo, ranked_value(last)));
    for (int g = tid; g < groups; g += kThreads) s.group_mass[g] = 0.0;
    __syncthreads();
    for (int j = tid >> 4; j < s.n_active; j += kThreads / 16) {
      const int g = s.active[j], lane = (g & 3) * 16 + (tid & 15);
      float v[16];
      load_chunk<T, VEC>(a, row, g >> 2, lane, v);
      double sum = 0.0;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const double w = v[e] >= lo && rank_of(v[e], index_of(g >> 2, lane, e)) >= last ? weight(v[e], top, scale) : 0.0;
        sum += w >= floor ? w : 0.0;
      }
#pragma unroll
      for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
      if ((tid & 15) == 0) s.group_mass[g] = sum;
    }
    __syncthreads();
    mass = 0.0;
    if (tid < chunks)
      for (int g = 0; g < kGroups; g++) mass += s.group_mass[kGroups * tid + g];
    upto = block_sums<double>(mass, s.sums, total);
    // (values that are not there do not stay below)
    m = lo;
  } else {
    m = -FLT_MAX;
  }

  // the chunk that the number falls into, and the place in it
  const double r = r_u * total;
  int c = block_least(tid < chunks && mass > 0.0 && upto > r ? tid : INT32_MAX, s);
  if (c == INT32_MAX) c = -block_least(tid < chunks && mass > 0.0 ? -tid : INT32_MAX, s);
  if (tid == c) s.sums[0] = upto - mass;
  __syncthreads();
  if (tid >= 64) return;
  double sum = s.sums[0], chosen = 0.0;
  float v[16];
  load_chunk<T, VEC>(a, row, c, tid, v);
  int at = -1;
  for (int q = 0; q < 4; q++) {
    double w[4], mine = 0.0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = q == 0 ? v[e] : q == 1 ? v[4 + e] : q == 2 ? v[8 + e] : v[12 + e];
      const bool in = x != -INFINITY && (!cut || (x >= m && rank_of(x, index_of(c, tid, 4 * q + e)) >= last));
      w[e] = in ? weight(x, top, scale) : 0.0;
      if (cut && w[e] < floor) w[e] = 0.0;
      mine += w[e];
    }
    double run = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double up = __shfl_up(run, d, 64);
      if (tid >= d) run += up;
    }
    double before = sum + (run - mine);
    int place = -1, end = -1;
    double pw = 0.0, ew = 0.0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      before += w[e];
      if (w[e] > 0.0) {
        end = index_of(c, tid, 4 * q + e);
        ew = w[e];
        if (place < 0 && before > r) {
          place = end;
          pw = w[e];
        }
      }
    }
    const uint64_t hits = __ballot(place >= 0);
    if (hits) {
      const int l = __builtin_ctzll(hits);
      at = __shfl(place, l, 64);
      chosen = __shfl(pw, l, 64);
      break;
    }
    // (the sums of the chunk, in another order, can end below r: the last value with a weight)
    const uint64_t ends = __ballot(end >= 0);
    if (ends) {
      const int l = 63 - __builtin_clzll(ends);
      at = __shfl(end, l, 64);
      chosen = __shfl(ew, l, 64);
    }
    sum += __shfl(run, 63, 64);
  }
  if (tid == 0) answer(a, row, at, chosen / total);
}

template <int T>
hipError_t launch_type(const SampleArgs& a, hipStream_t st) {
  const int chunks = (a.vocab + kChunk - 1) / kChunk;
  int bits = 0;
  while (((int64_t)1 << bits) < a.vocab) bits++;
  const dim3 grid((unsigned)((chunks + 3) / 4), (unsigned)a.rows);
  if (a.vec) {
    sample_chunks_kernel<T, true><<<grid, 256, 0, st>>>(a, chunks);
    sample_rows_kernel<T, true><<<(unsigned)a.rows, kThreads, 0, st>>>(a, chunks, bits);
  } else {
    sample_chunks_kernel<T, false><<<grid, 256, 0, st>>>(a, chunks);
    sample_rows_kernel<T, false><<<(unsigned)a.rows, kThreads, 0, st>>>(a, chunks, bits);
  }
  return hipGetLastError();
}

}  // namespace

int64_t sample_most_vocab() { return kMostVocab; }

size_t sample_plan(SampleArgs& a, void* ws) {
  const size_t chunks = (size_t)a.rows * ((a.vocab + kChunk - 1) / kChunk);
  a.masses = (double*)ws;
  a.maxima = (float*)((uintptr_t)ws + chunks * sizeof(double));
  return chunks * (sizeof(double) + kGroups * sizeof(float));
}

hipError_t launch_sample(const SampleArgs& a, int dtype, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  switch (dtype) {
    case QMM_X_F16: return launch_type<QMM_X_F16>(a, st);
    case QMM_X_BF16: return launch_type<QMM_X_BF16>(a, st);
    default: return launch_type<QMM_X_F32>(a, st);
  }
}

}  // namespace qmm
