// pages.hip — the page tables of a batch's sequences and the batch's rows, kept
// and made on the device: a step cuts sequences back, gives their pages to the
// stack of free ones, takes pages for the new tokens and says for every row of
// the batch which sequence, position and cache slot it has.
//
//   kept_b = ceil(keep_b / page), held_b = ceil(len_b / page),
//   need_b = ceil((keep_b + new_b) / page) - kept_b
// Freed page j (sequences and their pages in order) goes to free[F - 1 - j], F
// the count with all of them; page j taken (in the same order) comes from
// free[F - 1 - j]. So a step that cuts what the step before it added finds the
// same pages again, and the order of the stack never depends on timing.
//
// One workgroup plans: the running sums over the sequences (freed pages, rows,
// pages needed) in LDS, then the pages that change hands, one a thread, each
// finding its sequence by a binary search in those sums. Rows of a large batch
// are a second launch over the CUs.
//
// A step moves a few KiB and computes next to nothing: what it takes is a launch (2.6 us
// empty) and the latencies one after another of the loads, scans, searches and stores
// (8 sequences of one new token each 4.2 us), and with hundreds of sequences the one
// CU's instructions (256 sequences, 10240 rows 13.5 us).
#include <hip/hip_runtime.h>

#include "../../include/qmm.h"
#include "mv_common.h"
#include "wave_sums.h"

namespace qmm {

namespace {

constexpr int kMostThreads = 1024;
constexpr int kAtOnce = 2;  // pages a thread moves at once

// Running sums over the workgroup's threads (in `v`'s own type), and the total.
template <typename T>
__device__ __forceinline__ T block_sums(T v, T* wave_sums, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const T s = qmm::wave_sums(v);
  __syncthreads();  // the sums of the call before are read
  if (lane == 63) wave_sums[wave] = s;
  __syncthreads();
  T before = 0;
  total = 0;
  for (int w = 0; w < waves; w++) {
    const T x = wave_sums[w];
    if (w < wave) before += x;
    total += x;
  }
  return before + s - v;
}

// The last b < n with starts[b] <= j, for N numbers at once (starts ascending,
// starts[0] = 0; `top` the largest power of two below n, or 0).
__device__ __forceinline__ int top_step(int n) { return n > 1 ? 1 << (31 - __builtin_clz(n - 1)) : 0; }
template <int N>
__device__ __forceinline__ void owners(const int32_t* starts, int n, int top, const int32_t j[N], int b[N]) {
#pragma unroll
  for (int u = 0; u < N; u++) b[u] = 0;
  for (int step = top; step >= 1; step >>= 1) {
    int32_t s[N];
#pragma unroll
    for (int u = 0; u < N; u++) s[u] = starts[min(b[u] + step, n - 1)];
#pragma unroll
    for (int u = 0; u < N; u++)
      if (b[u] + step < n && s[u] <= j[u]) b[u] += step;
  }
}
__device__ __forceinline__ int owner(const int32_t* starts, int n, int top, int32_t j) {
  int b[1];
  owners<1>(starts, n, top, &j, b);
  return b[0];
}

// Pages that hold n positions (at most 2^30, so that nothing passes 32 bits).
__device__ __forceinline__ int32_t pages_of(const PagesArgs& a, int32_t n) {
  return (n + (1 << a.page_bits) - 1) >> a.page_bits;
}

__device__ __forceinline__ void write_row(const PagesArgs& a, int64_t t, int b, int32_t pos) {
  int64_t slot = -1;
  if (pos >= 0) {
    const int32_t p = a.tables[b * (int32_t)a.table_stride + (pos >> a.page_bits)];
    if (p >= 0) slot = ((int64_t)p << a.page_bits) + (pos & ((1 << a.page_bits) - 1));
  }
  a.slots[t] = slot;
  if (a.positions) a.positions[t] = pos;
  if (a.seq) a.seq[t] = b;
}

// s_* hold the sequences' running sums, s_keep what each keeps.
__global__ __launch_bounds__(kMostThreads) void pages_plan_kernel(PagesArgs a, int with_rows) {
  // (all of it dynamic: a limit raised to the CU's 160 KiB leaves no room for more)
  extern __shared__ int64_t lds[];
  const int n = a.seqs, tid = threadIdx.x, threads = blockDim.x;
  int64_t* const wave_sums = lds;             // [kMostThreads / 64]
  int32_t* const s_keep = (int32_t*)(lds + kMostThreads / 64);  // [n]
  int32_t* const s_freed = s_keep + n;        // [n + 1] pages given back before b
  int32_t* const s_need = s_freed + n + 1;    // [n + 1] pages taken before b
  int32_t* const s_rows = s_need + n + 1;     // [n + 1] rows before b
  int32_t* const s_took = s_rows + n + 1;     // [n] tokens taken, -1: refused
  const int64_t cap = a.row_pages << a.page_bits;
  const int top = top_step(n);

  int64_t freed_before = 0, rows_before = 0;
  for (int b0 = 0; b0 < n; b0 += threads) {
    const int b = b0 + tid;
    int32_t len = 0, keep = 0;
    int64_t add = 0;
    if (b < n) {
      len = (int32_t)max((int64_t)0, min((int64_t)a.lens[b], cap));
      keep = a.keep ? a.keep[b] : len;
      if (keep < 0 || keep > len) keep = len;
      add = a.fresh ? max(0, a.fresh[b]) : 0;
      s_keep[b] = keep;
    }
    const int32_t back = pages_of(a, len) - pages_of(a, keep);
    int64_t total;
    const int64_t f = freed_before + block_sums<int64_t>(back, wave_sums, total);
    freed_before += total;
    const int64_t r = rows_before + block_sums<int64_t>(add, wave_sums, total);
    rows_before += total;
    if (b < n) {
      s_freed[b] = (int32_t)f;
      s_rows[b] = (int32_t)min(r, a.tokens);
      const bool fits = r + add <= a.tokens && keep + add <= cap;
      s_took[b] = fits ? (int32_t)add : -1;
    }
  }
  const int32_t freed = (int32_t)freed_before;
  if (tid == 0) {
    s_freed[n] = freed;
    s_rows[n] = (int32_t)min(rows_before, a.tokens);
  }
  const int64_t count = max((int64_t)0, min((int64_t)a.free_count[0], a.pool));
  const int64_t have = min(count + freed, a.pool);

  int64_t need_before = 0;
  for (int b0 = 0; b0 < n; b0 += threads) {
    const int b = b0 + tid;
    int32_t keep = 0, took = 0;
    if (b < n) {
      keep = s_keep[b];
      took = s_took[b];
    }
    const int32_t want = took > 0 ? pages_of(a, keep + took) - pages_of(a, keep) : 0;
    int64_t total;
    const int64_t before = need_before + block_sums<int64_t>(want, wave_sums, total);
    need_before += total;
    if (b < n) {
      // the sequences whose pages are there are the first ones: behind them nothing more is taken
      s_need[b] = (int32_t)min(before, have);
      if (want > 0 && before + want > have) s_took[b] = -1;
    }
  }
  // (a refused sequence's share of what is left is taken by none)
  if (tid == 0) s_need[n] = (int32_t)min(need_before, have);
  __syncthreads();

  // the pages given back, on top of the stack, the first of them its end; two
  // a thread at once, so that their searches and loads overlap (eight take no less: a search is 80 instructions)
  for (int32_t j0 = tid; j0 < freed; j0 += kAtOnce * threads) {
    int32_t* entry[kAtOnce];
    int32_t p[kAtOnce], j[kAtOnce];
    int of[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) j[u] = min(j0 + u * threads, freed - 1);
    owners<kAtOnce>(s_freed, n, top, j, of);
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const int b = of[u];
      entry[u] = a.tables + b * (int32_t)a.table_stride + pages_of(a, s_keep[b]) + (j[u] - s_freed[b]);
      p[u] = *entry[u];
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const int64_t at = have - 1 - (j0 + u * threads);
      if (j0 + u * threads >= freed) break;
      if (at >= 0) a.free_pages[at] = p[u];
      *entry[u] = -1;
    }
  }
  __syncthreads();
  int32_t popped = 0;
  const int32_t wanted = s_need[n];
  for (int32_t j0 = tid; j0 < wanted; j0 += kAtOnce * threads) {
    int32_t* entry[kAtOnce];
    int32_t p[kAtOnce], j[kAtOnce];
    int of[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) j[u] = min(j0 + u * threads, wanted - 1);
    owners<kAtOnce>(s_need, n, top, j, of);
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const int b = of[u];
      const bool takes = j0 + u * threads < wanted && s_took[b] >= 0;
      entry[u] = takes ? a.tables + b * (int32_t)a.table_stride + pages_of(a, s_keep[b]) + (j[u] - s_need[b]) : nullptr;
      p[u] = a.free_pages[have - 1 - j[u]];
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; u++)
      if (entry[u]) {
        *entry[u] = p[u];
        popped = j0 + u * threads + 1;
      }
  }
  int64_t total;
  // (each thread's last page: the most of them is what left the stack)
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) popped = max(popped, __shfl_xor(popped, d, 64));
  __syncthreads();
  if ((tid & 63) == 0) wave_sums[tid >> 6] = popped;
  __syncthreads();
  total = 0;
  for (int w = 0; w < threads >> 6; w++) total = max(total, wave_sums[w]);
  if (tid == 0) a.free_count[0] = (int32_t)(have - total);
  for (int b = tid; b < n; b += threads) {
    a.lens[b] = s_keep[b] + max(0, s_took[b]);
    a.taken[b] = max(0, s_took[b]);
  }
  for (int b = tid; b <= n; b += threads) a.q_starts[b] = s_rows[b];
  if (!with_rows) return;
  for (int64_t t = tid; t < a.tokens; t += threads) {
    if (t >= s_rows[n]) {
      write_row(a, t, -1, -1);
    } else {
      const int b = owner(s_rows, n, top, (int32_t)t);
      write_row(a, t, b, s_took[b] < 0 ? -1 : s_keep[b] + ((int32_t)t - s_rows[b]));
    }
  }
}

// A large batch's rows, from what the plan left: a sequence that took nothing
// but has rows was refused.
__global__ __launch_bounds__(256) void pages_rows_kernel(PagesArgs a) {
  extern __shared__ int32_t s_rows[];
  for (int b = threadIdx.x; b <= a.seqs; b += 256) s_rows[b] = a.q_starts[b];
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  if (t >= s_rows[a.seqs]) {
    write_row(a, t, -1, -1);
    return;
  }
  const int b = owner(s_rows, a.seqs, top_step(a.seqs), (int32_t)t);
  const int32_t took = a.taken[b];
  write_row(a, t, b, took == 0 ? -1 : a.lens[b] - took + ((int32_t)t - s_rows[b]));
}

}  // namespace

int pages_most_seqs() { return 4096; }

hipError_t launch_pages_step(const PagesArgs& a, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  const size_t lds = kMostThreads / 64 * sizeof(int64_t) + (5 * (size_t)a.seqs + 3) * sizeof(int32_t);
  if (lds > 64 * 1024) {
    const hipError_t e = set_max_dynamic_lds<pages_plan_kernel>();
    if (e != hipSuccess) return e;
  }
  // (us in one launch / two: 1536 rows 10.4 / 12.4, 3840 12.4 / 12.5, 6400 14.6 / 12.7, 16384 30 / 16)
  const bool one = a.tokens <= 4 * kMostThreads;
  int64_t threads = one && a.tokens > a.seqs ? a.tokens : a.seqs;
  threads = threads > kMostThreads || !one ? kMostThreads : threads < 64 ? 64 : (threads + 63) / 64 * 64;
  pages_plan_kernel<<<1, (unsigned)threads, lds, st>>>(a, one ? 1 : 0);
  if (!one)
    pages_rows_kernel<<<(unsigned)((a.tokens + 255) / 256), 256, ((size_t)a.seqs + 1) * sizeof(int32_t), st>>>(a);
  return hipGetLastError();
}

}  // namespace qmm
