// attend.hip — causal attention of each sequence's new tokens over its pages
// of the Q8_0 cache (kv_cache.hip): grouped heads, a sliding window, a learned
// sink a head, ragged batches. The launches' choice and the join of a context's
// parts; the kernels are attend_few.hip's and attend_chunk.hip's.
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m))
// over the positions j of the sequence with pos - window < j <= pos, m their
// largest s_j. A row that no position is left to is zero.
//
// q, keys (code * scale), values and weights are f16 operands of the matrix
// cores, each rounded once; scores, maxima, sums and outputs are f32. The
// rounding, 2^-11 of a value, is an eighth of the half step that a code's own
// rounding leaves (1 / 254 of its block's largest); f16 outputs end 4e-4 to
// 5e-4 from 64 bits (an exact sum's rounding: 2e-4), f32 ones from f32 queries
// 5.4e-4 to 5.6e-4. f32 operands run at a 16th of the rate.
#include "attend.h"

namespace qmm {

namespace {

// A wave joins 64 / (hd / 4) rows, 4 dims a lane. G == 4: the parts of those
// rows are dealt to the workgroup's 4 waves in turn and joined in LDS (many
// parts); G == 1: each wave takes all parts of rows of its own.
template <int G>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, int lo_rows, int hi_rows, AttendParts p) {
  const int hd = a.c.hd, per = hd / 4, fit = 64 / per;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane / per, e = 4 * (lane - sub * per), first = G > 1 ? wave : 0;
  // rows of one kv head of a sequence, block after block
  const int64_t row_of_head = ((int64_t)blockIdx.x * (4 / G) + (G > 1 ? 0 : wave)) * fit + sub;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int block = (int)(row_of_head / p.rows), row = (int)(row_of_head - (int64_t)block * p.rows);
  int64_t q0;
  int nq, kv, pos0;
  sequence(a, b, q0, nq, kv, pos0);
  const int rows = nq * a.group;
  const int cut = cut_index(a, p, b * a.c.heads + kvh, block);
  const bool on = sub < fit && cut >= 0 && rows > lo_rows && rows <= hi_rows && row_of_head < rows;
  float top = -INFINITY, sum = 0.0f;
  f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (on) {
    const int64_t i0 = part_row(p, cut, first, row), step = G * (int64_t)p.rows;
    const int n = (p.parts - first + G - 1) / G;
#pragma unroll 4
    for (int s = 0; s < n; s++) {
      const int64_t i = i0 + s * step;
      const float m = p.ml[2 * i], l = p.ml[2 * i + 1];
      const f4v o = *(const f4v*)(p.o + i * hd + e);
      const float mx = fmaxf(top, m), base = mx == -INFINITY ? 0.0f : mx;
      const float fa = weight_of(a, top, base), fb = weight_of(a, m, base);
      top = mx;
      sum = sum * fa + l * fb;
      acc = acc * fa + o * fb;
    }
  }
  if constexpr (G > 1) {
    __shared__ f4v s_o[G][64];
    __shared__ float s_m[G][64], s_l[G][64];
    s_o[wave][lane] = acc;
    s_m[wave][lane] = top;
    s_l[wave][lane] = sum;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < G; w++) top = fmaxf(top, s_m[w][lane]);
    const float base = top == -INFINITY ? 0.0f : top;
    sum = 0.0f;
    acc = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < G; w++) {
      const float f = weight_of(a, s_m[w][lane], base);
      sum += s_l[w][lane] * f;
      acc += s_o[w][lane] * f;
    }
  }
  if (!on) return;
  const int r = (int)row_of_head, i = token_of(a, r), head = kvh * a.group + r - i * a.group;
  float out[4];
  finish_row<4>(a, head, top, sum, (const float*)&acc, out);
  store_out4(a, (q0 + i) * a.os + (int64_t)head * hd + e, out);
}

// A block that shares have split: its pieces from the share that began it to
// the one that ended it. 4 dims a lane, 64 / (hd / 4) rows a wave.
__global__ __launch_bounds__(256) void attend_join_shares_kernel(AttendArgs a, AttendParts p) {
  const int w = blockIdx.x;
  const int4 split = p.split[w];
  if (split.w < 0) return;
  const int hd = a.c.hd, per = hd / 4, fit = 64 / per;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane / per, e = 4 * (lane - sub * per), row = (blockIdx.y * 4 + wave) * fit + sub;
  const int b = split.x, kvh = split.y, r = split.z * kShareRows + row;
  int64_t q0;
  int nq, kv, pos0;
  sequence(a, b, q0, nq, kv, pos0);
  if (sub >= fit || row >= kShareRows || r >= nq * a.group) return;
  float top = -INFINITY, sum = 0.0f;
  f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int v = w; v <= split.w; v++) {
    const int64_t i = share_row(v == w ? 2 * w + 1 : 2 * v, row);
    const float m = p.ml[2 * i], l = p.ml[2 * i + 1];
    const f4v o = *(const f4v*)(p.o + i * hd + e);
    const float mx = fmaxf(top, m), base = mx == -INFINITY ? 0.0f : mx;
    const float fa = weight_of(a, top, base), fb = weight_of(a, m, base);
    top = mx;
    sum = sum * fa + l * fb;
    acc = acc * fa + o * fb;
  }
  const int i = token_of(a, r), head = kvh * a.group + r - i * a.group;
  float out[4];
  finish_row<4>(a, head, top, sum, (const float*)&acc, out);
  store_out4(a, (q0 + i) * a.os + (int64_t)head * hd + e, out);
}

// How a call runs: the sequences of at most `few` query rows a kv head on the
// few-row kernel (0: none), the others on the chunk kernel.
struct Plan {
  int few, few_parts, chunk_rows, chunk_blocks, chunk_cut, chunk_parts, shares;
};

int clamp_parts(int64_t want, int64_t most) {
  const int64_t p = want < most ? want : most;
  return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
}

// Steps that a block of `rows` query rows takes at most.
int64_t most_steps(const AttendArgs& a, int rows) {
  int64_t span = a.max_kv;
  if (a.window > 0 && a.window + rows / a.group + 1 < span) span = a.window + rows / a.group + 1;
  return (span + kTile - 1) / kTile;
}

Plan plan_of(const AttendArgs& a, int cus) {
  Plan p{};
  const int64_t rows = (int64_t)a.max_q * a.group, heads = (int64_t)a.seqs * a.c.heads;
  if (rows > kFewRows) {
    // blocks of 256 rows lay a step's keys and values down once for 8 waves;
    // over short contexts twice as many workgroups are worth more (us, 256 /
    // 128 rows: 512 tokens over 4096, 32 heads on 8 of 128 dims, 67 / 71; 2000 and 1333 over
    // 7777 and 5832, 64 on 8 of 128, 866 / 937; 1000 over 1000, 32 on 8 of 64, 35 / 32; 8 x 64
    // over 2000, 64 on 8 of 64, 50 / 48)
    p.chunk_rows = a.c.hd <= 128 && rows > kShareRows && most_steps(a, kShareRows) >= 32 ? kShareRows : 128;
    p.chunk_blocks = (int)((rows + p.chunk_rows - 1) / p.chunk_rows);
    const int64_t slots = (int64_t)cus * (p.chunk_rows > 128 || a.c.hd > 128 ? 1 : 2), n = heads * p.chunk_blocks;
    const double work = (double)(a.max_kv + 1024) * a.group * (double)n;  // in 64 bits
    if (p.chunk_rows == kShareRows && n > slots && n < 6 * slots && work < 1e17) {
      // a few rounds of the CUs: equal shares, so that the last round is whole and
      // sequences shorter than max_q and max_kv leave no CU idle (us, shares /
      // blocks, 64 heads on 8 of 128 dims: 2000 and 1333 tokens over 7777 and 5832 751 / 887; all of one length
      // 0 to 3 % slower: 2 x 2000 over 7777 985 / 981, 4000 over 7777 831 / 809). Many
      // rounds fill up by themselves, and their short blocks' beginnings count
      // more (7777 over 7777 1338 / 1083); fewer blocks than CUs are cut evenly
      // (512 over 4096, 32 heads on 8, 76 / 56).
      p.shares = cus;
    } else {
      // parts that fill the CUs, of 8 steps at least: of every block where those
      // are few, otherwise of what is left behind the last whole round of the CUs,
      // those blocks alone, so that the parts are never more than a round holds
      // (65 sequences of 5 tokens over 8192, 64 heads on 8 of 128, leave 8 blocks:
      // 301 us, 381 with that block of all 520 heads cut, over 554 MB of partial results)
      const int64_t left = n <= slots ? n : n % slots;
      p.chunk_parts = left ? clamp_parts(slots / left, most_steps(a, p.chunk_rows) / 8) : 1;
      p.chunk_cut = p.chunk_parts > 1 ? (int)left : 0;
    }
    if (a.seqs > 1) p.few = 16;  // one-token sequences beside a prompt
  } else {
    p.few = rows <= 16 ? 16 : kFewRows;
  }
  if (p.few) {
    // parts until two workgroups a CU are there, of one step a wave at least,
    // of four where the CUs have one each without, and none up to two steps a
    // wave (the join is a launch of 4 us, as much again for the host; graph
    // replays, us, 32 heads on 8 of 128 dims, the 16 64 on 8: 1 sequence of 500 whole 11.3, in 2 parts 10.8; of 2000 in 8
    // 11.1, in 2 18.1; 4 of 1000 in 4 10.6, whole 16.2; 16 of 8000 in 4 51.5, in 2
    // 68.1; 32 of 1000 whole 17.0, in 2 19.5)
    const int64_t steps = most_steps(a, p.few);
    p.few_parts = steps <= 2 * kFewWaves
                      ? 1
                      : clamp_parts(2 * cus / heads, steps / (heads < cus ? kFewWaves : 4 * kFewWaves));
  }
  return p;
}

// The partial results of `cut` blocks at ws: bytes, and where they lie.
size_t parts_at(const AttendArgs& a, int parts, int rows, int blocks, int cut, void* ws, AttendParts& p) {
  const int heads = a.seqs * a.c.heads;
  p = AttendParts{nullptr, nullptr, parts, rows, blocks, cut, cut / heads, cut % heads, nullptr, 0};
  if (parts <= 1) return 0;
  const size_t n = (size_t)cut * parts * rows;
  p.o = (float*)ws;
  p.ml = (float*)((uintptr_t)ws + n * a.c.hd * sizeof(float));  // (integers: a plan has no workspace)
  return n * (a.c.hd + 2) * sizeof(float);
}

// And those of `shares`.
size_t shares_at(const AttendArgs& a, int shares, void* ws, AttendParts& p) {
  p = AttendParts{(float*)ws, nullptr, 1, kShareRows, 0, 0, 0, 0, nullptr, shares};
  const size_t n = (size_t)2 * shares * kShareRows, sums = n * (a.c.hd + 2) * sizeof(float);
  p.ml = (float*)((uintptr_t)ws + n * a.c.hd * sizeof(float));
  p.split = (int4*)((uintptr_t)ws + sums);
  return sums + shares * sizeof(int4);
}

hipError_t join(const AttendArgs& a, int lo, int hi, const AttendParts& p, hipStream_t st) {
  // (us, parts dealt to 4 waves / all to one wave, 32 heads on 8 of 128 dims: 4 parts of 512 tokens' 64
  // blocks 11.9 / 7.8, 31 of one token's 32 heads 4.2 / 5.1, 64 of them 5.2 / 10.9)
  const bool deal = p.parts > 8;
  const int fit = 64 / (a.c.hd / 4) * (deal ? 1 : 4);
  const int64_t heads = (int64_t)a.seqs * a.c.heads, most = (int64_t)a.max_q * a.group;
  const int64_t held = (p.cut + heads - 1) / heads * p.rows, rows = most < held ? most : held;
  const dim3 grid((unsigned)((rows + fit - 1) / fit), (unsigned)a.c.heads, (unsigned)a.seqs);
  if (deal)
    attend_join_kernel<4><<<grid, 256, 0, st>>>(a, lo, hi, p);
  else
    attend_join_kernel<1><<<grid, 256, 0, st>>>(a, lo, hi, p);
  return hipGetLastError();
}

}  // namespace

bool attend_fits(const AttendArgs& a) {
  const int64_t rows = (int64_t)a.max_q * a.group;
  const int64_t heads = (int64_t)a.seqs * a.c.heads;
  return rows <= (int64_t)32000 * 128 && rows * a.group < ((int64_t)1 << 32) &&
         heads < ((int64_t)1 << 23);  // workgroups of 512 threads in a launch's x, which wraps at 2^32
}

size_t attend_workspace_bytes(const AttendArgs& a, int cus) {
  const Plan p = plan_of(a, cus);
  AttendParts q;
  const size_t few = p.few ? parts_at(a, p.few_parts, p.few, 1, a.seqs * a.c.heads, nullptr, q) : 0;
  const size_t chunk = p.shares ? shares_at(a, p.shares, nullptr, q) : p.chunk_blocks ? parts_at(a, p.chunk_parts, p.chunk_rows, p.chunk_blocks, p.chunk_cut, nullptr, q) : 0;
  return few > chunk ? few : chunk;  // one after the other
}

hipError_t launch_attend(const AttendArgs& a, int cus, void* ws, hipStream_t st) {
  const Plan p = plan_of(a, cus);
  AttendParts q;
  hipError_t e = hipSuccess;
  if (p.shares) {
    shares_at(a, p.shares, ws, q);
    e = launch_attend_chunk(a, p.few, q, st);
    if (e == hipSuccess) {
      const int rows = 4 * (64 / (a.c.hd / 4));
      attend_join_shares_kernel<<<dim3((unsigned)p.shares, (unsigned)((kShareRows + rows - 1) / rows)), 256, 0, st>>>(a, q);
      e = hipGetLastError();
    }
  } else if (p.chunk_blocks) {
    parts_at(a, p.chunk_parts, p.chunk_rows, p.chunk_blocks, p.chunk_cut, ws, q);
    e = launch_attend_chunk(a, p.few, q, st);
    if (e == hipSuccess && q.parts > 1) e = join(a, p.few, INT32_MAX, q, st);
  }
  if (p.few && e == hipSuccess) {
    parts_at(a, p.few_parts, p.few, 1, a.seqs * a.c.heads, ws, q);
    e = launch_attend_few(a, 0, p.few, q, st);
    if (e == hipSuccess && q.parts > 1) e = join(a, 0, p.few, q, st);
  }
  return e;
}

}  // namespace qmm
