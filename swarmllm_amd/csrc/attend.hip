// attend.hip — causal attention of each sequence's new tokens over its pages
// of the Q8_0 cache (kv_cache.hip): grouped heads, a sliding window, a learned
// sink a head, ragged batches (the reference's split-KV decode attention,
// kernels/decode_attn.cu:257-612, over its f16 cache). The launches' choice
// and the join of a context's parts; the kernels are attend_few.hip's and
// attend_chunk.hip's.
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m))
// over the positions j of the sequence with pos - window < j <= pos, m their
// largest s_j. A row that no position is left to is zero.
#include "attend.h"

namespace qmm {

namespace {

// 4 dims of a row a thread, over the parts in order.
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, int lo_rows, int hi_rows, AttendParts p) {
  const int hd = a.c.hd, per = hd / 4;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t pr = x / per;
  const int e = 4 * (int)(x - pr * per);
  const int64_t hb = pr / p.rows;  // (head of a sequence, block)
  const int row = (int)(pr - hb * p.rows);
  const int64_t hs = hb / p.blocks;
  const int block = (int)(hb - hs * p.blocks);
  const int64_t b = hs / a.c.heads;
  if (b >= a.seqs) return;
  int64_t q0;
  int nq, kv;
  sequence(a, (int)b, q0, nq, kv);
  const int rows = nq * a.group, r = block * p.rows + row;
  if (rows <= lo_rows || rows > hi_rows || r >= rows) return;
  float top = -INFINITY;
  for (int s = 0; s < p.parts; s++) top = fmaxf(top, p.ml[2 * part_row(p, hs, block, s, row)]);
  const float base = top == -INFINITY ? 0.0f : top;
  f4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f;
  for (int s = 0; s < p.parts; s++) {
    const int64_t i = part_row(p, hs, block, s, row);
    const float f = exp2_fast(p.ml[2 * i] - base);
    sum += p.ml[2 * i + 1] * f;
    acc += *(const f4v*)(p.o + i * hd + e) * f;
  }
  const int i = r / a.group, head = (int)(hs - b * a.c.heads) * a.group + r - i * a.group;
  float out[4];
  finish_row<4>(a, head, top, sum, (const float*)&acc, out);
  store_out4(a, (q0 + i) * a.os + (int64_t)head * hd + e, out);
}

// How a call runs: the sequences of at most `few` query rows a kv head on the
// few-row kernel (0: none), the others on the chunk kernel.
struct Plan {
  int few, few_parts, chunk_blocks, chunk_parts;
};

int clamp_parts(int64_t want, int64_t most) {
  const int64_t p = want < most ? want : most;
  return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
}

Plan plan_of(const AttendArgs& a, int cus) {
  Plan p{};
  const int64_t rows = (int64_t)a.max_q * a.group, heads = (int64_t)a.seqs * a.c.heads;
  int64_t span = a.max_kv;  // the positions that a row block's rows see at most
  if (rows > kFewRows) {
    if (a.window > 0 && a.window + kChunkRows / a.group + 1 < span) span = a.window + kChunkRows / a.group + 1;
    const int64_t tiles = (span + kTile - 1) / kTile;
    p.chunk_blocks = (int)((rows + kChunkRows - 1) / kChunkRows);
    // parts until two workgroups a CU are there, of 8 steps at least
    p.chunk_parts = clamp_parts(2 * cus / (heads * p.chunk_blocks), tiles / 8);
    if (a.seqs > 1) p.few = 16;  // one-token sequences beside a prompt
  } else {
    p.few = rows <= 16 ? 16 : kFewRows;
  }
  if (p.few) {
    span = a.max_kv;
    if (a.window > 0 && a.window + p.few / a.group + 1 < span) span = a.window + p.few / a.group + 1;
    // parts until two workgroups a CU are there, of 4 steps a wave at least
    p.few_parts = clamp_parts(2 * cus / heads, ((span + kTile - 1) / kTile) / 16);
  }
  return p;
}

// The partial results at ws: bytes, and where they lie.
size_t parts_at(const AttendArgs& a, int parts, int rows, int blocks, void* ws, AttendParts& p) {
  p = AttendParts{nullptr, nullptr, parts, rows, blocks};
  if (parts <= 1) return 0;
  const size_t n = (size_t)a.seqs * a.c.heads * blocks * parts * rows;
  p.o = (float*)ws;
  p.ml = p.o + n * a.c.hd;
  return n * (a.c.hd + 2) * sizeof(float);
}

hipError_t join(const AttendArgs& a, int lo, int hi, const AttendParts& p, hipStream_t st) {
  const int64_t threads = (int64_t)a.seqs * a.c.heads * p.blocks * p.rows * (a.c.hd / 4);
  attend_join_kernel<<<dim3((unsigned)((threads + 255) / 256)), 256, 0, st>>>(a, lo, hi, p);
  return hipGetLastError();
}

}  // namespace

bool attend_fits(const AttendArgs& a) {
  const int64_t rows = (int64_t)a.max_q * a.group;
  const int64_t heads = (int64_t)a.seqs * a.c.heads;
  return rows <= (int64_t)65535 * kChunkRows && heads * (rows + kChunkRows) * (a.c.hd / 4) < ((int64_t)1 << 39) &&
         heads < ((int64_t)1 << 31);
}

size_t attend_workspace_bytes(const AttendArgs& a, int cus) {
  const Plan p = plan_of(a, cus);
  AttendParts q;
  const size_t few = p.few ? parts_at(a, p.few_parts, p.few, 1, nullptr, q) : 0;
  const size_t chunk = p.chunk_blocks ? parts_at(a, p.chunk_parts, kChunkRows, p.chunk_blocks, nullptr, q) : 0;
  return few > chunk ? few : chunk;  // one after the other
}

hipError_t launch_attend(const AttendArgs& a, int cus, void* ws, hipStream_t st) {
  const Plan p = plan_of(a, cus);
  AttendParts q;
  hipError_t e = hipSuccess;
  if (p.chunk_blocks) {
    parts_at(a, p.chunk_parts, kChunkRows, p.chunk_blocks, ws, q);
    e = launch_attend_chunk(a, p.few, q, st);
    if (e == hipSuccess && q.parts > 1) e = join(a, p.few, INT32_MAX, q, st);
  }
  if (p.few && e == hipSuccess) {
    parts_at(a, p.few_parts, p.few, 1, ws, q);
    e = launch_attend_few(a, 0, p.few, q, st);
    if (e == hipSuccess && q.parts > 1) e = join(a, 0, p.few, q, st);
  }
  return e;
}

}  // namespace qmm
