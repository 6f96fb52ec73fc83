// attend.hip — causal attention of each sequence's new tokens over its pages
// of the Q8_0 cache (kv_cache.hip): grouped heads, a sliding window, a learned
// sink a head, ragged batches (the reference's split-KV decode attention,
// kernels/decode_attn.cu:257-612, over its f16 cache).
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m))
// over the positions j of the sequence with pos - window < j <= pos, m their
// largest s_j (or the sink). A row that no position is left to is zero.
#include "../../include/qmm.h"
#include "attend.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// One wave a query row and head: 64 positions at a time, a lane a position
// for the scores, then a lane a dim for the values.
template <int T>
__global__ __launch_bounds__(64) void attend_row_kernel(AttendArgs a) {
  __shared__ float s_p[64];
  __shared__ int64_t s_slot[64];
  const CachePlanes& c = a.c;
  const int lane = threadIdx.x, head = blockIdx.y, b = blockIdx.z;
  int64_t q0;
  int nq, kv;
  sequence(a, b, q0, nq, kv);
  const int i = blockIdx.x;
  if (i >= nq) return;
  const int64_t pos = (int64_t)kv - nq + i;
  const int kvh = head / a.group;
  const int64_t row = q0 + i;
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t first = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  for (int64_t j0 = first; j0 <= pos; j0 += 64) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    int64_t slot = -1;
    if (j <= pos) {
      const int64_t page = page_of(a, b, j);
      if (page >= 0) {
        const int at = (int)(j % c.page);
        slot = (page * c.heads + kvh) * c.page + at;
        float dot = 0.0f;
        for (int e = 0; e < c.hd; e++)
          dot = __builtin_fmaf(load1<T>(a.q, row * a.qs + head * a.qhs + e),
                               (float)c.k_codes[slot * c.hd + e] * h2f(c.k_scales[slot * (c.hd / 32) + (e >> 5)]), dot);
        s = dot * a.scale * kLog2e;
      }
    }
    float mt = s;
    for (int x = 32; x >= 1; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x, kWave));
    if (mt == -INFINITY) continue;  // uniform: the wave's own maximum
    const float mn = fmaxf(m, mt), f = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * f + wave_sum(p);
    s_p[lane] = p;
    s_slot[lane] = slot;
    __syncthreads();
    for (int u = 0; u < 4; u++) {
      const int e = lane + 64 * u;
      if (e >= c.hd) break;
      float acc = o[u] * f;
      for (int t = 0; t < 64; t++) {
        if (s_slot[t] < 0) continue;
        const int64_t ph = s_slot[t] / c.page;
        const int at = (int)(s_slot[t] - ph * c.page);
        acc = __builtin_fmaf(s_p[t], (float)c.v_codes[(ph * c.hd + e) * c.page + at] *
                                         h2f(c.v_scales[(ph * (c.hd / 32) + (e >> 5)) * c.page + at]), acc);
      }
      o[u] = acc;
    }
    __syncthreads();
  }
  if (a.sinks && l > 0.0f) {
    const float sk = a.sinks[head] * kLog2e, mn = fmaxf(m, sk), f = exp2f(m - mn);
    l = l * f + exp2f(sk - mn);
    for (int u = 0; u < 4; u++) o[u] *= f;
  }
  for (int u = 0; u < 4; u++) {
    const int e = lane + 64 * u;
    if (e < c.hd) store1(a.out, a.odt, row * a.os + head * c.hd + e, l > 0.0f ? o[u] / l : 0.0f);
  }
}

}  // namespace

size_t attend_workspace_bytes(const AttendArgs&, int) { return 0; }

hipError_t launch_attend(const AttendArgs& a, int cus, void* ws, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  const dim3 grid((unsigned)a.max_q, (unsigned)a.heads, (unsigned)a.seqs);
  switch (a.qdt) {
    case QMM_X_F32: attend_row_kernel<QMM_X_F32><<<grid, 64, 0, st>>>(a); break;
    case QMM_X_F16: attend_row_kernel<QMM_X_F16><<<grid, 64, 0, st>>>(a); break;
    default: attend_row_kernel<QMM_X_BF16><<<grid, 64, 0, st>>>(a); break;
  }
  return hipGetLastError();
}

}  // namespace qmm
