// norm.hip — residual addition and root-mean-square norm with the 8-bit
// activation of the products as its output, and such an activation read back.
//
// For each row: h = T(x + r) (one f32 addition, rounded to the stream's type
// T), ss = sum h^2, rs = f32(1 / sqrt(ss / k + eps)), y = f32(f32(h * rs) * w),
// and the codes, scales and sums of y as the activation quantizers write them
// (q8k_block_wave, q8_0_code): the planes equal qmm_quantize_act's of y bit
// for bit. The sum runs in 64 bits, and in one order for all the launch shapes
// that a row length can take (each of 16 sums takes every 16th block of 256
// values, a lane's values in turn, then the lanes', then the sums from the first
// on), so a row's bits do not follow from its batch. Built without FP
// contraction, which would join h * rs * w otherwise.
//
// A lane holds 4 consecutive values, a wave a 256-value block at a time (16-
// or 8-byte loads, whole lines), so a Q8_K block is one wave's and a Q8_0
// block 8 lanes'. A row stays in registers between its two passes, so what
// bounds a batch is its bytes: 2000 rows of 8192 f32 values with a residual take
// 49-51 us, 213 MB at 4.2-4.35 TB/s (a copy reaches 4.8). One row of 4096 takes
// 3.9-4.2 us (an empty launch 2.6), 77 of 2880 bf16 values 4.6-5.5.
#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

struct NormArgs {
  const void* x;
  const void* r;  // may be null
  const float* w;
  void* h;  // may be null, or x or r themselves
  void* y;  // may be null
  int8_t* codes;  // may be null: no activation
  float* d;
  void* sums;
  int64_t xs, rs, hs, ys, k, rows;
  float eps, qmax;
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// Four sums over the wave's lanes in wave_sum64's order; lanes 16 j and up
// hold that of v[j].
__device__ __forceinline__ double wave_sums64(const double v[4], int lane) {
  const bool b5 = lane & 32, b4 = lane & 16;
  const double a0 = (b5 ? v[2] : v[0]) + __shfl_xor(b5 ? v[0] : v[2], 32, kWave);
  const double a1 = (b5 ? v[3] : v[1]) + __shfl_xor(b5 ? v[1] : v[3], 32, kWave);
  double s = (b4 ? a1 : a0) + __shfl_xor(b4 ? a0 : a1, 16, kWave);
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor(s, m, kWave);
  return s;
}

// The 4 values at element e of a row (h as stored: rounded to T), and h out.
template <int T, bool VEC>
__device__ __forceinline__ void load_h(const NormArgs& a, int64_t row, int64_t e, float v[4]) {
  load4<T, VEC>(a.x, row * a.xs + e, v);
  if (a.r) {
    float u[4];
    load4<T, VEC>(a.r, row * a.rs + e, u);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = round_to<T>(v[i] + u[i]);
  }
}

// The norm and quantization of the 4 values at element e. All lanes of the
// wave call; `on` is the same for all 8 lanes of a 32-value block (and, for
// Q8_K, for the wave).
template <int LAYOUT, bool VEC>
__device__ __forceinline__ void emit(const NormArgs& a, int64_t row, int64_t e, bool on, const float h[4], float rs,
                                     int ydt) {
  const int lane = threadIdx.x & 63;
  float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (on) {
    float w[4];
    load4<QMM_X_F32, VEC>(a.w, e, w);
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = (h[i] * rs) * w[i];
    if (a.y) store4<VEC>(a.y, ydt, row * a.ys + e, y);
  }
  if (!a.codes) return;
  if (LAYOUT == ACT_Q8K) {
    uint32_t c;
    int32_t s16;
    float d;
    q8k_block_wave(y, lane, a.qmax, c, s16, d);
    if (!on) return;
    *(uint32_t*)(a.codes + row * a.k + e) = c;
    if ((lane & 3) == 0) ((int16_t*)a.sums)[(row * a.k + e) >> 4] = (int16_t)s16;
    if (lane == 0) a.d[(row * a.k + e) >> 8] = d;
  } else {
    float m = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
    uint32_t mb = __float_as_uint(fmaxf(m, 0.0f));
    mb = max(mb, dpp_u<0xB1>(mb));   // pairs
    mb = max(mb, dpp_u<0x4E>(mb));   // quads
    mb = max(mb, dpp_u<0x141>(mb));  // the two quads of 8 lanes
    const float d = __uint_as_float(mb) / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    const uint32_t c = pack4_i8(q8_0_code(y[0] * id), q8_0_code(y[1] * id), q8_0_code(y[2] * id), q8_0_code(y[3] * id));
    int32_t s = __builtin_amdgcn_sdot4((int)c, 0x01010101, 0, false);
    s += (int32_t)dpp_u<0xB1>((uint32_t)s);
    s += (int32_t)dpp_u<0x4E>((uint32_t)s);
    s += (int32_t)dpp_u<0x141>((uint32_t)s);
    if (!on) return;
    *(uint32_t*)(a.codes + row * a.k + e) = c;
    if ((lane & 7) == 0) {
      a.d[(row * a.k + e) >> 5] = h2f(f2h(d));
      ((int32_t*)a.sums)[(row * a.k + e) >> 5] = s;
    }
  }
}

// WPR waves a row, NB blocks of 256 values a wave (NB == 0: any number, the
// row read a second time). A workgroup of fewer than 4 waves a row takes
// several rows.
template <int T, int LAYOUT, int WPR, int NB, bool VEC>
__global__ __launch_bounds__(WPR < 4 ? 256 : WPR * 64) void rms_norm_act_kernel(NormArgs a, int ydt) {
  constexpr int kRows = WPR < 4 ? 4 / WPR : 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = wave % WPR;
  const int64_t row = wide_block() * kRows + wave / WPR;
  const bool row_on = row < a.rows;  // no early return: the waves of a row meet at a barrier
  constexpr int kHeld = NB ? NB : 1;
  constexpr int kSums = WPR == 4 ? 4 : 1;  // 16 of a row that more than one wave takes
  static_assert(WPR == 1 || WPR * kSums == 16, "the same 16 in each shape");
  float h[kHeld][4];
  double sums[kSums] = {};
  const int64_t e0 = (int64_t)sub * 256 + 4 * lane;
  if (row_on) {
    if (NB) {
#pragma unroll
      for (int b = 0; b < kHeld; b++) {
        const int64_t e = e0 + (int64_t)b * WPR * 256;
        if (e < a.k) load_h<T, VEC>(a, row, e, h[b]);
      }
#pragma unroll
      for (int b = 0; b < kHeld; b++) {
        const int64_t e = e0 + (int64_t)b * WPR * 256;
        if (e < a.k) {
          if (a.h) store4<VEC>(a.h, T, row * a.hs + e, h[b]);
#pragma unroll
          for (int i = 0; i < 4; i++)
            sums[b % kSums] = __builtin_fma((double)h[b][i], (double)h[b][i], sums[b % kSums]);
        }
      }
    } else {
      for (int64_t e = e0; e < a.k; e += WPR * 256) {
        load_h<T, VEC>(a, row, e, h[0]);
        if (a.h) store4<VEC>(a.h, T, row * a.hs + e, h[0]);
#pragma unroll
        for (int i = 0; i < 4; i++) sums[0] = __builtin_fma((double)h[0][i], (double)h[0][i], sums[0]);
      }
    }
  }
  double ss;
  if constexpr (kSums == 4)
    ss = wave_sums64(sums, lane);
  else
    ss = wave_sum64(sums[0]);
  if (WPR > 1) {
    __shared__ double s_ss[16];
    if ((lane & (64 / kSums - 1)) == 0) s_ss[sub + WPR * (lane / (64 / kSums))] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < 16; i++) ss += s_ss[i];
  }
  if (!row_on) return;
  const float rs = (float)(1.0 / sqrt(ss / (double)a.k + (double)a.eps));
  if (NB) {
#pragma unroll
    for (int b = 0; b < kHeld; b++) {
      const int64_t e = e0 + (int64_t)b * WPR * 256;
      if (e - 4 * lane < a.k) emit<LAYOUT, VEC>(a, row, e, e < a.k, h[b], rs, ydt);
    }
  } else {
    // h from where this lane left it (x itself where nothing was added or kept)
    for (int64_t e = e0; e - 4 * lane < a.k; e += WPR * 256) {
      if (e < a.k) {
        if (a.h)
          load4<T, VEC>(a.h, row * a.hs + e, h[0]);
        else
          load_h<T, VEC>(a, row, e, h[0]);
      }
      emit<LAYOUT, VEC>(a, row, e, e < a.k, h[0], rs, ydt);
    }
  }
}

template <int T, int LAYOUT, int WPR, int NB>
hipError_t launch_vec(const NormArgs& a, int ydt, bool vec, hipStream_t st) {
  constexpr int kRows = WPR < 4 ? 4 / WPR : 1;
  const int64_t groups = (a.rows + kRows - 1) / kRows;
  if (groups >= ((int64_t)1 << 36)) return hipErrorInvalidValue;
  const dim3 grid = wide_grid(groups), block(WPR < 4 ? 256 : WPR * 64);
  if (vec)
    rms_norm_act_kernel<T, LAYOUT, WPR, NB, true><<<grid, block, 0, st>>>(a, ydt);
  else
    rms_norm_act_kernel<T, LAYOUT, WPR, NB, false><<<grid, block, 0, st>>>(a, ydt);
  return hipGetLastError();
}

// A wave a row up to 1024 values (four rows a workgroup, no barrier). Longer
// rows: 16 waves, so that a lane holds as little as it can and a row's latency
// is shortest, but 4 waves of up to 8 blocks where the rows fill the CUs by
// themselves (512 and more: what counts then is the loads in flight).
template <int T, int LAYOUT>
hipError_t launch_shape(const NormArgs& a, int ydt, bool vec, hipStream_t st) {
  const int64_t blocks = (a.k + 255) / 256;
  if (blocks <= 4) return launch_vec<T, LAYOUT, 1, 4>(a, ydt, vec, st);
  if (blocks <= 32 && a.rows >= 512) return launch_vec<T, LAYOUT, 4, 8>(a, ydt, vec, st);
  if (blocks <= 16) return launch_vec<T, LAYOUT, 16, 1>(a, ydt, vec, st);
  if (blocks <= 64) return launch_vec<T, LAYOUT, 16, 4>(a, ydt, vec, st);
  return launch_vec<T, LAYOUT, 16, 0>(a, ydt, vec, st);
}

template <int T>
hipError_t launch_type(const NormArgs& a, bool q8k, int ydt, bool vec, hipStream_t st) {
  return q8k ? launch_shape<T, ACT_Q8K>(a, ydt, vec, st) : launch_shape<T, ACT_Q8_0>(a, ydt, vec, st);
}

// 8 values a lane: code * d (the block's scale), rounded to the output's type.
template <int LAYOUT>
__global__ __launch_bounds__(256) void dequantize_act_kernel(const int8_t* __restrict__ codes,
                                                             const float* __restrict__ d, void* __restrict__ out,
                                                             int odt, int vec, int64_t n) {
  const int64_t e = (wide_block() * 256 + threadIdx.x) * 8;
  if (e >= n) return;
  const uint2 c = *(const uint2*)(codes + e);
  const float s = d[e >> (LAYOUT == ACT_Q8K ? 8 : 5)];
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[i] = (float)(int8_t)(c.x >> (8 * i)) * s;
    v[4 + i] = (float)(int8_t)(c.y >> (8 * i)) * s;
  }
  if (vec) {
    store8(out, odt, e, v);
  } else {
    store4<false>(out, odt, e, v);
    store4<false>(out, odt, e + 4, v + 4);
  }
}

bool vec_ok(const void* p, int64_t stride, int dtype) {
  return p == nullptr || ((uintptr_t)p % (4 * value_bytes(dtype)) == 0 && stride % 4 == 0);
}

}  // namespace

hipError_t launch_rms_norm_act(const void* x, int dtype, int64_t xs, const void* r, int64_t rs, const float* w,
                               float eps, void* h, int64_t hs, void* xq, int layout, void* y, int ydt, int64_t ys,
                               int64_t k, int64_t rows, float qmax, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  NormArgs a{};
  if (xq) {
    const ActPlanes p = act_planes(layout, xq, k, rows);
    a.codes = p.codes;
    a.d = p.d;
    a.sums = p.sums;
  }
  a.x = x; a.r = r; a.w = w; a.h = h; a.y = y;
  a.xs = xs; a.rs = rs; a.hs = hs; a.ys = ys; a.k = k; a.rows = rows;
  a.eps = eps; a.qmax = qmax;
  const bool vec = vec_ok(x, xs, dtype) && vec_ok(r, rs, dtype) && vec_ok(h, hs, dtype) && vec_ok(y, ys, ydt) &&
                   vec_ok(w, 0, QMM_X_F32);
  const bool q8k = layout == ACT_Q8K && xq;
  switch (dtype) {
    case QMM_X_F32: return launch_type<QMM_X_F32>(a, q8k, ydt, vec, st);
    case QMM_X_F16: return launch_type<QMM_X_F16>(a, q8k, ydt, vec, st);
    case QMM_X_BF16: return launch_type<QMM_X_BF16>(a, q8k, ydt, vec, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_dequantize_act(const void* xq, int layout, void* out, int odt, int64_t k, int64_t rows,
                                 hipStream_t st) {
  QMM_NOTE_LAUNCH();
  const ActPlanes p = act_planes(layout, (void*)xq, k, rows);
  const int64_t n = k * rows, groups = (n + 2047) / 2048;
  if (groups >= ((int64_t)1 << 36)) return hipErrorInvalidValue;
  const int vec = (uintptr_t)out % 16 == 0;
  if (layout == ACT_Q8K)
    dequantize_act_kernel<ACT_Q8K><<<wide_grid(groups), 256, 0, st>>>(p.codes, p.d, out, odt, vec, n);
  else
    dequantize_act_kernel<ACT_Q8_0><<<wide_grid(groups), 256, 0, st>>>(p.codes, p.d, out, odt, vec, n);
  return hipGetLastError();
}

}  // namespace qmm
