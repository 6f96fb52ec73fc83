// kv_cache.hip — keys and values quantized to Q8_0 as they are written into a
// paged cache, and read back (the reference keeps them as f16:
// kv_write_f16, kernels/kv_append.cu:33).
//
// Per 32 values of a head: d32 = amax / 127 (amax over the finite values, at
// most kTop), codes
// clamp(round(v / d32), -127, 127) with halves away from zero, NaN as 0, and
// d = f16(d32): the wire codec's blocks. A value reads back as code * d.
//
// The planes: K codes [pages][heads][page][hd], scales [..][page][hd / 32]:
// a key lies along hd, the axis that q . k contracts. V codes
// [pages][heads][hd][page], scales [..][hd / 32][page]: values lie along the
// tokens, the axis that p . v contracts. Built without FP contraction.
#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

// 127 * 515.5: 127 times the next f16 scale, 516, is past the largest f16, so
// with this cap every cached value is a finite f16.
constexpr float kTop = 65468.5f;

__device__ __forceinline__ uint32_t cache_code(float v, float inv) {
  const float q = roundf(v * inv);  // half away from zero
  if (q != q) return 0;
  return (uint32_t)(uint8_t)(int8_t)(q < -127.0f ? -127.0f : (q > 127.0f ? 127.0f : q));
}

// The block of 32 values that 8 lanes hold, 4 each: its codes and scale.
__device__ __forceinline__ uint32_t q8_block8(const float v[4], uint16_t& d) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) m = fmaxf(m, __builtin_isfinite(v[i]) ? fabsf(v[i]) : 0.0f);
  uint32_t mb = __float_as_uint(m);
  mb = max(mb, dpp_u<0xB1>(mb));
  mb = max(mb, dpp_u<0x4E>(mb));
  mb = max(mb, dpp_u<0x141>(mb));
  const float amax = fminf(__uint_as_float(mb), kTop);
  const float s = amax / 127.0f, inv = s == 0.0f ? 0.0f : 1.0f / s;
  d = f2h(s);
  return cache_code(v[0], inv) | (cache_code(v[1], inv) << 8) | (cache_code(v[2], inv) << 16) |
         (cache_code(v[3], inv) << 24);
}

// 8 lanes a block of 32 values of one token's head, K's in blockIdx.y 0, V's in 1.
template <int T, bool VEC>
__global__ __launch_bounds__(256) void cache_write_kernel(CachePlanes c, const void* __restrict__ k,
                                                          const void* __restrict__ v, int64_t ks, int64_t khs,
                                                          int64_t vs, int64_t vhs,
                                                          const int64_t* __restrict__ slots, int64_t tokens) {
  const int per = c.heads * (c.hd / 4);  // lanes a token
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = g / per;
  if (t >= tokens) return;  // whole 8-lane groups
  const int u = (int)(g - t * per), head = u / (c.hd / 4), e = 4 * (u - head * (c.hd / 4));
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= c.pages * c.page) return;
  const int64_t page = slot / c.page;
  const int at = (int)(slot - page * c.page);
  const int64_t ph = page * c.heads + head;
  float x[4];
  uint16_t d;
  if (blockIdx.y == 0) {
    load4<T, VEC>(k, t * ks + head * khs + e, x);
    const uint32_t q = q8_block8(x, d);
    *(uint32_t*)(c.k_codes + (ph * c.page + at) * c.hd + e) = q;
    if ((e & 31) == 0) c.k_scales[(ph * c.page + at) * (c.hd / 32) + (e >> 5)] = d;
  } else {
    load4<T, VEC>(v, t * vs + head * vhs + e, x);
    const uint32_t q = q8_block8(x, d);
#pragma unroll
    for (int i = 0; i < 4; i++) c.v_codes[(ph * c.hd + e + i) * c.page + at] = (int8_t)(q >> (8 * i));
    if ((e & 31) == 0) c.v_scales[(ph * (c.hd / 32) + (e >> 5)) * c.page + at] = d;
  }
}

// The same grid reading: a slot outside the cache reads as zeros.
__global__ __launch_bounds__(256) void cache_read_kernel(CachePlanes c, const int64_t* __restrict__ slots,
                                                         void* __restrict__ k, void* __restrict__ v, int odt, int vec,
                                                         int64_t tokens) {
  const int per = c.heads * (c.hd / 4);
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = g / per;
  if (t >= tokens) return;
  const int u = (int)(g - t * per), head = u / (c.hd / 4), e = 4 * (u - head * (c.hd / 4));
  const int64_t slot = slots[t];
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (slot >= 0 && slot < c.pages * c.page) {
    const int64_t page = slot / c.page;
    const int at = (int)(slot - page * c.page);
    const int64_t ph = page * c.heads + head;
    if (blockIdx.y == 0) {
      const uint32_t q = *(const uint32_t*)(c.k_codes + (ph * c.page + at) * c.hd + e);
      const float d = h2f(c.k_scales[(ph * c.page + at) * (c.hd / 32) + (e >> 5)]);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (float)(int8_t)(q >> (8 * i)) * d;
    } else {
      const float d = h2f(c.v_scales[(ph * (c.hd / 32) + (e >> 5)) * c.page + at]);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (float)c.v_codes[(ph * c.hd + e + i) * c.page + at] * d;
    }
  }
  void* out = blockIdx.y == 0 ? k : v;
  const int64_t o = (t * c.heads + head) * c.hd + e;
  if (vec)
    store4<true>(out, odt, o, x);
  else
    store4<false>(out, odt, o, x);
}

bool vec_ok(const void* p, int64_t s, int64_t hs, int dtype) {
  return (uintptr_t)p % (4 * value_bytes(dtype)) == 0 && s % 4 == 0 && hs % 4 == 0;
}

template <int T>
hipError_t launch_write(const CachePlanes& c, const void* k, const void* v, int64_t ks, int64_t khs, int64_t vs,
                        int64_t vhs, const int64_t* slots, int64_t tokens, dim3 grid, hipStream_t st) {
  if (vec_ok(k, ks, khs, T) && vec_ok(v, vs, vhs, T))
    cache_write_kernel<T, true><<<grid, 256, 0, st>>>(c, k, v, ks, khs, vs, vhs, slots, tokens);
  else
    cache_write_kernel<T, false><<<grid, 256, 0, st>>>(c, k, v, ks, khs, vs, vhs, slots, tokens);
  return hipGetLastError();
}

bool cache_grid(const CachePlanes& c, int64_t tokens, dim3& grid) {
  const int64_t per = (int64_t)c.heads * (c.hd / 4);
  if (tokens > ((int64_t)1 << 40) / per) return false;
  const int64_t groups = (tokens * per + 255) / 256;
  grid = dim3((unsigned)groups, 2);
  return groups < ((int64_t)1 << 31);
}

}  // namespace

hipError_t launch_cache_write(const CachePlanes& c, const void* k, const void* v, int dtype, int64_t ks, int64_t khs,
                              int64_t vs, int64_t vhs, const int64_t* slots, int64_t tokens, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  dim3 grid;
  if (!cache_grid(c, tokens, grid)) return hipErrorInvalidValue;
  switch (dtype) {
    case QMM_X_F32: return launch_write<QMM_X_F32>(c, k, v, ks, khs, vs, vhs, slots, tokens, grid, st);
    case QMM_X_F16: return launch_write<QMM_X_F16>(c, k, v, ks, khs, vs, vhs, slots, tokens, grid, st);
    case QMM_X_BF16: return launch_write<QMM_X_BF16>(c, k, v, ks, khs, vs, vhs, slots, tokens, grid, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_cache_read(const CachePlanes& c, const int64_t* slots, int64_t tokens, void* k, void* v, int odt,
                             hipStream_t st) {
  QMM_NOTE_LAUNCH();
  dim3 grid;
  if (!cache_grid(c, tokens, grid)) return hipErrorInvalidValue;
  const int vec = vec_ok(k, 0, 0, odt) && vec_ok(v, 0, 0, odt);
  cache_read_kernel<<<grid, 256, 0, st>>>(c, slots, k, v, odt, vec, tokens);
  return hipGetLastError();
}

}  // namespace qmm
