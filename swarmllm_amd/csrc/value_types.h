// value_types.h — loads and stores of the float types an operator takes
// (qmm_x_dtype: f16, bf16, f32), 4 or 8 values at a time.
#pragma once

#include "../../include/qmm.h"
#include "qmm_device.h"

namespace qmm {

inline __host__ __device__ int value_bytes(int dtype) { return dtype == QMM_X_F32 ? 4 : 2; }
inline bool value_type_ok(int dtype) { return dtype == QMM_X_F16 || dtype == QMM_X_BF16 || dtype == QMM_X_F32; }

// A launch's threads in x stay below 2^32 (a larger grid wraps around without an
// error): up to 2^21 workgroups in x, of any size, and y for the rest.
inline dim3 wide_grid(int64_t groups) {
  const int64_t x = groups < ((int64_t)1 << 21) ? groups : (int64_t)1 << 21;
  return dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
}
__device__ __forceinline__ int64_t wide_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// bf16 bits of v, to nearest even; NaN stays a (quiet) NaN.
__device__ __forceinline__ uint16_t f2bf(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float bf2f(uint32_t b) { return __uint_as_float(b << 16); }
// f16 bits of v, to nearest even.
__device__ __forceinline__ uint16_t f2h_rn(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

template <int T>
__device__ __forceinline__ float round_to(float v) {
  if (T == QMM_X_F16) return h2f(f2h_rn(v));
  if (T == QMM_X_BF16) return bf2f(f2bf(v));
  return v;
}

template <int T>
__device__ __forceinline__ float widen(uint32_t b) {
  return T == QMM_X_F16 ? h2f((uint16_t)b) : bf2f(b & 0xFFFFu);
}
__device__ __forceinline__ uint32_t narrow(int dtype, float v) { return dtype == QMM_X_F16 ? f2h_rn(v) : f2bf(v); }

// Values [i, i + 4) of an array of type T. VEC: its base and i are aligned
// to 4 values; otherwise a value at a time.
template <int T, bool VEC>
__device__ __forceinline__ void load4(const void* p, int64_t i, float v[4]) {
  if (T == QMM_X_F32) {
    const float* f = (const float*)p + i;
    if (VEC) {
      const float4 t = *(const float4*)f;
      v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = f[e];
    }
  } else {
    const uint16_t* f = (const uint16_t*)p + i;
    if (VEC) {
      const uint2 t = *(const uint2*)f;
      v[0] = widen<T>(t.x & 0xFFFFu); v[1] = widen<T>(t.x >> 16);
      v[2] = widen<T>(t.y & 0xFFFFu); v[3] = widen<T>(t.y >> 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = widen<T>(f[e]);
    }
  }
}

template <int T>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  return T == QMM_X_F32 ? ((const float*)p)[i] : widen<T>(((const uint16_t*)p)[i]);
}
__device__ __forceinline__ void store1(void* p, int dtype, int64_t i, float v) {
  if (dtype == QMM_X_F32)
    ((float*)p)[i] = v;
  else
    ((uint16_t*)p)[i] = (uint16_t)narrow(dtype, v);
}

template <bool VEC>
__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, const float v[4]) {
  if (dtype == QMM_X_F32) {
    float* f = (float*)p + i;
    if (VEC) {
      *(float4*)f = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) f[e] = v[e];
    }
  } else {
    uint16_t* f = (uint16_t*)p + i;
    if (VEC) {
      *(uint2*)f = make_uint2(narrow(dtype, v[0]) | (narrow(dtype, v[1]) << 16),
                              narrow(dtype, v[2]) | (narrow(dtype, v[3]) << 16));
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) f[e] = (uint16_t)narrow(dtype, v[e]);
    }
  }
}

// 8 values at a 16-byte aligned place.
__device__ __forceinline__ void store8(void* p, int dtype, int64_t i, const float v[8]) {
  if (dtype == QMM_X_F32) {
    *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = narrow(dtype, v[2 * e]) | (narrow(dtype, v[2 * e + 1]) << 16);
    *(uint4*)((uint16_t*)p + i) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

}  // namespace qmm
