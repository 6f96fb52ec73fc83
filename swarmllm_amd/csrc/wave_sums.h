// wave_sums.h — running sums over a wave's lanes on the vector unit.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qmm {

// Running sums over the wave's lanes: within 16, then 15 -> the next 16, 31 -> the upper half.
template <int CTL, int ROWS, typename T>
__device__ __forceinline__ T lane_shift(T v) {
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); i++) w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[i], CTL, ROWS, 0xF, true);
  __builtin_memcpy(&v, w, sizeof(T));
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_sums(T v) {
  v += lane_shift<0x111, 0xF>(v);
  v += lane_shift<0x112, 0xF>(v);
  v += lane_shift<0x114, 0xF>(v);
  v += lane_shift<0x118, 0xF>(v);
  v += lane_shift<0x142, 0xA>(v);
  v += lane_shift<0x143, 0xC>(v);
  return v;
}

}  // namespace qmm
