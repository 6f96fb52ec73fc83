// kv_cache.hip — keys and values quantized to Q8_0 as they are written into a
// paged cache, and read back.
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
//
// What bounds both directions is memory. A workgroup takes 64 tokens of one
// head, its K (blockIdx.z 0) or its V (1). K moves straight through. V turns
// from rows of a token to rows of a dim in LDS, and where 16 tokens in a row have
// 16 consecutive positions (a prompt's do but at its ends) a lane moves them
// as one 16-byte piece; other tokens go a byte at a time. 32768 tokens of 8 x
// 128 values read back as f16 in 46 us (206 MB at 4.5 TB/s; a byte at a time
// 136 us), 2000 tokens' f32 rows written in 10.1-10.9 us (18.3) and read in 6-7 (11.2).
// A few tokens (a decode step's) take kernels of their own, a token a workgroup
// and nothing between its slot and its stores: 8 tokens 3.7 us each way, 8 on
// the tiles.
#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace qmm {

namespace {

// 127 * 515.5: 127 times the next f16 scale, 516, is past the largest f16, so
// with this cap every cached value is a finite f16.
constexpr float kTop = 65468.5f;
constexpr int kTokens = 64;  // of a workgroup
constexpr int kMaxHd = 256;

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

// The slots of a workgroup's tokens (-1: none, or outside the cache) and, a
// bit each, which groups of 16 tokens are 16 consecutive positions of a page
// from a multiple of 16 on. Ends with a barrier.
struct TileSlots {
  int64_t slot[kTokens];
  uint32_t runs;
};
__device__ __forceinline__ void load_slots(const CachePlanes& c, const int64_t* slots, int64_t t0, int64_t tokens,
                                           TileSlots& s) {
  const int tid = threadIdx.x;
  if (tid < kTokens) {  // the first wave, whole
    const int64_t v = t0 + tid < tokens ? slots[t0 + tid] : -1;
    const int64_t slot = v < 0 || v >= c.pages * c.page ? -1 : v;
    s.slot[tid] = slot;
    const int64_t first = __shfl(slot, tid & 48, kWave);
    const uint64_t ok = __ballot(first >= 0 && (first & 15) == 0 && slot == first + (tid & 15));
    uint32_t runs = 0;
#pragma unroll
    for (int g = 0; g < 4; g++) runs |= (uint32_t)(((ok >> (16 * g)) & 0xFFFF) == 0xFFFF) << g;
    if (tid == 0) s.runs = runs;
  }
  __syncthreads();
}

// 4 x 4 bytes turned: byte j of r[i] from byte i of r[j].
__device__ __forceinline__ void turn4(uint32_t r[4]) {
  const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), d = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  r[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  r[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  r[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  r[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Where a slot's page begins for a head, in units of a page's head.
struct Place {
  int64_t ph;
  int at;
};
__device__ __forceinline__ Place place_of(const CachePlanes& c, int64_t slot, int head) {
  const int bits = __builtin_ctz(c.page);
  return Place{(slot >> bits) * c.heads + head, (int)(slot & (c.page - 1))};
}

// Few tokens: blockIdx.x a token, 4 values a lane (a block's 8 lanes together),
// V's codes stored byte by byte. No LDS and no barrier between a slot and its
// stores.
template <int T, bool VEC>
__global__ __launch_bounds__(256) void cache_write_token_kernel(CachePlanes c, const void* __restrict__ k,
                                                                const void* __restrict__ v, int64_t ks, int64_t khs,
                                                                int64_t vs, int64_t vhs,
                                                                const int64_t* __restrict__ slots) {
  const int lanes = c.hd / 4, u = (int)(blockIdx.y * 256 + threadIdx.x), head = (int)((uint32_t)u / (uint32_t)lanes);
  if (head >= c.heads) return;  // whole 8-lane groups
  const int e = 4 * (u - head * lanes);
  const int64_t t = blockIdx.x, slot = slots[t];
  const bool is_v = blockIdx.z != 0;
  float f[4];
  uint16_t d;
  if (is_v)
    load4<T, VEC>(v, t * vs + head * vhs + e, f);
  else
    load4<T, VEC>(k, t * ks + head * khs + e, f);
  if (slot < 0 || slot >= c.pages * c.page) return;
  const uint32_t q = q8_block8(f, d);
  const Place w = place_of(c, slot, head);
  if (!is_v) {
    const int64_t row = w.ph * c.page + w.at;
    *(uint32_t*)(c.k_codes + row * c.hd + e) = q;
    if ((e & 31) == 0) c.k_scales[row * (c.hd / 32) + (e >> 5)] = d;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) c.v_codes[(w.ph * c.hd + e + i) * c.page + w.at] = (int8_t)(q >> (8 * i));
    if ((e & 31) == 0) c.v_scales[(w.ph * (c.hd / 32) + (e >> 5)) * c.page + w.at] = d;
  }
}

template <int T, bool VEC>
__global__ __launch_bounds__(256) void cache_write_kernel(CachePlanes c, const void* __restrict__ k,
                                                          const void* __restrict__ v, int64_t ks, int64_t khs,
                                                          int64_t vs, int64_t vhs,
                                                          const int64_t* __restrict__ slots, int64_t tokens) {
  constexpr int kRow = 17;  // words of a dim's 64 tokens, one more against bank conflicts
  __shared__ TileSlots s;
  __shared__ uint32_t s_codes[kMaxHd * kRow];
  __shared__ __attribute__((aligned(16))) uint16_t s_scales[kMaxHd / 32 * kTokens];
  const int tid = threadIdx.x, head = blockIdx.y, hd = c.hd, lanes = hd / 4;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens;
  const bool is_v = blockIdx.z != 0;
  const int here = tokens - t0 < kTokens ? (int)(tokens - t0) : kTokens;
  load_slots(c, slots, t0, tokens, s);
  // 4 tokens of 4 dims a lane; a block's 8 lanes stay together
  for (int x = tid; x < (here + 3) / 4 * lanes; x += 256) {
    const int t = 4 * (x / lanes), e = 4 * (x - t / 4 * lanes);
    float f[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (t + i < here) {
        if (is_v)
          load4<T, VEC>(v, (t0 + t + i) * vs + head * vhs + e, f[i]);
        else
          load4<T, VEC>(k, (t0 + t + i) * ks + head * khs + e, f[i]);
      } else {
        f[i][0] = f[i][1] = f[i][2] = f[i][3] = 0.0f;
      }
    }
    uint32_t q[4];
    uint16_t d[4];
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = q8_block8(f[i], d[i]);
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int64_t slot = t + i < here ? s.slot[t + i] : -1;
        if (slot < 0) continue;
        const Place w = place_of(c, slot, head);
        const int64_t row = w.ph * c.page + w.at;
        *(uint32_t*)(c.k_codes + row * hd + e) = q[i];
        if ((e & 31) == 0) c.k_scales[row * (hd / 32) + (e >> 5)] = d[i];
      }
    } else {
      turn4(q);
#pragma unroll
      for (int i = 0; i < 4; i++) s_codes[(e + i) * kRow + t / 4] = q[i];
      if ((e & 31) == 0)
        *(uint2*)(s_scales + (e >> 5) * kTokens + t) = make_uint2(d[0] | ((uint32_t)d[1] << 16), d[2] | ((uint32_t)d[3] << 16));
    }
  }
  if (!is_v) return;
  __syncthreads();
  // 16 tokens of a dim (then of a block's scales) at a time
  for (int x = tid; x < 4 * (hd + hd / 32); x += 256) {
    const int g = x & 3, r = x >> 2;
    if (16 * g >= here) continue;
    const bool run = (s.runs >> g) & 1;
    if (r < hd) {
      const uint32_t* q = s_codes + r * kRow + 4 * g;
      if (run) {
        const Place w = place_of(c, s.slot[16 * g], head);
        *(uint4*)(c.v_codes + (w.ph * hd + r) * c.page + w.at) = make_uint4(q[0], q[1], q[2], q[3]);
      } else {
        for (int i = 0; i < 16; i++) {
          const int64_t slot = s.slot[16 * g + i];
          if (slot < 0) continue;
          const Place w = place_of(c, slot, head);
          c.v_codes[(w.ph * hd + r) * c.page + w.at] = (int8_t)(q[i >> 2] >> (8 * (i & 3)));
        }
      }
    } else {
      const uint16_t* d = s_scales + (r - hd) * kTokens + 16 * g;
      if (run) {
        const Place w = place_of(c, s.slot[16 * g], head);
        uint4* o = (uint4*)(c.v_scales + (w.ph * (hd / 32) + r - hd) * c.page + w.at);
        o[0] = ((const uint4*)d)[0];
        o[1] = ((const uint4*)d)[1];
      } else {
        for (int i = 0; i < 16; i++) {
          const int64_t slot = s.slot[16 * g + i];
          if (slot < 0) continue;
          const Place w = place_of(c, slot, head);
          c.v_scales[(w.ph * (hd / 32) + r - hd) * c.page + w.at] = d[i];
        }
      }
    }
  }
}

// 8 values a lane to out + o.
__device__ __forceinline__ void put8(void* out, int odt, int vec, int64_t o, const float x[8]) {
  if (vec) {
    store8(out, odt, o, x);
  } else {
    store4<false>(out, odt, o, x);
    store4<false>(out, odt, o + 4, x + 4);
  }
}

// Few tokens: blockIdx.x a token, 8 values a lane.
__global__ __launch_bounds__(256) void cache_read_token_kernel(CachePlanes c, const int64_t* __restrict__ slots,
                                                               void* __restrict__ k, void* __restrict__ v, int odt,
                                                               int vec) {
  const int lanes = c.hd / 8, u = (int)(blockIdx.y * 256 + threadIdx.x), head = (int)((uint32_t)u / (uint32_t)lanes);
  if (head >= c.heads) return;
  const int e = 8 * (u - head * lanes);
  const int64_t t = blockIdx.x, slot = slots[t];
  const bool is_v = blockIdx.z != 0;
  float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (slot >= 0 && slot < c.pages * c.page) {
    const Place w = place_of(c, slot, head);
    if (!is_v) {
      const int64_t row = w.ph * c.page + w.at;
      const uint2 q = *(const uint2*)(c.k_codes + row * c.hd + e);
      const float d = h2f(c.k_scales[row * (c.hd / 32) + (e >> 5)]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f[i] = (float)(int8_t)(q.x >> (8 * i)) * d;
        f[4 + i] = (float)(int8_t)(q.y >> (8 * i)) * d;
      }
    } else {
      const float d = h2f(c.v_scales[(w.ph * (c.hd / 32) + (e >> 5)) * c.page + w.at]);
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = (float)c.v_codes[(w.ph * c.hd + e + i) * c.page + w.at] * d;
    }
  }
  put8(is_v ? v : k, odt, vec, (t * c.heads + head) * c.hd + e, f);
}

__global__ __launch_bounds__(256) void cache_read_kernel(CachePlanes c, const int64_t* __restrict__ slots,
                                                         void* __restrict__ k, void* __restrict__ v, int odt, int vec,
                                                         int64_t tokens) {
  __shared__ TileSlots s;
  // V's codes turned back to rows of a token, the scales of a block beside them
  __shared__ __attribute__((aligned(16))) int8_t s_codes[kTokens * (kMaxHd + 8)];
  __shared__ __attribute__((aligned(16))) uint16_t s_scales[kMaxHd / 32 * kTokens];
  const int tid = threadIdx.x, head = blockIdx.y, hd = c.hd, lanes = hd / 8;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens;
  const bool is_v = blockIdx.z != 0;
  const int here = tokens - t0 < kTokens ? (int)(tokens - t0) : kTokens;
  const int row = hd + 8;
  load_slots(c, slots, t0, tokens, s);
  if (is_v) {
    // 16 tokens of 4 dims at a time, then of a block's scales
    for (int x = tid; x < 4 * (hd / 4 + hd / 32); x += 256) {
      const int g = x / (hd / 4 + hd / 32), r = x - g * (hd / 4 + hd / 32);
      if (16 * g >= here) continue;
      const bool run = (s.runs >> g) & 1;
      if (r < hd / 4) {
        int8_t* q = s_codes + 16 * g * row + 4 * r;
        if (run) {
          const Place w = place_of(c, s.slot[16 * g], head);
          const int8_t* src = c.v_codes + (w.ph * hd + 4 * r) * c.page + w.at;
          uint4 u[4];
#pragma unroll
          for (int i = 0; i < 4; i++) u[i] = *(const uint4*)(src + i * c.page);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t m[4] = {(&u[0].x)[i], (&u[1].x)[i], (&u[2].x)[i], (&u[3].x)[i]};
            turn4(m);
#pragma unroll
            for (int j = 0; j < 4; j++) *(uint32_t*)(q + (4 * i + j) * row) = m[j];
          }
        } else {
          for (int i = 0; i < 16; i++) {
            const int64_t slot = s.slot[16 * g + i];
            if (slot < 0) continue;
            const Place w = place_of(c, slot, head);
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; j++)
              m |= (uint32_t)(uint8_t)c.v_codes[(w.ph * hd + 4 * r + j) * c.page + w.at] << (8 * j);
            *(uint32_t*)(q + i * row) = m;
          }
        }
      } else {
        const int blk = r - hd / 4;
        uint16_t* d = s_scales + blk * kTokens + 16 * g;
        if (run) {
          const Place w = place_of(c, s.slot[16 * g], head);
          const uint4* o = (const uint4*)(c.v_scales + (w.ph * (hd / 32) + blk) * c.page + w.at);
          ((uint4*)d)[0] = o[0];
          ((uint4*)d)[1] = o[1];
        } else {
          for (int i = 0; i < 16; i++) {
            const int64_t slot = s.slot[16 * g + i];
            if (slot < 0) continue;
            const Place w = place_of(c, slot, head);
            d[i] = c.v_scales[(w.ph * (hd / 32) + blk) * c.page + w.at];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int x = tid; x < here * lanes; x += 256) {
    const int t = x / lanes, e = 8 * (x - t * lanes);
    const int64_t slot = s.slot[t];
    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};  // a slot outside the cache reads as zeros
    if (slot >= 0) {
      uint2 q;
      float d;
      if (is_v) {
        q = *(const uint2*)(s_codes + t * row + e);
        d = h2f(s_scales[(e >> 5) * kTokens + t]);
      } else {
        const Place w = place_of(c, slot, head);
        const int64_t at = w.ph * c.page + w.at;
        q = *(const uint2*)(c.k_codes + at * hd + e);
        d = h2f(c.k_scales[at * (hd / 32) + (e >> 5)]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f[i] = (float)(int8_t)(q.x >> (8 * i)) * d;
        f[4 + i] = (float)(int8_t)(q.y >> (8 * i)) * d;
      }
    }
    put8(is_v ? v : k, odt, vec, ((t0 + t) * c.heads + head) * hd + e, f);
  }
}

bool vec_ok(const void* p, int64_t s, int64_t hs, int dtype) {
  return (uintptr_t)p % (4 * value_bytes(dtype)) == 0 && s % 4 == 0 && hs % 4 == 0;
}

// The kernels a token at a time take up to 2^19 keys' values: past that the
// tiles' 16-byte pieces pay for their barriers (graph replays, us, token /
// tile: 8 x 128, 8 consecutive tokens written 3.2 / 7.9, read 2.7 / 6.4; 512
// of them 6.0 / 6.9 and 3.9 / 5.1; 1024 9.7 / 7.2 and 5.8 / 5.5; 512 apart from
// each other 10.7 / 15.6 and 6.0 / 18.2).
bool few_values(const CachePlanes& c, int64_t tokens) { return tokens <= ((int64_t)1 << 19) / (c.heads * (int64_t)c.hd); }

dim3 token_grid(const CachePlanes& c, int64_t tokens, int per) {
  return dim3((unsigned)tokens, (unsigned)((c.heads * (c.hd / per) + 255) / 256), 2);
}
dim3 tile_grid(const CachePlanes& c, int64_t tokens) {
  return dim3((unsigned)(tokens / kTokens + (tokens % kTokens != 0)), (unsigned)c.heads, 2);
}

template <int T, bool VEC>
hipError_t launch_write(const CachePlanes& c, const void* k, const void* v, int64_t ks, int64_t khs, int64_t vs,
                        int64_t vhs, const int64_t* slots, int64_t tokens, hipStream_t st) {
  if (few_values(c, tokens))
    cache_write_token_kernel<T, VEC><<<token_grid(c, tokens, 4), 256, 0, st>>>(c, k, v, ks, khs, vs, vhs, slots);
  else
    cache_write_kernel<T, VEC><<<tile_grid(c, tokens), 256, 0, st>>>(c, k, v, ks, khs, vs, vhs, slots, tokens);
  return hipGetLastError();
}

template <int T>
hipError_t launch_write_type(const CachePlanes& c, const void* k, const void* v, int64_t ks, int64_t khs, int64_t vs,
                             int64_t vhs, const int64_t* slots, int64_t tokens, hipStream_t st) {
  return vec_ok(k, ks, khs, T) && vec_ok(v, vs, vhs, T)
             ? launch_write<T, true>(c, k, v, ks, khs, vs, vhs, slots, tokens, st)
             : launch_write<T, false>(c, k, v, ks, khs, vs, vhs, slots, tokens, st);
}

}  // namespace

hipError_t launch_cache_write(const CachePlanes& c, const void* k, const void* v, int dtype, int64_t ks, int64_t khs,
                              int64_t vs, int64_t vhs, const int64_t* slots, int64_t tokens, hipStream_t st) {
  QMM_NOTE_LAUNCH();
  switch (dtype) {
    case QMM_X_F32: return launch_write_type<QMM_X_F32>(c, k, v, ks, khs, vs, vhs, slots, tokens, st);
    case QMM_X_F16: return launch_write_type<QMM_X_F16>(c, k, v, ks, khs, vs, vhs, slots, tokens, st);
    case QMM_X_BF16: return launch_write_type<QMM_X_BF16>(c, k, v, ks, khs, vs, vhs, slots, tokens, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_cache_read(const CachePlanes& c, const int64_t* slots, int64_t tokens, void* k, void* v, int odt,
                             hipStream_t st) {
  QMM_NOTE_LAUNCH();
  const int vec = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0;
  if (few_values(c, tokens))
    cache_read_token_kernel<<<token_grid(c, tokens, 8), 256, 0, st>>>(c, slots, k, v, odt, vec);
  else
    cache_read_kernel<<<tile_grid(c, tokens), 256, 0, st>>>(c, slots, k, v, odt, vec, tokens);
  return hipGetLastError();
}

}  // namespace qmm
