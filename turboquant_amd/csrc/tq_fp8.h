// The 8-bit cache: e4m3 with a power of two for every block of 16 tokens and KV head.
//   2^e: the smallest that brings the block's largest finite value to 448 at most; the byte e + 127 is kept, -117 <= e <= 119
// The scale being a power of two, value / scale is exact, and e4m3 has an exponent of its own: a scale between two powers would gain nothing.
#pragma once

#include "tq_step.h"

namespace tq {

typedef uint32_t f8_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t f8_u32x4 __attribute__((ext_vector_type(4)));
typedef float f8_f32x2 __attribute__((ext_vector_type(2)));

constexpr int F8_LOWEST = -117, F8_HIGHEST = 119, F8_BIAS = 127;

// Element strides (bytes, too); channels lie one behind another, rows start on 16-byte boundaries.  Scales: (num_blocks, H) contiguous.
struct Fp8Cache {
  uint8_t *k, *v;
  uint8_t *k_scales, *v_scales;
  int64_t s_blk, s_h;
  int32_t s_t;
  int32_t H, d;
};

// the exponent of the scale of a block whose largest finite value is `largest`
__device__ __forceinline__ int f8_exponent(float largest) {
  if (largest == 0.0f) return F8_LOWEST;
  int x;
  const float m = frexpf(largest, &x);                        // largest = m 2^x, 0.5 <= m < 1; 448 = 0.875 2^9
  const int e = x - 9 + (m > 0.875f ? 1 : 0);
  return e < F8_LOWEST ? F8_LOWEST : (e > F8_HIGHEST ? F8_HIGHEST : e);
}
__device__ __forceinline__ float f8_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
// The scale that a byte says.  2^-127 and 2^127 are never written: a cache that is all zeros has the one, and the other is what a byte that nobody wrote says at most, so that
// zeros in place of its block's values stay zeros (2^128 is infinite).
__device__ __forceinline__ float f8_scale(uint32_t byte) { return byte == 0 ? 0x1p-127f : __uint_as_float((byte < 254u ? byte : 254u) << 23); }
// what has no e4m3 number of its size becomes the largest; NaN stays
__device__ __forceinline__ float f8_clamp(float x) { return x > 448.0f ? 448.0f : (x < -448.0f ? -448.0f : x); }
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(a), f8_clamp(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(c), f8_clamp(d), r, true);
  return (uint32_t)r;
}
__device__ __forceinline__ void f8_unpack4(uint32_t x, float* y) {
  const f8_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  y[0] = a[0]; y[1] = a[1]; y[2] = b[0]; y[3] = b[1];
}

// what the entry points check of a cache, and its description
inline int fp8_cache_init(Fp8Cache* c, void* k, void* v, void* k_scales, void* v_scales, int H, int d, int64_t s_blk, int64_t s_t, int64_t s_h) {
  if (!k || !v || !k_scales || !v_scales) return TQ_ENULL;
  if (H <= 0 || d <= 0) return TQ_EINVAL;
  if (d != 64 && d != 128 && d != 192 && d != 256) return TQ_EUNSUPPORTED;
  if (s_blk < 0 || s_t < 0 || s_h < 0 || s_t > (1 << 24) || s_blk % 16 || s_t % 16 || s_h % 16 || (((uintptr_t)k | (uintptr_t)v) & 15)) return TQ_EUNSUPPORTED;
  c->k = (uint8_t*)k; c->v = (uint8_t*)v; c->k_scales = (uint8_t*)k_scales; c->v_scales = (uint8_t*)v_scales;
  c->s_blk = s_blk; c->s_h = s_h; c->s_t = (int32_t)s_t; c->H = H; c->d = d;
  return TQ_OK;
}

}  // namespace tq
