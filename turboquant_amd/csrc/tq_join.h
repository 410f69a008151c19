// Splits of a row of attention -> the row:  out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i  over its first `used` splits.
#pragma once

#include "tq_common.h"

namespace tq {

constexpr int JOIN_MAX_SPLITS = 1024, JOIN_FEW = 16;

template <int DT>
__device__ __forceinline__ void join_store(void* out, int64_t at, const float4& x) {
  if constexpr (DT == TQ_F32) {
    *(float4*)((float*)out + at) = x;
  } else {
    Elem<DT>::store(out, at, x.x);
    Elem<DT>::store(out, at + 1, x.y);
    Elem<DT>::store(out, at + 2, x.z);
    Elem<DT>::store(out, at + 3, x.w);
  }
}

// Few splits, 64 at most: a wavefront per row, a lane knows the factor of its split (ml of lane < used; -inf, 0 behind them).  A split's numerators
// lie `apart` floats behind the one's before it; AHEAD of them are on their way at a time.
template <int DT, int AHEAD = 8>
__device__ __forceinline__ void join_few(const float* accs, int64_t apart, int d, void* out, int64_t row, int used, const float2& ml) {
  const int lane = (int)threadIdx.x & 63;
  const float top = wave_max_fast(ml.x), ref = top == -INFINITY ? 0.0f : top;
  const float f = __builtin_amdgcn_exp2f(ml.x - ref), sum = wave_sum_fast(f * ml.y), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int quads = d >> 2;
  for (int q = lane; q < quads; q += 64) {
    const float* acc = accs + q * 4;
    float4 o = make_float4(0, 0, 0, 0);
    for (int i0 = 0; i0 < used; i0 += AHEAD) {               // (the last one over again behind the end)
      float4 x[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) x[i] = *(const float4*)(acc + (i0 + i < used ? i0 + i : used - 1) * apart);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const bool in = i0 + i < used;                       // (where not, a numerator of zero: a factor of zero would make NaN of an infinite one)
        const float g = in ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (i0 + i) & 63)) : 0.0f;
        o.x = fmaf(g, in ? x[i].x : 0.0f, o.x); o.y = fmaf(g, in ? x[i].y : 0.0f, o.y);
        o.z = fmaf(g, in ? x[i].z : 0.0f, o.z); o.w = fmaf(g, in ? x[i].w : 0.0f, o.w);
      }
    }
    join_store<DT>(out, row * d + q * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  }
}

// Many splits: a workgroup per row and 64 channels, sixteen lanes to a split, sixteen splits at a time.
template <int DT>
__device__ __forceinline__ void join_many(const float2* ml, int64_t ml_apart, const float* accs, int64_t apart, int d, void* out, int64_t row, int used, int slice,
                                          float* s_f, float* s_red, float4* s_o) {
  const int tid = (int)threadIdx.x;
  float top = -INFINITY;
  for (int i = tid; i < used; i += 256) top = fmaxf(top, ml[i * ml_apart].x);
  top = wave_max_fast(top);
  if ((tid & 63) == 0) s_red[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int i = tid; i < used; i += 256) {
    const float2 x = ml[i * ml_apart];
    const float f = __builtin_amdgcn_exp2f(x.x - ref);
    s_f[i] = f;
    sum += f * x.y;
  }
  sum = wave_sum_fast(sum);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = sum;
  __syncthreads();
  sum = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int quad = tid & 15, share = tid >> 4;
  const float* acc = accs + slice * 64 + quad * 4;
  float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 8
  for (int i = share; i < used; i += 16) {
    const float4 x = *(const float4*)(acc + i * apart);
    const float f = s_f[i];
    o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
  }
  s_o[tid] = o;
  __syncthreads();
  if (share != 0) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    const float4 x = s_o[i * 16 + quad];
    o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
  }
  join_store<DT>(out, row * d + slice * 64 + quad * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// workgroups that join rows
inline int64_t join_groups(int64_t rows, int n_split, int d) {
  return n_split <= 1 ? 0 : (n_split <= JOIN_FEW ? (rows + 3) / 4 : rows * (d / 64));
}

}  // namespace tq
