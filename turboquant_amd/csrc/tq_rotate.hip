// The norm of every head of queries and keys and the rotation by position, in one pass.
//
//   y = x / sqrt(mean x^2 + eps) w       (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * inv_freq of the pair
//
// A group of lanes - head_dim / 8, to the next power of two - takes a head of a token: a lane four pairs, so that the halves a rotation brings
// together are one lane's already and the norm is a sum over neighbouring lanes.  Channels behind the rotated ones are pairs, too, that do not turn.
// An angle is the same for all heads: a workgroup works out the sines and cosines of its tokens once, one a thread, into LDS, behind the loads of its
// first heads.  In turns and 64 bits, position * (inv_freq / 2 pi) less its whole turns: at position 2^20 an angle in 32 bits would be 0.03 off.
// All sums, norms and rotations in 32 bits, one rounding at the end.  Bound by the memory system.
#include "tq_common.h"

#include <algorithm>

namespace tq {

struct Rotate {
  const void* in[2];       // queries, keys: (rows, H, d), element strides
  void* out[2];
  const void* weight[2];   // (d) or null: no norm
  int64_t in_t[2], in_h[2], out_t[2], out_h[2];
  const void* positions;   // (rows) int32 or int64
  const double* inv_freq;  // (rotary / 2)
  int64_t rows;
  int32_t H[2], d, rotary, wide_positions, tokens;
  float eps;
};

constexpr int ROTATE_TOKENS = 4, ROTATE_PAIRS = 256;        // of a workgroup; most of a head (d 512)

typedef uint32_t ro_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t ro_u32x4 __attribute__((ext_vector_type(4)));

// four neighbouring channels
template <int DT>
struct Four {
  ro_u32x2 x;
  __device__ __forceinline__ void load(const void* p, int64_t at) { x = *(const ro_u32x2*)((const uint16_t*)p + at); }
  __device__ __forceinline__ float get(int i) const {
    const uint16_t h = (uint16_t)(x[i >> 1] >> (i & 1 ? 16 : 0));
    return DT == TQ_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
  }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* y) {
    ro_u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r[i] = DT == TQ_BF16 ? (uint32_t)f32_to_bf16_bits(y[2 * i]) | (uint32_t)f32_to_bf16_bits(y[2 * i + 1]) << 16
                           : (uint32_t)f32_to_f16_bits(y[2 * i]) | (uint32_t)f32_to_f16_bits(y[2 * i + 1]) << 16;
    *(ro_u32x2*)((uint16_t*)p + at) = r;
  }
};
template <>
struct Four<TQ_F32> {
  float4 x;
  __device__ __forceinline__ void load(const void* p, int64_t at) { x = *(const float4*)((const float*)p + at); }
  __device__ __forceinline__ float get(int i) const { return i == 0 ? x.x : (i == 1 ? x.y : (i == 2 ? x.z : x.w)); }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* y) { *(float4*)((float*)p + at) = make_float4(y[0], y[1], y[2], y[3]); }
};

// LANES: of a head.  INTER: pairs are neighbours (2 i, 2 i + 1), not the two halves (i, i + rotary / 2).
template <int DT, int LANES, bool INTER>
__global__ void __launch_bounds__(256) rotate_kernel(const Rotate a) {
  constexpr int GROUPS = 256 / LANES, AHEAD = 4;
  __shared__ float2 s_turn[ROTATE_TOKENS][ROTATE_PAIRS];
  const int tid = (int)threadIdx.x, lane = tid % LANES, group = tid / LANES;
  const int64_t token0 = (int64_t)blockIdx.x * a.tokens;
  const int tokens = a.rows - token0 < a.tokens ? (int)(a.rows - token0) : a.tokens;
  const int heads = a.H[0] + a.H[1], items = tokens * heads, half = a.rotary >> 1;
  // a lane's pairs: first channels c0 .. c0 + 3, second ones c1 .. c1 + 3 (neighbours: the eight from c0 on)
  const int pair = lane * 4;
  const bool there = pair * 2 < a.d, turns = pair < half;
  const int rest = (a.d - a.rotary) >> 1;
  const int c0 = INTER ? pair * 2 : (turns ? pair : a.rotary + pair - half), c1 = INTER ? c0 + 4 : c0 + (turns ? half : rest);

  struct Item { int which, token, head; };
  const auto item = [&](int n) __attribute__((always_inline)) {
    Item i;
    i.token = n / heads;
    i.head = n - i.token * heads;
    i.which = i.head >= a.H[0];
    if (i.which) i.head -= a.H[0];
    return i;
  };
  Four<DT> A[AHEAD], B[AHEAD];
  const auto load = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int n = n0 + k * GROUPS;
      if (n < items && there) {
        const Item i = item(n);
        const int64_t at = (token0 + i.token) * a.in_t[i.which] + i.head * a.in_h[i.which];
        A[k].load(a.in[i.which], at + c0);
        B[k].load(a.in[i.which], at + c1);
      }
    }
  };
  load(group);
  for (int n = tid; n < tokens * half; n += 256) {
    const int t = n / half, p = n - t * half;
    const int64_t pos = a.wide_positions ? ((const int64_t*)a.positions)[token0 + t] : ((const int32_t*)a.positions)[token0 + t];
    const double turn = (double)pos * (a.inv_freq[p] * 0.15915494309189533577);
    float sin, cos;
    sincospif(2.0f * (float)(turn - rint(turn)), &sin, &cos);
    s_turn[t][p] = make_float2(cos, sin);
  }
  float w[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (a.weight[i] && there) {
      Four<DT> x, y;
      x.load(a.weight[i], c0);
      y.load(a.weight[i], c1);
#pragma unroll
      for (int j = 0; j < 4; ++j) { w[i][j] = x.get(j); w[i][4 + j] = y.get(j); }
    }
  __syncthreads();
  for (int n0 = group; n0 < items; n0 += AHEAD * GROUPS) {
    float y[AHEAD][8];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) { y[k][j] = A[k].get(j); y[k][4 + j] = B[k].get(j); }
    const int next = n0 + AHEAD * GROUPS;
    if (next < items) load(next);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int n = n0 + k * GROUPS;
      if (n >= items) break;                                 // (the same for a head's lanes)
      const Item i = item(n);
      if (a.weight[i.which]) {
        float sum = 0.0f;
        if (there)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum = fmaf(y[k][j], y[k][j], sum);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float r = rsqrtf(sum / (float)a.d + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[k][j] = y[k][j] * r * (i.which ? w[1][j] : w[0][j]);
      }
      if (there) {
        if (turns) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 cs = s_turn[i.token][pair + j];
            float& p = y[k][INTER ? 2 * j : j];
            float& q = y[k][INTER ? 2 * j + 1 : 4 + j];
            const float b = p;
            p = p * cs.x - q * cs.y;
            q = q * cs.x + b * cs.y;
          }
        }
        const int64_t at = (token0 + i.token) * a.out_t[i.which] + i.head * a.out_h[i.which];
        Four<DT>::store(a.out[i.which], at + c0, y[k]);
        Four<DT>::store(a.out[i.which], at + c1, y[k] + 4);
      }
    }
  }
}

template <int DT, int LANES>
static int launch_rotate(const Rotate& a, bool inter, unsigned grid, hipStream_t st) {
  if (inter) rotate_kernel<DT, LANES, true><<<dim3(grid), dim3(256), 0, st>>>(a);
  else rotate_kernel<DT, LANES, false><<<dim3(grid), dim3(256), 0, st>>>(a);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
template <int DT>
static int launch_rotate(const Rotate& a, bool inter, unsigned grid, hipStream_t st) {
  if (a.d <= 64) return launch_rotate<DT, 8>(a, inter, grid, st);
  if (a.d <= 128) return launch_rotate<DT, 16>(a, inter, grid, st);
  if (a.d <= 256) return launch_rotate<DT, 32>(a, inter, grid, st);
  return launch_rotate<DT, 64>(a, inter, grid, st);
}

}  // namespace tq

extern "C" int tq_rotate_heads(const void* q, const void* k, int dtype, int64_t rows, int Hq, int Hkv, int d, int64_t qs_t, int64_t qs_h, int64_t ks_t,
                               int64_t ks_h, const void* positions, int wide_positions, const double* inv_freq, int rotary_dim, int interleaved,
                               const void* q_weight, const void* k_weight, float eps, void* q_out, int64_t qo_t, int64_t qo_h, void* k_out, int64_t ko_t,
                               int64_t ko_h, void* stream) {
  using namespace tq;
  if (dtype < TQ_F32 || dtype > TQ_BF16 || rows < 0 || rows > INT32_MAX || Hq < 0 || Hkv < 0 || Hq + (int64_t)Hkv <= 0 || Hq + (int64_t)Hkv > (1 << 24)) return TQ_EINVAL;
  if (d <= 0 || rotary_dim < 0 || rotary_dim > d) return TQ_EINVAL;
  if (d % 8 || d > 512 || rotary_dim % 8) return TQ_EUNSUPPORTED;
  if ((Hq && (!q || !q_out)) || (Hkv && (!k || !k_out)) || !positions || (rotary_dim && !inv_freq)) return TQ_ENULL;
  // rows on 8-byte boundaries (fp32: 16), four channels at a time
  const int64_t bytes = dtype == TQ_F32 ? 16 : 8, piece = 4;
  const int64_t strides[8] = {qs_t, qs_h, ks_t, ks_h, qo_t, qo_h, ko_t, ko_h};
  for (const int64_t s : strides)
    if (s < 0 || s % piece) return TQ_EUNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)q_weight | (uintptr_t)k_weight) % bytes) return TQ_EUNSUPPORTED;
  if (rows == 0) return TQ_OK;
  // Few tokens: one a workgroup, so that there are workgroups for the compute units; the sines of many are worked out 256 at a time.
  Rotate a{{q, k}, {q_out, k_out}, {q_weight, k_weight}, {qs_t, ks_t}, {qs_h, ks_h}, {qo_t, ko_t}, {qo_h, ko_h}, positions, inv_freq, rows, {Hq, Hkv}, d,
           rotary_dim, wide_positions, rows < 1024 ? 1 : ROTATE_TOKENS, eps};
  const unsigned grid = (unsigned)((rows + a.tokens - 1) / a.tokens);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == TQ_F32) return launch_rotate<TQ_F32>(a, interleaved != 0, grid, st);
  if (dtype == TQ_F16) return launch_rotate<TQ_F16>(a, interleaved != 0, grid, st);
  return launch_rotate<TQ_BF16>(a, interleaved != 0, grid, st);
}
