// The norm of every head of queries and keys and the rotation by position, in one pass.
//
//   y = x / sqrt(mean x^2 + eps) w       (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * inv_freq of the pair
//
// A group of lanes takes a head of a token, a lane 4 PIECES pairs: the halves that a rotation brings together are one lane's already, and the norm is a sum
// over neighbouring lanes.  Channels behind the rotated ones are pairs, too, that do not turn.
// An angle is the same for all heads: a workgroup works out the sines and cosines of its tokens once, one a thread, into LDS, behind the loads of its
// first heads.  In turns and 64 bits, position * (inv_freq / 2 pi) less its whole turns: at position 2^20 an angle in 32 bits would be 0.03 off.
// All sums, norms and rotations in 32 bits, one rounding at the end.  Bound by the memory system: 16384 tokens, 40 and 8 heads of 128, bf16 with norms, 403 MB in 80 us,
// 5.0 TB/s (a large copy: 5.1); with four pairs a lane, 8 bytes a load, 145 us.  A step of 64 tokens, 5.8 us, is a launch, the positions' latency and the sines.
#include "tq_step.h"

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

// two numbers to 16 bits, nearest even
template <int DT>
__device__ __forceinline__ uint32_t ro_pack(float a, float b) {
  if constexpr (DT == TQ_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
  }
}

// 4 N neighbouring channels
template <int DT, int N>
struct Channels {
  typedef uint32_t words __attribute__((ext_vector_type(2 * N)));
  words x;
  __device__ __forceinline__ void load(const void* p, int64_t at) { x = *(const words*)((const uint16_t*)p + at); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = x[i >> 1];
    if constexpr (DT == TQ_BF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    else return f16_bits_to_f32((uint16_t)(w >> (i & 1 ? 16 : 0)));
  }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* y) {
    words r;
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) r[i] = ro_pack<DT>(y[2 * i], y[2 * i + 1]);
    *(words*)((uint16_t*)p + at) = r;
  }
};
template <int N>
struct Channels<TQ_F32, N> {
  float4 x[N];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *(const float4*)((const float*)p + at + 4 * i);
  }
  __device__ __forceinline__ float get(int i) const { const float4& v = x[i >> 2]; return (i & 3) == 0 ? v.x : ((i & 3) == 1 ? v.y : ((i & 3) == 2 ? v.z : v.w)); }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* y) {
#pragma unroll
    for (int i = 0; i < N; ++i) *(float4*)((float*)p + at + 4 * i) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
  }
};

// sum over LANES neighbouring lanes
template <int LANES>
__device__ __forceinline__ float ro_sum(float v) {
  v = lanes_sum_dpp<(LANES < 16 ? LANES : 16)>(v);
  if constexpr (LANES > 16) v += __shfl_xor(v, 16, 64);
  if constexpr (LANES > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

// LANES: of a head; a lane has N runs of four pairs.  INTER: pairs are neighbours (2 i, 2 i + 1), not the two halves (i, i + rotary / 2).
template <int DT, int LANES, int N, bool INTER>
__global__ void __launch_bounds__(256) rotate_kernel(const Rotate a) {
  constexpr int GROUPS = 256 / LANES, AHEAD = N == 1 ? 4 : 3, W = 4 * N;
  __shared__ float2 s_turn[ROTATE_TOKENS][ROTATE_PAIRS];
  const int tid = (int)threadIdx.x, lane = tid % LANES, group = tid / LANES;
  const int64_t token0 = (int64_t)blockIdx.x * a.tokens;
  const int tokens = a.rows - token0 < a.tokens ? (int)(a.rows - token0) : a.tokens;
  const int heads = a.H[0] + a.H[1], half = a.rotary >> 1;
  // a lane's pairs: first channels c0 .. c0 + W - 1, second ones c1 .. c1 + W - 1 (neighbours: the 2 W from c0 on)
  const int pair = lane * W;
  const bool there = pair * 2 < a.d, turns = pair < half;
  const int rest = (a.d - a.rotary) >> 1;
  const int c0 = INTER ? pair * 2 : (turns ? pair : a.rotary + pair - half), c1 = INTER ? c0 + W : c0 + (turns ? half : rest);

  // a group's heads are GROUPS apart, over the workgroup's tokens
  struct Item { int token, head; };
  const int over = GROUPS / heads, left = GROUPS - over * heads;
  const auto next = [&](Item i) __attribute__((always_inline)) {
    i.token += over;
    i.head += left;
    if (i.head >= heads) { i.head -= heads; ++i.token; }
    return i;
  };
  Channels<DT, N> A[AHEAD], B[AHEAD];
  const auto load = [&](Item i) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (i.token < tokens && there) {
        const bool key = i.head >= a.H[0];
        const int64_t at = (token0 + i.token) * (key ? a.in_t[1] : a.in_t[0]) + (key ? i.head - a.H[0] : i.head) * (key ? a.in_h[1] : a.in_h[0]);
        const void* from = key ? a.in[1] : a.in[0];
        A[k].load(from, at + c0);
        B[k].load(from, at + c1);
      }
      i = next(i);
    }
    return i;
  };
  Item now = {group / heads, group - group / heads * heads}, ahead = load(now);
  for (int n = tid; n < tokens * half; n += 256) {
    const int t = n / half, p = n - t * half;
    const int64_t pos = a.wide_positions ? ((const int64_t*)a.positions)[token0 + t] : ((const int32_t*)a.positions)[token0 + t];
    const double turn = (double)pos * (a.inv_freq[p] * 0.15915494309189533577);
    float sin, cos;
    sincospif(2.0f * (float)(turn - rint(turn)), &sin, &cos);
    s_turn[t][p] = make_float2(cos, sin);
  }
  Channels<DT, N> w[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (a.weight[i] && there) {
      w[i][0].load(a.weight[i], c0);
      w[i][1].load(a.weight[i], c1);
    }
  const float mean = 1.0f / (float)a.d;
  __syncthreads();
  while (now.token < tokens) {
    float y[AHEAD][2 * W];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int j = 0; j < W; ++j) { y[k][j] = A[k].get(j); y[k][W + j] = B[k].get(j); }
    if (ahead.token < tokens) ahead = load(ahead);
    else ahead.token = tokens;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (now.token >= tokens) break;                        // (the same for a head's lanes)
      const bool key = now.head >= a.H[0];
      if (key ? a.weight[1] : a.weight[0]) {
        float sum = 0.0f;
        if (there)
#pragma unroll
          for (int j = 0; j < 2 * W; ++j) sum = fmaf(y[k][j], y[k][j], sum);
        sum = ro_sum<LANES>(sum);
        const float r = rsqrtf(fmaf(sum, mean, a.eps));
#pragma unroll
        for (int j = 0; j < W; ++j) {
          y[k][j] = y[k][j] * r * (key ? w[1][0].get(j) : w[0][0].get(j));
          y[k][W + j] = y[k][W + j] * r * (key ? w[1][1].get(j) : w[0][1].get(j));
        }
      }
      if (there) {
        if (turns) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float2 cs = s_turn[now.token][pair + j];
            float& p = y[k][INTER ? 2 * j : j];
            float& q = y[k][INTER ? 2 * j + 1 : W + j];
            const float b = p;
            p = fmaf(p, cs.x, -(q * cs.y));
            q = fmaf(q, cs.x, b * cs.y);
          }
        }
        const int64_t at = (token0 + now.token) * (key ? a.out_t[1] : a.out_t[0]) + (key ? now.head - a.H[0] : now.head) * (key ? a.out_h[1] : a.out_h[0]);
        void* to = key ? a.out[1] : a.out[0];
        Channels<DT, N>::store(to, at + c0, y[k]);
        Channels<DT, N>::store(to, at + c1, y[k] + W);
      }
      now = next(now);
    }
  }
}

template <int DT, int LANES, int N>
static int launch_rotate(const Rotate& a, bool inter, unsigned grid, hipStream_t st) {
  if (inter) rotate_kernel<DT, LANES, N, true><<<dim3(grid), dim3(256), 0, st>>>(a);
  else rotate_kernel<DT, LANES, N, false><<<dim3(grid), dim3(256), 0, st>>>(a);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
// wide: eight pairs a lane, 16 bytes a load (fp32: two of them), where sizes, strides and addresses allow it
template <int DT>
static int launch_rotate(const Rotate& a, bool inter, bool wide, unsigned grid, hipStream_t st) {
  if (wide) {
    if (a.d <= 64) return launch_rotate<DT, 4, 2>(a, inter, grid, st);
    if (a.d <= 128) return launch_rotate<DT, 8, 2>(a, inter, grid, st);
    if (a.d <= 256) return launch_rotate<DT, 16, 2>(a, inter, grid, st);
    return launch_rotate<DT, 32, 2>(a, inter, grid, st);
  }
  if (a.d <= 64) return launch_rotate<DT, 8, 1>(a, inter, grid, st);
  if (a.d <= 128) return launch_rotate<DT, 16, 1>(a, inter, grid, st);
  if (a.d <= 256) return launch_rotate<DT, 32, 1>(a, inter, grid, st);
  return launch_rotate<DT, 64, 1>(a, inter, grid, st);
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
  if ((rows + a.tokens - 1) / a.tokens > STEP_MAX_GROUPS) return TQ_EINVAL;
  const unsigned grid = (unsigned)((rows + a.tokens - 1) / a.tokens);
  hipStream_t st = (hipStream_t)stream;
  bool wide = d % 16 == 0 && rotary_dim % 16 == 0 && ((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)q_weight | (uintptr_t)k_weight) % 16 == 0;
  for (const int64_t s : strides) wide = wide && s % (dtype == TQ_F32 ? 4 : 8) == 0;
  if (dtype == TQ_F32) return launch_rotate<TQ_F32>(a, interleaved != 0, wide, grid, st);
  if (dtype == TQ_F16) return launch_rotate<TQ_F16>(a, interleaved != 0, wide, grid, st);
  return launch_rotate<TQ_BF16>(a, interleaved != 0, wide, grid, st);
}
