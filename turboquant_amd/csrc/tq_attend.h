// Attention of a step's rows over a paged cache - the engine's exact blocks in fp16 or bf16, or the 8-bit cache -, causal, within a sliding window and
// a few first tokens (sinks).
//   row i of a sequence with `run` rows and `len` tokens stands at p = len - run + i and sees token t if t <= p and (t > p - window or t < sinks)
#pragma once

#include "tq_fp8.h"

namespace tq {

constexpr int ATTEND_ALL = INT32_MAX;      // a window that leaves nothing out

struct Attend {
  Step s;
  const void *k, *v;                       // element strides
  const uint8_t *k_scales, *v_scales;      // 8-bit cache: (num_blocks, H)
  int64_t s_blk, s_h;
  int32_t s_t, H, d;
  const void* q;                           // (rows, Hq, d)
  void* out;
  int32_t Hq, G, window, sinks;
  int32_t n_split, chunk;                  // splits of a unit's tokens, blocks of a split (more where there are more tokens than planned for)
  int32_t fill;                            // rows of no sequence become zeros
  float scale2;                            // scale x log2 e: the softmax is one of powers of two
  int64_t units;                           // rows' units that the grid has room for
  float* acc;                              // (rows, Hq, n_split, d): numerators of a split; unused with one split
  float2* ml;                              // (rows, Hq, n_split): its maximum (log2) and its sum; ATTEND_EMPTY, ATTEND_REST in the sum's place
};
constexpr float ATTEND_EMPTY = -1.0f;      // a split without tokens (these are the last ones of a row)
constexpr float ATTEND_REST = -2.0f;       // of a row of no sequence, in its first split

// The row with the lowest position that `unit rows` row .. row + n - 1 (of a sequence's run * G, heads of a token side by side) have, and what they see
struct AttendUnit {
  int b, h;
  int64_t row;             // of the sequence's first row in the step
  int first, rows;         // unit rows: the first of them (token row * G + head), how many
  int low, high;           // positions of the first and the last
  int tokens;              // up to the last's own token, as far as the table goes
};
// Blocks of TB tokens that a unit sees any token of: `front` from token 0 on (sinks), then from `from` on
template <int TB>
struct AttendBlocks {
  int front, from, count;
  __device__ __forceinline__ AttendBlocks(const Attend& a, const AttendUnit& u) {
    const int all = (u.tokens + TB - 1) / TB;
    from = (u.low >= a.window ? u.low - a.window + 1 : 0) / TB;
    from = from < all ? from : all;
    front = ((u.tokens < a.sinks ? u.tokens : a.sinks) + TB - 1) / TB;
    front = front < from ? front : from;
    count = front + all - from;
  }
  __device__ __forceinline__ int operator[](int i) const { return i < front ? i : i - front + from; }
};
// the last position that row p does not see for its window (tokens up to it are seen only below `sinks`)
__device__ __forceinline__ int attend_behind(const Attend& a, int p) { return p >= a.window ? p - a.window : -1; }

__host__ __device__ __forceinline__ int attend_per_split(int blocks, int n_split, int chunk) {
  const int least = (blocks + n_split - 1) / n_split;
  return least > chunk ? least : chunk;
}

// Unit u of units of M rows: whose rows they are.  false: there are fewer; *u counts on from behind the last.
template <int M>
__device__ __forceinline__ bool attend_unit(const Attend& a, int64_t* u, AttendUnit* t) {
  int64_t j = 0;
  StepRun r;
  if (!a.s.starts) {
    const int per = (a.G + M - 1) / M;
    if (*u >= (int64_t)a.s.B * per) { *u -= (int64_t)a.s.B * per; return false; }
    t->b = (int)(*u / per);
    j = *u - (int64_t)t->b * per;
  } else if (!step_unit(a.s, u, &t->b, &j, [&](const StepRun& x) { return ((int64_t)x.run * a.G + M - 1) / M; })) {
    return false;
  }
  // (all of it is the same for the whole wavefront, which only the scalar registers say to the compiler: its tables' entries are scalar loads then)
  t->b = __builtin_amdgcn_readfirstlane(t->b);
  j = step_uniform(j);
  r = step_run(a.s, t->b);
  r.row = step_uniform(r.row);
  r.run = __builtin_amdgcn_readfirstlane(r.run);
  r.len = __builtin_amdgcn_readfirstlane(r.len);
  t->row = r.row;
  t->first = (int)(j * M);
  const int64_t left = (int64_t)r.run * a.G - j * M;
  t->rows = left < M ? (int)left : M;
  t->low = r.token() + t->first / a.G;
  t->high = r.token() + (t->first + t->rows - 1) / a.G;
  const int cap = step_cap(a.s);
  t->tokens = t->high < 0 ? 0 : (t->high + 1 < cap ? t->high + 1 : cap);
  return true;
}

// Units behind the last sequence's, of which this is number `number` of `others`: rows of no sequence, KV head h's part of them
template <int D>
__device__ __forceinline__ void attend_rest(const Attend& a, int split, int h, int64_t number, int64_t others) {
  if (split) return;
  int64_t front;
  const int64_t rest = step_rest(a.s, &front);
  for (int64_t n = number; n < rest; n += others) {
    const int64_t row = step_rest_row(a.s, front, rest, n) * a.Hq + h * a.G;
    if (a.n_split > 1) {
      for (int g = (int)threadIdx.x; g < a.G; g += 256) a.ml[(row + g) * a.n_split] = make_float2(-INFINITY, ATTEND_REST);
    } else if (a.fill) {
      for (int c = (int)threadIdx.x; c < a.G * D / 2; c += 256) ((uint32_t*)((uint16_t*)a.out + row * D))[c] = 0;
    }
  }
}

template <int QT, bool F8> int launch_attend_few(const Attend& a, int tiles, unsigned grid, hipStream_t stream);
template <int QT, bool F8> int launch_attend_rows(const Attend& a, unsigned grid, hipStream_t stream);

}  // namespace tq
