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
  int32_t n_split, chunk;                  // splits of a unit's tokens at most, blocks of a split (more where there are more tokens than planned for)
  int32_t target, cap;                     // where sequences differ: items of a head to share their blocks out to (0: as planned), splits of one of them at most
  float share;                             // 1 / target
  int32_t fill;                            // rows of no sequence become zeros
  float scale2;                            // scale x log2 e: the softmax is one of powers of two
  int32_t units;                           // units that the plan has room for
  int32_t items;                           // (unit, split) pairs that the grid has room for, for each KV head
  // Partial results, where a row may have several, and of every row how many: 0 where it is no sequence's, 1 where it is in `out` already.  As planned, a row has n_split
  // places of its own.  Shared out anew, a workgroup has `part` places, if its unit is split at all: for a KV head there are less than 2 target such shares, since a unit is
  // split only if it has more blocks than a share, of which all units have `target`.
  float* acc;                              // (places, d): numerators
  float2* ml;                              // (places): maximum (log2) and sum
  int2* shares;                            // (rows, Hq): shared out anew the first of its workgroups; number | row in the unit << 16 | planned << 24; null: all rows have one
  int32_t part, parts;                     // rows that a unit has at most; workgroups of split units that there is room for, for each KV head
};

// Infinities and NaN among the values.  A row's weights are 0 where it sees nothing, and 0 times them is NaN: where the rows of a unit see different tokens
// (blocks at their own positions and at the window's edge), such values are put to zero before the product, and the rows that see them get them added
// at the end, read once more.  A block that all rows see whole takes them as they are.
//   16 or 8 bits each: the numbers of x that are finite
template <int DT>
__device__ __forceinline__ uint32_t attend_finite(uint32_t x) {
  // (an exponent of all ones, in e4m3 all ones but the sign: a carry into the sign's place tells)
  if constexpr (DT == TQ_E4M3) return x & ~(((((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu);
  else if constexpr (DT == TQ_BF16) return x & ~(((((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu);
  else return x & ~(((((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u) >> 15) * 0xffffu);
}
//   number i of x if it is not finite, else 0
template <int DT>
__device__ __forceinline__ float attend_not_finite(f8_u32x2 x, int i) {
  if constexpr (DT == TQ_E4M3) {
    return (x[0] >> i * 8 & 0x7f) == 0x7f ? NAN : 0.0f;
  } else {
    const uint32_t n = x[i >> 1] >> (i & 1) * 16 & 0xffff;
    if constexpr (DT == TQ_BF16) return (n & 0x7f80) == 0x7f80 ? __uint_as_float(n << 16) : 0.0f;
    else return (n & 0x7c00) == 0x7c00 ? __uint_as_float((n & 0x8000) << 16 | 0x7f800000u | (n & 0x3ff) << 13) : 0.0f;
  }
}

// What a workgroup works on: `rows` rows of a sequence's run * G (the heads of a token side by side), from `first` on, and a share of the tokens they see
struct AttendUnit {
  int b;
  int64_t row;             // of the sequence's first row in the step
  int first, rows;
  int low, high;           // positions of the first and the last
  int tokens;              // up to the last's own token, as far as the table goes
  int split, splits;       // which share, of how many (before it is known how many there are tokens for)
  bool planned;            // shares as the host planned them
  int place;               // shared out anew: which of the shares of split units it is
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

// the j-th unit of M rows of a run
template <int M>
__device__ __forceinline__ void attend_unit(const Attend& a, const StepRun& r, int64_t j, AttendUnit* t) {
  t->row = r.row;
  t->first = (int)(j * M);
  const int64_t left = (int64_t)r.run * a.G - j * M;
  t->rows = left < M ? (int)left : M;
  t->low = r.token() + t->first / a.G;
  t->high = r.token() + (t->first + t->rows - 1) / a.G;
  const int cap = step_cap(a.s);
  t->tokens = t->high < 0 ? 0 : (t->high + 1 < cap ? t->high + 1 : cap);
}
template <int M>
__device__ __forceinline__ int attend_units(const Attend& a, const StepRun& r) { return (int)(((int64_t)r.run * a.G + M - 1) / M); }
// Blocks that the last unit of a run, which sees the most, sees; with a window those of the rows that the unit may have at most.
template <int M, int TB>
__device__ __forceinline__ int attend_most(const Attend& a, const StepRun& r) {
  AttendUnit t;
  const int cap = step_cap(a.s), reach = (M - 1) / a.G + 1;
  t.tokens = r.len < cap ? r.len : cap;
  t.low = r.len - 1 - reach;
  return r.run ? AttendBlocks<TB>(a, t).count : 0;
}
// ceil(blocks / chunk), 1 .. most.  (By a reciprocal: a division for each of four sequences a lane is half the time that looking them up takes.  One off
// where numbers pass 24 bits is as good a share.)
struct AttendSplits {
  int chunk, most;
  float inverse;
  __device__ __forceinline__ AttendSplits(int chunk, int most) : chunk(chunk), most(most), inverse(__builtin_amdgcn_rcpf((float)chunk)) {}
  __device__ __forceinline__ int operator()(int blocks) const {
    int n = (int)((float)blocks * inverse);
    n += n * chunk < blocks;
    return n < 1 ? 1 : (n > most ? most : n);
  }
};

// Item `n` of a step: whose rows, which share of their tokens.  false: there are fewer; it is then number *over of *others that are left over, if any.
// Shares are planned by the longest sequence there may be, the first shares of all units in front of the second ones (with the shares of a unit next to
// each other 32 sequences of 8192 took 120 us, so 106).  Where up to 256 sequences turn out to differ, their blocks are shared out anew, `target` items for each
// KV head in all, so that no workgroup has much more to do than another, and none starts for nothing.
template <int M, int TB>
__device__ __forceinline__ bool attend_item(const Attend& a, int n, AttendUnit* t, int* over, int* others) {
  int unit = 0;
  StepRun run;
  *over = *others = 0;
  t->split = (unsigned)n / (unsigned)a.units;
  int u = n - t->split * a.units;                            // of the units, as planned
  t->planned = true;
  t->splits = a.n_split;
  t->place = 0;
  if (!a.s.starts && a.target == 0) {
    if (t->split >= a.n_split) return false;
    const int per = (a.G + M - 1) / M;
    t->b = (unsigned)u / (unsigned)per;
    unit = u - t->b * per;
    run = step_run(a.s, t->b);
    run.len = __builtin_amdgcn_readfirstlane(run.len);
  } else {
    StepRun r[4];
    int blocks[4];
    bool found = false;
    // (behind the last share there is an item for rows of no sequence, if there are no units left over: as many units as there may be are then all met)
    const bool rest = n == a.units * a.n_split;
    if (rest) u = a.units;
    const int given = u;
    for (int base = 0; base < a.s.B && !found; base += STEP_ROUND) {
      step_runs(a.s, base, r);
      int count[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) count[i] = base + i * 64 < a.s.B && r[i].run ? attend_units<M>(a, r[i]) : 0;
      if (a.target > 0) {                                     // (a single round)
        float total = 0.0f, longest = 0.0f, units = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          blocks[i] = 0;
          if (base + i * 64 >= a.s.B) continue;
          blocks[i] = attend_most<M, TB>(a, r[i]);
          const float x = (float)count[i], y = (float)blocks[i];
          total = fmaf(x, y, total);
          units += x;
          longest = fmaxf(longest, y);
        }
        total = wave_sum_fast(total);
        longest = wave_max_fast(longest);
        if (longest * wave_sum_fast(units) * 7 > total * 8) {  // (by more than an eighth)
          // (few rows: not less than 512 tokens, of which a wavefront has four turns, nor so little that the longest sequence would have more shares than it may; many: not less
          // than 2048 tokens, 32 turns, since the join of many rows takes its time)
          const float least = M > 32 ? 32.0f : fmaxf(16.0f, ceilf(longest * (1.0f / (float)a.cap)));
          const AttendSplits splits((int)fminf(fmaxf(ceilf(total * a.share), least), 1e9f), a.cap);
#pragma unroll
          for (int i = 0; i < 4; ++i) count[i] *= splits(blocks[i]);
          t->planned = false;
          int j = n;
          found = step_find(a.s, base, r, count, &j, &t->b, &unit, &run);
          if (!found) {
            *over = j;
            *others = a.items - (n - j);
            return false;
          }
          t->splits = __builtin_amdgcn_readfirstlane(splits(attend_most<M, TB>(a, run)));
          t->split = unit % t->splits;
          if (t->splits > 1) {
            int split[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split[i] = splits(blocks[i]) > 1 ? count[i] : 0;
            t->place = __builtin_amdgcn_readfirstlane(step_before(a.s, split, t->b) + unit);
            if (t->place - t->split + t->splits > a.parts) return false;      // (starts that do not ascend: more than there may be)
          }
          unit = unit / t->splits;
          break;
        }
      }
      found = step_find(a.s, base, r, count, &u, &t->b, &unit, &run);
    }
    if (t->planned && t->split >= a.n_split && !rest) return false;
    if (!found) {
      if (t->split == 0 || rest) {
        *over = u;
        *others = a.units + 1 - (given - u);
      }
      return false;
    }
    if (t->planned && rest) return false;                    // (more units than there may be: starts that do not ascend)
  }
  // (all of it is the same for the whole wavefront, which only the scalar registers say to the compiler: its tables' entries are scalar loads then)
  t->b = __builtin_amdgcn_readfirstlane(t->b);
  t->split = __builtin_amdgcn_readfirstlane(t->split);
  attend_unit<M>(a, run, __builtin_amdgcn_readfirstlane(unit), t);
  return true;
}

// A unit's share of its blocks: [first, last) of the list, and how many shares there are blocks for (one at least)
struct AttendShare {
  int first, last, used;
  __device__ __forceinline__ AttendShare(const Attend& a, const AttendUnit& u, int count) {
    int per = (count + u.splits - 1) / u.splits;
    if (u.planned && per < a.chunk) per = a.chunk;
    per = per < 1 ? 1 : per;
    used = count < 1 ? 1 : (count + per - 1) / per;
    first = u.split * per < count ? u.split * per : count;
    last = first + per < count ? first + per : count;
  }
};
// Where the partial result of a unit's row r lies, `row` of the step's rows x heads; and what the join is told of a row
__device__ __forceinline__ int64_t attend_place(const Attend& a, const AttendUnit& u, int h, int r, int64_t row) {
  return u.planned ? row * a.n_split + u.split : ((int64_t)u.place * a.H + h) * a.part + r;
}
__device__ __forceinline__ int2 attend_told(const Attend& a, const AttendUnit& u, int h, int r, int used) {
  return make_int2(u.place * a.H + h, used | r << 16 | (u.planned ? 1 << 24 : 0));
}
// Items behind the last sequence's, of which this is number `number` of `others`: rows of no sequence, KV head h's part of them
template <int D>
__device__ __forceinline__ void attend_rest(const Attend& a, int h, int number, int64_t others) {
  if (others <= 0) return;
  int64_t front;
  const int64_t rest = step_rest(a.s, &front);
  for (int64_t n = number; n < rest; n += others) {
    const int64_t row = step_rest_row(a.s, front, rest, n) * a.Hq + h * a.G;
    if (a.shares)
      for (int g = (int)threadIdx.x; g < a.G; g += 256) a.shares[row + g] = make_int2(0, 0);
    if (a.fill)
      for (int c = (int)threadIdx.x; c < a.G * D / 2; c += 256) ((uint32_t*)((uint16_t*)a.out + row * D))[c] = 0;
  }
}

template <int QT, bool F8> int launch_attend_few(const Attend& a, int tiles, unsigned grid, hipStream_t stream);
template <int QT, bool F8> int launch_attend_rows(const Attend& a, unsigned grid, hipStream_t stream);

}  // namespace tq
