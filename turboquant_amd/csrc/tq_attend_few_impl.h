// Attention of few rows - one token of a sequence, or a few - over a paged cache (instantiated by one file per types).
//
// A unit is 16 NT rows of a KV head: the query heads of a token side by side, tokens one behind another; they are the columns of the matrix
// instructions.  A workgroup's four wavefronts take 32 tokens each at a time, straight from memory into the operands, as the decode kernel of the exact
// cache does it: no shared memory and no barrier in the loop, the next block's keys and values on their way in registers.
//   scores    tokens are rows; a lane reads 16 bytes of ONE token's key.  8 bits: those are 16 channels, two steps of 32, and the queries lie in registers
//             in that order; two numbers become 16-bit ones in an instruction (e4m3 is a subset of both), the block's scale multiplies the score.
//   values    channels are rows; a lane reads its channels of its 8 tokens and turns them around in registers.  8 bits: half as many byte permutes, and the
//             conversion to bf16 multiplies by the block's scale for nothing; bf16 for fp16 queries, too, whose range the scale might leave.
//   softmax   one pass, running maximum and sum per row, all in 32 bits; weights go in as a high and a low half (ex_split).
//
// Bound by the memory system, whose 5.5 TB/s (a large read) it comes near where there is enough of it: one token of 32 sequences of 8192, 32 query heads on
// 8 of 128, 8 bits: 538 MB in 107 us with the join's 5 (5.0 TB/s); bf16 blocks, the last 4096 of 32 sequences of 32768: as many bytes, 103 us.
// One sequence of 131072, 16 query heads on 2 of 256, 8 bits: 134 MB in 35 us, of which the first loads and the join are 8.  One of 700: 10 us, the chain of length,
// table, keys, values and the join's launch.  Several rows on 8 bits are bound by instructions: 24 sequences of 61 .. 16000, 5 rows, 20 columns of the 32, fp16 queries, 154 MB
// in 54 us, where 32 tokens of a wavefront are 48 matrix instructions and 300 of the vector unit's (64 conversions, 24 permutes, the weights' halves).
#pragma once

#include "tq_attend.h"
#include "tq_exact_impl.h"

namespace tq {

// two e4m3 numbers (the lower or the upper half of x) as 16-bit ones, times a power of two
template <int QT, bool UPPER>
__device__ __forceinline__ uint32_t f8_widen(uint32_t x, float scale) {
  if constexpr (QT == TQ_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, UPPER));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, UPPER));
}

// Wavefronts on a SIMD.  (16 bits, 128 channels, rows at different positions: at three 8 registers are spilled, 2 rows of 24 sequences of 61 .. 16000 78 us, at two 71; 4 rows of 32 of
// 8192 214 / 199)
template <bool F8, int D, int NT, bool APART>
constexpr int attend_few_waves() {
  if (!F8 && D == 128 && NT == 1 && APART) return 2;
  if (NT == 1) return F8 ? (D <= 64 ? 4 : (D <= 128 ? 3 : 2)) : (D <= 64 ? 4 : (D <= 128 ? 3 : (D <= 192 ? 2 : 1)));
  return F8 ? (D <= 64 ? 3 : (D <= 128 ? 2 : 1)) : (D <= 64 ? 3 : (D <= 128 ? 2 : 1));
}

// APART: rows of a unit may stand at different positions (not one token of each sequence)
template <int QT, bool F8, int D, int NT, bool APART>
__global__ void __launch_bounds__(256, (attend_few_waves<F8, D, NT, APART>())) attend_few_kernel(const Attend a) {
  constexpr int PT = F8 ? TQ_BF16 : QT;                      // of the value product
  constexpr int VT = F8 ? TQ_E4M3 : QT;                      // of the cache
  constexpr int SIZE = F8 ? 1 : 2, PAGES = 2, TB = 32;
  constexpr int KLOADS = D * SIZE / 64, KSTEPS = D / 32;     // 16-byte pieces of a key that a lane reads; steps of 32 channels
  constexpr int TILES = D / 16;
  constexpr int WIDE = F8 ? 0 : D / 128, NARROW = F8 ? 0 : (D - WIDE * 128) / 64;
  constexpr int VWORDS = D / 64;                             // 8 bits: words of a token that a lane reads
  typedef uint32_t vword __attribute__((ext_vector_type(VWORDS == 3 ? 4 : VWORDS)));

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int col = lane & 15, quarter = lane >> 4;
  // Two heads' rows share a line of 128 bytes where a row is 64 or 192: they go to one of the eight dies, whose L2 the line is in then, eight workgroups apart (sixteen of
  // them are eight pairs, and so are those behind the last sixteen).  8 bits, 32 sequences of 8192, 32 heads on 8: of 64 92 -> 63 us, of 192 175 -> 170; 16 sequences, 32 on 32 of 64 173 -> 118.
  constexpr bool PAIRS = F8 && (D == 64 || D == 192);
  const bool paired = PAIRS && a.H % 2 == 0;
  unsigned at = blockIdx.x;
  if (paired) {
    const unsigned from = at & ~15u, r = at - from, half = (gridDim.x - from < 16u ? gridDim.x - from : 16u) / 2u;
    at = from + (r < half ? 2u * r : 2u * (r - half) + 1u);
  }
  const int item = (int)(at / (unsigned)a.H), x = (int)(at - (unsigned)item * (unsigned)a.H);
  AttendUnit u;
  int over, others;
  if (!attend_item<16 * NT, TB>(a, item, &u, &over, &others)) {
    attend_rest<D>(a, x, over, others);
    return;
  }
  // Which KV head: not the same for all that a compute unit has at a time (as planned, shares of one unit), whose addresses would all be the same in the bits
  // that tell heads apart.  32 sequences of 8192, 8 heads of 128, 8 bits: 122 us with head x, 119 with x + unit, 107 so.
  const int h = (int)((unsigned)(x + (u.planned ? u.split : item) * (paired ? 2 : 1)) % (unsigned)a.H);
  const AttendBlocks<TB> list(a, u);
  const AttendShare share(a, u, list.count);
  if (u.split >= share.used) return;
  const int first = share.first, last = share.last;

  // this lane's rows: one of each column tile
  bool live[NT];
  int64_t row[NT];                                           // (token row, head) of the step
  int at_p[NT], behind[NT];                                  // what the row sees: t <= at_p and (t > behind or t < sinks)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 16 + col;
    live[n] = r < u.rows;
    const int x = u.first + (live[n] ? r : 0), i = x / a.G;
    row[n] = (u.row + i) * a.Hq + h * a.G + (x - i * a.G);
    at_p[n] = u.low + (i - u.first / a.G);
    behind[n] = attend_behind(a, at_p[n]);
  }
  if (a.shares && u.split == 0 && wave == 0 && quarter == 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (live[n]) a.shares[row[n]] = attend_told(a, u, h, n * 16 + col, share.used);
  }
  const int32_t* table = a.s.table + u.b * a.s.table_step;

  // Scores are multiplied by their factor at once, or, 256 channels and one tile of columns, in the exponential, where the queries take a negative scale's sign or zero, so that the
  // scores' order is that of their products (one sequence of 131072, 16 heads on 2 of 256, 8 bits 36.8 / 34.5 us; 32 windows of 4096, bf16, 208 / 200; but one tile of 64
  // channels, 32 of 8192, 8 bits 91.8 / 95.2, and 128 of bf16, 2 rows of 24 sequences, 78.9 / 93.4, since registers are spilled; two tiles of 128, 5 rows, 54.8 / 56.1).
  constexpr bool LATER = D == 256 && NT == 1;
  const float scale = LATER ? (a.scale2 == 0.0f ? 1.0f : fabsf(a.scale2)) : a.scale2;
  ex_u32x4 Q[NT][KSTEPS];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      Q[n][s] = ex_u32x4{0, 0, 0, 0};
      const int c = F8 ? (s >> 1) * 64 + quarter * 16 + (s & 1) * 8 : s * 32 + quarter * 8;
      if (live[n]) Q[n][s] = *(const ex_u32x4*)((const uint16_t*)a.q + row[n] * D + c);
      if constexpr (LATER) {
        const uint32_t sign = a.scale2 < 0.0f ? 0x80008000u : 0u, some = a.scale2 == 0.0f ? 0u : 0xffffffffu;
#pragma unroll
        for (int i = 0; i < 4; ++i) Q[n][s][i] = (Q[n][s][i] & some) ^ sign;
      }
    }
  ex_f32x4 O[NT][TILES];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) O[n][t] = ex_f32x4{0, 0, 0, 0};
    m[n] = -INFINITY;
    l[n] = 0.0f;
  }

  // a block's two pages: where they lie, their scales, how many of their tokens count
  struct Pages {
    int64_t at[PAGES];
    uint32_t scales;                                         // lane l's: of page l & 1, of its keys or (l & 2) its values
    int valid[PAGES], t0;
    bool whole;
  };
  struct Entries {
    int32_t page[PAGES];
    int blk;
  };
  const int last_page = u.tokens > 0 ? (u.tokens - 1) / TQ_PAGE_TOKENS : 0;
  const int low_behind = attend_behind(a, u.high), unit_behind = attend_behind(a, u.low);
  // (table entries are read two blocks ahead, without a condition around them: those behind the last block are the last page's)
  const auto entries = [&](Entries& x, int i) __attribute__((always_inline)) {
    x.blk = list[i];
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      const int page = x.blk * PAGES + p;
      x.page[p] = step_entry(table, page < last_page ? page : last_page);
    }
  };
  const auto find = [&](Pages& x, const Entries& e) __attribute__((always_inline)) {
    x.t0 = e.blk * TB;
    x.whole = x.t0 + TB - 1 <= u.low && (x.t0 > low_behind || x.t0 + TB <= a.sinks);
    int64_t page[PAGES];
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      const int left = u.tokens - (e.blk * PAGES + p) * TQ_PAGE_TOKENS;
      x.valid[p] = left < 0 ? 0 : (left > TQ_PAGE_TOKENS ? TQ_PAGE_TOKENS : left);
      page[p] = e.page[p];
      if (page[p] < 0 || page[p] >= a.s.num_blocks) { page[p] = 0; x.valid[p] = 0; }
      x.whole &= x.valid[p] == TQ_PAGE_TOKENS;
      x.at[p] = (page[p] * a.s_blk + h * a.s_h) * SIZE;
    }
    if constexpr (F8) x.scales = (lane & 2 ? a.v_scales : a.k_scales)[(lane & 1 ? page[1] : page[0]) * a.H + h];
  };

  const uint32_t step = (uint32_t)a.s_t * SIZE;
  const uint32_t krow = (uint32_t)col * step + quarter * 16, vrow = (uint32_t)(quarter * 4) * step;
  ex_u32x4 K[PAGES][KLOADS];
  ex_u32x4 V[WIDE > 0 ? WIDE : 1][8];
  ex_u32x2 VN[8];
  vword VB[8];
  const auto load_keys = [&](const Pages& x) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
#pragma unroll
      for (int s = 0; s < KLOADS; ++s) K[p][s] = *(const ex_u32x4*)((const char*)a.k + x.at[p] + krow + s * 64);
  };
  const auto load_values = [&](const Pages& x) __attribute__((always_inline)) {
    if constexpr (F8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint8_t* from = (const uint8_t*)a.v + x.at[i >> 2] + vrow + (i & 3) * step + col * (VWORDS * 4);
        if constexpr (VWORDS == 3) {
          typedef uint32_t three __attribute__((ext_vector_type(3), aligned(4)));
          const three y = *(const three*)from;
          VB[i] = vword{y[0], y[1], y[2], 0};
        } else {
          VB[i] = *(const vword*)from;
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < WIDE; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) V[c][i] = *(const ex_u32x4*)((const char*)a.v + x.at[i >> 2] + vrow + (i & 3) * step + (c * 128 + col * 8) * 2);
      if constexpr (NARROW > 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) VN[i] = *(const ex_u32x2*)((const char*)a.v + x.at[i >> 2] + vrow + (i & 3) * step + (WIDE * 128 + col * 4) * 2);
      }
    }
  };

  bool odd = false;                                          // values that are not finite have been put to zero
  Pages now, next;
  Entries ahead;
  if (first + wave < last) {
    entries(ahead, first + wave);
    find(now, ahead);
    load_keys(now);
    load_values(now);
    entries(ahead, first + wave + 4);
  }
  for (int blk = first + wave; blk < last; blk += 4) {
    const bool more = blk + 4 < last;
    if (more) find(next, ahead);
    entries(ahead, blk + 8);
    float k_scale[PAGES], v_scale[PAGES];
    if constexpr (F8) {
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        k_scale[p] = scale * f8_scale((uint32_t)__builtin_amdgcn_readlane((int)now.scales, p));
        if constexpr (LATER) k_scale[p] = fmaxf(k_scale[p], 0x1p-149f);      // (two small ones may be nothing together, and nothing times a masked score's -inf is NaN)
        v_scale[p] = f8_scale((uint32_t)__builtin_amdgcn_readlane((int)now.scales, 2 + p));
      }
    }
    // ---- scores ----
    ex_f32x4 S[NT][PAGES];
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
#pragma unroll
      for (int n = 0; n < NT; ++n) S[n][p] = ex_f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        ex_u32x4 k;
        if constexpr (F8) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x = K[p][s >> 1][(s & 1) * 2 + w];
            k[w * 2] = f8_widen<QT, false>(x, 1.0f);
            k[w * 2 + 1] = f8_widen<QT, true>(x, 1.0f);
          }
        } else {
          k = K[p][s];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) S[n][p] = ex_mfma<QT>(k, Q[n][s], S[n][p]);
      }
    }
    if (more) load_keys(next);
    // ---- weights of this lane's rows: tokens quarter * 4 + i of each page ----
    ex_u32x4 P[NT], L[NT];                                   // high and low halves
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = -INFINITY, pr[PAGES][4];
#pragma unroll
      for (int p = 0; p < PAGES; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[p][i] = LATER ? S[n][p][i] : S[n][p][i] * (F8 ? k_scale[p] : scale);
      if (!now.whole) {
#pragma unroll
        for (int p = 0; p < PAGES; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int in = quarter * 4 + i, t = now.t0 + p * TQ_PAGE_TOKENS + in;
            const bool seen = (in < now.valid[p]) & (t <= at_p[n]) & ((t > behind[n]) | (t < a.sinks));
            pr[p][i] = seen ? pr[p][i] : -INFINITY;
          }
      }
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        if constexpr (LATER) {
          top = fmaxf(top, fmaxf(fmaxf(pr[p][0], pr[p][1]), fmaxf(pr[p][2], pr[p][3])) * (F8 ? k_scale[p] : scale));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, pr[p][i]);
        }
      }
      top = fmaxf(m[n], ex_quad_max(top));
      if (__any(top > m[n] + EX_SLACK)) {
        const float move = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[n] - top);
        l[n] *= move;
#pragma unroll
        for (int t = 0; t < TILES; ++t) O[n][t] *= move;
        m[n] = top;
      }
      const float ref = m[n] == -INFINITY ? 0.0f : m[n] - ex_lift<PT>();
#pragma unroll
      for (int p = 0; p < PAGES; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[p][i] = __builtin_amdgcn_exp2f(LATER ? fmaf(pr[p][i], F8 ? k_scale[p] : scale, -ref) : pr[p][i] - ref);
          l[n] += pr[p][i];
        }
#pragma unroll
      for (int p = 0; p < PAGES; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t hi, lo;
          ex_split<PT>(pr[p][2 * i], pr[p][2 * i + 1], &hi, &lo);
          P[n][p * 2 + i] = hi;
          L[n][p * 2 + i] = lo;
        }
    }
    // ---- values; those of tokens that no row of the unit sees are put to zero, since NaN times nothing is NaN ----
    if (!now.whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int in = quarter * 4 + (i & 3), t = now.t0 + (i >> 2) * TQ_PAGE_TOKENS + in;
        const uint32_t keep = (in < now.valid[i >> 2]) & ((t > unit_behind) | (t < a.sinks)) ? 0xffffffffu : 0u;
        if constexpr (F8) VB[i] &= keep;
#pragma unroll
        for (int c = 0; c < WIDE; ++c) V[c][i] &= keep;
        if constexpr (NARROW > 0) VN[i] &= keep;
      }
      if (APART && u.low != u.high) {
        uint32_t bad = 0;
        const auto finite = [&](uint32_t x) __attribute__((always_inline)) {
          const uint32_t y = attend_finite<VT>(x);
          bad |= x ^ y;
          return y;
        };
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (F8)
#pragma unroll
            for (int w = 0; w < VWORDS; ++w) VB[i][w] = finite(VB[i][w]);
#pragma unroll
          for (int c = 0; c < WIDE; ++c)
#pragma unroll
            for (int w = 0; w < 4; ++w) V[c][i][w] = finite(V[c][i][w]);
          if constexpr (NARROW > 0)
#pragma unroll
            for (int w = 0; w < 2; ++w) VN[i][w] = finite(VN[i][w]);
        }
        odd |= __any(bad != 0) != 0;
      }
    }
    if constexpr (F8) {
#pragma unroll
      for (int w = 0; w < VWORDS; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ex_u32x4 f[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = __builtin_amdgcn_perm(VB[2 * j + 1][w], VB[2 * j][w], half ? 0x07030602u : 0x05010400u);
            f[0][j] = f8_widen<TQ_BF16, false>(x, v_scale[j >> 1]);
            f[1][j] = f8_widen<TQ_BF16, true>(x, v_scale[j >> 1]);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int t = w * 4 + half * 2 + k;
#pragma unroll
            for (int n = 0; n < NT; ++n) O[n][t] = ex_mfma<PT>(f[k], P[n], ex_mfma<PT>(f[k], L[n], O[n][t]));
          }
        }
    } else {
#pragma unroll
      for (int c = 0; c < WIDE; ++c) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          ex_u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(V[c][2 * j + 1][t >> 1], V[c][2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int n = 0; n < NT; ++n) O[n][c * 8 + t] = ex_mfma<PT>(f, P[n], ex_mfma<PT>(f, L[n], O[n][c * 8 + t]));
        }
      }
      if constexpr (NARROW > 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          ex_u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(VN[2 * j + 1][t >> 1], VN[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int n = 0; n < NT; ++n) O[n][WIDE * 8 + t] = ex_mfma<PT>(f, P[n], ex_mfma<PT>(f, L[n], O[n][WIDE * 8 + t]));
        }
      }
    }
    if (more) load_values(next);
    now = next;
  }
  if (APART && odd) {
    for (int blk = first + wave; blk < last; blk += 4) {
      entries(ahead, blk);
      find(now, ahead);
      if (now.whole) continue;
      for (int in = 0; in < TB; ++in) {
        const int p = in / TQ_PAGE_TOKENS, t = now.t0 + in;
        if ((in & (TQ_PAGE_TOKENS - 1)) >= (p ? now.valid[1] : now.valid[0])) continue;
        const char* from = (const char*)a.v + (p ? now.at[1] : now.at[0]) + (uint32_t)(in & (TQ_PAGE_TOKENS - 1)) * step;
#pragma unroll
        for (int c = 0; c < TILES; c += 4)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ex_u32x2 x;
            if constexpr (F8) x[0] = x[1] = *(const uint32_t*)(from + (quarter * 4 + i) * TILES + c);
            else x = *(const ex_u32x2*)(from + ex_channel<WIDE>(c, quarter, i) * 2);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if ((t <= at_p[n]) & ((t > behind[n]) | (t < a.sinks)))
#pragma unroll
                for (int k = 0; k < 4; ++k) O[n][c + k][i] += attend_not_finite<VT>(x, k);
          }
      }
    }
  }

  // ---- the four wavefronts: to a common maximum, then summed pairwise (2, 3 -> 0, 1 -> 0) ----
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __align__(16) ex_f32x4 s_acc[2][TILES][64];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n) __syncthreads();
    const float sum_lane = ex_quad_sum(l[n]);
    if (quarter == 0) { s_m[wave][col] = m[n]; s_l[wave][col] = sum_lane; }
    __syncthreads();
    const float M = fmaxf(fmaxf(s_m[0][col], s_m[1][col]), fmaxf(s_m[2][col], s_m[3][col]));
    const float ref = M == -INFINITY ? 0.0f : M;
    const float f = __builtin_amdgcn_exp2f(m[n] - ref);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += s_l[w][col] * __builtin_amdgcn_exp2f(s_m[w][col] - ref);
#pragma unroll
    for (int t = 0; t < TILES; ++t) O[n][t] *= f;
    if (wave >= 2)
#pragma unroll
      for (int t = 0; t < TILES; ++t) s_acc[wave - 2][t][lane] = O[n][t];
    __syncthreads();
    if (wave < 2)
#pragma unroll
      for (int t = 0; t < TILES; ++t) O[n][t] += s_acc[wave][t][lane];
    __syncthreads();
    if (wave == 1)
#pragma unroll
      for (int t = 0; t < TILES; ++t) s_acc[0][t][lane] = O[n][t];
    __syncthreads();
    if (wave == 0 && live[n]) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) O[n][t] += s_acc[0][t][lane];
      const int64_t slot = attend_place(a, u, h, n * 16 + col, row[n]);
      if (share.used > 1 && quarter == 0) a.ml[slot] = make_float2(M - ex_lift<PT>(), sum);
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      float* acc = a.acc + slot * D;
#pragma unroll
      for (int t = 0; t < TILES; t += 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = F8 ? (quarter * 4 + i) * TILES + t : ex_channel<WIDE>(t, quarter, i);      // and the three after it
          const ex_f32x4 x = {O[n][t][i], O[n][t + 1][i], O[n][t + 2][i], O[n][t + 3][i]};
          if (share.used > 1) *(ex_f32x4*)(acc + c) = x;
          else *(ex_u32x2*)((uint16_t*)a.out + row[n] * D + c) = ex_u32x2{ex_pack<QT>(x[0] * inv, x[1] * inv), ex_pack<QT>(x[2] * inv, x[3] * inv)};
        }
    }
  }
}

template <int QT, bool F8>
int launch_attend_few(const Attend& a, int tiles, unsigned grid, hipStream_t stream) {
#define TQ_ATTEND_D(D)                                                                                 \
  case D:                                                                                              \
    if (a.s.starts) {                                                                                  \
      if (tiles == 1) attend_few_kernel<QT, F8, D, 1, true><<<dim3(grid), dim3(256), 0, stream>>>(a);  \
      else attend_few_kernel<QT, F8, D, 2, true><<<dim3(grid), dim3(256), 0, stream>>>(a);             \
    } else {                                                                                           \
      if (tiles == 1) attend_few_kernel<QT, F8, D, 1, false><<<dim3(grid), dim3(256), 0, stream>>>(a); \
      else attend_few_kernel<QT, F8, D, 2, false><<<dim3(grid), dim3(256), 0, stream>>>(a);            \
    }                                                                                                  \
    break
  switch (a.d) {
    TQ_ATTEND_D(64); TQ_ATTEND_D(128); TQ_ATTEND_D(192); TQ_ATTEND_D(256);
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_ATTEND_D
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

}  // namespace tq
