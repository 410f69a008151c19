// Attention of many rows - prompts, chunks of them, dozens of query heads on one KV head - over a paged cache (instantiated by one file per types).
//
// A unit is 128 rows of a KV head: the query heads of a token side by side, tokens one behind another.  A wavefront takes 32 of them, each a column of
// its matrix instructions; the workgroup's keys and values go through LDS, 64 tokens at a time, in 16 bits whatever the cache holds, two buffers in turn:
// the next tokens are on their way while these are worked on - 16 bits straight to LDS (through registers 64 channels take 338 us for 285, 128 509 for 469, 256 1264
// for 1107; two sequences of 8192, 2048 rows, 32 query heads on 8), 8 bits in registers to be converted -, and a turn has one barrier.
//   scores    S^T = K Q^T: tokens are rows.  A lane has 32 of the 64 scores of a row, its neighbour 32 lanes on the others.
//   softmax   one pass, running maximum and sum per row in 32 bits; the reference moves by 2^8 at a time (EX_SLACK).
//   values    O^T = V^T P^T: the contraction takes the tokens in the order in which a lane holds the weights already, so that no weight changes its lane;
//             the transposing LDS read brings values in that order.
// Weights are rounded once, to 16 bits, half a step of 2^-9 (fp16: 2^-12) that a sum over many averages out; a high and a low half, as the kernel of few
// rows has them, would be half as many matrix instructions again.  Numerators and sum are of the same rounded weights, so that what all tokens' values have in common
// comes out as it is (sums of the weights as they were before: 64 channels 288 -> 299 us, 256 1058 -> 1069, 128 and 192 the same).  8 bits for fp16 queries: bf16 values, whose range the block's scale
// needs, and there the weights are two halves: one of bf16 would be eight times coarser than the output.
// Instructions of a wavefront follow one another: those of the vector unit stand between the matrix instructions (weights and values of the next sixteen tokens
// beside the product of these; 256 channels 1541 -> 1331 us), keys are read four ahead, and turns come in pairs, so that buffers are constants in addresses
// (64 channels 354 -> 345 us).
// Bound by both kinds of instructions of two wavefronts on a SIMD (192 and 256 channels: one): a turn of 128 channels is 1024 cycles of matrix instructions and 144 vector ones, 32 of
// them exponentials.  bf16, 128 channels: 481 GFLOP in 460 us, 1.05 PFLOP/s, where a large product of the library reaches 1.40; with a window of 4096, one prompt of 8192, 413 in
// 415; 64 channels 0.81, 192 0.83, 256 0.90 PFLOP/s; 8 bits, 128 channels 1.01 (fp16 queries with their two halves 0.73).  The clock falls as they are busier: with 16 bits straight to LDS a launch takes a fifth
// fewer cycles and a tenth less time.  Eight wavefronts to a workgroup, which would load half as
// often, 460 us, too; two tiles of rows to a wavefront, which would read LDS half as often, 64 channels 274, 128 627 (at one wavefront on a SIMD half of its registers are the
// accumulators', and scores are copied out of them).  Without its reads of LDS a turn of 128 channels would take 0.78 of its time, without its loads 0.87, without exponentials 0.91.
// With 32 tokens a turn and three wavefronts on a SIMD 128 channels take 413 us for 419 with the window and 511 for 467 without (512 workgroups at a time become 768, of 1024); the
// next turn's scores computed ahead of this one's products take 41 - 264 registers more than there are.
// LDS: 16-byte pieces of a row change places by the row (rows_key_turn, rows_value_turn), so that reads do not meet in a bank, and 16 bits on their way in do not either; the stores of
// converted 8 bits do, two to a bank (2.95e7 cycles of 1.18e8 that LDS is busy; see there).
#pragma once

#include "tq_attend.h"
#include "tq_attend_few_impl.h"

#include <type_traits>

namespace tq {

typedef float ro_f32x16 __attribute__((ext_vector_type(16)));
typedef short ro_s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ ro_f32x16 rows_mfma(ex_u32x4 a, ex_u32x4 b, ro_f32x16 c) {
  if constexpr (DT == TQ_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ex_bf16x8, a), __builtin_bit_cast(ex_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ex_f16x8, a), __builtin_bit_cast(ex_f16x8, b), c, 0, 0, 0);
}

// sum + both of two 16-bit numbers (fp16's small ones count)
template <int DT>
__device__ __forceinline__ float rows_add(uint32_t x, float sum) {
  if constexpr (DT == TQ_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, x), b2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
  }
}

constexpr int ROWS_TOKENS = 64;
template <int D> constexpr int rows_lds() { return 2 * 2 * ROWS_TOKENS * D * 2; }

// Where piece c (16 bytes, 8 channels) of a token's row lies.  Rows of 256 and 512 bytes begin in the same bank, of 128 and 384 in one of two.
// Keys: 16 lanes read the same piece of 16 rows.  Values: 16 lanes read 32 bytes of 4 rows, the 16 beside them the next 32.
template <int D> __device__ __forceinline__ int rows_key_turn(int t) { return D % 128 == 0 ? (t & 15) : ((t >> 1) & 7); }
template <int D> __device__ __forceinline__ int rows_value_turn(int t) { return D % 128 == 0 ? (t & 3) << 2 : ((t >> 1) & 1) << 2; }

// HALVES: weights go into the product as a high and a low half
template <int QT, bool F8, int D, bool HALVES>
__global__ void __launch_bounds__(256, (D <= 128 ? 2 : 1)) attend_rows_kernel(const Attend a) {
  constexpr int PT = F8 ? TQ_BF16 : QT;                      // of the value product
  constexpr bool FOLD = F8 && QT == TQ_BF16;                 // a key's scale goes into the key
  constexpr int VT = F8 ? TQ_E4M3 : QT;                      // of the cache
  constexpr int SIZE = F8 ? 1 : 2, ROW = D * 2;              // bytes of an element in the cache, of a row in LDS
  constexpr int LANES = D * SIZE / 16, LOADS = ROWS_TOKENS * LANES / 256;
  constexpr int KSTEPS = D / 16, TILES = D / 32, M = 128;
  constexpr int KAHEAD = 4;                                  // reads of keys that are on their way at a time
  constexpr int HALF = ROWS_TOKENS * ROW;                    // keys or values of a turn
  extern __shared__ __attribute__((aligned(16))) char s_rows[];

  const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 31, half = lane >> 5;
  // (the last units of a sequence have the most tokens: they begin first)
  // (units of a KV head follow one another on a die, whose L2 has its blocks: with two heads that share lines on each, as few rows have them, 8 bits of 64 channels 320 -> 345 us,
  // of 192 1031 -> 1228)
  const unsigned turn_of = blockIdx.x / (unsigned)a.H;
  const int h = (int)(blockIdx.x - turn_of * (unsigned)a.H);
  const int item = a.items - 1 - (int)turn_of;
  AttendUnit u;
  int over, others;
  if (!attend_item<M, ROWS_TOKENS>(a, item, &u, &over, &others)) {
    attend_rest<D>(a, h, over, others);
    return;
  }
  const AttendBlocks<ROWS_TOKENS> list(a, u);
  const AttendShare share(a, u, list.count);
  if (u.split >= share.used) return;
  const int first = share.first, last = share.last;

  // this lane's row
  const int r = wave * 32 + col, x = u.first + (r < u.rows ? r : 0), token = x / a.G;
  const bool live = r < u.rows;
  const int64_t row = (u.row + token) * a.Hq + h * a.G + (x - token * a.G);
  const int at_p = u.low + (token - u.first / a.G), behind = attend_behind(a, at_p);
  if (a.shares && u.split == 0 && half == 0 && live) a.shares[row] = attend_told(a, u, h, r, share.used);
  // the wavefront's first and last positions
  const int r0 = wave * 32, r1 = r0 + 31;
  const bool busy = r0 < u.rows;
  const int w_low = u.low + (u.first + r0) / a.G - u.first / a.G, w_high = u.low + (u.first + (r1 < u.rows ? r1 : u.rows - 1)) / a.G - u.first / a.G;
  const int w_behind_low = attend_behind(a, w_low), w_behind_high = attend_behind(a, w_high);
  const int32_t* table = a.s.table + u.b * a.s.table_step;

  // (a negative scale turns the queries and one of zero clears them, so that the scores' order is that of their products)
  const float f = a.scale2 == 0.0f ? 1.0f : fabsf(a.scale2);
  const uint32_t sign = a.scale2 < 0.0f ? 0x80008000u : 0u, keep = a.scale2 == 0.0f ? 0u : 0xffffffffu;
  ex_u32x4 Q[KSTEPS];
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) {
    Q[s] = ex_u32x4{0, 0, 0, 0};
    if (live) Q[s] = *(const ex_u32x4*)((const uint16_t*)a.q + row * D + s * 16 + half * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) Q[s][i] = (Q[s][i] & keep) ^ sign;
  }
  ro_f32x16 O[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[t][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  // ---- a turn's tokens: table entries, loads into registers, registers into LDS ----
  const int last_page = u.tokens > 0 ? (u.tokens - 1) / TQ_PAGE_TOKENS : 0;
  struct Turn {
    ex_u32x4 entry;                                          // (an array would be memory where a wavefront picks one of them)
    int t0;
  };
  const auto entries = [&](Turn& x, int i) __attribute__((always_inline)) {
    const int at = i < last ? i : last - 1, blk = list[at < 0 ? 0 : at];      // (a unit without tokens: block 0, of which nothing is used)
    x.t0 = blk * ROWS_TOKENS;
    if (blk * 4 + 3 <= last_page) {
      x.entry = step_entries(table, blk * 4);
    } else {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int page = blk * 4 + p;
        x.entry[p] = (uint32_t)step_entry(table, page < last_page ? page : last_page);
      }
    }
  };
  // (scalar instructions are a wavefront's time as well: 64-bit products for each load were a fifth of it)
  const uint32_t in_cache = a.s.num_blocks < 0x80000000ll ? (uint32_t)a.s.num_blocks : 0x80000000u;
  const uint64_t block_bytes = (uint64_t)a.s_blk * SIZE, head_bytes = (uint64_t)h * a.s_h * SIZE;
  const uint32_t step = (uint32_t)a.s_t * SIZE;
  // all of a turn's tokens are the sequence's, in blocks of the cache
  const auto complete = [&](const Turn& x) __attribute__((always_inline)) {
    const uint32_t p = x.entry[0] > x.entry[1] ? x.entry[0] : x.entry[1], q = x.entry[2] > x.entry[3] ? x.entry[2] : x.entry[3];
    return x.t0 + ROWS_TOKENS <= u.tokens && (p > q ? p : q) < in_cache;
  };
  // The i-th load of a lane: 16 bytes of token token_of of the turn.  16 bits: they go to LDS directly, a wavefront's 1 KB to 1 KB of it, and a lane reads
  // the piece that belongs where its bytes land; a wavefront's tokens are one page's.  Lanes' places in a page repeat with every load, with 512 bytes a row every
  // two and with 192 channels every three.
  // 8 bits go through registers: rows of a power of two of pieces have one place in all pages, with 192 channels lanes work it out load by load.
  constexpr bool EVEN = D != 192;
  constexpr int APART = 256 / LANES, PER = F8 ? 2 : 1;       // tokens from a load to the next; pieces of 8 channels in one
  const auto token_of = [&](int i) __attribute__((always_inline)) { return EVEN ? tid / LANES + i * APART : (i * 256 + tid) / LANES; };
  const auto piece_of = [&](int i) __attribute__((always_inline)) { return EVEN ? tid % LANES : (i * 256 + tid) % LANES; };
  const auto entry_of = [&](const Turn& x, int i) __attribute__((always_inline)) {
    if constexpr (EVEN) {
      constexpr int OWN = 64 / LANES;                        // tokens of a wavefront's load
      if constexpr (OWN < 8) return x.entry[i * APART / 16];
      else if constexpr (OWN < 16) return wave < 2 ? x.entry[i * APART / 16] : x.entry[i * APART / 16 + 1];
      else return wave < 2 ? (wave < 1 ? x.entry[0] : x.entry[1]) : (wave < 3 ? x.entry[2] : x.entry[3]);
    } else {
      const int p = F8 ? token_of(i) >> 4 : (i * 4 + wave) / 6;
      return p < 2 ? (p < 1 ? x.entry[0] : x.entry[1]) : (p < 3 ? x.entry[2] : x.entry[3]);
    }
  };
  // 16 bits
  constexpr int PLACES = D == 192 ? 3 : (D == 256 ? 2 : 1);
  uint32_t key_at[PLACES], value_at[PLACES];
  const uint32_t lds0 = (uint32_t)(uintptr_t)s_rows;
  // 8 bits
  constexpr int HELD = F8 ? LOADS : 1;
  ex_u32x4 KR[HELD], VR[HELD];
  uint32_t ks[HELD], vs[HELD];
  uint32_t next_g[4];                                        // fp16 queries: the scales of the next turn's keys, and of these
  float g[4];
  const uint32_t here = EVEN ? (uint32_t)(tid / LANES % 16) * step + (uint32_t)(tid % LANES) * 16 : 0;
  if constexpr (!F8) {
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int t = (i * 256 + tid) / LANES, piece = (i * 256 + tid) % LANES;
      key_at[i] = (uint32_t)(t & 15) * step + (uint32_t)(piece ^ rows_key_turn<D>(t)) * 16;
      value_at[i] = (uint32_t)(t & 15) * step + (uint32_t)(piece ^ rows_value_turn<D>(t)) * 16;
    }
  }
  const auto load = [&](const Turn& x, uint32_t to) __attribute__((always_inline)) {
    if constexpr (F8 && !FOLD)
#pragma unroll
      for (int p = 0; p < 4; ++p) next_g[p] = a.k_scales[(uint64_t)(x.entry[p] < in_cache ? x.entry[p] : 0u) * a.H + h];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t e = entry_of(x, i), page = e < in_cache ? e : 0u;      // (a block that is there; its tokens are masked)
      const uint64_t block = page * block_bytes + head_bytes;
      if constexpr (F8) {
        uint32_t at = here + (APART < 16 ? (uint32_t)(i * APART % 16) * step : 0u);
        if constexpr (!EVEN) at = (uint32_t)(token_of(i) & 15) * step + (uint32_t)piece_of(i) * 16;
        KR[i] = *(const ex_u32x4*)((const char*)a.k + block + at);
        VR[i] = *(const ex_u32x4*)((const char*)a.v + block + at);
        ks[i] = a.k_scales[(uint64_t)page * a.H + h];
        vs[i] = a.v_scales[(uint64_t)page * a.H + h];
      } else {
        const uint32_t m0 = lds0 + to + (uint32_t)(i * 256 + wave * 64) * 16;
        ex_row_to_lds((const char*)a.k + block, key_at[i % PLACES], m0);
        ex_row_to_lds((const char*)a.v + block, value_at[i % PLACES], m0 + HALF);
      }
    }
  };
  const int t_here = tid / LANES, c_here = tid % LANES * PER;
  const uint32_t key_to = (uint32_t)(t_here * ROW + (c_here ^ rows_key_turn<D>(t_here)) * 16), value_to = (uint32_t)(t_here * ROW + (c_here ^ rows_value_turn<D>(t_here)) * 16);
  // all rows of the unit see all of a turn's tokens
  const int behind_low = attend_behind(a, u.low), behind_high = attend_behind(a, u.high);
  const auto seen_whole = [&](const Turn& x) __attribute__((always_inline)) {
    return x.t0 + ROWS_TOKENS - 1 <= u.low && (x.t0 > behind_high || x.t0 + ROWS_TOKENS <= a.sinks) && complete(x);
  };
  bool odd = false;                                          // this wavefront has put values that are not finite to zero
  // where all rows do not: values of tokens that nobody sees are zeros - what lies in their slots may be NaN -, and so are those that are not finite
  const auto sanitise = [&](const Turn& x, int i, ex_u32x4 v) __attribute__((always_inline)) {
    const int t = x.t0 + token_of(i);
    if (!((t < u.tokens) & (entry_of(x, i) < in_cache) & ((t > behind_low) | (t < a.sinks)))) v = ex_u32x4{0, 0, 0, 0};
    if (u.low != u.high) {
      ex_u32x4 y;
#pragma unroll
      for (int w = 0; w < 4; ++w) y[w] = attend_finite<VT>(v[w]);
      odd |= __any(((y[0] ^ v[0]) | (y[1] ^ v[1]) | (y[2] ^ v[2]) | (y[3] ^ v[3])) != 0) != 0;
      v = y;
    }
    return v;
  };
  const auto store = [&](int i, bool whole, char* to) __attribute__((always_inline)) {
    if constexpr (!F8) {
      ex_arrived();
      if (!whole) {
        Turn x;
        entries(x, i);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          ex_u32x4* const v = (ex_u32x4*)(to + HALF + (i * 256 + tid) * 16);
          *v = sanitise(x, i, *v);
        }
      }
    } else {
      if (!whole) {
        Turn x;
        entries(x, i);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) VR[i] = sanitise(x, i, VR[i]);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        uint32_t k = (key_to ^ (uint32_t)(rows_key_turn<D>(i * APART) * 16)) + (uint32_t)(i * APART * ROW), v = value_to + (uint32_t)(i * APART * ROW);
        if constexpr (!EVEN) {
          const int t = token_of(i), c = piece_of(i) * PER;
          k = (uint32_t)(t * ROW + (c ^ rows_key_turn<D>(t)) * 16);
          v = (uint32_t)(t * ROW + (c ^ rows_value_turn<D>(t)) * 16);
        }
        char *const kt = to, *const vt = to + HALF;
        const float kf = FOLD ? f8_scale(ks[i]) : 1.0f, vf = f8_scale(vs[i]);
        // (eight lanes store together, every second piece of 256 bytes, so that half of the banks have two: to have four of the lanes begin with the other
        // piece leaves no conflict and takes longer, 536 us for 522)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ex_u32x4 y, z;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            y[w * 2] = f8_widen<QT, false>(KR[i][j * 2 + w], kf);
            y[w * 2 + 1] = f8_widen<QT, true>(KR[i][j * 2 + w], kf);
            z[w * 2] = f8_widen<TQ_BF16, false>(VR[i][j * 2 + w], vf);
            z[w * 2 + 1] = f8_widen<TQ_BF16, true>(VR[i][j * 2 + w], vf);
          }
          *(ex_u32x4*)(kt + (k ^ (uint32_t)(j * 16))) = y;
          *(ex_u32x4*)(vt + (v ^ (uint32_t)(j * 16))) = z;
        }
      }
    }
  };
  // ---- a lane's places in LDS: the other steps and tiles lie where a few of the place's bits differ ----
  const int j16 = lane & 15;
  const uint32_t key_from = (uint32_t)(col * ROW + (half ^ rows_key_turn<D>(col)) * 16);
  const uint32_t value_from = (uint32_t)(HALF + (half * 4 + (j16 >> 2)) * ROW + ((D % 128 == 0 ? j16 >> 2 : j16 >> 3) * 4 + ((lane >> 4) & 1) * 2 + ((j16 & 3) >> 1)) * 16 + (j16 & 1) * 8);
  constexpr int KPLACES = D % 128 == 0 ? 8 : 4, VPLACES = D % 128 == 0 ? 4 : 2;
  uint32_t kp[KPLACES], vp[VPLACES];
#pragma unroll
  for (int s = 0; s < KPLACES; ++s) kp[s] = key_from ^ (uint32_t)(s * 32);
#pragma unroll
  for (int t = 0; t < VPLACES; ++t) vp[t] = value_from ^ (uint32_t)(t * 64);

  Turn ahead;                                                // table entries of the turn behind the one that is worked on
  entries(ahead, first);
  int t0 = ahead.t0;
  bool whole = seen_whole(ahead);
  if (first < last) {
    load(ahead, 0);
    store(first, whole, s_rows);
    if constexpr (F8 && !FOLD)
#pragma unroll
      for (int p = 0; p < 4; ++p) g[p] = f8_scale(next_g[p]);
  }
  entries(ahead, first + 1);
  __syncthreads();
  // A wavefront that is further in its turn goes first: 64 channels 292 -> 275 us, 128 476 -> 460, 256 1106 -> 1098, 8 bits 128 508 -> 490; but 64 channels of 8 bits, whose
  // turn is conversions for the most part, 327 -> 360.
  const auto priority = [](auto p) __attribute__((always_inline)) {
    if constexpr (!F8 || D > 64) __builtin_amdgcn_s_setprio(decltype(p)::value);
  };
  const auto turn = [&](int i, auto which) __attribute__((always_inline)) {
    char* const buffer = s_rows + decltype(which)::value * 2 * HALF;
    char* const other = s_rows + (decltype(which)::value ^ 1) * 2 * HALF;
    const bool more = i + 1 < last;
    // (first of all, since scalar loads and reads of LDS have one counter: the keys would wait for them)
    Turn after;
    entries(after, i + 2);
    if (more) load(ahead, (decltype(which)::value ^ 1) * 2 * HALF);
    const int next_t0 = ahead.t0;
    const bool next_whole = seen_whole(ahead);
    ahead = after;
    // what this wavefront's rows see of the turn: nothing, all of it, or some
    const int t1 = t0 + ROWS_TOKENS - 1;
    const bool any = busy && t0 <= w_high && (t1 > w_behind_low || t0 < a.sinks);
    if (any) {
      bool clear = whole;
      if (!whole && t1 <= w_low && (t0 > w_behind_high || t1 < a.sinks)) {
        Turn now;
        entries(now, i);
        clear = complete(now);
      }
      priority(std::integral_constant<int, 1>());
      ro_f32x16 S[2];
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int e = 0; e < 16; ++e) S[T][e] = 0.0f;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
        for (int T = 0; T < 2; ++T)
          S[T] = rows_mfma<QT>(*(const ex_u32x4*)(buffer + kp[s % KPLACES] + (s / KPLACES) * KPLACES * 32 + T * 32 * ROW), Q[s], S[T]);
      __builtin_amdgcn_sched_group_barrier(0x100, KAHEAD, 0);
#pragma unroll
      for (int i = 0; i < 2 * KSTEPS - KAHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, KAHEAD, 0);
      ex_u32x4 V[2][TILES];
      const auto values = [&](int at) __attribute__((always_inline)) {
#pragma unroll
        for (int ct = 0; ct < TILES; ++ct) {
          char* from = buffer + vp[ct % VPLACES] + (ct / VPLACES) * VPLACES * 64 + at * 16 * ROW;
          typedef __attribute__((address_space(3))) ro_s16x4* lds4;
          const ro_s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)from);
          const ro_s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(from + 8 * ROW));
          const ex_u32x2 lo = __builtin_bit_cast(ex_u32x2, x), hi = __builtin_bit_cast(ex_u32x2, y);
          V[at & 1][ct] = ex_u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      };
      values(0);
      if constexpr (F8 && !FOLD)
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int e = 0; e < 8; ++e) S[p >> 1][(p & 1) * 8 + e] *= g[p];
      if (!clear) {
        Turn now;
        entries(now, i);
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int t = t0 + T * 32 + (e >> 2) * 8 + half * 4 + (e & 3);
            const bool seen = (t <= at_p) & (t < u.tokens) & ((t > behind) | (t < a.sinks)) & (now.entry[T * 2 + (e >> 3)] < in_cache);
            S[T][e] = seen ? S[T][e] : -INFINITY;
          }
      }
      priority(std::integral_constant<int, 2>());
      float top = -INFINITY;
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, S[T][e]);
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(m, fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * f);
      if (__any(top > m + EX_SLACK)) {
        const float move = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        l *= move;
#pragma unroll
        for (int t = 0; t < TILES; ++t) O[t] *= move;
        m = top;
      }
      const float ref = m == -INFINITY ? 0.0f : m - ex_lift<PT>();
      // Sixteen tokens at a time: the weights and values of the next while the matrix instructions of these run.
      ex_u32x4 P[2], L[2];
      const auto weights = [&](int at) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float x = __builtin_amdgcn_exp2f(fmaf(S[at >> 1][(at & 1) * 8 + i], f, -ref)), y = __builtin_amdgcn_exp2f(fmaf(S[at >> 1][(at & 1) * 8 + i + 1], f, -ref));
          if constexpr (HALVES) {
            l += x;
            l += y;
            uint32_t hi, lo;
            ex_split<PT>(x, y, &hi, &lo);
            P[at & 1][i >> 1] = hi;
            L[at & 1][i >> 1] = lo;
          } else {
            P[at & 1][i >> 1] = ex_pack<PT>(x, y);
          }
        }
      };
      weights(0);
      priority(std::integral_constant<int, 3>());
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int at = 0; at < 4; ++at) {
        if (at < 3) {
          values(at + 1);
          weights(at + 1);
        }
        if constexpr (!HALVES)                               // (behind the next weights: right behind their own rounding 256 channels take 1081 us for 1069)
#pragma unroll
          for (int i = 0; i < 4; ++i) l = rows_add<PT>(P[at & 1][i], l);
#pragma unroll
        for (int ct = 0; ct < TILES; ++ct) {
          if constexpr (HALVES) O[ct] = rows_mfma<PT>(V[at & 1][ct], L[at & 1], O[ct]);
          O[ct] = rows_mfma<PT>(V[at & 1][ct], P[at & 1], O[ct]);
        }
        if (at < 3) {
#pragma unroll
          for (int ct = 0; ct < TILES; ++ct) {
            __builtin_amdgcn_sched_group_barrier(0x008, HALVES ? 2 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, ((HALVES ? 28 : 20) + TILES - 1) / TILES, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    priority(std::integral_constant<int, 0>());
    if (more) store(i + 1, next_whole, other);
    if constexpr (F8 && !FOLD)
#pragma unroll
      for (int p = 0; p < 4; ++p) g[p] = f8_scale(next_g[p]);
    __syncthreads();
    t0 = next_t0;
    whole = next_whole;
  };
  for (int i = first; i < last; i += 2) {
    turn(i, std::integral_constant<int, 0>());
    if (i + 1 < last) turn(i + 1, std::integral_constant<int, 1>());
  }
  if (u.low != u.high) {                                     // (all that remains of the buffers: whether any wavefront has)
    if (tid == 0) *(uint32_t*)s_rows = 0;
    __syncthreads();
    if (odd) *(uint32_t*)s_rows = 1;
    __syncthreads();
    if (*(const uint32_t*)s_rows) {
      for (int i = first; i < last; ++i) {
        Turn now;
        entries(now, i);
        if (seen_whole(now)) continue;
        for (int in = 0; in < ROWS_TOKENS && now.t0 + in < u.tokens; ++in) {
          const int t = now.t0 + in;
          const uint32_t page = (uint32_t)step_entry(table, t / TQ_PAGE_TOKENS);
          if (page >= in_cache) continue;
          const char* from = (const char*)a.v + page * block_bytes + head_bytes + (uint32_t)(in % TQ_PAGE_TOKENS) * step;
          const bool sees = (t <= at_p) & ((t > behind) | (t < a.sinks));
#pragma unroll
          for (int c = 0; c < TILES; ++c)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const int at = (c * 32 + (e >> 2) * 8 + half * 4) * SIZE;
              ex_u32x2 x;
              if constexpr (F8) x[0] = x[1] = *(const uint32_t*)(from + at);
              else x = *(const ex_u32x2*)(from + at);
              if (sees)
#pragma unroll
                for (int k = 0; k < 4; ++k) O[c][e + k] += attend_not_finite<VT>(x, k);
            }
        }
      }
    }
  }

  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  const float sum = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  if (!live) return;
  const int64_t slot = attend_place(a, u, h, r, row);
  if (share.used > 1 && half == 0) a.ml[slot] = make_float2(m - ex_lift<PT>(), sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  float* acc = a.acc + slot * D;
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int c = t * 32 + (e >> 2) * 8 + half * 4;         // and the three after it
      const ex_f32x4 y = {O[t][e], O[t][e + 1], O[t][e + 2], O[t][e + 3]};
      if (share.used > 1) *(ex_f32x4*)(acc + c) = y;
      else *(ex_u32x2*)((uint16_t*)a.out + row * D + c) = ex_u32x2{ex_pack<QT>(y[0] * inv, y[1] * inv), ex_pack<QT>(y[2] * inv, y[3] * inv)};
    }
}

template <int QT, bool F8, int D, bool HALVES>
int launch_attend_rows_h(const Attend& a, unsigned grid, hipStream_t stream) {
  static std::atomic<uint64_t> ready{0};
  if (const int rc = exact_allow_lds((const void*)attend_rows_kernel<QT, F8, D, HALVES>, rows_lds<D>(), ready)) return rc;
  attend_rows_kernel<QT, F8, D, HALVES><<<dim3(grid), dim3(256), rows_lds<D>(), stream>>>(a);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
// Two halves for fp16 queries over 8 bits, and for a decode step's, so that its results are as good with dozens of heads on one as with a few (bf16, 32 sequences of 8192, 64 heads on one of
// 128 33.1 -> 34.6 us, 128 heads 43.7 -> 52.1; 16 of 8192, 128 on 2 of 256 59.8 -> 70.3).
template <int QT, bool F8, int D>
int launch_attend_rows_d(const Attend& a, unsigned grid, hipStream_t stream) {
  if ((F8 && QT == TQ_F16) || !a.s.starts) return launch_attend_rows_h<QT, F8, D, true>(a, grid, stream);
  return launch_attend_rows_h<QT, F8, D, F8 && QT == TQ_F16>(a, grid, stream);
}

template <int QT, bool F8>
int launch_attend_rows(const Attend& a, unsigned grid, hipStream_t stream) {
  switch (a.d) {
    case 64: return launch_attend_rows_d<QT, F8, 64>(a, grid, stream);
    case 128: return launch_attend_rows_d<QT, F8, 128>(a, grid, stream);
    case 192: return launch_attend_rows_d<QT, F8, 192>(a, grid, stream);
    case 256: return launch_attend_rows_d<QT, F8, 256>(a, grid, stream);
    default: return TQ_EUNSUPPORTED;
  }
}

}  // namespace tq
