// Decode attention over a paged exact cache for dozens of query heads on a KV head (instantiated by one file per 16-bit type).
//
// The mathematics and the operand layouts are those of tq_exact_impl.h; what differs is who reads.  There a workgroup reads keys and values for
// sixteen heads, straight into registers: with 128 heads on one latent of 576 channels that is eight passes over the cache.  Here a workgroup
// of four wavefronts, one tile of sixteen heads each, shares a block of 32 tokens in LDS: the cache is read once for 64 heads, from memory for the first
// 64 and from the die's cache for the others, which exact_place puts next to each other.
//   * A wavefront owns its heads for the whole range of tokens - scores, softmax, accumulators -, so that nothing is exchanged or joined
//     between wavefronts.  576 channels: 72 registers of queries, 144 of accumulators and a chunk of values twice, one wavefront per SIMD (with two,
//     of eight tiles in a workgroup, 256 registers each were not enough, and the spills' waits drained the loads ahead).
//   * Blocks lie in LDS twice: while one is worked on, the next is filled by LDS-direct loads, which all wavefronts issue in turn.  One barrier per
//     block: behind it everybody's part of this block has arrived and everybody is done with the other.
//   * A row takes one 16-byte piece more than it has: rows then start 16 bytes apart in the banks, and the sixteen rows of a key operand are read
//     without conflicts.
// Bound at 576 channels by what a wavefront issues and its reads of LDS, one wavefront per SIMD: 16 sequences of 8192 tokens, 128 heads, bf16, 114 us for
// 302 MB (2.6 TB/s; as a plain read 56) and 38.7 GFLOP (340 TFLOP/s; as a large product 35 us), the values' half of them done twice (104 us with weights in one number).
// Workgroups of two and eight tiles were slower or no faster (B x heads, bf16, lengths of 8192, weights in one number): 32 x 128 of 256: 175 us with two, 96 with four, 114 with
// eight; 32 x 128 of 128: 109, 57, 57; 32 x 32 of 576, where half of four tiles are empty: 135, 126.
#pragma once

#include <type_traits>

#include "tq_exact_impl.h"

namespace tq {

constexpr int HEADS_TILES = 4;                      // wavefronts of a workgroup, a tile of sixteen heads each

// Where a block's rows lie in LDS, in 16-byte pieces.  Up to 448 channels they follow one another, and a load takes 64 pieces wherever a row ends.  512 and
// 576 channels: a load takes the first 64 pieces of ONE row, whose address is the wavefront's (a scalar and the lane's constant; with divisions by
// the length of a row the loads were 250 of a block's 815 vector instructions), and with 576 another takes the last 8 of eight rows.
// Values of 576 channels are read 64 channels at a time, 16 registers instead of 32 (with 128, 30 of 256 were spilled, and a wait for a spilled
// register is one for the next block): 8 bytes a lane, so that four rows should be half the banks apart.
template <int D>
struct HeadsLds {
  static constexpr bool ROWS = D >= 512;
  static constexpr int WIDE = D / 128;         // chunks of 128 value channels
  static constexpr int PIECES = D / 8;
  static constexpr int KROW = (ROWS ? 64 : PIECES) + 1, VROW = (ROWS ? 64 : PIECES) + (WIDE ? 1 : 2);
  static constexpr int LOADS = ROWS ? 32 + (PIECES > 64 ? 4 : 0) : (32 * VROW + 63) / 64;                  // of a block's keys, or values
  static constexpr int KTAIL = 32 * KROW * 16, VTAIL = 32 * VROW * 16;                                     // bytes before the rows' ends
  static constexpr int KBYTES = ROWS ? KTAIL + (LOADS - 32) * 1024 : LOADS * 1024, VBYTES = ROWS ? VTAIL + (LOADS - 32) * 1024 : LOADS * 1024;
  static constexpr int BYTES = 2 * (KBYTES + VBYTES);
  static_assert(PIECES == 72 || PIECES <= 64, "the ends of eight rows fill a load");
};

// the value, computed where it stands: what is made of it does not stay in registers from one turn to the next
__device__ __forceinline__ int ex_anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int DT, int D>
__global__ void __launch_bounds__(HEADS_TILES * 64, D <= 256 ? 2 : 1) exact_heads_kernel(const ExactDecode a) {
  constexpr int TW = HEADS_TILES;
  using Lds = HeadsLds<D>;
  constexpr int KSTEPS = D / 32, TILES = D / 16, WIDE = Lds::WIDE, NARROW = (D - WIDE * 128) / 64;
  constexpr int KROW = Lds::KROW, VROW = Lds::VROW, LOADS = Lds::LOADS, TURN = Lds::KBYTES + Lds::VBYTES;
  constexpr int DEPTH = D > 256 ? 16 : 8;                    // key operands on their way from LDS
  extern __shared__ __align__(16) unsigned char s_blocks[];  // [2 turns][keys, values]

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int split, group, h, b;
  if (!exact_place(a, &split, &group, &h, &b)) return;
  const int len = exact_len(a.c, b);
  const int blocks = (len + 31) / 32;
  const int per = exact_blocks_per_split(blocks, a.n_split, a.chunk);
  const int first = split * per < blocks ? split * per : blocks, last = first + per < blocks ? first + per : blocks;
  if (first >= last && a.n_split > 1) return;                // (the whole workgroup)

  const int head0 = (group * TW + wave) * EXACT_HEADS;       // of the KV head's G query heads
  const int64_t row0 = (int64_t)b * a.Hq + h * a.G + head0;
  const int32_t* table = a.c.table + b * a.c.table_step;
  const uint32_t step = (uint32_t)a.c.s_t * 2;
  const uint32_t lds0 = (uint32_t)(uintptr_t)s_blocks;

  ex_u32x4 Q[KSTEPS];
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) {
    const int lane = (int)threadIdx.x & 63;
    Q[s] = ex_u32x4{0, 0, 0, 0};
    if (head0 + (lane & 15) < a.G) Q[s] = *(const ex_u32x4*)((const char*)a.q + ((row0 + (lane & 15)) * D) * 2 + s * 64 + (lane >> 4) * 16);
  }
  ex_f32x4 O[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) O[t] = ex_f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  ExactPages<2> now, next;
  const uint32_t head_off = (uint32_t)((int)threadIdx.x & 63) * 16;        // a lane's part of a row
  // This wavefront's loads of a block, NL of them, number u.  (Issued in a row they hold it up for 128 clocks each, 2300 of a block's 7000: they are spread
  // over the block before.)
  constexpr int ROW_LOADS = 64 / TW, END_LOADS = LOADS > 32 ? 8 / TW : 0;
  constexpr int NL = Lds::ROWS ? ROW_LOADS + END_LOADS : (2 * LOADS + TW - 1) / TW;
  const auto fetch = [&](const ExactPages<2>& at, int turn, int u) __attribute__((always_inline)) {
    if constexpr (Lds::ROWS) {
      if (u < ROW_LOADS) {
        // row wave + i TW of a page: keys of both pages, then values
        const int side = u / (ROW_LOADS / 2), p = u / (ROW_LOADS / 4) & 1, i = u % (ROW_LOADS / 4);
        const int row = wave + i * TW, row_bytes = (side ? VROW : KROW) * 16;
        ex_row_to_lds((const char*)(side ? a.c.v : a.c.k) + at.at[p] + (uint64_t)((uint32_t)row * step), head_off,
                      lds0 + (uint32_t)(turn * TURN + (side ? Lds::KBYTES : 0) + (p * 16 + row) * row_bytes));
      } else {
        // the ends of rows r .. r + 7: keys of both pages, then values; a key's pieces change places by its row, for the banks
        const int ln = ex_anew((int)threadIdx.x & 63);
        const int n = (u - ROW_LOADS) * TW + wave, r = (n & 3) * 8;
        const bool value = n >= 4;
        const uint32_t off = (uint32_t)((r & 8) + (ln >> 3)) * step + (64 + (value ? ln & 7 : (ln & 7) ^ (ln >> 3))) * 16;
        const uint32_t to = lds0 + (uint32_t)(turn * TURN + (value ? Lds::KBYTES + Lds::VTAIL : Lds::KTAIL) + r * 128);
        ex_row_to_lds((const char*)(value ? a.c.v : a.c.k) + (r < 16 ? at.at[0] : at.at[1]), off, to);
      }
    } else {
      const int n = u * TW + wave;                           // keys first
      if (2 * LOADS % TW != 0 && n >= 2 * LOADS) return;
      const int ln = ex_anew((int)threadIdx.x & 63);         // (places are computed anew: there are no registers to keep them in)
      const bool value = n >= LOADS;
      const int k = value ? n - LOADS : n, piece = k * 64 + ln;
      int r = value ? piece / VROW : piece / KROW, p = piece - r * (value ? VROW : KROW);
      r = r < 32 ? r : 31;                                   // (what fills the last load up, and the pieces between two rows: of no use, but there)
      p = p < Lds::PIECES ? p : Lds::PIECES - 1;
      const char* from = (const char*)(value ? a.c.v : a.c.k) + (r < 16 ? at.at[0] : at.at[1]) + ((uint32_t)(r & 15) * step + (uint32_t)p * 16);
      ex_to_lds(from, lds0 + (uint32_t)(turn * TURN + (value ? Lds::KBYTES : 0) + k * 1024));
    }
  };
  // table entries are read two blocks ahead, as vector loads behind a block's own: they have arrived with it
  int32_t entry[2] = {-1, -1};
  if (first < last) {
    now.find(a.c, table, len, first, h, 2);
#pragma unroll
    for (int u = 0; u < NL; ++u) fetch(now, 0, u);
    ExactPages<2>::entries(entry, table, len, first + 1);
  }
  const auto block = [&](auto more, int blk, int turn) __attribute__((always_inline)) {
    ex_arrived();
    __syncthreads();
    constexpr bool MORE = decltype(more)::value;
    constexpr int STEPS = 2 * KSTEPS + TILES;                // matrix instructions of a block
    if constexpr (MORE) {
      entry[0] = __builtin_amdgcn_readfirstlane(entry[0]);
      entry[1] = __builtin_amdgcn_readfirstlane(entry[1]);
      next.place(a.c, entry, len, blk + 1, h, 2);
      ExactPages<2>::entries(entry, table, len, blk + 2);
    }
    const auto load_ahead = [&](int g) __attribute__((always_inline)) {        // behind matrix instruction g
      if constexpr (MORE) {
#pragma unroll
        for (int u = 0; u < NL; ++u)
          if (u >= NL * g / STEPS && u < NL * (g + 1) / STEPS) fetch(next, turn ^ 1, u);
      }
    };
    if (!now.whole) {
      // values of tokens without weight are put to zero where they lie, since NaN times nothing is NaN
#pragma unroll 1
      for (int r = 0; r < 32; ++r) {
        if ((r & 15) < (r < 16 ? now.valid[0] : now.valid[1])) continue;
        unsigned char* to = s_blocks + turn * TURN + Lds::KBYTES;
        for (int p = (int)threadIdx.x; p < Lds::PIECES; p += TW * 64)
          *(ex_u32x4*)(to + (p < 64 || !Lds::ROWS ? (r * VROW + p) * 16 : Lds::VTAIL + r * 128 + (p - 64) * 16)) = ex_u32x4{0, 0, 0, 0};
      }
      __syncthreads();
    }
    const int lane = ex_anew((int)threadIdx.x & 63), col = lane & 15, quarter = lane >> 4;
    // (a lane's first key and value piece: all others are constants away)
    const unsigned char* kb = s_blocks + (turn * TURN + (col * KROW + quarter) * 16);
    const unsigned char* vb = s_blocks + (turn * TURN + Lds::KBYTES + quarter * 4 * VROW * 16);
    // ---- scores ----
    const auto key = [&](int p, int s) __attribute__((always_inline)) {
      if (Lds::ROWS && s >= 16)                              // the last eight pieces
        return *(const ex_u32x4*)(s_blocks + turn * TURN + Lds::KTAIL + (p * 16 + col) * 128 + ((((s - 16) * 4 + quarter) ^ (col & 7)) * 16));
      return *(const ex_u32x4*)(kb + (p * 16 * KROW + s * 4) * 16);
    };
    const auto value = [&](int c, int i) __attribute__((always_inline)) {                  // chunk of 128 channels, token
      return *(const ex_u32x4*)(vb + (((i >> 2) * 16 + (i & 3)) * VROW + c * 16) * 16 + col * 16);
    };
    const auto value_end = [&](int i) __attribute__((always_inline)) {                     // the last 64 channels
      const int r = (i >> 2) * 16 + (i & 3);                 // (and quarter * 4)
      if (Lds::ROWS) return *(const ex_u32x2*)(s_blocks + turn * TURN + Lds::KBYTES + Lds::VTAIL + r * 128 + quarter * 512 + col * 8);
      return *(const ex_u32x2*)(vb + (r * VROW + WIDE * 16) * 16 + col * 8);
    };
    // (the compiler would read each operand right before its use and wait for it: the order is held down by the barriers for the scheduler)
    constexpr int N = 2 * KSTEPS, PRE = N < DEPTH ? N : DEPTH;
    ex_f32x4 S[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    ex_u32x4 kf[PRE];
#pragma unroll
    for (int i = 0; i < PRE; ++i) kf[i] = key(i & 1, i >> 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      S[i & 1] = ex_mfma<DT>(kf[i % PRE], Q[i >> 1], S[i & 1]);
      if (i + PRE < N) kf[i % PRE] = key((i + PRE) & 1, (i + PRE) >> 1);
      load_ahead(i);
      if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
    ex_u32x4 x[2][8];
    if constexpr (WIDE > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[0][i] = value(0, i);
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- weights ----
    float top = -INFINITY, pr[2][4];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float s2 = S[p][i] * a.scale2;
        pr[p][i] = now.whole || quarter * 4 + i < now.valid[p] ? s2 : -INFINITY;
        top = fmaxf(top, pr[p][i]);
      }
    if (a.scores && head0 + col < a.G) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int page = blk * 2 + p;
        if (page < a.score_pages)
          *(ex_f32x4*)(a.scores + ((((int64_t)b * a.c.H + h) * a.score_pages + page) * a.G + head0) * TQ_PAGE_TOKENS + (col * TQ_PAGE_TOKENS + quarter * 4)) =
              ex_f32x4{pr[p][0], pr[p][1], pr[p][2], pr[p][3]};
      }
    }
    top = fmaxf(m, ex_quad_max(top));
    if (__any(top > m + EX_SLACK)) {
      const float move = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      l *= move;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        if constexpr (D > 256) asm volatile("" : "+a"(O[t]));  // (they lie in the other half of the registers and would be copied out in every turn)
        O[t] *= move;
      }
      m = top;
    }
    const float ref = m == -INFINITY ? 0.0f : m - ex_lift<DT>();
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[p][i] = __builtin_amdgcn_exp2f(pr[p][i] - ref);
        l += pr[p][i];
      }
    ex_u32x4 P, L;                                           // high and low halves
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t hi, lo;
        ex_split<DT>(pr[p][2 * i], pr[p][2 * i + 1], &hi, &lo);
        P[p * 2 + i] = hi;
        L[p * 2 + i] = lo;
      }
    // ---- values ----
    ex_u32x2 y[8];
#pragma unroll
    for (int c = 0; c < WIDE; ++c) {
      if (c + 1 < WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[(c + 1) & 1][i] = value(c + 1, i);
      } else if constexpr (NARROW > 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = value_end(i);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const ex_u32x4* v = x[c & 1];
        ex_u32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(v[2 * j + 1][t >> 1], v[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
        O[c * 8 + t] = ex_mfma<DT>(f, P, ex_mfma<DT>(f, L, O[c * 8 + t]));
        load_ahead(N + c * 8 + t);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (NARROW > 0) {
      if constexpr (WIDE == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = value_end(i);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        ex_u32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(y[2 * j + 1][t >> 1], y[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
        O[WIDE * 8 + t] = ex_mfma<DT>(f, P, ex_mfma<DT>(f, L, O[WIDE * 8 + t]));
        load_ahead(N + WIDE * 8 + t);
      }
    }
    now = next;
  };
  int turn = 0;
  for (int blk = first; blk + 1 < last; ++blk, turn ^= 1) block(std::true_type{}, blk, turn);
  if (first < last) block(std::false_type{}, last - 1, turn);
  l = ex_quad_sum(l);
  const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  if (head0 + col >= a.G) return;
  exact_store<DT, D, WIDE>(a, O, m - ex_lift<DT>(), l, row0 + col, split, quarter);
}

template <int DT>
int launch_exact_heads(const ExactDecode& a, hipStream_t stream) {
  const dim3 grid((unsigned)exact_grid(a)), block(HEADS_TILES * 64);
#define TQ_HEADS_D(D)                                                                                       \
  case D: {                                                                                                 \
    const auto kern = exact_heads_kernel<DT, D>;                                                            \
    static std::atomic<uint64_t> ready{0};                                                                  \
    if (const int rc = exact_allow_lds((const void*)kern, HeadsLds<D>::BYTES, ready)) return rc;            \
    kern<<<grid, block, HeadsLds<D>::BYTES, stream>>>(a);                                                   \
    break;                                                                                                  \
  }
  switch (a.c.d) {
    TQ_HEADS_D(64) TQ_HEADS_D(128) TQ_HEADS_D(192) TQ_HEADS_D(256) TQ_HEADS_D(320) TQ_HEADS_D(384) TQ_HEADS_D(448) TQ_HEADS_D(512) TQ_HEADS_D(576)
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_HEADS_D
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

}  // namespace tq
