// The page-streaming kernel of decode attention over a paged exact cache (instantiated by one file per element type).
//
//   s[t] = scale q . k_t     out = sum_t exp(s[t] - m) v_t / sum_t exp(s[t] - m)     for the G query heads of a KV head at once
//
// A wavefront takes 32 tokens (fp32: 16) at a time, straight from memory into the operands of its matrix instructions - no shared memory, no
// barrier in the loop:
//   scores    tokens are rows, heads columns: a lane reads 16 bytes of the key of ONE token, which is its part of the row operand as it lies;
//             the queries stay in registers as the column operand.  A lane gets scores of one head: four tokens of each sixteen.
//   values    channels are rows, heads columns, tokens the contraction, in the order in which the lane holds the weights already: no weight
//             changes its lane.  A lane reads 8 neighbouring channels (4 in the last 64 of an odd multiple of 64) of each of
//             its 8 tokens - sixteen lanes a whole row - and turns the 8 x 8 block of halves around in registers (32 byte
//             permutes a block of 128 channels); row r of channel tile t is channel 8 r + t, so the tiles need no exchange between lanes.
//             fp32: a lane's four channels of a token are the row operands of four instructions as they are.
//   softmax   one pass: running maximum and sum per head; a lane's accumulators all belong to its head, so a move of the maximum is a
//             scalar of the lane.  Maximum, sum, scores and numerators are fp32.  The matrix instruction takes 16-bit weights: they go in as two
//             numbers, a high and a low half (ex_split), so that what is rounded away is 2^-15 (fp16: 2^-21) of a weight
//             (rounded once, 2^-8 and 2^-11, outputs were a third and a fifth further from 64 bits than fp32 weights' are).  Twice the products of
//             the values: nothing that shows at sixteen heads, 8 us of 114 with 128 heads on one of 576 channels.
// Bound by the memory system.  bf16, 16 sequences of 8192, 32 query on 8 KV heads of 128: 117 us for 546 MB, 4.7 TB/s where a large read reaches 5.4; one of
// 131072, 16 on 2 heads of 256: 62 us, 4.4 TB/s; fp16, 96 of 61 .. 8190, 40 on 8 heads of 128: 145 - 155 us, 4.4 - 4.7 TB/s, the rest the ends of short
// sequences; fp32, 8 of 1500 .. 2048, 16 heads of 64: 28 us, 4.2 TB/s.  One of 700 tokens: 5.4 us, a launch and four latencies one behind another (length,
// table entry, keys and values, the join of the four wavefronts).
// Registers before LDS: with the next block's keys and values on their way in registers a wavefront needs no barrier; with table entries read behind
// a condition the compiler waited for them at once, and with them for the block on its way.
// Tokens behind the length and those of a block number outside the cache have no weight; what lies in their slots is not used in any
// product, so that NaN left there stays there.
#pragma once

#include "tq_exact.h"

namespace tq {

// lane l's 16 bytes land at m0 + 16 l.  The compiler sees neither the load nor its write to LDS: ex_arrived() waits for it.
__device__ __forceinline__ void ex_to_lds(const void* from, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(from), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void ex_row_to_lds(const void* base, uint32_t off, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void ex_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

typedef float ex_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t ex_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t ex_u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 ex_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 ex_f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ ex_f32x4 ex_mfma(ex_u32x4 a, ex_u32x4 b, ex_f32x4 c) {
  static_assert(DT == TQ_BF16 || DT == TQ_F16, "16-bit elements");
  if constexpr (DT == TQ_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ex_bf16x8, a), __builtin_bit_cast(ex_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ex_f16x8, a), __builtin_bit_cast(ex_f16x8, b), c, 0, 0, 0);
}

// two weights to the cache's type, nearest even
template <int DT>
__device__ __forceinline__ uint32_t ex_pack(float lo, float hi) {
  if constexpr (DT == TQ_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 r = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, r);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 r = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, r);
  }
}

// Two weights as the sum of two numbers each of the cache's type.  The high one is cut, never rounded up, and always less than the weight, so that the low one
// is positive where the weight is: with a low part of zero, or one below zero, an infinite value would give NaN (0 x inf, inf - inf) where it has to give
// infinity.  fp16: less by 2^-24 at least, below which a low part would be rounded to nothing; a weight below 2^-25 is nothing in either half, 2^-31 of the
// largest and less.
template <int DT>
__device__ __forceinline__ void ex_split(float a, float b, uint32_t* hi, uint32_t* lo) {
  if constexpr (DT == TQ_BF16) {
    const uint32_t ua = __builtin_elementwise_sub_sat(__float_as_uint(a), 1u), ub = __builtin_elementwise_sub_sat(__float_as_uint(b), 1u);
    *hi = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    *lo = ex_pack<DT>(a - __uint_as_float(ua & 0xffff0000u), b - __uint_as_float(ub & 0xffff0000u));
  } else {
    constexpr float LESS = 1.0f - 0x1p-22f;
    const auto h = __builtin_amdgcn_cvt_pkrtz(fmaxf(fmaf(a, LESS, -0x1p-24f), 0.0f), fmaxf(fmaf(b, LESS, -0x1p-24f), 0.0f));
    *hi = __builtin_bit_cast(uint32_t, h);
    *lo = ex_pack<DT>(a - (float)h[0], b - (float)h[1]);
  }
}

// maximum / sum over the four lanes that hold a head (16 lanes apart)
__device__ __forceinline__ float ex_quad_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float ex_quad_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The reference of the powers of two moves up when a head's maximum has passed it by more than 2^EX_SLACK, not with every new maximum: accumulators
// are multiplied seldom, and weights are up to 2^EX_SLACK large.  fp16 weights are multiplied by 2^6 besides, which keeps the largest
// under fp16's 2^16: without it a long context's many small ones would round to nothing.
constexpr float EX_SLACK = 8.0f;
template <int DT> __device__ __forceinline__ constexpr float ex_lift() { return DT == TQ_F16 ? 6.0f : 0.0f; }

// Channel of accumulator element i (0..3) of channel tile `tile` in a lane of quarter `quarter`: WIDE chunks of 128 channels, whose tiles'
// rows are 8 channels apart, then chunks of 64, 4 apart.
template <int WIDE>
__device__ __forceinline__ int ex_channel(int tile, int quarter, int i) {
  if (tile < WIDE * 8) return (tile >> 3) * 128 + (quarter * 4 + i) * 8 + (tile & 7);
  const int t = tile - WIDE * 8;
  return WIDE * 128 + (t >> 2) * 64 + (quarter * 4 + i) * 4 + (t & 3);
}
template <int DT, int D> constexpr int ex_wide() { return DT == TQ_F32 ? 0 : D / 128; }

// A wavefront's accumulators of one head: the output, or the split's numerators with its maximum and sum.  The tiles of a chunk hold
// neighbouring channels, so that a lane writes 16 bytes at a time.
template <int DT, int D, int WIDE = ex_wide<DT, D>()>
__device__ __forceinline__ void exact_store(const ExactDecode& a, const ex_f32x4* O, float top, float sum, int64_t row, int split, int quarter) {
  if (quarter == 0) a.ml[row * a.n_split + split] = make_float2(top, sum);
  const bool one = a.n_split == 1;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  float* acc = a.acc + (row * a.n_split + split) * D;
#pragma unroll
  for (int t = 0; t < D / 16; t += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = ex_channel<WIDE>(t, quarter, i);         // and the three after it
      const ex_f32x4 x = {O[t][i], O[t + 1][i], O[t + 2][i], O[t + 3][i]};
      if (!one) {
        *(ex_f32x4*)(acc + c) = x;
      } else if constexpr (DT == TQ_F32) {
        *(ex_f32x4*)((float*)a.out + row * D + c) = x * inv;
      } else {
        *(ex_u32x2*)((uint16_t*)a.out + row * D + c) = ex_u32x2{ex_pack<DT>(x[0] * inv, x[1] * inv), ex_pack<DT>(x[2] * inv, x[3] * inv)};
      }
    }
}

template <int DT, int D>
constexpr int exact_waves_per_simd() { return D <= 64 ? 4 : (D <= 128 ? 3 : (D <= 256 ? 2 : 1)); }

// A block's pages: where they lie, and how many of their tokens count (none of a page behind the sequence or outside the cache: its loads
// go to block 0, which is there, and what they bring is masked)
template <int PAGES>
struct ExactPages {
  int64_t at[PAGES];                                         // byte offset of the KV head's first row
  int valid[PAGES];
  bool whole;
  __device__ __forceinline__ void find(const ExactCache& c, const int32_t* table, int len, int blk, int h, int size) {
    int32_t entry[PAGES];
    entries(entry, table, len, blk);
    place(c, entry, len, blk, h, size);
  }
  // (no condition around the loads: behind one they would be waited for at once.  Pages behind the sequence have its last entry, and no tokens.)
  static __device__ __forceinline__ void entries(int32_t* entry, const int32_t* table, int len, int blk) {
    const int last = len > 0 ? (len - 1) / TQ_PAGE_TOKENS : 0;
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      const int page = blk * PAGES + p;
      entry[p] = table[page < last ? page : last];
    }
  }
  __device__ __forceinline__ void place(const ExactCache& c, const int32_t* entry, int len, int blk, int h, int size) {
    whole = true;
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      const int left = len - (blk * PAGES + p) * TQ_PAGE_TOKENS;
      valid[p] = left < 0 ? 0 : (left > TQ_PAGE_TOKENS ? TQ_PAGE_TOKENS : left);
      int64_t page = entry[p];
      if (page < 0 || page >= c.num_blocks) { page = 0; valid[p] = 0; }
      whole &= valid[p] == TQ_PAGE_TOKENS;
      at[p] = (page * c.s_blk + h * c.s_h) * size;
    }
  }
};

template <int DT, int D>
__global__ void __launch_bounds__(256, (exact_waves_per_simd<DT, D>())) exact_decode_kernel(const ExactDecode a) {
  constexpr bool F32 = DT == TQ_F32;
  constexpr int TB = exact_tokens<DT>(), PAGES = TB / TQ_PAGE_TOKENS;
  constexpr int SIZE = F32 ? 4 : 2;
  constexpr int KSTEPS = D * SIZE / 64;                      // 16-byte pieces that a lane reads of a key
  constexpr int TILES = D / 16;                              // channel tiles
  constexpr int WIDE = ex_wide<DT, D>(), NARROW = (D - WIDE * 128) / 64;
  constexpr int VTOKENS = F32 ? 4 : 8;                       // tokens of a lane
  constexpr bool AHEAD = D <= 256;                           // keys and values are read a block ahead (above, their registers are the accumulators')
  constexpr bool QUERIES_IN_LDS = D == 256;                  // (two wavefronts per SIMD: 256 registers)

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int col = lane & 15, quarter = lane >> 4;            // head of the group; which four tokens of sixteen
  int split, group, h, b;
  if (!exact_place(a, &split, &group, &h, &b)) return;

  const int len = exact_len(a.c, b);
  const int blocks = (len + TB - 1) / TB;
  const int per = exact_blocks_per_split(blocks, a.n_split, a.chunk);
  const int first = split * per < blocks ? split * per : blocks, last = first + per < blocks ? first + per : blocks;
  if (first >= last && a.n_split > 1) return;

  const int head = group * EXACT_HEADS + col;                // of the KV head's G query heads
  const bool live = head < a.G;
  const int64_t row = (int64_t)b * a.Hq + h * a.G + head;
  const int32_t* table = a.c.table + b * a.c.table_step;

  __shared__ ex_u32x4 s_q[QUERIES_IN_LDS ? KSTEPS : 1][64];
  ex_u32x4 Q[QUERIES_IN_LDS ? 1 : KSTEPS];
  const auto query = [&](int s) __attribute__((always_inline)) {
    ex_u32x4 x = {0, 0, 0, 0};
    if (live) x = *(const ex_u32x4*)((const char*)a.q + (row * D) * SIZE + s * 64 + quarter * 16);
    return x;
  };
  if constexpr (QUERIES_IN_LDS) {
    for (int s = wave; s < KSTEPS; s += 4) s_q[s][lane] = query(s);
    __syncthreads();
  } else {
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) Q[s] = query(s);
  }
  ex_f32x4 O[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) O[t] = ex_f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  const uint32_t step = (uint32_t)a.c.s_t * SIZE;
  const uint32_t krow = (uint32_t)col * step + quarter * 16, vrow = (uint32_t)(quarter * 4) * step;
  ex_u32x4 K[PAGES][KSTEPS];
  ex_u32x4 V[WIDE > 0 ? WIDE : 1][VTOKENS];                  // (fp32: one chunk of 64 after another, below)
  ex_u32x2 VN[VTOKENS];
  ex_f32x4 VF[F32 ? NARROW : 1][4];
  const auto load_key = [&](const ExactPages<PAGES>& at, int p, int s) __attribute__((always_inline)) {
    K[p][s] = *(const ex_u32x4*)((const char*)a.c.k + at.at[p] + krow + s * 64);
  };
  const auto load_keys = [&](const ExactPages<PAGES>& at) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) load_key(at, p, s);
  };
  const auto load_chunk = [&](const ExactPages<PAGES>& at, int c) __attribute__((always_inline)) {      // of 128 channels (fp32: 64)
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) VF[c][i] = *(const ex_f32x4*)((const char*)a.c.v + at.at[0] + vrow + i * step + (c * 64 + col * 4) * SIZE);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) V[c][i] = *(const ex_u32x4*)((const char*)a.c.v + at.at[i >> 2] + vrow + (i & 3) * step + (c * 128 + col * 8) * SIZE);
    }
  };
  const auto load_narrow = [&](const ExactPages<PAGES>& at) __attribute__((always_inline)) {
    if constexpr (!F32 && NARROW > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) VN[i] = *(const ex_u32x2*)((const char*)a.c.v + at.at[i >> 2] + vrow + (i & 3) * step + (WIDE * 128 + col * 4) * SIZE);
    }
  };
  constexpr int CHUNKS = F32 ? NARROW : WIDE;
  const auto load_values = [&](const ExactPages<PAGES>& at) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) load_chunk(at, c);
    load_narrow(at);
  };

  ExactPages<PAGES> now, next;
  if (first + wave < last) {
    now.find(a.c, table, len, first + wave, h, SIZE);
    if constexpr (AHEAD) {
      load_keys(now);
      load_values(now);
    }
  }
  for (int blk = first + wave; blk < last; blk += 4) {
    const bool more = blk + 4 < last;
    if (more) next.find(a.c, table, len, blk + 4, h, SIZE);
    int q_lane = lane;
    if constexpr (QUERIES_IN_LDS) asm volatile("" : "+v"(q_lane));        // (the compiler would read them once, into registers that are not there)
    // ---- scores; the next block's keys are on their way as soon as this one's are used ----
    ex_f32x4 S[PAGES];
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      S[p] = ex_f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        if constexpr (!AHEAD) load_key(now, p, s);
        const ex_u32x4 q = QUERIES_IN_LDS ? s_q[QUERIES_IN_LDS ? s : 0][q_lane] : Q[QUERIES_IN_LDS ? 0 : s];
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            S[p] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(K[p][s][i]), __uint_as_float(q[i]), S[p], 0, 0, 0);
        } else {
          S[p] = ex_mfma<DT>(K[p][s], q, S[p]);
        }
      }
    }
    if (AHEAD && more) load_keys(next);
    // ---- weights of this lane's head: tokens quarter * 4 + i of each page ----
    float top = -INFINITY, pr[PAGES][4];
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float s2 = S[p][i] * a.scale2;
        pr[p][i] = now.whole || quarter * 4 + i < now.valid[p] ? s2 : -INFINITY;
        top = fmaxf(top, pr[p][i]);
      }
    if (a.scores && live) {
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        const int page = blk * PAGES + p;
        if (page < a.score_pages)
          *(ex_f32x4*)(a.scores + ((((int64_t)b * a.c.H + h) * a.score_pages + page) * a.G + head) * TQ_PAGE_TOKENS + quarter * 4) =
              ex_f32x4{pr[p][0], pr[p][1], pr[p][2], pr[p][3]};
      }
    }
    top = fmaxf(m, ex_quad_max(top));
    if (__any(top > m + EX_SLACK)) {
      const float move = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      l *= move;
#pragma unroll
      for (int t = 0; t < TILES; ++t) O[t] *= move;
      m = top;
    }
    const float ref = m == -INFINITY ? 0.0f : m - ex_lift<DT>();
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[p][i] = __builtin_amdgcn_exp2f(pr[p][i] - ref);
        l += pr[p][i];
      }
    // ---- values; those of tokens without weight are put to zero, since NaN times nothing is NaN ----
    if constexpr (F32) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        if constexpr (!AHEAD) load_chunk(now, c);
        if (!now.whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (quarter * 4 + i >= now.valid[0]) VF[c][i] = ex_f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) O[c * 4 + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(VF[c][i][t], pr[0][i], O[c * 4 + t], 0, 0, 0);
      }
    } else {
      ex_u32x4 P, L;                                         // high and low halves
#pragma unroll
      for (int p = 0; p < PAGES; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t hi, lo;
          ex_split<DT>(pr[p][2 * i], pr[p][2 * i + 1], &hi, &lo);
          P[p * 2 + i] = hi;
          L[p * 2 + i] = lo;
        }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        if constexpr (!AHEAD) load_chunk(now, c);
        if (!now.whole) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (quarter * 4 + (i & 3) >= now.valid[i >> 2]) V[c][i] = ex_u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          ex_u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            f[j] = __builtin_amdgcn_perm(V[c][2 * j + 1][t >> 1], V[c][2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
          O[c * 8 + t] = ex_mfma<DT>(f, P, ex_mfma<DT>(f, L, O[c * 8 + t]));
        }
      }
      if constexpr (NARROW > 0) {
        if constexpr (!AHEAD) load_narrow(now);
        if (!now.whole) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (quarter * 4 + (i & 3) >= now.valid[i >> 2]) VN[i] = ex_u32x2{0, 0};
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          ex_u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            f[j] = __builtin_amdgcn_perm(VN[2 * j + 1][t >> 1], VN[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
          O[WIDE * 8 + t] = ex_mfma<DT>(f, P, ex_mfma<DT>(f, L, O[WIDE * 8 + t]));
        }
      }
    }
    if (AHEAD && more) load_values(next);
    now = next;
  }

  // ---- the four wavefronts of the workgroup: to a common maximum, then summed pairwise (2, 3 -> 0, 1 -> 0) ----
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __align__(16) ex_f32x4 s_acc[2][TILES][64];
  l = ex_quad_sum(l);
  if (quarter == 0) { s_m[wave][col] = m; s_l[wave][col] = l; }
  __syncthreads();
  const float M = fmaxf(fmaxf(s_m[0][col], s_m[1][col]), fmaxf(s_m[2][col], s_m[3][col]));
  const float ref = M == -INFINITY ? 0.0f : M;
  const float f = __builtin_amdgcn_exp2f(m - ref);
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += s_l[w][col] * __builtin_amdgcn_exp2f(s_m[w][col] - ref);
#pragma unroll
  for (int t = 0; t < TILES; ++t) O[t] *= f;
  if (wave >= 2)
#pragma unroll
    for (int t = 0; t < TILES; ++t) s_acc[wave - 2][t][lane] = O[t];
  __syncthreads();
  if (wave < 2)
#pragma unroll
    for (int t = 0; t < TILES; ++t) O[t] += s_acc[wave][t][lane];
  __syncthreads();
  if (wave == 1)
#pragma unroll
    for (int t = 0; t < TILES; ++t) s_acc[0][t][lane] = O[t];
  __syncthreads();
  if (wave != 0 || !live) return;
#pragma unroll
  for (int t = 0; t < TILES; ++t) O[t] += s_acc[0][t][lane];
  exact_store<DT, D>(a, O, M - ex_lift<DT>(), sum, row, split, quarter);
}

template <int DT>
int launch_exact_decode(const ExactDecode& a, hipStream_t stream) {
  const dim3 grid((unsigned)exact_grid(a)), block(256);
#define TQ_EXACT_D(D) \
  case D: exact_decode_kernel<DT, D><<<grid, block, 0, stream>>>(a); break
  switch (a.c.d) {
    TQ_EXACT_D(64); TQ_EXACT_D(128); TQ_EXACT_D(192); TQ_EXACT_D(256); TQ_EXACT_D(320); TQ_EXACT_D(384);
    TQ_EXACT_D(448); TQ_EXACT_D(512); TQ_EXACT_D(576); TQ_EXACT_D(640); TQ_EXACT_D(704); TQ_EXACT_D(768);
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_EXACT_D
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

}  // namespace tq
