// Decode attention over a paged exact cache for dozens of query heads on a KV head (instantiated by one file per 16-bit type).
//
// The mathematics and the operand layouts are those of tq_exact_impl.h; what differs is who reads.  There a workgroup reads keys and values for
// sixteen heads, straight into registers: with 128 heads on one latent of 576 channels that is eight passes over the cache.  Here a workgroup
// of TW wavefronts, one tile of sixteen heads each, shares a block of 32 tokens in LDS: the cache is read once for 16 TW heads.
//   * A wavefront owns its heads for the whole range of tokens - scores, softmax, accumulators -, so that nothing is exchanged or joined
//     between wavefronts.  576 channels: 72 registers of queries, 144 of accumulators, two wavefronts per SIMD.
//   * Blocks lie in LDS twice: while one is worked on, the next is filled by LDS-direct loads, which all wavefronts issue in turn.  One barrier per
//     block: behind it everybody's part of this block has arrived and everybody is done with the other.
//   * A row takes one 16-byte piece more than it has: rows then start 16 bytes apart in the banks, and the sixteen rows of a key operand are read
//     without conflicts.
#pragma once

#include "tq_exact_impl.h"

namespace tq {

// lane l's 16 bytes land at m0 + 16 l.  The compiler sees neither the load nor its write to LDS: ex_arrived() waits for it.
__device__ __forceinline__ void ex_to_lds(const void* from, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(from), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void ex_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Values of more than 512 channels are read 64 channels at a time, 16 registers instead of 32 (with 128, 30 of 256 were spilled, and a wait for a spilled
// register is one for the next block): 8 bytes a lane, so that four rows should be half the banks apart.
__host__ __device__ constexpr int heads_wide(int d) { return d > 512 ? 0 : d / 128; }
__host__ __device__ constexpr int heads_key_row(int d) { return d / 8 + 1; }
__host__ __device__ constexpr int heads_value_row(int d) { return d / 8 + (heads_wide(d) ? 1 : 2); }
__host__ __device__ constexpr int heads_loads(int d) { return (32 * heads_value_row(d) + 63) / 64; }          // of a block's keys, or values
__host__ __device__ constexpr int heads_lds(int d) { return 4 * heads_loads(d) * 1024; }

// the value, computed where it stands: what is made of it does not stay in registers from one turn to the next
__device__ __forceinline__ int ex_anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int DT, int D, int TW>
__global__ void __launch_bounds__(TW * 64, TW == 8 || D <= 256 ? 2 : 1) exact_heads_kernel(const ExactDecode a) {
  constexpr int KSTEPS = D / 32, TILES = D / 16, WIDE = heads_wide(D), NARROW = (D - WIDE * 128) / 64;
  constexpr int KROW = heads_key_row(D), VROW = heads_value_row(D), LOADS = heads_loads(D), BUF = LOADS * 1024;
  static_assert((32 * KROW + 63) / 64 <= LOADS, "keys take no more loads than values");
  constexpr float LIFT = DT == TQ_F16 ? 14.0f : 0.0f;        // (as in tq_exact_impl.h)
  extern __shared__ __align__(16) unsigned char s_blocks[];  // [2 turns][keys, values][LOADS KB]

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
  const auto fetch = [&](const ExactPages<2>& at, int turn) __attribute__((always_inline)) {
    const int ln = ex_anew((int)threadIdx.x & 63);           // (the places in a block are computed anew: there are no registers to keep them in)
#pragma unroll
    for (int i = 0; i < 2 * LOADS; i += TW) {
      const int n = i + wave;                                // this wavefront's load: keys first
      if (2 * LOADS % TW != 0 && n >= 2 * LOADS) break;
      const bool value = n >= LOADS;
      const int k = value ? n - LOADS : n, piece = k * 64 + ln;
      int r = value ? piece / VROW : piece / KROW, p = piece - r * (value ? VROW : KROW);
      r = r < 32 ? r : 31;                                   // (what fills the last load up, and the pieces between two rows: of no use, but there)
      p = p < D / 8 ? p : D / 8 - 1;
      const char* from = (const char*)(value ? a.c.v : a.c.k) + (r < 16 ? at.at[0] : at.at[1]) + ((uint32_t)(r & 15) * step + (uint32_t)p * 16);
      ex_to_lds(from, lds0 + (uint32_t)(turn * 2 * BUF + n * 1024));
      if constexpr (D > 512) __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (first < last) {
    now.find(a.c, table, len, first, h, 2);
    fetch(now, 0);
  }
  for (int blk = first, turn = 0; blk < last; ++blk, turn ^= 1) {
    ex_arrived();
    __syncthreads();
    if (blk + 1 < last) {
      next.find(a.c, table, len, blk + 1, h, 2);
      fetch(next, turn ^ 1);
    }
    const int lane = ex_anew((int)threadIdx.x & 63), col = lane & 15, quarter = lane >> 4;
    // (a lane's first key and value piece: all others are constants away)
    const unsigned char *kb = s_blocks + (turn * 2 * BUF + (col * KROW + quarter) * 16), *vb = s_blocks + (turn * 2 * BUF + BUF + (quarter * 4 * VROW + col) * 16);
    // ---- scores ----
    ex_f32x4 S[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        S[p] = ex_mfma<DT>(*(const ex_u32x4*)(kb + (p * 16 * KROW + s * 4) * 16), Q[s], S[p]);
      if (D > 256 && s & 1) __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);                       // (values are not read into registers that keys still need)
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
    if (__any(top > m)) {
      const float move = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      l *= move;
#pragma unroll
      for (int t = 0; t < TILES; ++t) O[t] *= move;
      m = top;
    }
    const float ref = m == -INFINITY ? 0.0f : m - LIFT;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[p][i] = __builtin_amdgcn_exp2f(pr[p][i] - ref);
        l += pr[p][i];
      }
    ex_u32x4 P;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i) P[p * 2 + i] = ex_pack<DT>(pr[p][2 * i], pr[p][2 * i + 1]);
    // ---- values ----
#pragma unroll
    for (int c = 0; c < WIDE; ++c) {
      ex_u32x4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = *(const ex_u32x4*)(vb + (((i >> 2) * 16 + (i & 3)) * VROW + c * 16) * 16);
        if (!now.whole && quarter * 4 + (i & 3) >= now.valid[i >> 2]) x[i] = ex_u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        ex_u32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(x[2 * j + 1][t >> 1], x[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
        O[c * 8 + t] = ex_mfma<DT>(f, P, O[c * 8 + t]);
      }
      if constexpr (D > 256) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int c = 0; c < NARROW; ++c) {
      ex_u32x2 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = *(const ex_u32x2*)(vb - col * 8 + (((i >> 2) * 16 + (i & 3)) * VROW + WIDE * 16 + c * 8) * 16);
        if (!now.whole && quarter * 4 + (i & 3) >= now.valid[i >> 2]) x[i] = ex_u32x2{0, 0};
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        ex_u32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(x[2 * j + 1][t >> 1], x[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
        O[WIDE * 8 + c * 4 + t] = ex_mfma<DT>(f, P, O[WIDE * 8 + c * 4 + t]);
      }
      if constexpr (D > 256) __builtin_amdgcn_sched_barrier(0);
    }
    now = next;
  }
  l = ex_quad_sum(l);
  const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  if (head0 + col >= a.G) return;
  exact_store<DT, D, WIDE>(a, O, m - LIFT, l, row0 + col, split, quarter);
}

template <int DT>
int launch_exact_heads(const ExactDecode& a, int tw, hipStream_t stream) {
  const dim3 grid((unsigned)exact_grid(a)), block(tw * 64);
#define TQ_HEADS_TW(D, TW)                                                                                                  \
  {                                                                                                                         \
    const auto kern = exact_heads_kernel<DT, D, TW>;                                                                        \
    static std::atomic<uint64_t> ready{0};                                                                                  \
    if (const int rc = exact_allow_lds((const void*)kern, heads_lds(D), ready)) return rc;                                  \
    kern<<<grid, block, heads_lds(D), stream>>>(a);                                                                         \
    break;                                                                                                                  \
  }
#define TQ_HEADS_D(D)                                                                 \
  case D:                                                                             \
    if (tw == 8) TQ_HEADS_TW(D, 8)                                                    \
    if (tw == 4) TQ_HEADS_TW(D, 4)                                                    \
    TQ_HEADS_TW(D, 2)
  switch (a.c.d) {
    TQ_HEADS_D(64) TQ_HEADS_D(128) TQ_HEADS_D(192) TQ_HEADS_D(256) TQ_HEADS_D(320) TQ_HEADS_D(384) TQ_HEADS_D(448) TQ_HEADS_D(512) TQ_HEADS_D(576)
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_HEADS_D
#undef TQ_HEADS_TW
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

}  // namespace tq
