// Softmax weights of a window of queries, summed over the window and the heads of a KV head, in two passes over the keys:
//
//   rows r = (w, g): w of the newest W' = min(W, rows of the sequence, its length) queries, g of the G heads on the KV head
//   first   m_r = max_t s_rt,  l_r = sum_t 2^(s_rt - m_r)          s_rt = scale log2 e  q_r . k_t  for t <= length - W' + w
//   second  weights[t] += sum_r 2^(s_rt - m_r) / l_r
//
// The scores are computed twice rather than stored: at W = 32 and four heads of 128 on a KV head a token's scores are 512 bytes, which would be written and
// read, and its key, which is read again, 256.
// Tokens are rows of the matrix instruction, (query, head) rows its columns; those stay in registers, window_tiles() tiles of 16 per wavefront.  The
// wavefronts of a workgroup stand side by side on the tiles, and, with few of those, on the tokens.  Keys lie in LDS twice, filled by LDS-direct loads
// a turn ahead: read from memory as operands, they came from the L1 once for every wavefront, 16 lines of 64 bytes a load, and that was the bound.
// Bound by reads of LDS, matrix instructions and the exponentials in turn: bf16, four sequences of 32768, 32 / 8 heads of 128, 32 queries: 66 us the first pass,
// 5 the join, 68 the second; a pass is 268 MB (4.0 TB/s) and 34 GFLOP (520 TFLOP/s).  fp16, nine of 17 .. 4099, 16 / 2 heads of 256, 64 queries: 20 + 5 + 20 us
// for 13 MB: the longest sequence's workgroups.  One of 1500: 7.1 + 3.5 + 8.4 us, three launches of latencies.
// In the first pass a lane keeps maximum and sum of its own tokens (four of each sixteen) and joins them with the three other lanes of its
// row at the end; in the second it sums its columns' weights of its tokens, over the tiles in registers, over lanes once per block.
#pragma once

#include "tq_exact_heads_impl.h"
#include "tq_exact_window.h"

namespace tq {

constexpr int WINDOW_TOKENS = 1024;             // tokens whose sums a workgroup of the second pass holds at a time

// A block's keys in LDS: rows one behind another, a row's 16-byte pieces in an order of its own, so that the sixteen rows of an operand lie in
// different banks: with an even number of bank widths to a row, piece p of row r is the (p ^ r)-th of its sixteen; with an odd one, the
// (p ^ r / 2)-th of its eight.
template <int PIECES>
__device__ __forceinline__ int window_place(int p, int r) {
  return PIECES % 16 == 0 ? p ^ (r & 15) : p ^ (r >> 1 & 7);
}

template <int DT, int D, int WAVES, bool ADD>
__global__ void __launch_bounds__(WAVES * 64, window_waves_per_simd(DT, D, WAVES)) exact_window_kernel(const ExactWindow a) {
  constexpr bool F32 = DT == TQ_F32;
  constexpr int TB = exact_tokens<DT>(), PAGES = TB / TQ_PAGE_TOKENS, SIZE = F32 ? 4 : 2;
  constexpr int KSTEPS = D * SIZE / 64, NT = window_tiles(DT, D), PIECES = D * SIZE / 16;
  constexpr int BLOCK = window_block_bytes(D), PAGE_LOADS = PIECES / 4;        // LDS-direct loads of a page: 64 pieces each
  extern __shared__ __align__(16) unsigned char s_keys[];    // [2 turns][wavefronts side by side on tokens][BLOCK]
  __shared__ float s_w[ADD ? WAVES : 1][ADD ? WINDOW_TOKENS : 1];

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int col = lane & 15, quarter = lane >> 4;
  unsigned id = blockIdx.x;
  int group0 = 0, groups = a.row_groups;
  if (!ADD) { group0 = (int)(id % (unsigned)a.row_groups); id /= (unsigned)a.row_groups; groups = 1; }
  // (splits of a sequence on different dies, as in decode)
  const unsigned pairs = (unsigned)(a.c.H * a.B);
  const int split = (int)(id / pairs), pair = (int)((id % pairs + (unsigned)split) % pairs);
  const int h = pair % a.c.H, b = pair / a.c.H;

  const int len = __builtin_amdgcn_readfirstlane(exact_len(a.c, b));
  const int blocks = (len + TB - 1) / TB, per = exact_blocks_per_split(blocks, a.n_split, a.chunk);
  const int first = split * per < blocks ? split * per : blocks, last = first + per < blocks ? first + per : blocks;
  // the rows of the window
  int64_t r0 = a.starts[b], r1 = a.starts[b + 1];
  r0 = r0 < 0 ? 0 : r0;
  r1 = r1 > a.rows ? a.rows : r1;
  const int64_t run = r1 > r0 ? r1 - r0 : 0;
  int W = a.W < len ? a.W : len;
  W = run < W ? (int)run : W;
  const int n_rows = W * a.G;
  const int tile_wave = wave % a.tile_waves, token_wave = wave / a.tile_waves, token_waves = a.waves / a.tile_waves;
  const int32_t* table = a.c.table + b * a.c.table_step;
  const int64_t row_at = (int64_t)b * a.c.H + h;
  const int padded = a.row_tiles * 16;
  if (first >= last || n_rows == 0) return;                  // (the same for the whole workgroup)
  const uint32_t step = (uint32_t)a.c.s_t * SIZE, lds0 = (uint32_t)(uintptr_t)s_keys;

  // A turn: token_waves blocks from `blk` on.  Lane l knows the table entry of the turn's page l (behind the sequence, where nothing counts, its
  // last; a condition around the load would have it waited for at once, and with it the keys that are on their way).
  const int last_page = (len - 1) / TQ_PAGE_TOKENS;
  const auto entries = [&](int blk) __attribute__((always_inline)) {
    const int page = blk * PAGES + lane;
    return table[page < last_page ? page : last_page];
  };
  const uint32_t in_cache = a.c.num_blocks < 0x80000000ll ? (uint32_t)a.c.num_blocks : 0x80000000u;
  const auto there = [&](int entry, int p) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_readlane(entry, p) < in_cache; };
  // A wavefront's loads of a turn are numbers wave, wave + waves, ...: page n / PAGE_LOADS, 64 pieces of it.  A lane's place in its page is the same in
  // every turn; the first FIXED of them stay in registers (computed anew they were 40 instructions a load, and the loads a quarter of a turn).
  constexpr int FIXED = 5;
  const int turn_loads = token_waves * PAGES * PAGE_LOADS;
  const char* head = (const char*)a.c.k + h * a.c.s_h * SIZE;
  const uint64_t block_bytes = (uint64_t)a.c.s_blk * SIZE;
  const auto place = [&](int n) __attribute__((always_inline)) {
    const int piece = n % PAGE_LOADS * 64 + lane, r = piece / PIECES, at = piece - r * PIECES;
    return (uint32_t)r * step + (uint32_t)window_place<PIECES>(at, r) * 16;
  };
  uint32_t fixed[FIXED];
#pragma unroll
  for (int i = 0; i < FIXED; ++i) fixed[i] = place(wave + i * a.waves);
  const auto load = [&](int entry, int turn, int n, uint32_t off) __attribute__((always_inline)) {
    const int p = n / PAGE_LOADS;
    uint32_t page = (uint32_t)__builtin_amdgcn_readlane(entry, p);
    page = page < in_cache ? page : 0;                       // (a block that is there; its tokens are masked)
    ex_row_to_lds(head + page * block_bytes, off, lds0 + (uint32_t)(turn * token_waves * BLOCK + n * 1024));
  };
  const auto fetch = [&](int entry, int turn) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FIXED; ++i)
      if (wave + i * a.waves < turn_loads) load(entry, turn, wave + i * a.waves, fixed[i]);
    for (int n = wave + FIXED * a.waves; n < turn_loads; n += a.waves) load(entry, turn, n, place(n));
  };

  for (int sub = first; sub < last; sub += ADD ? WINDOW_TOKENS / TB : last - first) {
    const int sub_end = ADD && sub + WINDOW_TOKENS / TB < last ? sub + WINDOW_TOKENS / TB : last;
    if (ADD) {
      __syncthreads();
      for (int i = (int)threadIdx.x; i < (sub_end - sub) * TB; i += a.waves * 64)
        for (int k = 0; k < a.tile_waves; ++k) s_w[k][i] = 0.0f;
      __syncthreads();
    }
    for (int grp = group0; grp < group0 + groups; ++grp) {
      if (grp * a.tile_waves * NT * 16 >= n_rows) break;     // (the same for the whole workgroup)
      const int tile0 = (grp * a.tile_waves + tile_wave) * NT;
      const bool busy = tile0 * 16 < n_rows;                 // (a wavefront without rows still fetches and waits with the others)
      if (ADD && grp > group0) __syncthreads();              // (the turns of the group before have been read)
      int entry = entries(sub);
      fetch(entry, 0);
      int entry_next = entries(sub + token_waves);
      ex_u32x4 Q[NT][KSTEPS];
      float mx[NT], sm[NT];                                  // first pass: maximum (unscaled) and sum; second: maximum (log2) and 1 / sum of the row
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int r = (tile0 + t) * 16 + col;
        const bool live = r < n_rows;
        mx[t] = ADD ? 0.0f : -INFINITY;
        sm[t] = 0.0f;
        if (ADD && live) {
          const float2 st = a.stat[row_at * padded + r];
          mx[t] = st.x;
          sm[t] = st.y;
        }
        if constexpr (window_staged(DT, D, WAVES)) {
          if (a.tile_waves == a.waves) {
            // A tile's rows by way of LDS, a wavefront for itself; offsets from the tile's first row.  (A row behind the last is the last one over again: its
            // scores are hidden.)
            const int row0 = (tile0 + t) * 16 < n_rows ? (tile0 + t) * 16 : n_rows - 1, w0 = row0 / a.G;
            const char* base = (const char*)a.q + (((r1 - W + w0) * a.Hq + h * a.G + (row0 - w0 * a.G)) * D) * SIZE;
            const uint32_t row_bytes = D * SIZE, turn_bytes = (uint32_t)(a.Hq - a.G) * row_bytes;
            const uint32_t to = lds0 + (uint32_t)(2 * BLOCK + wave * 16 * D * SIZE);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // (the tile before has been read)
#pragma unroll
            for (int n = 0; n < PIECES / 4; ++n) {
              const int piece = n * 64 + lane, in = piece / PIECES, at = piece - in * PIECES;
              const int rr = row0 + in < n_rows ? row0 + in : n_rows - 1;
              const uint32_t turns = (a.G == 1 ? (uint32_t)rr : __umulhi((uint32_t)rr, a.per_head)) - (uint32_t)w0;
              ex_row_to_lds(base, (uint32_t)(rr - row0) * row_bytes + turns * turn_bytes + (uint32_t)window_place<PIECES>(at, in) * 16, to + n * 1024);
            }
            ex_arrived();
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s)
              Q[t][s] = *(const ex_u32x4*)(s_keys + 2 * BLOCK + wave * 16 * D * SIZE + (col * PIECES + window_place<PIECES>(s * 4 + quarter, col)) * 16) ^ a.flip;
            continue;
          }
        }
        const int w = live ? r / a.G : 0, g = r - w * a.G;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
          Q[t][s] = ex_u32x4{0, 0, 0, 0};
          if (live) Q[t][s] = *(const ex_u32x4*)((const char*)a.q + (((r1 - W + w) * a.Hq + h * a.G + g) * D) * SIZE + s * 64 + quarter * 16);
          // (a negative scale is the queries'; and with something done to them they have arrived before the loop: where it waited for them, it waited for the keys
          // on their way, 65 -> 90 us)
          Q[t][s] ^= a.flip;
        }
      }
      const bool full_tiles = (tile0 + NT) * 16 <= n_rows;
      for (int turn0 = sub, turn = 0; turn0 < sub_end; turn0 += token_waves, turn ^= 1) {
        ex_arrived();
        __syncthreads();                                     // everybody's loads of this turn are there, everybody is done with the other
        const int now = entry;
        entry = entry_next;
        if (turn0 + token_waves < sub_end) fetch(entry, turn ^ 1);
        entry_next = entries(turn0 + 2 * token_waves);       // (always: behind a condition it would be waited for)
        const int blk = turn0 + token_wave, t0 = blk * TB;
        if (!busy || blk >= sub_end) continue;
        int valid[PAGES];
        bool whole = full_tiles && t0 + TB <= len - W + 1;   // every row sees every token
#pragma unroll
        for (int p = 0; p < PAGES; ++p) {
          const int left = len - t0 - p * TQ_PAGE_TOKENS;
          valid[p] = !there(now, token_wave * PAGES + p) || left < 0 ? 0 : (left > TQ_PAGE_TOKENS ? TQ_PAGE_TOKENS : left);
          whole &= valid[p] == TQ_PAGE_TOKENS;
        }
        const unsigned char* keys = s_keys + (turn * token_waves + token_wave) * BLOCK;
        const auto key = [&](int p, int s) __attribute__((always_inline)) {
          return *(const ex_u32x4*)(keys + ((p * 16 + col) * PIECES + window_place<PIECES>(s * 4 + quarter, col)) * 16);
        };
        ex_f32x4 S[NT][PAGES];
#pragma unroll
        for (int p = 0; p < PAGES; ++p) {
#pragma unroll
          for (int t = 0; t < NT; ++t) S[t][p] = ex_f32x4{0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KSTEPS; ++s) {
            const ex_u32x4 kf = key(p, s);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  S[t][p] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[i]), __uint_as_float(Q[t][s][i]), S[t][p], 0, 0, 0);
              } else {
                S[t][p] = ex_mfma<DT>(kf, Q[t][s], S[t][p]);
              }
            }
          }
        }
        // hidden scores have no weight; blocks that every row sees whole are left as they are
        if (!whole) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int r = (tile0 + t) * 16 + col;
            const int end = r < n_rows ? len - W + r / a.G + 1 : 0;          // tokens that the row of this lane's column sees
#pragma unroll
            for (int p = 0; p < PAGES; ++p)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int in = quarter * 4 + i;
                if (!(in < valid[p] && t0 + p * TQ_PAGE_TOKENS + in < end)) S[t][p][i] = -INFINITY;
              }
          }
        }
        if constexpr (!ADD) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float top = mx[t];
#pragma unroll
            for (int p = 0; p < PAGES; ++p)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, S[t][p][i]);
            const float ref = top == -INFINITY ? 0.0f : top * a.scale2;
            float sum = sm[t] * __builtin_amdgcn_exp2f(fmaf(mx[t], a.scale2, -ref));
#pragma unroll
            for (int p = 0; p < PAGES; ++p)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(fmaf(S[t][p][i], a.scale2, -ref));
            sm[t] = sum;
            mx[t] = top;
          }
        } else {
#pragma unroll
          for (int p = 0; p < PAGES; ++p) {
            ex_f32x4 add = {0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) add[i] = fmaf(__builtin_amdgcn_exp2f(fmaf(S[t][p][i], a.scale2, -mx[t])), sm[t], add[i]);
            // over the sixteen rows of the tiles
#pragma unroll
            for (int i = 0; i < 4; ++i) add[i] = lanes_sum_dpp<16>(add[i]);
            if (col == 0) {
              ex_f32x4* to = (ex_f32x4*)&s_w[tile_wave][(blk - sub) * TB + p * TQ_PAGE_TOKENS + quarter * 4];
              *to += add;
            }
          }
        }
      }
      if constexpr (!ADD) {
        if (!busy) continue;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float mine = mx[t] == -INFINITY ? -INFINITY : mx[t] * a.scale2;
          const float top = ex_quad_max(mine), ref = top == -INFINITY ? 0.0f : top;
          const float sum = ex_quad_sum(sm[t] * __builtin_amdgcn_exp2f(mine - ref));
          const int r = (tile0 + t) * 16 + col;
          if (quarter == 0 && r < n_rows) a.ml[(row_at * a.parts + split * token_waves + token_wave) * padded + r] = make_float2(top, sum);
        }
      }
    }
    if constexpr (ADD) {
      __syncthreads();
      float* w = a.weights + b * a.w_b + h * a.w_h;
      for (int i = (int)threadIdx.x; i < (sub_end - sub) * TB; i += a.waves * 64) {
        const int t = sub * TB + i;
        float add = 0.0f;
        for (int k = 0; k < a.tile_waves; ++k) add += s_w[k][i];
        if (t < len && t < a.L) w[t] += add;
      }
    }
  }
}

template <int DT>
int launch_exact_window(const ExactWindow& a, bool add, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.n_split * (add ? 1 : a.row_groups) * a.c.H * a.B)), block(a.waves * 64);
  const int lds = 2 * a.waves / a.tile_waves * window_block_bytes(a.c.d) +
                  (a.tile_waves == a.waves && window_staged(DT, a.c.d, a.waves) ? a.waves * window_tile_bytes(DT, a.c.d) : 0);
#define TQ_WINDOW(D, WAVES, ADD)                                                                                            \
  {                                                                                                                         \
    const auto kern = exact_window_kernel<DT, D, WAVES, ADD>;                                                               \
    static std::atomic<uint64_t> ready{0};                                                                                  \
    if (const int rc = exact_allow_lds((const void*)kern, WINDOW_LDS, ready)) return rc;                                    \
    kern<<<grid, block, lds, stream>>>(a);                                                                                  \
    break;                                                                                                                  \
  }
#define TQ_WINDOW_D(D)                                                                \
  case D:                                                                             \
    if (a.waves == 8 && add) TQ_WINDOW(D, 8, true)                                    \
    if (a.waves == 8) TQ_WINDOW(D, 8, false)                                          \
    if (add) TQ_WINDOW(D, 4, true)                                                    \
    TQ_WINDOW(D, 4, false)
  switch (a.c.d) {
    TQ_WINDOW_D(64) TQ_WINDOW_D(128) TQ_WINDOW_D(192) TQ_WINDOW_D(256) TQ_WINDOW_D(320) TQ_WINDOW_D(384)
    TQ_WINDOW_D(448) TQ_WINDOW_D(512) TQ_WINDOW_D(576) TQ_WINDOW_D(640) TQ_WINDOW_D(704) TQ_WINDOW_D(768)
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_WINDOW_D
#undef TQ_WINDOW
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

}  // namespace tq
