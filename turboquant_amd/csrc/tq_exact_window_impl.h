// Softmax weights of a window of queries, summed over the window and the heads of a KV head, in two passes over the keys:
//
//   rows r = (w, g): w of the newest W' = min(W, rows of the sequence, its length) queries, g of the G heads on the KV head
//   first   m_r = max_t s_rt,  l_r = sum_t 2^(s_rt - m_r)          s_rt = scale log2 e  q_r . k_t  for t <= length - W' + w
//   second  weights[t] += sum_r 2^(s_rt - m_r) / l_r
//
// The scores are computed twice rather than stored: at W = 32 and 32 heads of 128 a token's scores are 4 KB per KV head and its key 256 bytes.
// Tokens are rows of the matrix instruction and come from memory as they lie, as in decode; (query, head) rows are its columns and stay in
// registers, window_tiles() tiles of 16 per wavefront.  The four wavefronts of a workgroup stand side by side on the tiles, or, with few of them,
// on the tokens.  In the first pass a lane keeps maximum and sum of its own tokens (four of each sixteen) and joins them with the three other lanes of its
// row at the end; in the second it sums its columns' weights of its tokens, over the tiles in registers, over lanes once per block.
#pragma once

#include "tq_exact_impl.h"
#include "tq_exact_window.h"

namespace tq {

constexpr int WINDOW_TOKENS = 1024;             // tokens whose sums a workgroup of the second pass holds at a time

template <int DT, int D, bool ADD>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) exact_window_kernel(const ExactWindow a) {
  constexpr bool F32 = DT == TQ_F32;
  constexpr int TB = exact_tokens<DT>(), PAGES = TB / TQ_PAGE_TOKENS, SIZE = F32 ? 4 : 2;
  constexpr int KSTEPS = D * SIZE / 64, NT = window_tiles(DT, D);
  __shared__ float s_w[ADD ? 4 : 1][ADD ? WINDOW_TOKENS : 1];

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int col = lane & 15, quarter = lane >> 4;
  int id = (int)blockIdx.x;
  const int split = id % a.n_split; id /= a.n_split;
  int group0 = 0, groups = a.row_groups;
  if (!ADD) { group0 = id % a.row_groups; id /= a.row_groups; groups = 1; }
  const int h = id % a.c.H, b = id / a.c.H;

  const int len = exact_len(a.c, b);
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
  const int tile_wave = wave % a.tile_waves, token_wave = wave / a.tile_waves, token_waves = 4 / a.tile_waves;
  const int32_t* table = a.c.table + b * a.c.table_step;
  const int64_t row_at = (int64_t)b * a.c.H + h;
  const int padded = a.row_tiles * 16;
  if (first >= last || n_rows == 0) return;                  // (the same for the whole workgroup)

  for (int sub = first; sub < last; sub += ADD ? WINDOW_TOKENS / TB : last - first) {
    const int sub_end = ADD && sub + WINDOW_TOKENS / TB < last ? sub + WINDOW_TOKENS / TB : last;
    if (ADD) {
      __syncthreads();
      for (int i = (int)threadIdx.x; i < 4 * WINDOW_TOKENS; i += 256) s_w[0][i] = 0.0f;
      __syncthreads();
    }
    for (int grp = group0; grp < group0 + groups; ++grp) {
      const int tile0 = (grp * a.tile_waves + tile_wave) * NT;
      if (tile0 * 16 >= n_rows) continue;                    // (no barrier inside)
      ex_u32x4 Q[NT][KSTEPS];
      int end[NT];                                           // tokens that the row of this lane's column sees
      float mx[NT], sm[NT];                                  // first pass: maximum and sum; second: maximum and 1 / sum of the row
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int r = (tile0 + t) * 16 + col;
        const bool live = r < n_rows;
        const int w = live ? r / a.G : 0, g = r - w * a.G;
        end[t] = live ? len - W + w + 1 : 0;
        mx[t] = ADD ? 0.0f : -INFINITY;
        sm[t] = 0.0f;
        if (ADD && live) {
          const float2 st = a.stat[row_at * padded + r];
          mx[t] = st.x;
          sm[t] = st.y;
        }
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
          Q[t][s] = ex_u32x4{0, 0, 0, 0};
          if (live) Q[t][s] = *(const ex_u32x4*)((const char*)a.q + (((r1 - W + w) * a.Hq + h * a.G + g) * D) * SIZE + s * 64 + quarter * 16);
        }
      }
      const bool full_tiles = (tile0 + NT) * 16 <= n_rows;
      for (int blk = sub + token_wave; blk < sub_end; blk += token_waves) {
        const int t0 = blk * TB;
        bool whole = full_tiles && t0 + TB <= len - W + 1;   // every row sees every token
        const char* kp[PAGES];
        int valid[PAGES];
#pragma unroll
        for (int p = 0; p < PAGES; ++p) {
          const int left = len - t0 - p * TQ_PAGE_TOKENS;
          valid[p] = left < 0 ? 0 : (left > TQ_PAGE_TOKENS ? TQ_PAGE_TOKENS : left);
          int64_t page = left > 0 ? table[blk * PAGES + p] : 0;
          if (page < 0 || page >= a.c.num_blocks) { page = 0; valid[p] = 0; }
          whole &= valid[p] == TQ_PAGE_TOKENS;
          kp[p] = (const char*)a.c.k + (page * a.c.s_blk + h * a.c.s_h) * SIZE;
        }
        const uint32_t krow = (uint32_t)col * (uint32_t)a.c.s_t * SIZE + quarter * 16;
        ex_f32x4 S[NT][PAGES];
#pragma unroll
        for (int p = 0; p < PAGES; ++p) {
          const bool there = whole || col < valid[p];
#pragma unroll
          for (int t = 0; t < NT; ++t) S[t][p] = ex_f32x4{0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KSTEPS; ++s) {
            ex_u32x4 kf = {0, 0, 0, 0};
            if (there) kf = *(const ex_u32x4*)(kp[p] + krow + s * 64);
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
        // scores in powers of two; hidden ones have no weight
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int p = 0; p < PAGES; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int in = quarter * 4 + i;
              const float s2 = S[t][p][i] * a.scale2;
              S[t][p][i] = whole || (in < valid[p] && t0 + p * TQ_PAGE_TOKENS + in < end[t]) ? s2 : -INFINITY;
            }
        if constexpr (!ADD) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float top = mx[t];
#pragma unroll
            for (int p = 0; p < PAGES; ++p)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, S[t][p][i]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = sm[t] * __builtin_amdgcn_exp2f(mx[t] - ref);
#pragma unroll
            for (int p = 0; p < PAGES; ++p)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(S[t][p][i] - ref);
            sm[t] = sum;
            mx[t] = top;
          }
        } else {
          ex_f32x4 add[PAGES];
#pragma unroll
          for (int p = 0; p < PAGES; ++p) {
            add[p] = ex_f32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) add[p][i] = fmaf(__builtin_amdgcn_exp2f(S[t][p][i] - mx[t]), sm[t], add[p][i]);
            // over the sixteen rows of the tiles
#pragma unroll
            for (int i = 0; i < 4; ++i) add[p][i] = lanes_sum_dpp<16>(add[p][i]);
            if (col == 0) {
              float* to = &s_w[wave][(blk - sub) * TB + p * TQ_PAGE_TOKENS + quarter * 4];
#pragma unroll
              for (int i = 0; i < 4; ++i) to[i] += add[p][i];
            }
          }
        }
      }
      if constexpr (!ADD) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float top = ex_quad_max(mx[t]), ref = top == -INFINITY ? 0.0f : top;
          const float sum = ex_quad_sum(sm[t] * __builtin_amdgcn_exp2f(mx[t] - ref));
          const int r = (tile0 + t) * 16 + col;
          if (quarter == 0 && r < n_rows) a.ml[(row_at * a.parts + split * token_waves + token_wave) * padded + r] = make_float2(top, sum);
        }
      }
    }
    if constexpr (ADD) {
      __syncthreads();
      float* w = a.weights + b * a.w_b + h * a.w_h;
      for (int i = (int)threadIdx.x; i < (sub_end - sub) * TB; i += 256) {
        const int t = sub * TB + i;
        if (t < len && t < a.L) w[t] += (s_w[0][i] + s_w[1][i]) + (s_w[2][i] + s_w[3][i]);
      }
    }
  }
}

template <int DT>
int launch_exact_window(const ExactWindow& a, bool add, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.n_split * (add ? 1 : a.row_groups) * a.c.H * a.B)), block(256);
#define TQ_WINDOW_D(D)                                                                \
  case D:                                                                             \
    if (add) exact_window_kernel<DT, D, true><<<grid, block, 0, stream>>>(a);         \
    else exact_window_kernel<DT, D, false><<<grid, block, 0, stream>>>(a);            \
    break
  switch (a.c.d) {
    TQ_WINDOW_D(64); TQ_WINDOW_D(128); TQ_WINDOW_D(192); TQ_WINDOW_D(256); TQ_WINDOW_D(320); TQ_WINDOW_D(384);
    TQ_WINDOW_D(448); TQ_WINDOW_D(512); TQ_WINDOW_D(576); TQ_WINDOW_D(640); TQ_WINDOW_D(704); TQ_WINDOW_D(768);
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_WINDOW_D
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

}  // namespace tq
