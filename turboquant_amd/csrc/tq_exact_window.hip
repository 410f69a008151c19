// A window's weights over a paged exact cache: entry points, and the launch that joins the parts of a row.
#include "tq_exact_window.h"

#include <algorithm>
#include <cmath>

namespace tq {

// stat[r] = (M, 1 / sum_i 2^(m_i - M) l_i) over the parts of a row; a row that sees nothing has no weight to give.  Sixteen rows a workgroup, sixteen
// threads a row.
__global__ void __launch_bounds__(256) exact_window_join_kernel(const float2* ml, float2* stat, int parts, int padded, ExactCache c, int block_tokens,
                                                                int n_split, int chunk, int token_waves) {
  __shared__ float s_top[16][17], s_sum[16][17];
  const int r = (int)threadIdx.x & 15, share = (int)threadIdx.x >> 4;
  const int64_t at = (int64_t)blockIdx.x * 16, row = at / padded;
  const int in = (int)(at - row * padded) + r, len = exact_len(c, (int)(row / c.H));
  const int used = exact_splits_used((len + block_tokens - 1) / block_tokens, n_split, chunk) * token_waves;
  const float2* x = ml + row * parts * padded + in;
  float top = -INFINITY, sum = 0.0f;
  for (int p = share; p < used; p += 16) {
    const float2 v = x[(int64_t)p * padded];
    const float now = fmaxf(top, v.x), ref = now == -INFINITY ? 0.0f : now;
    sum = sum * __builtin_amdgcn_exp2f(top - ref) + v.y * __builtin_amdgcn_exp2f(v.x - ref);
    top = now;
  }
  s_top[share][r] = top;
  s_sum[share][r] = sum;
  __syncthreads();
  if (share != 0) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, s_top[i][r]);
  const float ref = top == -INFINITY ? 0.0f : top;
  sum = 0.0f;
  for (int i = 0; i < 16; ++i) sum += s_sum[i][r] * __builtin_amdgcn_exp2f(s_top[i][r] - ref);
  stat[at + r] = make_float2(ref, sum == 0.0f ? 0.0f : 1.0f / sum);
}

struct WindowPlan {
  int row_tiles, waves, tile_waves, row_groups, n_split, chunk, block_tokens, parts;
  size_t ml_at, stat_at, bytes;
};

static bool window_plan(WindowPlan* p, int dtype, int B, int Hq, int Hkv, int d, int W, int64_t max_len) {
  if (dtype < TQ_F32 || dtype > TQ_BF16 || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || d <= 0 || d % 64 || d > 768) return false;
  if (W <= 0 || W > 1024 || max_len < 0 || max_len > INT32_MAX - 64 || Hq / Hkv > 1024) return false;
  if ((int64_t)Hq * d > 1 << 25) return false;               // (sixteen rows of queries lie within 32 bits of each other)
  const int G = Hq / Hkv, NT = window_tiles(dtype, d);
  p->block_tokens = dtype == TQ_F32 ? 16 : 32;
  p->row_tiles = (W * G + 15) / 16;
  p->tile_waves = p->row_tiles > 4 * NT ? 8 : (p->row_tiles > 2 * NT ? 4 : (p->row_tiles > NT ? 2 : 1));
  p->row_groups = (p->row_tiles + p->tile_waves * NT - 1) / (p->tile_waves * NT);
  const int64_t blocks = std::max<int64_t>(1, (max_len + p->block_tokens - 1) / p->block_tokens);
  const int64_t pairs = std::max<int64_t>(1, (int64_t)B * Hkv);
  // the wavefronts that are left stand side by side on the tokens, as far as two turns of their blocks take no more than 64 KB (one block: any size)
  const int64_t token_waves = p->tile_waves >= 4 ? 1 : std::max(1, std::min(4 / p->tile_waves, 32768 / window_block_bytes(d)));
  p->waves = (int)(p->tile_waves * token_waves);
  // twice as many workgroups as the card holds: sequences differ in length (nine of 17 .. 4099 tokens, 16 / 2 heads of 256, a pass: 33 us with once as
  // many, 24 with twice, 24 with three times; four of 32768, 32 / 8 heads of 128, where nothing differs: 74, 81, 85); a block for every wavefront at least
  const int64_t resident = 256 * 4 * window_waves_per_simd(dtype, d, p->waves == 8 ? 8 : 4) / p->waves;
  int64_t n = std::max(2 * resident / pairs, (max_len + 4095) / 4096);
  n = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(n, (blocks + token_waves - 1) / token_waves), 4096));
  const int64_t chunk = ((blocks + n - 1) / n + token_waves - 1) / token_waves * token_waves;
  p->chunk = (int)chunk;
  p->n_split = (int)((blocks + chunk - 1) / chunk);
  p->parts = (int)(p->n_split * token_waves);
  const size_t rows = (size_t)B * Hkv * p->row_tiles * 16;
  p->ml_at = 0;
  p->stat_at = (rows * p->parts * sizeof(float2) + 255) & ~(size_t)255;
  p->bytes = p->stat_at + std::max<size_t>(256, (rows * sizeof(float2) + 255) & ~(size_t)255);
  return pairs * p->n_split * p->row_groups <= INT32_MAX && (int64_t)(rows / 16) <= INT32_MAX;
}

}  // namespace tq

extern "C" size_t tq_exact_window_bytes(int dtype, int B, int Hq, int Hkv, int d, int window, int64_t max_len) {
  tq::WindowPlan p;
  return tq::window_plan(&p, dtype, B, Hq, Hkv, d, window, max_len) ? p.bytes : 0;
}

extern "C" int tq_exact_window(const void* q, int dtype, int64_t rows, const int32_t* query_start_loc, int B, int Hq, int Hkv, int d, int window,
                               const void* k_cache, int64_t cs_blk, int64_t cs_t, int64_t cs_h, int64_t num_blocks, const int32_t* block_table,
                               int bt_stride, const int32_t* seq_lens, float sm_scale, int64_t max_len, float* weights, int64_t w_b, int64_t w_h,
                               int64_t weight_len, void* workspace, void* stream) {
  using namespace tq;
  if (!q || !query_start_loc || !weights) return TQ_ENULL;
  WindowPlan p;
  if (!window_plan(&p, dtype, B, Hq, Hkv, d, window, max_len)) return TQ_EINVAL;
  ExactWindow a{};
  const int rc = exact_cache_init(&a.c, k_cache, k_cache, dtype, Hkv, d, cs_blk, cs_t, cs_h, num_blocks, block_table, bt_stride, seq_lens);
  if (rc) return rc;
  if (rows < 0 || w_b < 0 || w_h < 0 || weight_len <= 0 || weight_len > INT32_MAX - 64) return TQ_EINVAL;
  if ((uintptr_t)q & 15) return TQ_EUNSUPPORTED;
  if (B == 0 || rows == 0) return TQ_OK;
  if (!workspace) return TQ_ENULL;
  if ((uintptr_t)workspace & 15) return TQ_EINVAL;
  a.q = q; a.starts = query_start_loc; a.rows = rows; a.B = B; a.Hq = Hq; a.G = Hq / Hkv; a.W = window;
  a.row_tiles = p.row_tiles; a.tile_waves = p.tile_waves; a.row_groups = p.row_groups; a.n_split = p.n_split; a.chunk = p.chunk; a.parts = p.parts;
  // (not zero: a hidden score of -inf stays one)
  a.scale2 = std::max(std::fabs(sm_scale) * 1.4426950408889634f, 1.17549435e-38f);
  a.flip = std::signbit(sm_scale) ? (dtype == TQ_F32 ? 0x80000000u : 0x80008000u) : 0u;
  a.waves = p.waves;
  a.per_head = (uint32_t)(((uint64_t)1 << 32) / (uint32_t)a.G + ((((uint64_t)1 << 32) % (uint32_t)a.G) != 0));
  a.ml = (float2*)((char*)workspace + p.ml_at);
  a.stat = (float2*)((char*)workspace + p.stat_at);
  a.weights = weights; a.w_b = w_b; a.w_h = w_h; a.L = (int)weight_len;
  hipStream_t st = (hipStream_t)stream;
  const auto pass = dtype == TQ_F32 ? launch_exact_window<TQ_F32> : (dtype == TQ_F16 ? launch_exact_window<TQ_F16> : launch_exact_window<TQ_BF16>);
  int done = pass(a, false, st);
  if (done) return done;
  const int padded = p.row_tiles * 16;
  exact_window_join_kernel<<<dim3((unsigned)((int64_t)B * Hkv * p.row_tiles)), dim3(256), 0, st>>>(a.ml, a.stat, p.parts, padded, a.c, p.block_tokens, p.n_split,
                                                                                                   p.chunk, p.waves / p.tile_waves);
  TQ_CHECK_LAUNCH();
  return pass(a, true, st);
}
