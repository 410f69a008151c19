// A window's weights over a paged exact cache: entry points, and the launch that joins the parts of a row.
#include "tq_exact_window.h"

#include <algorithm>

namespace tq {

// stat[r] = (M, 1 / sum_i 2^(m_i - M) l_i) over the parts of a row; a row that sees nothing has no weight to give
__global__ void __launch_bounds__(256) exact_window_join_kernel(const float2* ml, float2* stat, int parts, int padded, int64_t rows,
                                                                ExactCache c, int block_tokens, int n_split, int chunk, int token_waves) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * padded) return;
  const int64_t row = i / padded;
  const int r = (int)(i - row * padded), len = exact_len(c, (int)(row / c.H));
  const int used = exact_splits_used((len + block_tokens - 1) / block_tokens, n_split, chunk) * token_waves;
  float top = -INFINITY, sum = 0.0f;
  for (int p = 0; p < used; ++p) top = fmaxf(top, ml[(row * parts + p) * padded + r].x);
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int p = 0; p < used; ++p) {
    const float2 x = ml[(row * parts + p) * padded + r];
    sum += x.y * __builtin_amdgcn_exp2f(x.x - ref);
  }
  stat[i] = make_float2(ref, sum == 0.0f ? 0.0f : 1.0f / sum);
}

struct WindowPlan {
  int row_tiles, tile_waves, row_groups, n_split, chunk, block_tokens, parts;
  size_t ml_at, stat_at, bytes;
};

static bool window_plan(WindowPlan* p, int dtype, int B, int Hq, int Hkv, int d, int W, int64_t max_len) {
  if (dtype < TQ_F32 || dtype > TQ_BF16 || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || d <= 0 || d % 64 || d > 768) return false;
  if (W <= 0 || W > 1024 || max_len < 0 || max_len > INT32_MAX - 64 || Hq / Hkv > 1024) return false;
  const int G = Hq / Hkv, NT = window_tiles(dtype, d);
  p->block_tokens = dtype == TQ_F32 ? 16 : 32;
  p->row_tiles = (W * G + 15) / 16;
  p->tile_waves = p->row_tiles > 2 * NT ? 4 : (p->row_tiles > NT ? 2 : 1);
  p->row_groups = (p->row_tiles + p->tile_waves * NT - 1) / (p->tile_waves * NT);
  const int64_t blocks = std::max<int64_t>(1, (max_len + p->block_tokens - 1) / p->block_tokens);
  const int64_t pairs = std::max<int64_t>(1, (int64_t)B * Hkv);
  const int64_t token_waves = 4 / p->tile_waves;
  // four workgroups a compute unit of the second pass, up to 1024 tokens each; a block for every wavefront of a workgroup at least
  int64_t n = std::max((1024 + pairs - 1) / pairs, (max_len + 1023) / 1024);
  n = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(n, (blocks + 4 * token_waves - 1) / (4 * token_waves)), 4096));
  const int64_t chunk = (blocks + n - 1) / n;
  p->chunk = (int)chunk;
  p->n_split = (int)((blocks + chunk - 1) / chunk);
  p->parts = (int)(p->n_split * token_waves);
  const size_t rows = (size_t)B * Hkv * p->row_tiles * 16;
  p->ml_at = 0;
  p->stat_at = (rows * p->parts * sizeof(float2) + 255) & ~(size_t)255;
  p->bytes = p->stat_at + std::max<size_t>(256, (rows * sizeof(float2) + 255) & ~(size_t)255);
  return pairs * p->n_split * p->row_groups <= INT32_MAX && (int64_t)((rows + 255) / 256) <= INT32_MAX;
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
  a.scale2 = sm_scale * 1.4426950408889634f;
  a.ml = (float2*)((char*)workspace + p.ml_at);
  a.stat = (float2*)((char*)workspace + p.stat_at);
  a.weights = weights; a.w_b = w_b; a.w_h = w_h; a.L = (int)weight_len;
  hipStream_t st = (hipStream_t)stream;
  const auto pass = dtype == TQ_F32 ? launch_exact_window<TQ_F32> : (dtype == TQ_F16 ? launch_exact_window<TQ_F16> : launch_exact_window<TQ_BF16>);
  int done = pass(a, false, st);
  if (done) return done;
  const int padded = p.row_tiles * 16;
  const int64_t all = (int64_t)B * Hkv * padded;
  exact_window_join_kernel<<<dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st>>>(a.ml, a.stat, p.parts, padded, (int64_t)B * Hkv, a.c, p.block_tokens,
                                                                                      p.n_split, p.chunk, 4 / p.tile_waves);
  TQ_CHECK_LAUNCH();
  return pass(a, true, st);
}
