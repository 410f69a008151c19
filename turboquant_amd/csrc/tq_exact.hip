// Decode attention over a paged exact cache: entry points, and the launch that joins splits and adds weights.
#include "tq_exact.h"

#include <algorithm>

namespace tq {

// ---- splits -> outputs, scores -> weights ---------------------------------------------------------------------------------------------
// Row workgroups (first of the grid, none with a single split): out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i over a row's splits.
// Weight workgroups: weights[b, h, t] += sum over the heads of h of 2^(s_t - M) / sum, a thread per token, heads in order: no atomics, the same
// result every time.  Both only need what the page kernel left, so that they share a launch.
constexpr int JOIN_MAX_SPLITS = 1024, JOIN_TOKENS = 1024;

template <int DT>
__device__ __forceinline__ void exact_join_row(const ExactJoin& a, int row, float* s_f, float* s_red) {
  const int tid = (int)threadIdx.x, b = row / a.Hq;
  const int64_t most = (int64_t)a.table_row * TQ_PAGE_TOKENS;
  const int n = a.lens[b], len = n < 0 ? 0 : (n > most ? (int)most : n);
  const int used = exact_splits_used((len + a.block_tokens - 1) / a.block_tokens, a.n_split, a.chunk);
  const float2* ml = a.ml + (int64_t)row * a.n_split;
  // (every thread for itself: the maximum and the sum are a few hundred values of the L1)
  float top = -INFINITY;
  for (int i = tid; i < used; i += 256) top = fmaxf(top, ml[i].x);
  top = wave_max_fast(top);
  if ((tid & 63) == 0) s_red[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int i = tid; i < used; i += 256) {
    const float f = __builtin_amdgcn_exp2f(ml[i].x - ref);
    s_f[i] = f;
    sum += f * ml[i].y;
  }
  sum = wave_sum_fast(sum);
  __syncthreads();
  if ((tid & 63) == 0) s_red[tid >> 6] = sum;
  __syncthreads();
  sum = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;

  // four channels per thread; as many threads as are left share the splits
  const int quads = a.d >> 2, shares = 256 / quads, share = tid / quads, quad = tid - share * quads;
  float4 o = make_float4(0, 0, 0, 0);
  if (share < shares) {
    const float4* acc = (const float4*)(a.acc + (int64_t)row * a.n_split * a.d) + quad;
    for (int i = share; i < used; i += shares) {
      const float4 x = acc[(int64_t)i * quads];
      const float f = s_f[i];
      o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
    }
  }
  __shared__ float4 s_o[256];
  s_o[tid] = o;
  __syncthreads();
  if (share != 0) return;
  for (int i = 1; i < shares; ++i) {
    const float4 x = s_o[i * quads + quad];
    o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
  }
  const int64_t at = (int64_t)row * a.d + quad * 4;
  Elem<DT>::store(a.out, at, o.x * inv);
  Elem<DT>::store(a.out, at + 1, o.y * inv);
  Elem<DT>::store(a.out, at + 2, o.z * inv);
  Elem<DT>::store(a.out, at + 3, o.w * inv);
}

__device__ __forceinline__ void exact_add_weights(const ExactJoin& a, int id, float2* s_head) {
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int chunk = id % a.weight_chunks; id /= a.weight_chunks;
  const int h = id % a.H, b = id / a.H;
  const int64_t most = (int64_t)a.table_row * TQ_PAGE_TOKENS;
  const int n = a.lens[b], held = n < 0 ? 0 : (n > most ? (int)most : n);
  const int len = held < a.L ? held : a.L;
  const int t0 = chunk * JOIN_TOKENS;
  if (t0 >= len) return;
  const int used = exact_splits_used((held + a.block_tokens - 1) / a.block_tokens, a.n_split, a.chunk);
  for (int g = wave; g < a.G; g += 4) {
    const float2* ml = a.ml + ((int64_t)b * a.Hq + h * a.G + g) * a.n_split;
    float top = -INFINITY, sum = 0.0f;
    for (int i = lane; i < used; i += 64) top = fmaxf(top, ml[i].x);
    top = wave_max_fast(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    for (int i = lane; i < used; i += 64) sum += ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - ref);
    sum = wave_sum_fast(sum);
    if (lane == 0) s_head[g] = make_float2(ref, sum == 0.0f ? 0.0f : 1.0f / sum);
  }
  __syncthreads();
  float* w = a.weights + b * a.w_b + h * a.w_h;
  for (int t = t0 + tid; t < t0 + JOIN_TOKENS && t < len; t += 256) {
    const float* s = a.scores + (((int64_t)b * a.H + h) * a.score_pages + (t >> 4)) * a.G * TQ_PAGE_TOKENS + (t & 15);
    float add = 0.0f;
    for (int g = 0; g < a.G; ++g) add += __builtin_amdgcn_exp2f(s[g * TQ_PAGE_TOKENS] - s_head[g].x) * s_head[g].y;
    w[t] += add;
  }
}

template <int DT>
__global__ void __launch_bounds__(256) exact_join_kernel(const ExactJoin a, int rows) {
  __shared__ float2 s_two[JOIN_MAX_SPLITS];
  __shared__ float s_red[4];
  const int id = (int)blockIdx.x;
  if (id < rows) exact_join_row<DT>(a, id, (float*)s_two, s_red);
  else exact_add_weights(a, id - rows, s_two);
}

// ---- how a call is split ----------------------------------------------------------------------------------------------------------------
struct ExactPlan {
  int groups, n_split, chunk, block_tokens, score_pages;
  size_t ml_at, acc_at, scores_at, bytes;
};

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// n_split 0: chosen here.  score_len: tokens whose weights are wanted (0: none).  false: out of range.
static bool exact_plan(ExactPlan* p, int dtype, int B, int Hq, int Hkv, int d, int64_t max_len, int n_split, int64_t score_len) {
  if (dtype < TQ_F32 || dtype > TQ_BF16 || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || d <= 0 || d % 64 || d > 768) return false;
  if (max_len < 0 || max_len > INT32_MAX - 64 || n_split < 0 || n_split > JOIN_MAX_SPLITS || score_len < 0 || score_len > INT32_MAX - 64) return false;
  const int G = Hq / Hkv;
  if (G > JOIN_MAX_SPLITS) return false;
  p->block_tokens = dtype == TQ_F32 ? 16 : 32;
  p->groups = (G + EXACT_HEADS - 1) / EXACT_HEADS;
  const int64_t pairs = std::max<int64_t>(1, (int64_t)B * Hkv * p->groups);
  const int64_t blocks = std::max<int64_t>(1, (max_len + p->block_tokens - 1) / p->block_tokens);
  int64_t n = n_split;
  if (n == 0) {
    const int64_t resident = 256 * (d <= 64 ? 4 : (d <= 128 ? 3 : (d <= 256 ? 2 : 1)));
    n = std::max((resident + pairs - 1) / pairs, (max_len + 1023) / 1024);
    n = std::min<int64_t>(std::min<int64_t>(n, (blocks + 3) / 4), JOIN_MAX_SPLITS);
  }
  n = std::max<int64_t>(1, std::min(n, blocks));
  int64_t chunk = (blocks + n - 1) / n;
  if (n_split == 0) chunk = (chunk + 3) & ~(int64_t)3;                  // (a block for each of the four wavefronts)
  p->n_split = (int)std::max<int64_t>(1, (blocks + chunk - 1) / chunk);
  p->chunk = (int)chunk;
  p->score_pages = (int)((score_len + TQ_PAGE_TOKENS - 1) / TQ_PAGE_TOKENS);
  const size_t rows = (size_t)B * Hq;
  size_t at = 0;
  p->ml_at = at;      at = round256(at + rows * p->n_split * sizeof(float2));
  p->acc_at = at;     at = round256(at + (p->n_split > 1 ? rows * p->n_split * d * sizeof(float) : 0));
  p->scores_at = at;  at = round256(at + (size_t)B * Hkv * p->score_pages * G * TQ_PAGE_TOKENS * sizeof(float));
  p->bytes = at;
  const int64_t grid = (pairs * p->n_split + 8 * p->groups), join = (int64_t)rows + (int64_t)B * Hkv * ((score_len + JOIN_TOKENS - 1) / JOIN_TOKENS);
  return grid <= INT32_MAX && join <= INT32_MAX;
}

int exact_cache_init(ExactCache* c, const void* k, const void* v, int dtype, int H, int d, int64_t s_blk, int64_t s_t, int64_t s_h, int64_t num_blocks,
                     const int32_t* table, int bt_stride, const int32_t* lens) {
  if (!k || !v || !table || !lens) return TQ_ENULL;
  if (dtype < TQ_F32 || dtype > TQ_BF16 || H <= 0 || d <= 0 || num_blocks <= 0 || bt_stride == 0 || bt_stride == INT32_MIN) return TQ_EINVAL;
  const int64_t per16 = dtype == TQ_F32 ? 4 : 8;                        // elements of a 16-byte piece
  if (s_blk < 0 || s_t < 0 || s_h < 0 || s_t > (1 << 24)) return TQ_EUNSUPPORTED;
  if (s_blk % per16 || s_t % per16 || s_h % per16 || (((uintptr_t)k | (uintptr_t)v) & 15)) return TQ_EUNSUPPORTED;
  c->k = k; c->v = v; c->s_blk = s_blk; c->s_h = s_h; c->s_t = (int32_t)s_t; c->H = H; c->d = d; c->num_blocks = num_blocks;
  c->table = table; c->lens = lens;
  c->table_row = bt_stride < 0 ? -bt_stride : bt_stride;
  c->table_step = bt_stride < 0 ? 0 : bt_stride;
  return TQ_OK;
}

}  // namespace tq

extern "C" size_t tq_exact_decode_bytes(int dtype, int B, int Hq, int Hkv, int d, int64_t max_len, int n_split, int64_t weight_len) {
  tq::ExactPlan p;
  return tq::exact_plan(&p, dtype, B, Hq, Hkv, d, max_len, n_split, weight_len) ? p.bytes : 0;
}

extern "C" int tq_exact_decode(const void* q, int dtype, int B, int Hq, int Hkv, int d, const void* k_cache, const void* v_cache, int64_t cs_blk,
                               int64_t cs_t, int64_t cs_h, int64_t num_blocks, const int32_t* block_table, int bt_stride, const int32_t* seq_lens,
                               float sm_scale, int64_t max_len, float* weights, int64_t w_b, int64_t w_h, int64_t weight_len, void* out,
                               void* workspace, int n_split, void* stream) {
  using namespace tq;
  if (!q || !out) return TQ_ENULL;
  ExactPlan p;
  if (!exact_plan(&p, dtype, B, Hq, Hkv, d, max_len, n_split, weights ? weight_len : 0)) return TQ_EINVAL;
  ExactDecode a{};
  const int rc = exact_cache_init(&a.c, k_cache, v_cache, dtype, Hkv, d, cs_blk, cs_t, cs_h, num_blocks, block_table, bt_stride, seq_lens);
  if (rc) return rc;
  if (weights && (w_b < 0 || w_h < 0)) return TQ_EINVAL;
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15)) return TQ_EUNSUPPORTED;
  if (B == 0) return TQ_OK;
  if (!workspace) return TQ_ENULL;
  if ((uintptr_t)workspace & 15) return TQ_EINVAL;
  char* ws = (char*)workspace;
  a.q = q; a.out = out; a.B = B; a.Hq = Hq; a.G = Hq / Hkv; a.groups = p.groups; a.n_split = p.n_split; a.chunk = p.chunk;
  a.scale2 = sm_scale * 1.4426950408889634f;
  a.ml = (float2*)(ws + p.ml_at);
  a.acc = (float*)(ws + p.acc_at);
  a.scores = p.score_pages ? (float*)(ws + p.scores_at) : nullptr;
  a.score_pages = p.score_pages;
  hipStream_t st = (hipStream_t)stream;
  const int done = dtype == TQ_F32 ? launch_exact_decode<TQ_F32>(a, st)
                                   : (dtype == TQ_F16 ? launch_exact_decode<TQ_F16>(a, st) : launch_exact_decode<TQ_BF16>(a, st));
  if (done) return done;
  if (p.n_split == 1 && !p.score_pages) return TQ_OK;
  ExactJoin j{};
  j.lens = seq_lens; j.table_row = a.c.table_row; j.B = B; j.Hq = Hq; j.H = Hkv; j.G = a.G; j.d = d; j.n_split = p.n_split; j.chunk = p.chunk;
  j.block_tokens = p.block_tokens; j.acc = a.acc; j.ml = a.ml; j.out = out; j.scores = a.scores; j.score_pages = p.score_pages;
  j.weights = weights; j.w_b = w_b; j.w_h = w_h; j.L = p.score_pages ? (int)weight_len : 0;
  j.weight_chunks = (j.L + JOIN_TOKENS - 1) / JOIN_TOKENS;
  const int rows = p.n_split > 1 ? B * Hq : 0;
  const dim3 grid((unsigned)(rows + B * Hkv * j.weight_chunks)), block(256);
  if (dtype == TQ_F32) exact_join_kernel<TQ_F32><<<grid, block, 0, st>>>(j, rows);
  else if (dtype == TQ_F16) exact_join_kernel<TQ_F16><<<grid, block, 0, st>>>(j, rows);
  else exact_join_kernel<TQ_BF16><<<grid, block, 0, st>>>(j, rows);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
