// Decode attention over a paged exact cache: entry points, and the launch that joins splits and adds weights.
#include "tq_exact.h"
#include "tq_join.h"

#include <algorithm>

namespace tq {

// ---- splits -> outputs, scores -> weights ---------------------------------------------------------------------------------------------
// Rows (the first workgroups of the grid, none with a single split): out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i over a row's splits.
// Weights: weights[b, h, t] += sum over the heads of h of 2^(s_t - M) / sum, a thread per token, heads in order: no atomics, the same
// result every time.  Both only need what the page kernel left, so that they share a launch.  Bound by the chain of length, maxima, sums and numerators:
// 16 x 32 rows of four splits with the weights of 16 x 8 x 8192 tokens (25 MB) 8.2 us; 96 x 40 rows with those of 96 x 8 x 61 .. 8190 (44 MB) 18 - 20.
__device__ __forceinline__ int join_len(const ExactJoin& a, int b) {
  const int64_t most = (int64_t)a.table_row * TQ_PAGE_TOKENS;
  const int n = a.lens[b];
  return n < 0 ? 0 : (n > most ? (int)most : n);
}
__device__ __forceinline__ int join_used(const ExactJoin& a, int len) {
  return exact_splits_used((len + a.block_tokens - 1) / a.block_tokens, a.n_split, a.chunk);
}
// A thread's four tokens are neighbours: sixteen bytes of each head's scores.
__device__ __forceinline__ void exact_add_weights(const ExactJoin& a, int id, float2* s_head) {
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int chunk = id % a.weight_chunks; id /= a.weight_chunks;
  const int h = id % a.H, b = id / a.H;
  const int held = join_len(a, b), len = held < a.L ? held : a.L;
  const int t0 = chunk * a.weight_tokens;
  if (t0 >= len) return;
  const int used = join_used(a, held);
  for (int g = wave; g < a.G; g += 4) {
    const float2* ml = a.ml + ((int64_t)b * a.Hq + h * a.G + g) * a.n_split;
    float2 x = lane < used ? ml[lane] : make_float2(-INFINITY, 0.0f);
    float top = x.x;
    for (int i = lane + 64; i < used; i += 64) top = fmaxf(top, ml[i].x);
    top = wave_max_fast(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = x.y * __builtin_amdgcn_exp2f(x.x - ref);
    for (int i = lane + 64; i < used; i += 64) sum += ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - ref);
    sum = wave_sum_fast(sum);
    if (lane == 0) s_head[g] = make_float2(ref, sum == 0.0f ? 0.0f : 1.0f / sum);
  }
  __syncthreads();
  for (int t = t0 + tid * 4; t < t0 + a.weight_tokens && t < len; t += 1024) {
    const float* s = a.scores + (((int64_t)b * a.H + h) * a.score_pages + (t >> 4)) * a.G * TQ_PAGE_TOKENS + (t & 15);
    float4 add = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int g = 0; g < a.G; ++g) {
      const float4 x = *(const float4*)(s + g * TQ_PAGE_TOKENS);
      const float2 r = s_head[g];
      add.x = fmaf(__builtin_amdgcn_exp2f(x.x - r.x), r.y, add.x);
      add.y = fmaf(__builtin_amdgcn_exp2f(x.y - r.x), r.y, add.y);
      add.z = fmaf(__builtin_amdgcn_exp2f(x.z - r.x), r.y, add.z);
      add.w = fmaf(__builtin_amdgcn_exp2f(x.w - r.x), r.y, add.w);
    }
    float* w = a.weights + b * a.w_b + h * a.w_h + t;
    const int n = len - t;
    w[0] += add.x;
    if (n > 1) w[1] += add.y;
    if (n > 2) w[2] += add.z;
    if (n > 3) w[3] += add.w;
  }
}

template <int DT>
__global__ void __launch_bounds__(256) exact_join_kernel(const ExactJoin a, int row_groups) {
  __shared__ float2 s_two[JOIN_MAX_SPLITS];
  __shared__ float s_red[8];
  __shared__ float4 s_o[256];
  int id = (int)blockIdx.x;
  if (id >= row_groups) {
    exact_add_weights(a, id - row_groups, s_two);
  } else if (a.n_split <= JOIN_FEW) {
    id = id * 4 + ((int)threadIdx.x >> 6);
    if (id < a.B * a.Hq) {
      const int lane = (int)threadIdx.x & 63, used = join_used(a, join_len(a, id / a.Hq));
      join_few<DT>(a.acc + (int64_t)id * a.n_split * a.d, a.d, a.d, a.out, id, used, lane < used ? a.ml[(int64_t)id * a.n_split + lane] : make_float2(-INFINITY, 0.0f));
    }
  } else {
    const int slices = a.d >> 6;
    const int row = id / slices;
    join_many<DT>(a.ml + (int64_t)row * a.n_split, 1, a.acc + (int64_t)row * a.n_split * a.d, a.d, a.d, a.out, row, join_used(a, join_len(a, row / a.Hq)), id % slices, (float*)s_two, s_red, s_o);
  }
}

// Tokens of a weight workgroup: more than 1024 only where that leaves 2048 workgroups (a workgroup that finds its part of a short sequence empty
// still has to be dispatched: 96 sequences of 61 .. 8190 tokens, 8 KV heads: 26 us with 6144 workgroups, 20 with 2304)
static int64_t join_tokens(int64_t pairs, int64_t len) {
  const int64_t groups = pairs * ((len + 1023) / 1024);
  return 1024 * std::max<int64_t>(1, std::min<int64_t>(groups / 2048, 64));
}

// ---- how a call is split ----------------------------------------------------------------------------------------------------------------
struct ExactPlan {
  bool shared;                        // the kernel of 64 heads, not that of sixteen
  int groups, n_split, chunk, block_tokens, score_pages, weight_tokens;
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
  const int tiles = (G + EXACT_HEADS - 1) / EXACT_HEADS;
  // More than sixteen heads share their reads where the passes over the cache that this saves outweigh a start that is 2-4 us longer: from 64 MB, all
  // heads' passes together (bf16, one KV head, sixteen / 64 heads a workgroup; one sequence of 16384, 32 heads: d 128 17 MB 10.1 / 12.7 us, d 448 59 MB
  // 20.5 / 24.1, d 576 75 MB 27.1 / 24.4; 16 of 8192: 32 heads of 128 134 MB 22.8 / 23.7, 48 heads of 128 201 MB 25.9 / 26.2, of 192 302 MB 45 / 36, of 576
  // 906 MB 286 / 82).  d = 64 with 32 heads: 16.2 / 19.7 at 67 MB, never.
  const int64_t passes = (int64_t)tiles * d * 4 * std::max<int64_t>(1, (int64_t)B * Hkv);
  const bool shared = dtype != TQ_F32 && tiles > 1 && d <= 576 && (d > 64 || tiles > 2) && max_len > (int64_t(64) << 20) / passes;
  p->shared = shared;
  p->groups = shared ? (tiles + 3) / 4 : tiles;
  const int64_t pairs = std::max<int64_t>(1, (int64_t)B * Hkv * p->groups);
  const int64_t blocks = std::max<int64_t>(1, (max_len + p->block_tokens - 1) / p->block_tokens);
  // As many workgroups as the card holds, and no split of more than 1024 tokens: sequences differ in length (64 of up to 4096, 32 / 8 heads of 128: one
  // split 146 us, two 133, four 124, eight 124; all of 4096: 191.5, 190, 191, 197; four of 65536: 24 splits 213, 64 197).  The kernel of 64 heads fills the card
  // once: its splits are dear to join.
  int64_t n = n_split;
  if (n == 0) {
    const int64_t resident = 256 * (shared ? (d > 256 ? 1 : 2) : (d <= 64 ? 4 : (d <= 128 ? 3 : (d <= 256 ? 2 : 1))));
    n = std::max((resident + pairs - 1) / pairs, (max_len + 1023) / 1024);
    if (shared) n = (resident + pairs - 1) / pairs;
    n = std::min<int64_t>(std::min<int64_t>(n, (blocks + 3) / 4), JOIN_MAX_SPLITS);
  }
  n = std::max<int64_t>(1, std::min(n, blocks));
  int64_t chunk = (blocks + n - 1) / n;
  if (n_split == 0 && !shared) chunk = (chunk + 3) & ~(int64_t)3;                  // (a block for each of the four wavefronts)
  p->n_split = (int)std::max<int64_t>(1, (blocks + chunk - 1) / chunk);
  p->chunk = (int)chunk;
  p->weight_tokens = (int)join_tokens((int64_t)B * Hkv, score_len);
  p->score_pages = (int)((score_len + TQ_PAGE_TOKENS - 1) / TQ_PAGE_TOKENS);
  const size_t rows = (size_t)B * Hq;
  size_t at = 0;
  p->ml_at = at;      at = round256(at + rows * p->n_split * sizeof(float2));
  p->acc_at = at;     at = round256(at + (p->n_split > 1 ? rows * p->n_split * d * sizeof(float) : 0));
  p->scores_at = at;  at = round256(at + (size_t)B * Hkv * p->score_pages * G * TQ_PAGE_TOKENS * sizeof(float));
  p->bytes = at;
  const int64_t grid = (pairs * p->n_split + 8 * p->groups), join = join_groups((int64_t)rows, p->n_split, d) + (int64_t)B * Hkv * ((score_len + p->weight_tokens - 1) / p->weight_tokens);
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
  int done;
  if (p.shared)
    done = dtype == TQ_F16 ? launch_exact_heads<TQ_F16>(a, st) : launch_exact_heads<TQ_BF16>(a, st);
  else
    done = dtype == TQ_F32 ? launch_exact_decode<TQ_F32>(a, st)
                           : (dtype == TQ_F16 ? launch_exact_decode<TQ_F16>(a, st) : launch_exact_decode<TQ_BF16>(a, st));
  if (done) return done;
  if (p.n_split == 1 && !p.score_pages) return TQ_OK;
  ExactJoin j{};
  j.lens = seq_lens; j.table_row = a.c.table_row; j.B = B; j.Hq = Hq; j.H = Hkv; j.G = a.G; j.d = d; j.n_split = p.n_split; j.chunk = p.chunk;
  j.block_tokens = p.block_tokens; j.acc = a.acc; j.ml = a.ml; j.out = out; j.scores = a.scores; j.score_pages = p.score_pages;
  j.weights = weights; j.w_b = w_b; j.w_h = w_h; j.L = p.score_pages ? (int)weight_len : 0;
  j.weight_tokens = p.weight_tokens;
  j.weight_chunks = (j.L + j.weight_tokens - 1) / j.weight_tokens;
  const int rows = (int)join_groups((int64_t)B * Hq, p.n_split, d);
  const dim3 grid((unsigned)(rows + (int64_t)B * Hkv * j.weight_chunks)), block(256);
  if (dtype == TQ_F32) exact_join_kernel<TQ_F32><<<grid, block, 0, st>>>(j, rows);
  else if (dtype == TQ_F16) exact_join_kernel<TQ_F16><<<grid, block, 0, st>>>(j, rows);
  else exact_join_kernel<TQ_BF16><<<grid, block, 0, st>>>(j, rows);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
