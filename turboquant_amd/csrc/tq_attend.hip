// Attention of a step's rows over a paged cache: the plan, the entry points, and the launch that joins splits.
#include "tq_attend.h"
#include "tq_join.h"

#include <algorithm>

namespace tq {

struct AttendJoin {
  const float2* ml;
  const float* acc;
  void* out;
  int64_t rows;            // token rows x heads
  int32_t n_split, d, fill;
};

// Splits that a row has (those without tokens are the last ones), -1 for a row of no sequence
__device__ __forceinline__ int attend_used(const AttendJoin& a, int64_t row) {
  const float2* ml = a.ml + row * a.n_split;
  const int lane = (int)threadIdx.x & 63;
  int used = 0;
  for (int i0 = 0; i0 < a.n_split; i0 += 64) {
    const float y = i0 + lane < a.n_split ? ml[i0 + lane].y : ATTEND_EMPTY;
    if (i0 == 0 && __builtin_amdgcn_readfirstlane(__float_as_int(y)) == __float_as_int(ATTEND_REST)) return -1;
    const int n = __popcll(__ballot(!(y < 0.0f)));
    used += n;
    if (n < 64) break;
  }
  return used;
}

template <int DT>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendJoin a) {
  __shared__ float s_f[JOIN_MAX_SPLITS];
  __shared__ float s_red[8];
  __shared__ float4 s_o[256];
  const int lane = (int)threadIdx.x & 63;
  if (a.n_split <= JOIN_FEW) {
    const int64_t row = (int64_t)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
    if (row >= a.rows) return;
    const float2 none = make_float2(-INFINITY, 0.0f);
    float2 ml = lane < a.n_split ? a.ml[row * a.n_split + lane] : make_float2(-INFINITY, ATTEND_EMPTY);
    const bool rest = __builtin_amdgcn_readfirstlane(__float_as_int(ml.y)) == __float_as_int(ATTEND_REST);
    if (rest && !a.fill) return;
    const bool there = !rest && !(ml.y < 0.0f);              // (a sum may be NaN)
    const int used = __popcll(__ballot(there));
    join_few<DT>(a.acc, a.n_split, a.d, a.out, row, used, there ? ml : none);
  } else {
    const int slices = a.d >> 6;
    const int64_t row = blockIdx.x / (unsigned)slices;
    int used = attend_used(a, row);
    if (used < 0) {
      if (!a.fill) return;
      used = 0;
    }
    join_many<DT>(a.ml, a.acc, a.n_split, a.d, a.out, row, used, (int)(blockIdx.x % (unsigned)slices), s_f, s_red, s_o);
  }
}

// ---- how a call is split ----------------------------------------------------------------------------------------------------------------
struct AttendPlan {
  int tiles;                          // column tiles of the kernel of few rows; 0: the kernel of many
  int64_t units, grid;
  int n_split, chunk;
  size_t ml_at, acc_at, bytes;
};

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// starts: whether the rows are the sequences' as starts say, up to max_rows of one (else one row each).  n_split 0: chosen here.
static bool attend_plan(AttendPlan* p, int dtype, int cache, bool starts, int64_t rows, int B, int Hq, int Hkv, int d, int64_t max_len, int64_t max_rows,
                        int64_t window, int sinks, int n_split) {
  if ((dtype != TQ_F16 && dtype != TQ_BF16) || (cache != dtype && cache != TQ_E4M3) || rows < 0 || rows > INT32_MAX || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv)
    return false;
  if ((d != 64 && d != 128 && d != 192 && d != 256) || max_len < 0 || max_len > INT32_MAX - 64 || max_rows < 0 || window < 0 || sinks < 0 || n_split < 0 ||
      n_split > JOIN_MAX_SPLITS || (!starts && rows != B))
    return false;
  const int G = Hq / Hkv;
  if (G > 1024) return false;
  max_rows = starts ? std::max<int64_t>(1, std::min(max_rows, rows)) : 1;
  p->tiles = max_rows * G <= 16 ? 1 : (max_rows * G <= 32 ? 2 : 0);
  const int M = p->tiles ? 16 * p->tiles : 128, TB = p->tiles ? 32 : 64;
  p->units = starts ? (rows * G + M - 1) / M + B + 1 : (int64_t)B * ((G + M - 1) / M);
  // (of these, up to B are not met, and most of a short row's are)
  const int64_t busy = starts ? std::max<int64_t>(std::min<int64_t>(B, rows), (rows * G + M - 1) / M) : p->units;
  const int64_t pairs = std::max<int64_t>(1, busy * Hkv);
  int64_t tokens = std::max<int64_t>(max_len, 1);
  if (window > 0 && window < tokens) tokens = std::min(tokens, window + max_rows + std::min<int64_t>(sinks, tokens) + TB);
  const int64_t blocks = (tokens + TB - 1) / TB;
  int64_t n = n_split;
  if (n == 0) {
    if (p->tiles) {
      // Workgroups enough for the bytes that have to be on their way: one for each compute unit where a turn of its four wavefronts is 64 KB, two where it
      // is less (us; fp8, d 128, 8 heads, one sequence of 131072: 32 splits 67.7, 64 64.4, 128 65.4, 256 65.0; d 256, 2 heads: 64 47.6, 128 36.6, 256 38.5, 384 46.6;
      // bf16, d 128, one of 65536: 16 75.7, 32 53.7, 64 58.5), no split of more than 2048 tokens (fp8, 32 of 8192: 1 138, 2 114.6, 4 106.4, 8 105.2), and of
      // the next numbers of splits, while they leave 512 tokens, the first that leaves no compute unit without work in its last round (24 of 6000: 3 70.9, 4 62.9).
      const int64_t turn = 4 * TB * 2 * d * (cache == TQ_E4M3 ? 1 : 2), target = turn >= 65536 ? 256 : 512;
      n = std::max((target + pairs - 1) / pairs, (tokens + 2047) / 2048);
      double best = 0;
      for (int64_t i = n; i <= 2 * n && i <= std::max(n, tokens / 512); ++i) {
        const double full = double(pairs * i) / (256 * ((pairs * i + 255) / 256));
        if (full > best + 0.02) { best = full; n_split = (int)std::min<int64_t>(i, JOIN_MAX_SPLITS); }
        if (best >= 0.95) break;
      }
      n = std::min<int64_t>(n_split, (blocks + 3) / 4);
      n_split = 0;
    } else {
      n = (256 * (d <= 128 ? 2 : 1) + pairs - 1) / pairs;
      n = std::min<int64_t>(std::min<int64_t>(n, (blocks + 3) / 4), JOIN_MAX_SPLITS);
    }
  }
  n = std::max<int64_t>(1, std::min(n, blocks));
  int64_t chunk = (blocks + n - 1) / n;
  if (n_split == 0 && p->tiles) chunk = (chunk + 3) & ~(int64_t)3;                             // (a block for each of the four wavefronts)
  p->n_split = (int)std::max<int64_t>(1, (blocks + chunk - 1) / chunk);
  p->chunk = (int)chunk;
  const size_t all = (size_t)rows * Hq;
  size_t at = 0;
  p->ml_at = at;      at = round256(at + all * p->n_split * sizeof(float2));
  p->acc_at = at;     at = round256(at + (p->n_split > 1 ? all * p->n_split * d * sizeof(float) : 0));
  p->bytes = std::max<size_t>(at, 256);
  p->grid = p->units * Hkv * p->n_split;
  return p->grid <= INT32_MAX && join_groups((int64_t)all, p->n_split, d) <= INT32_MAX;
}

}  // namespace tq

extern "C" size_t tq_attend_bytes(int dtype, int cache, int starts, int64_t rows, int B, int Hq, int Hkv, int d, int64_t max_len, int64_t max_rows,
                                  int64_t window, int sinks, int n_split) {
  tq::AttendPlan p;
  return tq::attend_plan(&p, dtype, cache, starts != 0, rows, B, Hq, Hkv, d, max_len, max_rows, window, sinks, n_split) ? p.bytes : 0;
}

extern "C" int tq_attend(const void* q, int dtype, int64_t rows, const int32_t* query_start_loc, int B, int Hq, int Hkv, int d, int cache, const void* k_cache,
                         const void* v_cache, const uint8_t* k_scales, const uint8_t* v_scales, int64_t cs_blk, int64_t cs_t, int64_t cs_h,
                         int64_t num_blocks, const int32_t* block_table, int bt_stride, const int32_t* seq_lens, float sm_scale, int64_t max_len,
                         int64_t max_rows, int64_t window, int sinks, void* out, int fill, void* workspace, int n_split, void* stream) {
  using namespace tq;
  if (!q || !out || !k_cache || !v_cache) return TQ_ENULL;
  AttendPlan p;
  if (!attend_plan(&p, dtype, cache, query_start_loc != nullptr, rows, B, Hq, Hkv, d, max_len, max_rows, window, sinks, n_split)) return TQ_EINVAL;
  Attend a{};
  if (const int rc = step_init(&a.s, query_start_loc, rows, B, seq_lens, block_table, bt_stride, num_blocks)) return rc;
  if (cache == TQ_E4M3) {
    Fp8Cache c;
    if (const int rc = fp8_cache_init(&c, (void*)k_cache, (void*)v_cache, (void*)k_scales, (void*)v_scales, Hkv, d, cs_blk, cs_t, cs_h)) return rc;
  } else {
    if (cs_blk < 0 || cs_t < 0 || cs_h < 0 || cs_t > (1 << 24) || cs_blk % 8 || cs_t % 8 || cs_h % 8 || (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15))
      return TQ_EUNSUPPORTED;
  }
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15)) return TQ_EUNSUPPORTED;
  if (rows == 0) return TQ_OK;
  if (!workspace) return TQ_ENULL;
  if ((uintptr_t)workspace & 15) return TQ_EINVAL;
  a.k = k_cache; a.v = v_cache; a.k_scales = k_scales; a.v_scales = v_scales; a.s_blk = cs_blk; a.s_h = cs_h; a.s_t = (int32_t)cs_t; a.H = Hkv; a.d = d;
  a.q = q; a.out = out; a.Hq = Hq; a.G = Hq / Hkv;
  a.window = window <= 0 || window > INT32_MAX ? ATTEND_ALL : (int32_t)window;
  a.sinks = sinks; a.n_split = p.n_split; a.chunk = p.chunk; a.fill = fill; a.scale2 = sm_scale * 1.4426950408889634f;
  a.units = p.units;
  a.ml = (float2*)((char*)workspace + p.ml_at);
  a.acc = (float*)((char*)workspace + p.acc_at);
  hipStream_t st = (hipStream_t)stream;
  int rc;
  const unsigned g = (unsigned)p.grid;
  if (p.tiles) {
    if (cache == TQ_E4M3) rc = dtype == TQ_F16 ? launch_attend_few<TQ_F16, true>(a, p.tiles, g, st) : launch_attend_few<TQ_BF16, true>(a, p.tiles, g, st);
    else rc = dtype == TQ_F16 ? launch_attend_few<TQ_F16, false>(a, p.tiles, g, st) : launch_attend_few<TQ_BF16, false>(a, p.tiles, g, st);
  } else {
    if (cache == TQ_E4M3) rc = dtype == TQ_F16 ? launch_attend_rows<TQ_F16, true>(a, g, st) : launch_attend_rows<TQ_BF16, true>(a, g, st);
    else rc = dtype == TQ_F16 ? launch_attend_rows<TQ_F16, false>(a, g, st) : launch_attend_rows<TQ_BF16, false>(a, g, st);
  }
  if (rc || p.n_split == 1) return rc;
  const AttendJoin j{a.ml, a.acc, out, rows * Hq, p.n_split, d, fill};
  const dim3 grid((unsigned)join_groups(j.rows, p.n_split, d)), block(256);
  if (dtype == TQ_F16) attend_join_kernel<TQ_F16><<<grid, block, 0, st>>>(j);
  else attend_join_kernel<TQ_BF16><<<grid, block, 0, st>>>(j);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
