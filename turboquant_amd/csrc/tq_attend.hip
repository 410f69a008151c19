// Attention of a step's rows over a paged cache: the plan, the entry points, and the launch that joins splits.
#include "tq_attend.h"
#include "tq_join.h"

#include <algorithm>

namespace tq {

struct AttendJoin {
  const int2* shares;
  const float2* ml;
  const float* acc;
  void* out;
  int64_t rows;            // token rows x heads
  int32_t H, d, few, n_split, part, parts, cap;
};

// A row's shares, and where they lie.  (Rows whose starts do not ascend may have been nobody's work: what lies in their place is no share.)
struct AttendRow {
  int used;
  int64_t first, apart;
  __device__ __forceinline__ AttendRow(const AttendJoin& a, const int2& s, int64_t row) {
    used = s.y & 0xffff;
    if (s.y >> 24) {
      if (used > a.n_split) used = 0;
      first = row * a.n_split;
      apart = 1;
    } else {
      const int r = s.y >> 16 & 0xff;
      if (used > a.cap || r >= a.part || s.x < 0 || s.x + (int64_t)(used - 1) * a.H >= (int64_t)a.parts * a.H) used = 0;
      first = (int64_t)s.x * a.part + r;
      apart = (int64_t)a.H * a.part;
    }
  }
};

// A wavefront for each `few` rows, one after another; or (0) a workgroup per row and 64 channels.
template <int DT>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendJoin a) {
  __shared__ float s_f[JOIN_MAX_SPLITS];
  __shared__ float s_red[8];
  __shared__ float4 s_o[256];
  const int lane = (int)threadIdx.x & 63;
  if (a.few) {
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + ((int)threadIdx.x >> 6)) * a.few;
    int2 mine = make_int2(0, 0);
    if (lane < a.few && row0 + lane < a.rows) mine = a.shares[row0 + lane];
    // (fewer than two: there already, or a row of no sequence)
    for (uint64_t left = __ballot((mine.y & 0xffff) > 1); left; left &= left - 1) {
      const int i = __ffsll((unsigned long long)left) - 1;
      const AttendRow r(a, make_int2(__builtin_amdgcn_readlane(mine.x, i), __builtin_amdgcn_readlane(mine.y, i)), row0 + i);
      if (r.used < 2) continue;
      const float2 ml = lane < r.used ? a.ml[r.first + lane * r.apart] : make_float2(-INFINITY, 0.0f);
      join_few<DT, 16>(a.acc + r.first * a.d, r.apart * a.d, a.d, a.out, row0 + i, r.used, ml);
    }
  } else {
    const int slices = a.d >> 6;
    const int64_t row = blockIdx.x / (unsigned)slices;
    const int2 s = a.shares[row];
    const AttendRow r(a, make_int2(__builtin_amdgcn_readfirstlane(s.x), __builtin_amdgcn_readfirstlane(s.y)), row);
    if (r.used < 2) return;
    join_many<DT>(a.ml + r.first, r.apart, a.acc + r.first * a.d, r.apart * a.d, a.d, a.out, row, r.used, (int)(blockIdx.x % (unsigned)slices), s_f, s_red, s_o);
  }
}

// ---- how a call is split ----------------------------------------------------------------------------------------------------------------
struct AttendPlan {
  int tiles;                          // column tiles of the kernel of few rows; 0: the kernel of many
  int64_t units, items, grid;
  int n_split, chunk, target, cap, few, part, parts;
  size_t shares_at, ml_at, acc_at, bytes;
};

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// starts: whether the rows are the sequences' as starts say, up to max_rows of one (else one row each).  n_split 0: chosen here.
// Splits of the tokens of units of 128 rows: the least of what the model says they take, in us.  A turn is 1.15 (128 channels, a workgroup on a compute unit; up to the
// other half of them 1.35, since some get two; two on all of them 2.05, so that the second gains little; 192 and 256 channels have one, 1.2), and a join is a launch and the
// partial results' way out and back, 5 and 1 for 2 MB.  No split has less than four turns of 128 channels.  Measured (us; bf16, 32 query heads on 8 of 128, one sequence, 1 / 2 / 4 / 8 / 16 splits): 512
// tokens, 512 rows 20 / 26 / 31 / 39; 1024, 1024 30 / 41 / 54 / 64; 4096, 64 rows 82 / 50 / 32 / 24 / 23, 512 rows 82 / 71 / 58 / 64 / 89; 16384, 64 rows
// 309 / 165 / 90 / 54 / 42, 512 rows 305 / 199 / 152 / 158 / 175, 2048 rows 483 / 541 / 553 / 587 / 674.  Other types and sizes go by the same numbers: bf16 and 8 bits, bf16 and fp16 queries, 64, 128 and 256 channels, 512
// rows of 512, 64 and 512 of 4096 and 16384: never more than 9 % above the best of 1 .. 32 splits; 64 rows of 2048 at 256 channels, where the bound of four turns leaves four, 35 (fp16 queries over 8 bits 47) for 30 (35) with eight.
static int64_t attend_rows_splits(int64_t pairs, int64_t blocks, int64_t rows, int d) {
  const int64_t most = std::min<int64_t>(blocks * 128 / (4 * std::max(d, 128)), JOIN_MAX_SPLITS);
  const double channels = d / 128.0, mb = (double)rows * d * 4e-6;
  int64_t best = 1;
  double least = 0;
  for (int64_t n = 1; n <= std::max<int64_t>(most, 1); ++n) {
    const int64_t groups = pairs * n, turns = (blocks + n - 1) / n;
    double turn = groups <= 128 ? 1.15 : (groups <= 256 ? 1.35 : 2.05 * (double)((groups + 511) / 512));
    if (d > 128) turn = 1.2 * (double)((groups + 255) / 256);
    const double us = (double)turns * turn * channels + (n > 1 ? 5 + 0.5 * mb * (double)n : 0);
    if (n == 1 || us < least) { best = n; least = us; }
    if (groups > 512) break;                                 // (behind two on all compute units more of them are more rounds)
  }
  return best;
}

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
  // (every sequence with rows may have a last unit that is not full)
  const int64_t units = std::max<int64_t>(1, starts ? (rows * G + std::min<int64_t>(B, rows) * (M - 1)) / M : (int64_t)B * ((G + M - 1) / M));
  // (of these, up to B are not met, and most of a short row's are)
  const int64_t busy = starts ? std::max<int64_t>(std::min<int64_t>(B, rows), (rows * G + M - 1) / M) : units;
  const int64_t pairs = std::max<int64_t>(1, busy * Hkv);
  int64_t tokens = std::max<int64_t>(max_len, 1);
  if (window > 0 && window < tokens) tokens = std::min(tokens, window + max_rows + std::min<int64_t>(sinks, tokens) + TB);
  const int64_t blocks = (tokens + TB - 1) / TB;
  const int given = n_split;
  int64_t n = n_split;
  if (n == 0) {
    if (p->tiles) {
      // Workgroups enough for the bytes that have to be on their way: one for each compute unit where a turn of its four wavefronts is 64 KB, two where it
      // is less (us; fp8, d 128, 8 heads, one sequence of 131072: 32 splits 67.7, 64 64.4, 128 65.4, 256 65.0; d 256, 2 heads: 64 47.6, 128 36.6, 256 38.5, 384 46.6;
      // bf16, d 128, one of 65536: 16 75.7, 32 53.7, 64 58.5), no split of more than 2048 tokens (fp8, 32 of 8192: 1 138, 2 114.6, 4 106.4, 8 105.2) as long as that makes no more
      // than 4096 workgroups or four splits (d 128, splits of 2048 / so: fp8, 8 heads, 32 of 65536 752 / 737, 64 of 65536 1504 / 1449, 128 of 32768 1558 / 1481; 16 heads, 256 of 4096, one split 860, two 780,
      // four 742), and of the next numbers of splits, while they leave 512 tokens, the first that leaves no compute unit without work in its last round (24 of 6000: 3 70.9, 4 62.9).
      const int64_t turn = 4 * TB * 2 * d * (cache == TQ_E4M3 ? 1 : 2), target = turn >= 65536 ? 256 : 512;
      // Steps of more sequences than are shared out anew keep splits of 2048 tokens, since one may be far longer than the others, while partial results are 256 MiB at most.
      const int64_t most = B > STEP_ROUND ? ((int64_t)256 << 20) / (4 * std::max<int64_t>(1, rows * Hq * d)) : 4096 / pairs;
      n = std::max((target + pairs - 1) / pairs, std::min((tokens + 2047) / 2048, std::max<int64_t>(4, most)));
      double best = 0;
      for (int64_t i = n; i <= 2 * n && i <= std::max(n, tokens / 512); ++i) {
        const double full = double(pairs * i) / (256 * ((pairs * i + 255) / 256));
        if (full > best + 0.02) { best = full; n_split = (int)std::min<int64_t>(i, JOIN_MAX_SPLITS); }
        if (best >= 0.95) break;
      }
      n = std::min<int64_t>(n_split, (blocks + 3) / 4);
    } else {
      n = attend_rows_splits(pairs, blocks, rows * Hq, d);
    }
  }
  n = std::max<int64_t>(1, std::min(n, blocks));
  int64_t chunk = (blocks + n - 1) / n;
  if (!given && p->tiles) chunk = (chunk + 3) & ~(int64_t)3;                       // (a block for each of the four wavefronts)
  p->units = units;
  p->n_split = (int)std::max<int64_t>(1, (blocks + chunk - 1) / chunk);
  p->chunk = (int)chunk;
  // Sequences that differ (to find out takes a workgroup 1 - 2 us: not where 2048 tokens are the most that one has to itself) have their blocks shared out anew: 1024
  // items in all (us, as planned / shared out; fp8, 24 sequences of 61 .. 16000, 5 rows 75 / 54, one row 54 / 46; 96 of 61 .. 8190 86 / 81), and with many rows 512
  // (exact, 64 of 100 .. 20000, 64 rows 694 / 448).  A row has up to 64 of them where that leaves the join a wavefront for each row (above, a workgroup
  // for 64 channels of one), and of few rows up to 96, none of less than 512 tokens (without these bounds / with: 40 of 50 .. 6000, 16 heads on 2 of 256 36.5 / 25.2; 4 of
  // 1000 .. 100000, 32 on 4 41.9 / 38.0; 8 of 5000 .. 60000, 16 on 2 of 256 58.0 / 60.3).  Of many rows none has less than 2048 tokens (one turn at least / so; exact, 32 heads on 8
  // of 128: 24 of 300 .. 16000, 16 rows 116 / 101; 16 of 300 .. 5000, 64 rows 85 / 73; 3 of 300 .. 30000, 64 rows 57 / 62).
  const bool many = rows * Hq >= 512;
  p->target = p->cap = 0;
  if (!given && B > 1 && B <= STEP_ROUND && tokens > 2048) {
    p->target = (int)(((p->tiles ? 1024 : 512) + Hkv - 1) / Hkv);
    p->cap = (int)std::max<int64_t>(p->n_split, std::min<int64_t>((blocks + 3) / 4, many ? 64 : (p->tiles ? 96 : JOIN_MAX_SPLITS)));
  }
  // (one for rows of no sequence; 2: total and its share are rounded)
  p->items = std::max<int64_t>(units * p->n_split + (starts ? 1 : 0), p->target ? p->target + units + 3 : 0);
  const int most = std::max(p->n_split, p->cap);
  // (with many rows a sequence few are split: 131072 of which none is took 12 us with a wavefront each; 8 sequences of 300 .. 4000, 300 rows, 9600 rows of 32 heads, with eight rows each 105, with
  // four 99)
  p->few = most <= JOIN_FEW || (many && most <= 64) ? (p->tiles || p->n_split > 1 ? 1 : (int)std::min<int64_t>(8, std::max<int64_t>(1, rows * Hq / 16384))) : 0;
  const size_t all = (size_t)rows * Hq;
  p->grid = p->items * Hkv;
  // Partial results: as planned, each row's splits; shared out anew, those of split units (Attend), of which there are 2 target at most, and no more than all units have.
  // (4: total and its share are rounded.)
  p->part = (int)std::min<int64_t>(M, starts ? rows * G : G);
  p->parts = p->target ? (int)std::min<int64_t>(2 * p->target + 4, units * p->cap) : 0;
  const size_t places = most > 1 ? std::max(p->n_split > 1 ? all * p->n_split : 0, (size_t)p->parts * Hkv * p->part) : 0;
  size_t at = 0;
  p->shares_at = at;  at = round256(at + (most > 1 ? all * sizeof(int2) : 0));
  p->ml_at = at;      at = round256(at + places * sizeof(float2));
  p->acc_at = at;     at = round256(at + places * d * sizeof(float));
  p->bytes = std::max<size_t>(at, 256);
  const int64_t joins = most <= 1 ? 0 : (p->few ? (int64_t)(all + 4 * p->few - 1) / (4 * p->few) : (int64_t)all * (d / 64));
  return p->grid <= STEP_MAX_GROUPS && joins <= STEP_MAX_GROUPS && (int64_t)all * (d / 64) <= INT32_MAX;
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
  if (!(sm_scale > -0x1p127f && sm_scale < 0x1p127f)) return TQ_EINVAL;      // (masked scores are -inf, which a factor of NaN or infinity would not leave so)
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
  a.target = p.target; a.cap = p.cap; a.units = (int32_t)p.units; a.items = (int32_t)p.items; a.share = p.target ? 1.0f / p.target : 0.0f;
  const bool joined = std::max(p.n_split, p.cap) > 1;
  a.shares = joined ? (int2*)((char*)workspace + p.shares_at) : nullptr;
  a.part = p.part; a.parts = p.parts;
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
  if (rc || !joined) return rc;
  const AttendJoin j{a.shares, a.ml, a.acc, out, rows * Hq, Hkv, d, p.few, p.n_split, p.part, p.parts, p.cap};
  const dim3 grid((unsigned)(p.few ? (j.rows + 4 * p.few - 1) / (4 * p.few) : j.rows * (d / 64))), block(256);
  if (dtype == TQ_F16) attend_join_kernel<TQ_F16><<<grid, block, 0, st>>>(j);
  else attend_join_kernel<TQ_BF16><<<grid, block, 0, st>>>(j);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
