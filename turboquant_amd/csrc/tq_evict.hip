// Eviction from a cache by accumulated attention weight: which tokens stay, and their way to the front of the sequence's slots.
//
// Order of who stays, per sequence and KV head: first the sinks (positions below `sinks`) and the newest (positions from seen - recent on), then
// by weight; of two alike the one in the lower slot.  A weight that is no number comes last, +inf counts as the largest number, -0 as 0.
// The first `budget` of them stay.  Slots below the budget whose token goes are holes; the k-th hole takes the k-th of the tokens that stay
// behind the budget.  Tokens below it that stay do not move: with a budget kept up every few tokens only those few move, and since sources lie
// behind the budget and destinations before it, all moves of a row can run at once.
#include "tq_common.h"

#include <algorithm>

namespace tq {

constexpr int SEL_THREADS = 1024, SEL_BINS = 2048;

struct EvictSelect {
  const float* w;  int64_t w_b, w_h;            // (B, H, L) in
  const int32_t* pos;  int64_t p_b, p_h;
  const int32_t *lens, *seen;                   // seen null: the lengths
  int32_t B, H, L, budget, sinks, recent, moves;
  int32_t *lens_out, *count, *dst, *src;        // (B), (B, H), (B, H, moves) twice
  float* w_out;  int64_t wo_b, wo_h;            // may be the inputs themselves
  int32_t* pos_out;  int64_t po_b, po_h;
};

// larger is kept first; the largest value is that of a token kept whatever its weight
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int sinks, int newest) {
  if (pos < sinks || pos >= newest) return 0xffffffffu;
  w = w != w ? -INFINITY : fminf(w + 0.0f, 3.4028234663852886e38f);
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// inclusive sum over the workgroup's threads; *total = all of it
__device__ __forceinline__ uint32_t sel_scan(uint32_t v, uint32_t* s_wave, uint32_t* total) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = __shfl_up(v, o, 64);
    if (lane >= o) v += x;
  }
  __syncthreads();                              // (s_wave may still be read from the call before)
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < SEL_THREADS / 64; ++i) {
    const uint32_t x = s_wave[i];
    if (i < wave) before += x;
    all += x;
  }
  *total = all;
  return before + v;
}

__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const EvictSelect a) {
  __shared__ uint32_t s_bin[SEL_BINS];
  __shared__ uint32_t s_wave[SEL_THREADS / 64];
  __shared__ uint32_t s_found[2];
  const int tid = (int)threadIdx.x, h = (int)blockIdx.x % a.H, b = (int)blockIdx.x / a.H;
  const int held = a.lens[b], n = held < 0 ? 0 : (held > a.L ? a.L : held);
  const int seen = a.seen ? a.seen[b] : held;
  const int64_t newest64 = (int64_t)seen - a.recent;
  const int newest = newest64 < INT32_MIN ? INT32_MIN : (int)newest64;
  const float* w = a.w + b * a.w_b + h * a.w_h;
  const int32_t* pos = a.pos + b * a.p_b + h * a.p_h;
  float* w_out = a.w_out + b * a.wo_b + h * a.wo_h;
  int32_t* pos_out = a.pos_out + b * a.po_b + h * a.po_h;
  const int64_t row = (int64_t)b * a.H + h;
  int32_t *dst = a.dst + row * a.moves, *src = a.src + row * a.moves;
  const int left = n < a.budget ? n : a.budget;
  if (h == 0 && tid == 0) a.lens_out[b] = left;

  uint32_t moved = 0;
  if (n > a.budget && a.budget > 0) {
    // ---- the key of the last one that stays: three digits, from the highest ----
    uint32_t want = (uint32_t)a.budget, prefix = 0;
    int low = 21;                               // lowest bit of the digit
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass == 2 ? 10 : 11, above = low + bits;
      for (int i = tid; i < SEL_BINS; i += SEL_THREADS) s_bin[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += SEL_THREADS) {
        const uint32_t k = evict_key(w[i], pos[i], a.sinks, newest);
        if (above == 32 || (k >> above) == (prefix >> above)) atomicAdd(&s_bin[(k >> low) & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // from the highest bin down: the one in which the count reaches what is wanted
      const int hi = SEL_BINS - 1 - 2 * tid;    // this thread's two bins, in that order
      const uint32_t c0 = s_bin[hi], c1 = s_bin[hi - 1];
      uint32_t total;
      const uint32_t upto = sel_scan(c0 + c1, s_wave, &total), before = upto - c0 - c1;
      if (before < want && want <= upto) {
        const bool first = want <= before + c0;
        s_found[0] = (uint32_t)(first ? hi : hi - 1);
        s_found[1] = want - (first ? before : before + c0);
      }
      __syncthreads();
      prefix |= s_found[0] << low;
      want = s_found[1];                        // of the keys equal so far
      low = pass == 0 ? 10 : 0;
    }
    // ---- in slot order: who stays, holes and movers ----
    uint32_t ties = 0, holes = 0, movers = 0;
    for (int i0 = 0; i0 < n; i0 += SEL_THREADS) {
      const int i = i0 + tid;
      const bool in = i < n;
      const uint32_t k = in ? evict_key(w[i], pos[i], a.sinks, newest) : 0u;
      const bool tie = in && k == prefix;
      uint32_t total;
      const uint32_t rank = ties + sel_scan(tie, s_wave, &total);       // 1 for the first
      ties += total;
      const bool stays = in && (k > prefix || (tie && rank <= want));
      const bool hole = in && !stays && i < a.budget, mover = stays && i >= a.budget;
      const uint32_t at = sel_scan((uint32_t)hole | (uint32_t)mover << 16, s_wave, &total);
      const uint32_t hr = holes + (at & 0xffff), mr = movers + (at >> 16);
      if (hole) dst[hr - 1] = i;
      if (mover) src[mr - 1] = i;
      holes += total & 0xffff;
      movers += total >> 16;
    }
    moved = movers;
  }
  if (tid == 0) a.count[row] = (int32_t)moved;
  for (int i = (int)moved + tid; i < a.moves; i += SEL_THREADS) dst[i] = src[i] = -1;
  // ---- weights and positions of who stays: in place first, then the movers, then the slots that are free now ----
  if (w_out != w)
    for (int i = tid; i < left; i += SEL_THREADS) w_out[i] = w[i];
  if (pos_out != pos)
    for (int i = tid; i < left; i += SEL_THREADS) pos_out[i] = pos[i];
  __syncthreads();
  for (int i = tid; i < (int)moved; i += SEL_THREADS) {
    const int to = dst[i], of = src[i];
    w_out[to] = w[of];
    pos_out[to] = pos[of];
  }
  __syncthreads();
  for (int i = left + tid; i < a.L; i += SEL_THREADS) {
    w_out[i] = 0.0f;
    pos_out[i] = seen + (i - left);
  }
}

// ---- the moves ----------------------------------------------------------------------------------------------------------------------------

struct MoveList {
  const int32_t *count, *dst, *src;             // (B, H), (B, H, moves) twice
  int32_t B, H, moves;
  const int32_t* table;
  int64_t table_step;
  int32_t table_row;
  int64_t num_blocks;
};

__device__ __forceinline__ int64_t move_block(const MoveList& m, int b, int slot) {
  const int page = slot / TQ_PAGE_TOKENS;
  if (slot < 0 || page >= m.table_row) return -1;
  const int64_t blk = m.table[b * m.table_step + page];
  return blk < 0 || blk >= m.num_blocks ? -1 : blk;
}

struct MoveExact {
  MoveList m;
  char *k, *v;
  int64_t s_blk, s_t, s_h;                      // bytes
  int32_t pieces;                               // of 16 bytes in a row
};

constexpr int MOVE_TOKENS = 64;                 // moves of a workgroup

// a row's pieces by neighbouring threads, keys and values of a move in the same turn
__global__ void __launch_bounds__(256) move_exact_kernel(const MoveExact a) {
  __shared__ int64_t s_to[MOVE_TOKENS], s_of[MOVE_TOKENS];
  const int chunks = (a.m.moves + MOVE_TOKENS - 1) / MOVE_TOKENS;
  const int chunk = (int)(blockIdx.x % (unsigned)chunks), row = (int)(blockIdx.x / (unsigned)chunks), h = row % a.m.H, b = row / a.m.H;
  const int first = chunk * MOVE_TOKENS, count = a.m.count[row] < a.m.moves ? a.m.count[row] : a.m.moves;
  const int n = count - first < MOVE_TOKENS ? count - first : MOVE_TOKENS;
  if (n <= 0) return;
  if ((int)threadIdx.x < n) {
    const int to = a.m.dst[(int64_t)row * a.m.moves + first + threadIdx.x], of = a.m.src[(int64_t)row * a.m.moves + first + threadIdx.x];
    const int64_t tb = move_block(a.m, b, to), ob = move_block(a.m, b, of);
    const bool ok = tb >= 0 && ob >= 0;
    s_to[threadIdx.x] = ok ? tb * a.s_blk + (to % TQ_PAGE_TOKENS) * a.s_t + h * a.s_h : -1;
    s_of[threadIdx.x] = ok ? ob * a.s_blk + (of % TQ_PAGE_TOKENS) * a.s_t + h * a.s_h : -1;
  }
  __syncthreads();
  for (int i = (int)threadIdx.x; i < n * a.pieces; i += 256) {
    const int t = i / a.pieces, p = i - t * a.pieces;
    if (s_to[t] < 0) continue;
    const uint4 x = *(const uint4*)(a.k + s_of[t] + p * 16), y = *(const uint4*)(a.v + s_of[t] + p * 16);
    *(uint4*)(a.k + s_to[t] + p * 16) = x;
    *(uint4*)(a.v + s_to[t] + p * 16) = y;
  }
}

// Compressed pages: a workgroup owns a page that has holes, since the codes of its sixteen tokens share words.  A source in the same page is not
// disturbed: its bits are written back as they are.
struct MovePool {
  MoveList m;
  uint8_t* pool;
  tq_page_layout L;
  int32_t pages;                                // logical pages that may have holes
};

__global__ void __launch_bounds__(256) move_pool_kernel(const MovePool a) {
  __shared__ const uint8_t* s_of[TQ_PAGE_TOKENS];          // page of the slot's new token, null: the slot keeps its own
  __shared__ int s_slot[TQ_PAGE_TOKENS];
  __shared__ int s_any;
  const int page = (int)(blockIdx.x % (unsigned)a.pages), row = (int)(blockIdx.x / (unsigned)a.pages), h = row % a.m.H, b = row / a.m.H;
  const int count = a.m.count[row] < a.m.moves ? a.m.count[row] : a.m.moves;
  const int32_t *dst = a.m.dst + (int64_t)row * a.m.moves, *src = a.m.src + (int64_t)row * a.m.moves;
  const int64_t blk = move_block(a.m, b, page * TQ_PAGE_TOKENS);
  if (count <= 0 || blk < 0) return;
  // holes are in ascending order: the first in this page
  int lo = 0, hi = count;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (dst[mid] < page * TQ_PAGE_TOKENS) lo = mid + 1; else hi = mid;
  }
  if (threadIdx.x < TQ_PAGE_TOKENS) s_of[threadIdx.x] = nullptr;
  if (threadIdx.x == 0) s_any = 0;
  __syncthreads();
  const int64_t bytes = a.L.page_bytes;
  if (threadIdx.x < TQ_PAGE_TOKENS && lo + (int)threadIdx.x < count) {
    const int to = dst[lo + threadIdx.x], of = src[lo + threadIdx.x];
    const int64_t ob = move_block(a.m, b, of);
    if (to / TQ_PAGE_TOKENS == page && to >= 0 && ob >= 0) {
      s_of[to % TQ_PAGE_TOKENS] = a.pool + (ob * a.m.H + h) * bytes;
      s_slot[to % TQ_PAGE_TOKENS] = of % TQ_PAGE_TOKENS;
      s_any = 1;
    }
  }
  __syncthreads();
  if (!s_any) return;
  uint8_t* own = a.pool + (blk * a.m.H + h) * bytes;
  const int tid = (int)threadIdx.x, d = a.L.d, planes = a.L.mse_bits + 1, words = d >> 5, vb = a.L.value_bits;
  // key words, token by token
  for (int i = tid; i < TQ_PAGE_TOKENS * planes * words; i += 256) {
    const int n = i % TQ_PAGE_TOKENS, p = (i / TQ_PAGE_TOKENS) % planes, j = i / (TQ_PAGE_TOKENS * planes);
    if (s_of[n]) *(uint32_t*)(own + key_word_off(a.L, p, j, n)) = *(const uint32_t*)(s_of[n] + key_word_off(a.L, p, j, s_slot[n]));
  }
  for (int i = tid; i < TQ_PAGE_TOKENS * 2; i += 256) {
    const int n = i >> 1;
    if (s_of[n]) ((uint32_t*)(own + a.L.off_meta))[i] = ((const uint32_t*)(s_of[n] + a.L.off_meta))[s_slot[n] * 2 + (i & 1)];
  }
  // value codes: a word of a channel's field holds 32 / value_bits tokens
  const int per = 32 / vb, field = vb / 2;                 // words of a field
  const uint32_t mask = (1u << vb) - 1;
  for (int i = tid; i < d * field; i += 256) {
    const int c = i / field, k = i % field, off = vfield_off(a.L, c);
    uint32_t* to = (uint32_t*)(own + off) + k;
    uint32_t x = *to;
    for (int t = 0; t < per; ++t) {
      const int n = k * per + t;
      if (!s_of[n]) continue;
      const int s = s_slot[n];
      const uint32_t code = ((const uint32_t*)(s_of[n] + off))[s / per] >> (vb * (s % per)) & mask;
      x = (x & ~(mask << (vb * t))) | code << (vb * t);
    }
    *to = x;
  }
  const int groups = d / a.L.group_size, es = elem_bytes(a.L.dtype);
  for (int i = tid; i < groups * TQ_PAGE_TOKENS; i += 256) {
    const int g = i / TQ_PAGE_TOKENS, n = i % TQ_PAGE_TOKENS;
    if (!s_of[n]) continue;
    const int to = (g * TQ_PAGE_TOKENS + n) * es, of = (g * TQ_PAGE_TOKENS + s_slot[n]) * es;
    if (es == 4) {
      *(uint32_t*)(own + a.L.off_vscale + to) = *(const uint32_t*)(s_of[n] + a.L.off_vscale + of);
      *(uint32_t*)(own + a.L.off_vzero + to) = *(const uint32_t*)(s_of[n] + a.L.off_vzero + of);
    } else {
      *(uint16_t*)(own + a.L.off_vscale + to) = *(const uint16_t*)(s_of[n] + a.L.off_vscale + of);
      *(uint16_t*)(own + a.L.off_vzero + to) = *(const uint16_t*)(s_of[n] + a.L.off_vzero + of);
    }
  }
}

static int move_list(MoveList* m, const int32_t* count, const int32_t* dst, const int32_t* src, int B, int H, int moves, const int32_t* table,
                     int bt_stride, int64_t num_blocks) {
  if (!count || !dst || !src || !table) return TQ_ENULL;
  if (B < 0 || H <= 0 || moves < 0 || bt_stride == 0 || bt_stride == INT32_MIN || num_blocks <= 0) return TQ_EINVAL;
  m->count = count; m->dst = dst; m->src = src; m->B = B; m->H = H; m->moves = moves; m->table = table; m->num_blocks = num_blocks;
  m->table_row = bt_stride < 0 ? -bt_stride : bt_stride;
  m->table_step = bt_stride < 0 ? 0 : bt_stride;
  return TQ_OK;
}

}  // namespace tq

extern "C" int tq_evict_select(const float* weights, int64_t w_b, int64_t w_h, const int32_t* positions, int64_t p_b, int64_t p_h, const int32_t* seq_lens,
                               const int32_t* seen, int B, int H, int L, int budget, int sinks, int recent, int moves, int32_t* lens_out, int32_t* count,
                               int32_t* dst, int32_t* src, float* weights_out, int64_t wo_b, int64_t wo_h, int32_t* positions_out, int64_t po_b,
                               int64_t po_h, void* stream) {
  using namespace tq;
  if (!weights || !positions || !seq_lens || !lens_out || !count || !dst || !src || !weights_out || !positions_out) return TQ_ENULL;
  if (B < 0 || H <= 0 || L <= 0 || budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget) return TQ_EINVAL;
  if (w_b < 0 || w_h < 0 || p_b < 0 || p_h < 0 || wo_b < 0 || wo_h < 0 || po_b < 0 || po_h < 0 || L > INT32_MAX - 2 * SEL_THREADS) return TQ_EINVAL;
  if (moves < std::max(1, std::min(budget, L - budget)) || (int64_t)B * H > INT32_MAX) return TQ_EINVAL;
  if (B == 0) return TQ_OK;
  EvictSelect a{weights, w_b, w_h, positions, p_b, p_h, seq_lens, seen, B, H, L, budget, sinks, recent, moves, lens_out, count, dst, src,
                weights_out, wo_b, wo_h, positions_out, po_b, po_h};
  evict_select_kernel<<<dim3((unsigned)(B * H)), dim3(SEL_THREADS), 0, (hipStream_t)stream>>>(a);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

extern "C" int tq_move_tokens_exact(void* k_cache, void* v_cache, int dtype, int d, int64_t cs_blk, int64_t cs_t, int64_t cs_h, int64_t num_blocks,
                                    const int32_t* block_table, int bt_stride, const int32_t* count, const int32_t* dst, const int32_t* src, int B,
                                    int H, int moves, void* stream) {
  using namespace tq;
  if (!k_cache || !v_cache) return TQ_ENULL;
  if (dtype < TQ_F32 || dtype > TQ_BF16 || d <= 0) return TQ_EINVAL;
  MoveExact a{};
  const int rc = move_list(&a.m, count, dst, src, B, H, moves, block_table, bt_stride, num_blocks);
  if (rc) return rc;
  const int64_t size = elem_bytes(dtype);
  a.s_blk = cs_blk * size; a.s_t = cs_t * size; a.s_h = cs_h * size;
  if (cs_blk < 0 || cs_t < 0 || cs_h < 0 || d * size % 16 || a.s_blk % 16 || a.s_t % 16 || a.s_h % 16) return TQ_EUNSUPPORTED;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return TQ_EUNSUPPORTED;
  a.k = (char*)k_cache; a.v = (char*)v_cache; a.pieces = (int)(d * size / 16);
  if (B == 0 || moves == 0) return TQ_OK;
  const int64_t grid = (int64_t)B * H * ((moves + MOVE_TOKENS - 1) / MOVE_TOKENS);
  if (grid > INT32_MAX) return TQ_EINVAL;
  move_exact_kernel<<<dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream>>>(a);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

extern "C" int tq_move_tokens_pool(uint8_t* pool, int64_t num_pages, const tq_page_layout* layout, const int32_t* block_table, int bt_stride,
                                   const int32_t* count, const int32_t* dst, const int32_t* src, int B, int H, int moves, int budget, void* stream) {
  using namespace tq;
  if (!pool || !layout) return TQ_ENULL;
  if (budget <= 0) return TQ_EINVAL;
  if (layout->value_bits != 2 && layout->value_bits != 4 && layout->value_bits != 8) return TQ_EUNSUPPORTED;
  MovePool a{};
  const int rc = move_list(&a.m, count, dst, src, B, H, moves, block_table, bt_stride, num_pages);
  if (rc) return rc;
  a.pool = pool; a.L = *layout;
  const int64_t most = ((int64_t)budget + TQ_PAGE_TOKENS - 1) / TQ_PAGE_TOKENS;
  a.pages = (int)std::min<int64_t>(most, a.m.table_row);
  if (B == 0 || moves == 0) return TQ_OK;
  const int64_t grid = (int64_t)B * H * a.pages;
  if (grid > INT32_MAX) return TQ_EINVAL;
  move_pool_kernel<<<dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream>>>(a);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}
