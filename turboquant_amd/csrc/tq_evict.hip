// Eviction from a cache by accumulated attention weight: which tokens stay, and their way to the front of the sequence's slots.
//
// Order of who stays, per sequence and KV head: first the sinks (positions below `sinks`) and the newest (positions from seen - recent on), then
// by weight; of two alike the one in the lower slot.  A weight that is no number counts as -inf, +inf as the largest number, -0 as 0.
// The first `budget` of them stay.  Slots below the budget whose token goes are holes; the k-th hole takes the k-th of the tokens that stay
// behind the budget.  Tokens below it that stay do not move: with a budget kept up every few tokens only those few move, and since sources lie
// behind the budget and destinations before it, all moves of a row can run at once.
// Bound by latencies in a row, not by bytes: a digit is a count, a barrier, a sum over the bins, a barrier.  Digits of 11 bits: three of them, where 8 bits
// take four.  Counts of whole wavefronts whose keys fall into one bin are added once.
#include "tq_common.h"

#include <algorithm>

namespace tq {

constexpr int SEL_BINS = 2048;
// the digits of a key, from the highest: 11, 11 and 10 bits
__host__ __device__ constexpr int sel_low(int pass) { return pass == 0 ? 21 : (pass == 1 ? 10 : 0); }
__host__ __device__ constexpr int sel_bits(int pass) { return pass == 2 ? 10 : 11; }

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

// One row: its pointers and numbers
struct EvictRow {
  const float* w;
  const int32_t* pos;
  float* w_out;
  int32_t *pos_out, *dst, *src;
  int64_t row;
  int b, h, n, left, seen, newest;
  __device__ __forceinline__ EvictRow(const EvictSelect& a, int r) {
    row = r; h = r % a.H; b = r / a.H;
    const int held = a.lens[b];
    n = held < 0 ? 0 : (held > a.L ? a.L : held);
    left = n < a.budget ? n : a.budget;
    seen = a.seen ? a.seen[b] : held;
    const int64_t from = (int64_t)seen - a.recent;
    newest = from < INT32_MIN ? INT32_MIN : (int)from;
    w = a.w + b * a.w_b + h * a.w_h;
    pos = a.pos + b * a.p_b + h * a.p_h;
    w_out = a.w_out + b * a.wo_b + h * a.wo_h;
    pos_out = a.pos_out + b * a.po_b + h * a.po_h;
    dst = a.dst + row * a.moves;
    src = a.src + row * a.moves;
  }
};

// Weights and positions of a wavefront's J x 64 slots from `base` on (of slot 0 from `end` on).  All loads first, none behind a condition: one memory
// latency, not J of them.
template <int J>
__device__ __forceinline__ void sel_load(float (&w)[J], int (&pos)[J], const EvictRow& r, int base, int end) {
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = base + j * 64 + lane, at = i < end ? i : 0;
    w[j] = r.w[at];
    pos[j] = r.pos[at];
  }
#pragma unroll
  for (int j = 0; j < J; ++j) asm volatile("" : "+v"(w[j]), "+v"(pos[j]));
}
// counts a key's digit; a wavefront whose keys all fall into one bin adds once (sums that are all alike would be 64 turns of one address)
__device__ __forceinline__ void sel_count(uint32_t* bins, bool in, uint32_t digit) {
  const uint64_t who = __ballot(in);
  if (who == 0) return;
  const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)digit, __builtin_ctzll(who));
  if (__ballot(in && digit == first) == who) {
    if (((int)threadIdx.x & 63) == __builtin_ctzll(who)) atomicAdd(&bins[first], (uint32_t)__popcll(who));
  } else if (in) {
    atomicAdd(&bins[digit], 1u);
  }
}

// inclusive sum over a wavefront's lanes: within rows of sixteen, then the rows' ends into the rows behind them
__device__ __forceinline__ uint32_t lanes_scan16(uint32_t v) {
#define TQ_SCAN_STEP(ctrl, rows) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, true)
  TQ_SCAN_STEP(0x111, 0xF); TQ_SCAN_STEP(0x112, 0xF); TQ_SCAN_STEP(0x114, 0xF); TQ_SCAN_STEP(0x118, 0xF);
  return v;
}
__device__ __forceinline__ uint32_t lanes_scan(uint32_t v) {
  v = lanes_scan16(v);
  TQ_SCAN_STEP(0x142, 0xA); TQ_SCAN_STEP(0x143, 0xC);
#undef TQ_SCAN_STEP
  return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }

// Sums over the wavefronts in front of this one, and over all, of a count that each of them has.  (Up to sixteen, a lane each: in a workgroup of a
// thousand threads an instruction that all of them execute takes sixteen clocks.)
template <int WAVES>
__device__ __forceinline__ uint32_t sel_before(const uint32_t* s_wave, uint32_t* total) {
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t v = lanes_scan16(lane < WAVES ? s_wave[lane] : 0u);
  *total = lane_of(v, WAVES - 1);
  return wave > 0 ? lane_of(v, wave - 1) : 0u;
}

// inclusive sum over the workgroup's threads; *total = all of it
template <int THREADS>
__device__ __forceinline__ uint32_t sel_scan(uint32_t v, uint32_t* s_wave, uint32_t* total) {
  v = lanes_scan(v);
  __syncthreads();                              // (s_wave may still be read from the call before)
  if (((int)threadIdx.x & 63) == 63) s_wave[(int)threadIdx.x >> 6] = v;
  __syncthreads();
  return sel_before<THREADS / 64>(s_wave, total) + v;
}

// The bin, from the highest down, in which the count reaches `want`: s_found = {bin, how many of it are wanted}.  counts(bin, c): c[i] = keys in bin - i, for
// as many as a thread has.
template <int THREADS, class Counts>
__device__ __forceinline__ void sel_find(uint32_t want, Counts counts, uint32_t* s_wave, uint32_t* s_found) {
  constexpr int EACH = SEL_BINS / THREADS;
  const int hi = SEL_BINS - 1 - EACH * (int)threadIdx.x;
  uint32_t c[EACH], mine = 0, total;
  counts(hi, c);
#pragma unroll
  for (int i = 0; i < EACH; ++i) mine += c[i];
  uint32_t before = sel_scan<THREADS>(mine, s_wave, &total) - mine;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (before < want && want <= before + c[i]) {
      s_found[0] = (uint32_t)(hi - i);
      s_found[1] = want - before;
    }
    before += c[i];
  }
  __syncthreads();
}

// sums over the wavefronts in front, in slot order, of two counts that each of them has, and over all
template <int WAVES>
__device__ __forceinline__ uint2 sel_waves(uint2 v, uint32_t (*s_two)[WAVES], uint2* total) {
  __syncthreads();
  if (((int)threadIdx.x & 63) == 0) {
    s_two[0][(int)threadIdx.x >> 6] = v.x;
    s_two[1][(int)threadIdx.x >> 6] = v.y;
  }
  __syncthreads();
  uint2 before;
  before.x = sel_before<WAVES>(s_two[0], &total->x);
  before.y = sel_before<WAVES>(s_two[1], &total->y);
  return before;
}

// Keys of a wavefront's J x 64 neighbouring slots in registers: who of them stays, and the lists.  `ties`: keys equal to `last` in front of these slots;
// `holes`, `movers`: in front of the wavefront's slots, found by `offsets` from its own numbers.  mover(slot, rank, j) for all of the wavefront's movers,
// between(), hole(slot, rank, j) for its holes.  Returns bit j: slot j stays.
template <int J, class Offsets, class Mover, class Between, class Hole>
__device__ __forceinline__ uint32_t sel_lists(const uint32_t (&k)[J], int base, int n, int budget, uint32_t last, uint32_t want, uint32_t ties, Offsets offsets,
                                              Mover mover, Between between, Hole hole) {
  const int lane = (int)threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1;
  uint32_t stays = 0, holes = 0, movers = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = base + j * 64 + lane;
    const bool in = i < n, tie = in && k[j] == last;
    const uint64_t t = __ballot(tie);
    bool keep = in && k[j] > last;
    if (t) {
      keep = keep || (tie && ties + (uint32_t)__popcll(t & below) < want);
      ties += (uint32_t)__popcll(t);
    }
    stays |= (uint32_t)keep << j;
    holes += (uint32_t)__popcll(__ballot(in && !keep && i < budget));
    movers += (uint32_t)__popcll(__ballot(keep && i >= budget));
  }
  const uint2 at = offsets(make_uint2(holes, movers));
  holes = at.x; movers = at.y;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = base + j * 64 + lane;
    const bool is = (stays >> j & 1) && i >= budget;
    const uint64_t who = __ballot(is);
    if (who == 0) continue;                     // (the wavefront as one)
    if (is) mover(i, movers + (uint32_t)__popcll(who & below), j);
    movers += (uint32_t)__popcll(who);
  }
  between();
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = base + j * 64 + lane;
    const bool is = i < n && !(stays >> j & 1) && i < budget;
    const uint64_t who = __ballot(is);
    if (who == 0) continue;
    if (is) hole(i, holes + (uint32_t)__popcll(who & below), j);
    holes += (uint32_t)__popcll(who);
  }
  return stays;
}

// ---- a row in one workgroup: its weights and positions are read once and stay in registers, movers meet their holes in LDS ----
// 256 rows of 2064 slots, cut to 2048: 11 us (8.5 MB, 1.6 us as a copy): twenty barriers with a few loads or counts between them.
// `each` (up to J): 64 slots per wavefront and step, so that all wavefronts have some.
template <int THREADS, int J>
__global__ void __launch_bounds__(THREADS) evict_row_kernel(const EvictSelect a, int each) {
  constexpr int WAVES = THREADS / 64;
  __shared__ uint32_t s_bin[SEL_BINS];
  __shared__ uint32_t s_wave[WAVES], s_found[2];
  __shared__ uint32_t s_two[2][WAVES];
  __shared__ float2 s_mover[THREADS * J / 2];   // weight and position (as it is) of the n-th; no more than half of the slots move
  const int tid = (int)threadIdx.x, lane = tid & 63, base = (tid >> 6) * (each * 64);
  const EvictRow r(a, (int)blockIdx.x);
  if (r.h == 0 && tid == 0) a.lens_out[r.b] = r.left;
  uint32_t moved = 0;
  const int end = base + each * 64 < r.n ? base + each * 64 : r.n;            // of this wavefront's slots
  float w[J];
  int pos[J];
  if (r.n > 0) sel_load<J>(w, pos, r, base, end);
  uint32_t stays = 0xffffffffu;
  if (r.n > a.budget) {
    uint32_t k[J];
#pragma unroll
    for (int j = 0; j < J; ++j) k[j] = base + j * 64 + lane < end ? evict_key(w[j], pos[j], a.sinks, r.newest) : 0u;
    uint32_t want = (uint32_t)a.budget, last = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int low = sel_low(pass), above = low + sel_bits(pass);
      for (int i = tid; i < SEL_BINS; i += THREADS) s_bin[i] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; ++j)
        sel_count(s_bin, base + j * 64 + lane < end && (pass == 0 || (k[j] >> (above & 31)) == (last >> (above & 31))), (k[j] >> low) & ((1u << sel_bits(pass)) - 1));
      __syncthreads();
      sel_find<THREADS>(want, [&](int bin, uint32_t* c) {
#pragma unroll
        for (int i = 0; i < SEL_BINS / THREADS; ++i) c[i] = s_bin[bin - i];
      }, s_wave, s_found);
      last |= s_found[0] << low;
      want = s_found[1];
    }
    // ties in front of this wavefront's slots
    uint32_t ties = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) ties += (uint32_t)__popcll(__ballot(base + j * 64 + lane < end && k[j] == last));
    uint2 total;
    ties = sel_waves<WAVES>(make_uint2(ties, 0), s_two, &total).x;
    stays = sel_lists<J>(k, base, end, a.budget, last, want, ties, [&](uint2 mine) { return sel_waves<WAVES>(mine, s_two, &total); },
                         [&](int slot, uint32_t rank, int j) {
                           r.src[rank] = slot;
                           s_mover[rank] = make_float2(w[j], __int_as_float(pos[j]));
                         },
                         [] { __syncthreads(); },
                         [&](int slot, uint32_t rank, int) {
                           const float2 x = s_mover[rank];
                           r.dst[rank] = slot;
                           r.w_out[slot] = x.x;
                           r.pos_out[slot] = __float_as_int(x.y);
                         });
    moved = total.y;
  }
  // Who stays in place, the slots that are free now, the ends of the lists.  (In place, too: every wavefront has its slots in registers - where a row is
  // cut, behind barriers; where it is not, no slot that is written has been read.)
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = base + j * 64 + lane;
    if (i < end && i < r.left && (stays >> j & 1)) {
      if (r.w_out != r.w) r.w_out[i] = w[j];
      if (r.pos_out != r.pos) r.pos_out[i] = pos[j];
    }
  }
  for (int i = r.left + tid; i < a.L; i += THREADS) {
    r.w_out[i] = 0.0f;
    r.pos_out[i] = r.seen + (i - r.left);
  }
  if (tid == 0) a.count[r.row] = (int32_t)moved;
  for (int i = (int)moved + tid; i < a.moves; i += THREADS) r.dst[i] = r.src[i] = -1;
}

// ---- a long row in several workgroups ----
// A part is up to PART slots, all below the budget or none.  Three launches count the digits, each part into bins of its own (no atomics on memory, nothing to
// clear); a launch finds the digit of the one before by summing the parts.  A fourth writes the lists: what lies in front of a part follows
// from the parts' counts of larger keys and of ties.  It copies who stays where it is, movers leave their weight and position in the workspace, and a
// fifth puts those where the holes are and clears the slots behind the budget; weights and positions may be rewritten in place, since nothing is read
// from them there.
// Two rows of 131072: 5.6 + 7.7 + 6.8 + 12 + 3.9 us, of which 2 - 3 each are launch and first load; 32 of 32768: 7.1 + 8 + 7.4 + 12 + 4.9.  A digit's sums over the
// parts are read sixteen parts at a time (one behind another they were 12600 of a launch's 36000 clocks).
constexpr int PART_THREADS = 1024, PART_J = 8, PART = PART_THREADS * PART_J, PART_WAVES = PART_THREADS / 64;

struct EvictParts {
  int32_t below, parts;                         // parts below the budget, and in all
  uint32_t* bins;                               // (3 passes, rows, parts, SEL_BINS)
  uint32_t* larger;                             // (rows, parts): keys known to be larger than the last that stays
  uint32_t* found;                              // (3 passes, rows, 2)
  float* moved_w;                               // (rows, moves)
  int32_t* moved_pos;
};

__device__ __forceinline__ void part_slots(const EvictSelect& a, const EvictParts& q, const EvictRow& r, int part, int* first, int* end) {
  const int64_t from = part < q.below ? (int64_t)part * PART : (int64_t)a.budget + (int64_t)(part - q.below) * PART;
  const int64_t to = part < q.below && from + PART > a.budget ? a.budget : from + PART;
  *first = (int)(from < r.n ? from : r.n);
  *end = (int)(to < r.n ? to : r.n);
}

// (pass 3: the lists)
template <int PASS>
__global__ void __launch_bounds__(PART_THREADS) evict_part_kernel(const EvictSelect a, const EvictParts q) {
  __shared__ uint32_t s_bin[SEL_BINS];
  __shared__ uint32_t s_wave[PART_WAVES], s_found[2];
  __shared__ uint32_t s_two[2][PART_WAVES], s_part[2][64], s_front[4];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = (int)(blockIdx.x % (unsigned)q.parts);
  const EvictRow r(a, (int)(blockIdx.x / (unsigned)q.parts));
  const int64_t rows = (int64_t)a.B * a.H;
  if (PASS == 0 && part == 0 && r.h == 0 && tid == 0) a.lens_out[r.b] = r.left;
  if (r.n <= a.budget) return;                  // (the last launch does what there is to do)
  int first, end;
  part_slots(a, q, r, part, &first, &end);
  const int base = first + wave * (PART_J * 64);
  float w[PART_J];                              // (on their way while the digits are found)
  int pos[PART_J];
#pragma unroll
  for (int j = 0; j < PART_J; ++j) {
    const int i = base + j * 64 + lane, at = i < end ? i : 0;
    w[j] = r.w[at];
    pos[j] = r.pos[at];
  }
  uint32_t want = (uint32_t)a.budget, last = 0;
  if constexpr (PASS > 0) {
#pragma unroll
    for (int p = 0; p + 1 < PASS; ++p) {        // digits that earlier launches have found
      const uint32_t* f = q.found + (p * rows + r.row) * 2;
      last |= f[0] << sel_low(p);
      want = f[1];
    }
    const uint32_t* bins = q.bins + (((PASS - 1) * rows + r.row) * q.parts) * SEL_BINS;
    // (two neighbouring bins of sixteen parts on their way at a time)
    sel_find<PART_THREADS>(want, [&](int bin, uint32_t* c) {
      static_assert(SEL_BINS / PART_THREADS == 2, "two bins a thread");
      c[0] = c[1] = 0;
      for (int p0 = 0; p0 < q.parts; p0 += 16) {
        uint2 x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = *(const uint2*)(bins + (int64_t)(p0 + i < q.parts ? p0 + i : 0) * SEL_BINS + bin - 1);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (p0 + i < q.parts) { c[0] += x[i].y; c[1] += x[i].x; }
      }
    }, s_wave, s_found);
    const uint32_t digit = s_found[0];
    last |= digit << sel_low(PASS - 1);
    want = s_found[1];
    if (PASS < 3) {
      // every part's own: how many of its keys are larger by this digit
      uint32_t n = 0, total;
#pragma unroll
      for (int u = 0; u < SEL_BINS / PART_THREADS; ++u) {
        const int i = u * PART_THREADS + tid;
        const uint32_t c = bins[(int64_t)part * SEL_BINS + i];
        n += i > (int)digit ? c : 0;
      }
      sel_scan<PART_THREADS>(n, s_wave, &total);
      if (tid == 0) {
        uint32_t* larger = q.larger + r.row * q.parts + part;
        *larger = PASS == 1 ? total : *larger + total;
        if (part == 0) {
          uint32_t* f = q.found + ((PASS - 1) * rows + r.row) * 2;
          f[0] = digit;
          f[1] = want;
        }
      }
    }
  }
  uint32_t k[PART_J];
#pragma unroll
  for (int j = 0; j < PART_J; ++j) k[j] = base + j * 64 + lane < end ? evict_key(w[j], pos[j], a.sinks, r.newest) : 0u;
  if constexpr (PASS < 3) {
    constexpr int LOW = sel_low(PASS), ABOVE = (LOW + sel_bits(PASS)) & 31;
    for (int i = tid; i < SEL_BINS; i += PART_THREADS) s_bin[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PART_J; ++j)
      sel_count(s_bin, base + j * 64 + lane < end && (PASS == 0 || (k[j] >> ABOVE) == (last >> ABOVE)), (k[j] >> LOW) & ((1u << sel_bits(PASS)) - 1));
    __syncthreads();
    uint32_t* mine = q.bins + ((PASS * rows + r.row) * q.parts + part) * SEL_BINS;
    for (int i = tid; i < SEL_BINS; i += PART_THREADS) mine[i] = s_bin[i];
  } else {
    // Parts in slot order: keys that stay for sure and ties of each, a wavefront per part; then one wavefront, a lane per part, sums what lies in front of
    // this part.  64 parts at a time.
    const uint32_t digit = last & ((1u << sel_bits(2)) - 1);
    const uint32_t* bins = q.bins + ((2 * rows + r.row) * q.parts) * SEL_BINS;
    uint32_t ties = 0, ties_all = 0, holes = 0, movers = 0, all = 0;
    for (int p0 = 0; p0 < q.parts; p0 += 64) {
      for (int p = p0 + wave; p < q.parts && p < p0 + 64; p += PART_WAVES) {
        constexpr int U = (1 << sel_bits(2)) / 64;
        uint32_t x[U], n = 0, t = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = bins[(int64_t)p * SEL_BINS + u * 64 + lane];
        const uint32_t larger = q.larger[r.row * q.parts + p];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          n += u * 64 + lane > (int)digit ? x[u] : 0;
          t += u * 64 + lane == (int)digit ? x[u] : 0;
        }
        n = lane_of(lanes_scan(n), 63) + larger;
        t = lane_of(lanes_scan(t), 63);
        if (lane == 0) { s_part[0][p - p0] = n; s_part[1][p - p0] = t; }
      }
      __syncthreads();
      if (wave == 0) {
        const int p = p0 + lane;
        const uint32_t n = p < q.parts ? s_part[0][lane] : 0, t = p < q.parts ? s_part[1][lane] : 0;
        const uint32_t upto = ties_all + lanes_scan(t), before = upto - t;
        const uint32_t kept = n + (want > before ? (want - before < t ? want - before : t) : 0);
        const bool low = p < q.below;
        const uint32_t size = (uint32_t)(p + 1 < q.below ? PART : a.budget - (q.below - 1) * PART);
        const uint32_t h = lanes_scan(low ? size - kept : 0), m = lanes_scan(low || p >= q.parts ? 0 : kept);
        const int front = part - p0 < 0 ? 0 : (part - p0 < 64 ? part - p0 : 64);          // of these parts, in front of this one
        if (lane == 0) { s_front[0] = s_front[1] = s_front[2] = 0; }
        if (lane == front - 1) { s_front[0] = upto - ties_all; s_front[1] = h; s_front[2] = m; }
        if (lane == 63) s_front[3] = m;
        ties_all = lane_of(upto, 63);
      }
      __syncthreads();
      ties += s_front[0]; holes += s_front[1]; movers += s_front[2]; all += s_front[3];
    }
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < PART_J; ++j) mine += (uint32_t)__popcll(__ballot(base + j * 64 + lane < end && k[j] == last));
    uint2 total;
    ties += sel_waves<PART_WAVES>(make_uint2(mine, 0), s_two, &total).x;
    const uint32_t stays = sel_lists<PART_J>(k, base, end, a.budget, last, want, ties, [&](uint2 x) {
      const uint2 at = sel_waves<PART_WAVES>(x, s_two, &total);
      return make_uint2(holes + at.x, movers + at.y);
    }, [&](int slot, uint32_t rank, int j) {
      r.src[rank] = slot;
      q.moved_w[r.row * a.moves + rank] = w[j];
      q.moved_pos[r.row * a.moves + rank] = pos[j];
    }, [] {}, [&](int slot, uint32_t rank, int) { r.dst[rank] = slot; });
    if (part < q.below) {
#pragma unroll
      for (int j = 0; j < PART_J; ++j)
        if (stays >> j & 1) {
          const int i = base + j * 64 + lane;
          if (r.w_out != r.w) r.w_out[i] = w[j];
          if (r.pos_out != r.pos) r.pos_out[i] = pos[j];
        }
    }
    if (part == 0 && tid == 0) a.count[r.row] = (int32_t)all;
  }
}

// A thread for some of a row's numbers: its move of that number, its slot of that number if it is free or the row is left as it is, its place in the
// lists of moves if there is none.
constexpr int FINISH_SHARE = 1024;
__global__ void __launch_bounds__(256) evict_finish_kernel(const EvictSelect a, const EvictParts q, int shares) {
  const int share = (int)(blockIdx.x % (unsigned)shares);
  const EvictRow r(a, (int)(blockIdx.x / (unsigned)shares));
  const bool cut = r.n > a.budget;
  const int moved = cut ? a.count[r.row] : 0;
  if (share == 0 && threadIdx.x == 0 && !cut) a.count[r.row] = 0;
  constexpr int J = FINISH_SHARE / 256;
  int i[J], to[J], pos[J];
  float w[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    i[j] = share * FINISH_SHARE + j * 256 + (int)threadIdx.x;
    const bool move = i[j] < moved, copy = !cut && i[j] < r.left;
    to[j] = move ? r.dst[i[j]] : i[j];
    w[j] = move ? q.moved_w[r.row * a.moves + i[j]] : (copy ? r.w[i[j]] : 0.0f);
    pos[j] = move ? q.moved_pos[r.row * a.moves + i[j]] : (copy ? r.pos[i[j]] : 0);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (i[j] < moved || (!cut && i[j] < r.left)) {
      r.w_out[to[j]] = w[j];
      r.pos_out[to[j]] = pos[j];
    }
    if (i[j] >= r.left && i[j] < a.L) {
      r.w_out[i[j]] = 0.0f;
      r.pos_out[i[j]] = r.seen + (i[j] - r.left);
    }
    if (i[j] >= moved && i[j] < a.moves) r.dst[i[j]] = r.src[i[j]] = -1;
  }
}

// Slots of a row in one workgroup (32 rows of 32768: 53 us with one workgroup of 1024 threads each, 45 in parts)
constexpr int ROW_SLOTS = 16384;

struct EvictPlan { int below, parts, shares; size_t bins_at, larger_at, found_at, w_at, pos_at, bytes; };
static EvictPlan evict_plan(int64_t rows, int L, int budget, int moves) {
  EvictPlan p{};
  if (L <= ROW_SLOTS) return p;
  const int64_t front = std::min(L, budget);
  p.below = (int)((front + PART - 1) / PART);
  p.parts = p.below + (int)((L - front + PART - 1) / PART);
  p.shares = (int)(((int64_t)std::max(L, moves) + FINISH_SHARE - 1) / FINISH_SHARE);
  size_t at = 0;
  const auto take = [&](size_t n) { const size_t here = at; at = (at + n + 255) & ~(size_t)255; return here; };
  p.bins_at = take((size_t)3 * rows * p.parts * SEL_BINS * 4);
  p.larger_at = take((size_t)rows * p.parts * 4);
  p.found_at = take((size_t)3 * rows * 2 * 4);
  p.w_at = take((size_t)rows * moves * 4);
  p.pos_at = take((size_t)rows * moves * 4);
  p.bytes = at;
  return p;
}

// ---- rows of sequences that begin ----
// As many query rows in this step as tokens: nothing was there before it.  Weights 0, positions from 0 on, whatever an earlier sequence of the row has left.
// One launch in every step; where nothing begins a workgroup reads three numbers and ends: 2.0 us for 256 rows of 8192, 5.6 us where all begin (17 MB).
constexpr int BEGIN_SHARE = 4096;
struct EvictBegin {
  float* w;  int64_t w_b, w_h;
  int32_t* pos;  int64_t p_b, p_h;
  const int32_t *lens, *starts;
  int32_t H, L, shares;
};
__global__ void __launch_bounds__(256) evict_begin_kernel(const EvictBegin a) {
  const int share = (int)(blockIdx.x % (unsigned)a.shares), row = (int)(blockIdx.x / (unsigned)a.shares), h = row % a.H, b = row / a.H;
  const int64_t run = (int64_t)a.starts[b + 1] - a.starts[b];
  if (run <= 0 || run != a.lens[b]) return;
  float* w = a.w + b * a.w_b + h * a.w_h;
  int32_t* pos = a.pos + b * a.p_b + h * a.p_h;
  const int end = a.L - share * BEGIN_SHARE < BEGIN_SHARE ? a.L : (share + 1) * BEGIN_SHARE;
  for (int i = share * BEGIN_SHARE + (int)threadIdx.x; i < end; i += 256) {
    w[i] = 0.0f;
    pos[i] = i;
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

// A row's pieces by neighbouring threads, keys and values of a move in the same turn.  Bound by the memory system's rate for rows of 256 bytes here and there:
// 32 rows of sequences and heads cut from 32768 to 4096 (some 3600 moves each, 128-channel bf16, 117 MB read and written) 30 us, 3.9 TB/s; 512 moves 3.6.
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
// disturbed: its bits are written back as they are.  Bound by reads of 2 and 4 bytes from pages here and there: 32 rows cut from 32768 to 4096 (116,000 moves of
// 136 bytes, 32 MB read and written) 49 us.
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

extern "C" size_t tq_evict_select_bytes(int B, int H, int L, int budget, int moves) {
  if (B <= 0 || H <= 0 || L <= 0 || budget <= 0 || moves <= 0) return 0;
  return tq::evict_plan((int64_t)B * H, L, budget, moves).bytes;
}

extern "C" int tq_evict_select(const float* weights, int64_t w_b, int64_t w_h, const int32_t* positions, int64_t p_b, int64_t p_h, const int32_t* seq_lens,
                               const int32_t* seen, int B, int H, int L, int budget, int sinks, int recent, int moves, int32_t* lens_out, int32_t* count,
                               int32_t* dst, int32_t* src, float* weights_out, int64_t wo_b, int64_t wo_h, int32_t* positions_out, int64_t po_b,
                               int64_t po_h, void* workspace, void* stream) {
  using namespace tq;
  if (!weights || !positions || !seq_lens || !lens_out || !count || !dst || !src || !weights_out || !positions_out) return TQ_ENULL;
  if (B < 0 || H <= 0 || L <= 0 || budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget) return TQ_EINVAL;
  if (w_b < 0 || w_h < 0 || p_b < 0 || p_h < 0 || wo_b < 0 || wo_h < 0 || po_b < 0 || po_h < 0 || L > (1 << 30)) return TQ_EINVAL;
  if (moves < std::max(1, std::min(budget, L - budget)) || moves > (1 << 30) || (int64_t)B * H > INT32_MAX) return TQ_EINVAL;
  if (B == 0) return TQ_OK;
  const EvictSelect a{weights, w_b, w_h, positions, p_b, p_h, seq_lens, seen, B, H, L, budget, sinks, recent, moves, lens_out, count, dst, src,
                      weights_out, wo_b, wo_h, positions_out, po_b, po_h};
  hipStream_t st = (hipStream_t)stream;
  const int64_t rows = (int64_t)B * H;
  if (L <= ROW_SLOTS) {
    const dim3 grid((unsigned)rows);
    const auto each = [&](int threads) { return (L + threads - 1) / threads; };
    if (L <= 1024) evict_row_kernel<256, 4><<<grid, dim3(256), 0, st>>>(a, each(256));
    else if (L <= 4096) evict_row_kernel<512, 8><<<grid, dim3(512), 0, st>>>(a, each(512));
    else evict_row_kernel<1024, 16><<<grid, dim3(1024), 0, st>>>(a, each(1024));
    TQ_CHECK_LAUNCH();
    return TQ_OK;
  }
  const EvictPlan p = evict_plan(rows, L, budget, moves);
  if (!workspace) return TQ_ENULL;
  if ((uintptr_t)workspace & 15) return TQ_EINVAL;
  if (rows * p.parts > INT32_MAX || rows * p.shares > INT32_MAX) return TQ_EINVAL;
  char* ws = (char*)workspace;
  const EvictParts q{p.below, p.parts, (uint32_t*)(ws + p.bins_at), (uint32_t*)(ws + p.larger_at), (uint32_t*)(ws + p.found_at), (float*)(ws + p.w_at),
                     (int32_t*)(ws + p.pos_at)};
  const dim3 grid((unsigned)(rows * p.parts)), block(PART_THREADS);
  evict_part_kernel<0><<<grid, block, 0, st>>>(a, q);
  TQ_CHECK_LAUNCH();
  evict_part_kernel<1><<<grid, block, 0, st>>>(a, q);
  TQ_CHECK_LAUNCH();
  evict_part_kernel<2><<<grid, block, 0, st>>>(a, q);
  TQ_CHECK_LAUNCH();
  evict_part_kernel<3><<<grid, block, 0, st>>>(a, q);
  TQ_CHECK_LAUNCH();
  evict_finish_kernel<<<dim3((unsigned)(rows * p.shares)), dim3(256), 0, st>>>(a, q, p.shares);
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

extern "C" int tq_evict_begin(float* weights, int64_t w_b, int64_t w_h, int32_t* positions, int64_t p_b, int64_t p_h, const int32_t* seq_lens,
                              const int32_t* query_start_loc, int B, int H, int L, void* stream) {
  using namespace tq;
  if (!weights || !positions || !seq_lens || !query_start_loc) return TQ_ENULL;
  if (B < 0 || H <= 0 || L <= 0 || L > (1 << 30) || w_b < 0 || w_h < 0 || p_b < 0 || p_h < 0) return TQ_EINVAL;
  const int shares = (L + BEGIN_SHARE - 1) / BEGIN_SHARE;
  if ((int64_t)B * H > INT32_MAX || (int64_t)B * H * shares > INT32_MAX) return TQ_EINVAL;
  if (B == 0) return TQ_OK;
  const EvictBegin a{weights, w_b, w_h, positions, p_b, p_h, seq_lens, query_start_loc, H, L, shares};
  evict_begin_kernel<<<dim3((unsigned)((int64_t)B * H * shares)), dim3(256), 0, (hipStream_t)stream>>>(a);
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
