// A step of an engine over a paged cache: rows starts[b] .. starts[b + 1] - 1 of the step's tensors are sequence b's, the last of them its token
// lens[b] - 1, whose block is table[b][token / 16].  All of it lies in device memory; the host knows the number of rows and of sequences only.
#pragma once

#include "tq_common.h"

namespace tq {

constexpr int64_t STEP_MAX_GROUPS = (1 << 24) - 1;      // of 256: a launch has less than 2^32 threads

struct Step {
  const int32_t* starts;   // B + 1; null: one row per sequence
  const int32_t* lens;
  const int32_t* table;
  int64_t table_step;      // entries from one sequence's row to the next; 0: one row for all
  int64_t num_blocks;
  int32_t table_row;       // entries of a row
  int32_t B;
  int64_t rows;            // of the step's tensors
};

// Sequence b's rows: [row, row + run), the first of them token `token` (negative where a sequence has more rows than tokens).  What starts says is cut to
// the rows that there are.
struct StepRun {
  int64_t row;
  int32_t run, len;
  __device__ __forceinline__ int32_t token() const { return len - run; }
};
__device__ __forceinline__ StepRun step_run(const Step& s, int b) {
  StepRun r;
  const int n = s.lens[b];
  r.len = n < 0 ? 0 : (n > INT32_MAX - 64 ? INT32_MAX - 64 : n);      // (so that the next block's first token is a number, too)
  if (!s.starts) { r.row = b; r.run = 1; return r; }
  int64_t first = s.starts[b], end = s.starts[b + 1];
  first = first < 0 ? 0 : first;
  end = end > s.rows ? s.rows : end;
  r.row = first;
  r.run = end > first ? (int32_t)(end - first) : 0;
  return r;
}
// tokens that the table has blocks for
__device__ __forceinline__ int32_t step_cap(const Step& s) {
  const int64_t most = (int64_t)s.table_row * TQ_PAGE_TOKENS;
  return most > INT32_MAX ? INT32_MAX : (int32_t)most;
}
// Rows of no sequence: in front of the first one's and behind the last one's.  Their number, and the n-th of them.
__device__ __forceinline__ int64_t step_rest(const Step& s, int64_t* front) {
  *front = 0;
  if (!s.starts) return 0;
  int64_t a = s.starts[0], z = s.starts[s.B];
  a = a < 0 ? 0 : (a > s.rows ? s.rows : a);
  z = z < a ? a : (z > s.rows ? s.rows : z);
  *front = a;
  return a + s.rows - z;
}
__device__ __forceinline__ int64_t step_rest_row(const Step& s, int64_t front, int64_t rest, int64_t n) { return n < front ? n : n + s.rows - rest; }

// a number that is the same in all lanes, as a scalar
__device__ __forceinline__ int64_t step_uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// sums over the lanes up to each one, by row shifts and the two broadcasts of a row's last lane; the whole wavefront
__device__ __forceinline__ int step_sums(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Sequences are looked at 256 at a time, four a lane and 64 apart, so that their loads are on their way together.
constexpr int STEP_ROUND = 256;
__device__ __forceinline__ void step_runs(const Step& s, int base, StepRun (&r)[4]) {
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = base + i * 64 + lane;
    r[i].run = r[i].len = 0;
    r[i].row = 0;
    if (base + i * 64 < s.B && at < s.B) r[i] = step_run(s, at);
  }
}
// Of a round whose sequences have count[i] units each: which has unit *u (their sums fit 31 bits), which one of its units that is, and its rows.  false:
// none of them, and *u is less by all of theirs.
__device__ __forceinline__ bool step_find(const Step& s, int base, const StepRun (&r)[4], const int (&count)[4], int* u, int* b, int* j, StepRun* run) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (base + i * 64 >= s.B) break;
    const int upto = step_sums(count[i]), all = __builtin_amdgcn_readlane(upto, 63);
    if (*u < all) {
      const int owner = __ffsll((unsigned long long)__ballot(upto > *u)) - 1;
      *b = base + i * 64 + owner;
      *j = *u - (__builtin_amdgcn_readlane(upto, owner) - __builtin_amdgcn_readlane(count[i], owner));
      run->row = __builtin_amdgcn_readlane((int)r[i].row, owner);      // (a step has less than 2^31 rows)
      run->run = __builtin_amdgcn_readlane(r[i].run, owner);
      run->len = __builtin_amdgcn_readlane(r[i].len, owner);
      return true;
    }
    *u -= all;
  }
  return false;
}
// How many units the sequences in front of sequence b have, of a step's first round.
__device__ __forceinline__ int step_before(const Step& s, const int (&count)[4], int b) {
  int before = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i * 64 > b) break;
    const int upto = step_sums(count[i]), in = b - i * 64 < 64 ? b - i * 64 : 63;
    before += __builtin_amdgcn_readlane(upto, in) - (b - i * 64 < 64 ? __builtin_amdgcn_readlane(count[i], in) : 0);
  }
  return before;
}
// Unit `u` of a step whose sequence b has count(b) of them: its sequence, which one of them it is and the sequence's rows; false (and u less all of them) if there are fewer.
// A whole wavefront asks; u is the same in all lanes.
template <class Count>
__device__ __forceinline__ bool step_unit(const Step& s, int* u, int* b, int* j, StepRun* run, Count count) {
  for (int base = 0; base < s.B; base += STEP_ROUND) {
    StepRun r[4];
    step_runs(s, base, r);
    int c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = r[i].run ? count(r[i]) : 0;
    if (step_find(s, base, r, c, u, b, j, run)) return true;
  }
  return false;
}

// A table entry at a place that is the same for the whole wavefront: no launch writes its own table, so that this is a scalar load, which waits for no
// vector load in front of it.
__device__ __forceinline__ int32_t step_entry(const int32_t* table, int page) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)table)[page];
}
// four of them, one behind another
__device__ __forceinline__ uint32_t __attribute__((ext_vector_type(4))) step_entries(const int32_t* table, int page) {
  typedef uint32_t four __attribute__((ext_vector_type(4), aligned(4)));
  return *(const __attribute__((address_space(4))) four*)(uintptr_t)(table + page);
}

// what the entry points check of a step, and its description
inline int step_init(Step* s, const int32_t* starts, int64_t rows, int B, const int32_t* lens, const int32_t* table, int bt_stride, int64_t num_blocks) {
  if ((!table || !lens) && B > 0) return TQ_ENULL;           // (no sequence: nobody looks at either)
  if (B < 0 || rows < 0 || rows > INT32_MAX || num_blocks <= 0 || bt_stride == 0 || bt_stride == INT32_MIN) return TQ_EINVAL;
  s->starts = starts; s->lens = lens; s->table = table; s->rows = rows; s->B = B; s->num_blocks = num_blocks;
  s->table_row = bt_stride < 0 ? -bt_stride : bt_stride;
  s->table_step = bt_stride < 0 ? 0 : bt_stride;
  return TQ_OK;
}

}  // namespace tq
