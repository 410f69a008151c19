// A step's keys and values into the 8-bit cache, and back.
//
// A wavefront takes one block of 16 tokens of one KV head, keys or values: its lanes hold the block's rows 8 neighbouring channels at a time (16 bytes of
// 16-bit input, 8 of the cache), which is all of it, so that the largest value is a reduction over the wavefront and the block is read once.
// Tokens that a block held before the step keep their bytes unless the block's exponent grows: then they are rounded again from what they stand for.  It never shrinks before the
// block starts anew: what was rounded away for a token that is written over later does not come back.
// No two wavefronts write to one block of a head: a block belongs to one sequence.
// Bound by the memory system where there are prompts (32768 rows, 8 heads of 128, bf16: write 44 us, 201 MB in and out, read 38, a launch each: 403 MB in 84 us, 4.8 TB/s; a
// large copy reaches 5.1), by the chain of starts, lengths, table entry and rows where there are tokens (64 tokens: 4.6 and 5.2 us, of which a launch that does nothing is 2).
#include "tq_fp8.h"

#include <algorithm>

namespace tq {

struct Fp8Store {
  Step s;
  Fp8Cache c;
  const void *k, *v;       // write: (rows, H, d), element strides
  int64_t ks_t, ks_h, vs_t, vs_h;
  void *k_out, *v_out;     // read: (rows, H, d) contiguous
  int32_t parts;           // workgroups that share a block's heads
  int32_t fill;            // read: rows of no sequence become zeros
};

// tokens [first, end) of a sequence's run that lie in its n-th block of 16, and the block's row
struct Fp8Unit {
  int b, page, first, end;
  int64_t row;             // of token `first`
  bool any;
};
// blocks that a run touches; rows in front of token 0 count (reading, they are zeros)
__device__ __forceinline__ int store_blocks(const StepRun& r) {
  return r.run == 0 ? 0 : ((r.len - 1) >> 4) - (r.token() >> 4) + 1;
}
__device__ __forceinline__ bool store_unit(const Step& s, int u, Fp8Unit* t, int64_t* rest_unit) {
  int j = 0;
  StepRun r;
  const bool found = step_unit(s, &u, &t->b, &j, &r, [](const StepRun& x) { return store_blocks(x); });
  *rest_unit = u;
  if (!found) return false;
  const int first = r.token();
  t->page = (first >> 4) + j;
  t->first = j == 0 ? first : t->page * TQ_PAGE_TOKENS;
  t->end = (t->page + 1) * TQ_PAGE_TOKENS < r.len ? (t->page + 1) * TQ_PAGE_TOKENS : r.len;
  t->row = r.row + (t->first - first);
  return true;
}
// the block's number, or -1
__device__ __forceinline__ int64_t store_block(const Step& s, const Fp8Unit& t) {
  if (t.page < 0 || t.page >= s.table_row) return -1;
  const int64_t n = s.table[t.b * s.table_step + t.page];
  return n < 0 || n >= s.num_blocks ? -1 : n;
}

// 8 neighbouring channels
template <int DT>
struct Eight {
  f8_u32x4 x;
  __device__ __forceinline__ void load(const void* p, int64_t at) { x = *(const f8_u32x4*)((const uint16_t*)p + at); }
  __device__ __forceinline__ void none() { x = f8_u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float* y) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t h = (uint16_t)(x[i >> 1] >> (i & 1 ? 16 : 0));
      y[i] = DT == TQ_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
    }
  }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* y) {
    f8_u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = DT == TQ_BF16 ? (uint32_t)f32_to_bf16_bits(y[2 * i]) | (uint32_t)f32_to_bf16_bits(y[2 * i + 1]) << 16
                           : (uint32_t)f32_to_f16_bits(y[2 * i]) | (uint32_t)f32_to_f16_bits(y[2 * i + 1]) << 16;
    *(f8_u32x4*)((uint16_t*)p + at) = r;
  }
};
template <>
struct Eight<TQ_F32> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* p, int64_t at) { a = *(const float4*)((const float*)p + at); b = *(const float4*)((const float*)p + at + 4); }
  __device__ __forceinline__ void none() { a = b = make_float4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float* y) const { y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w; y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w; }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* y) {
    *(float4*)((float*)p + at) = make_float4(y[0], y[1], y[2], y[3]);
    *(float4*)((float*)p + at + 4) = make_float4(y[4], y[5], y[6], y[7]);
  }
};

template <int DT, int D>
__global__ void __launch_bounds__(256) fp8_write_kernel(const Fp8Store a) {
  constexpr int PIECES = D / 32, PER_ROW = D / 8;            // pieces of 8 channels: of a lane, of a row
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  Fp8Unit t;
  int64_t rest;
  if (!store_unit(a.s, (int)(blockIdx.x / a.parts), &t, &rest)) return;
  const int64_t block = store_block(a.s, t);
  if (block < 0) return;                                     // (rows in front of token 0 among them: their page has none)
  const int low = t.first - t.page * TQ_PAGE_TOKENS, high = t.end - t.page * TQ_PAGE_TOKENS;
  const int step = 4 * a.parts;
  for (int pair = (int)(blockIdx.x % a.parts) * 4 + wave; pair < 2 * a.c.H; pair += step) {
    const int h = pair >> 1;
    const bool values = pair & 1;
    const void* in = values ? a.v : a.k;
    const int64_t at = t.row * (values ? a.vs_t : a.ks_t) + h * (values ? a.vs_h : a.ks_h), s_t = values ? a.vs_t : a.ks_t;
    uint8_t* cache = (values ? a.c.v : a.c.k) + block * a.c.s_blk + h * a.c.s_h;
    uint8_t* scale = (values ? a.c.v_scales : a.c.k_scales) + block * a.c.H + h;
    Eight<DT> x[PIECES];
    int e_old = F8_LOWEST;
    if (low > 0) e_old = (int)*scale - F8_BIAS;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = i * 64 + lane, r = n / PER_ROW, c = (n - r * PER_ROW) * 8;
      if (r >= low && r < high) x[i].load(in, at + (int64_t)(r - low) * s_t + c);
      else x[i].none();
    }
    float largest = 0.0f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      float y[8];
      x[i].get(y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float size = fabsf(y[j]);
        largest = size < INFINITY && size > largest ? size : largest;
      }
    }
    int e = f8_exponent(wave_max_fast(largest));
    e_old = e_old < F8_LOWEST ? F8_LOWEST : (e_old > F8_HIGHEST ? F8_HIGHEST : e_old);
    e = e > e_old ? e : e_old;
    const float f = f8_power(-e);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = i * 64 + lane, r = n / PER_ROW, c = (n - r * PER_ROW) * 8;
      if (r >= low && r < high) {
        float y[8];
        x[i].get(y);
        *(f8_u32x2*)(cache + (int64_t)r * a.c.s_t + c) = f8_u32x2{f8_pack4(y[0] * f, y[1] * f, y[2] * f, y[3] * f), f8_pack4(y[4] * f, y[5] * f, y[6] * f, y[7] * f)};
      }
    }
    if (low > 0 && e > e_old) {                              // (the same for the whole wavefront)
      const float g = e - e_old > 126 ? 0.0f : f8_power(e_old - e);
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int n = i * 64 + lane, r = n / PER_ROW, c = (n - r * PER_ROW) * 8;
        if (r < low) {
          f8_u32x2* p = (f8_u32x2*)(cache + (int64_t)r * a.c.s_t + c);
          const f8_u32x2 was = *p;
          float y[8];
          f8_unpack4(was[0], y);
          f8_unpack4(was[1], y + 4);
          *p = f8_u32x2{f8_pack4(y[0] * g, y[1] * g, y[2] * g, y[3] * g), f8_pack4(y[4] * g, y[5] * g, y[6] * g, y[7] * g)};
        }
      }
    }
    if (lane == 0) *scale = (uint8_t)(e + F8_BIAS);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(256) fp8_read_kernel(const Fp8Store a) {
  constexpr int PIECES = D / 32, PER_ROW = D / 8;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  Fp8Unit t;
  int64_t rest, block = -1, front = 0, all = 0;
  const bool mine = store_unit(a.s, (int)(blockIdx.x / a.parts), &t, &rest);
  int low = 0, high = 0;
  if (mine) {
    block = store_block(a.s, t);
    low = t.first - t.page * TQ_PAGE_TOKENS;
    high = t.end - t.page * TQ_PAGE_TOKENS;
  } else {                                                    // sixteen rows of no sequence
    if (!a.fill) return;
    all = step_rest(a.s, &front);
    if (rest * TQ_PAGE_TOKENS >= all) return;
    high = all - rest * TQ_PAGE_TOKENS < TQ_PAGE_TOKENS ? (int)(all - rest * TQ_PAGE_TOKENS) : TQ_PAGE_TOKENS;
  }
  const int step = 4 * a.parts;
  for (int pair = (int)(blockIdx.x % a.parts) * 4 + wave; pair < 2 * a.c.H; pair += step) {
    const int h = pair >> 1;
    const bool values = pair & 1;
    const uint8_t* cache = (values ? a.c.v : a.c.k) + block * a.c.s_blk + h * a.c.s_h;
    const float f = block < 0 ? 0.0f : f8_scale((values ? a.c.v_scales : a.c.k_scales)[block * a.c.H + h]);
    void* out = values ? a.v_out : a.k_out;
    f8_u32x2 x[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = i * 64 + lane, r = n / PER_ROW, c = (n - r * PER_ROW) * 8;
      x[i] = f8_u32x2{0, 0};
      if (block >= 0 && r >= low && r < high) x[i] = *(const f8_u32x2*)(cache + (int64_t)r * a.c.s_t + c);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = i * 64 + lane, r = n / PER_ROW, c = (n - r * PER_ROW) * 8;
      if (r >= low && r < high) {
        const int64_t row = mine ? t.row + (r - low) : step_rest_row(a.s, front, all, rest * TQ_PAGE_TOKENS + r);
        float y[8];
        f8_unpack4(x[i][0], y);
        f8_unpack4(x[i][1], y + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= f;
        Eight<DT>::store(out, (row * a.c.H + h) * D + c, y);
      }
    }
  }
}

// Workgroups for a step of so many rows: the blocks that its sequences touch at most, and the rest rows'.  A block's heads are shared out to
// as many workgroups as bring the launch to a few for each compute unit, and to more where one would have over 32 KB of rows (32768 rows, us in one / in two / in four: 8 heads of 256, bf16,
// 128 KB, read 112 / 93 / 88; of 128, 64 KB, 39.6 / 38.1 / 40.0; of 64, 32 KB, 19.2 / 18.7 / 21.5).
static int64_t store_units(int64_t rows, int B) { return (rows + TQ_PAGE_TOKENS - 1) / TQ_PAGE_TOKENS + 2 * (int64_t)B + 1; }
static int store_parts(int64_t units, int H, int d, int dtype) {
  const int most = (2 * H + 3) / 4;
  const int64_t rows = 2ll * H * TQ_PAGE_TOKENS * d * (dtype == TQ_F32 ? 4 : 2);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, std::max<int64_t>((1024 + units - 1) / units, (rows + 32767) / 32768)));
}

template <int DT>
static int launch_store(const Fp8Store& a, bool write, int64_t grid, hipStream_t st) {
  const dim3 g((unsigned)grid), block(256);
#define TQ_STORE_D(D)                                             \
  case D:                                                         \
    if (write) fp8_write_kernel<DT, D><<<g, block, 0, st>>>(a);   \
    else fp8_read_kernel<DT, D><<<g, block, 0, st>>>(a);          \
    break
  switch (a.c.d) {
    TQ_STORE_D(64); TQ_STORE_D(128); TQ_STORE_D(192); TQ_STORE_D(256);
    default: return TQ_EUNSUPPORTED;
  }
#undef TQ_STORE_D
  TQ_CHECK_LAUNCH();
  return TQ_OK;
}

static int store(Fp8Store& a, int dtype, bool write, hipStream_t st) {
  if (a.s.rows == 0) return TQ_OK;
  const int64_t units = store_units(a.s.rows, a.s.B);
  a.parts = store_parts(units, a.c.H, a.c.d, dtype);
  if (units * a.parts > STEP_MAX_GROUPS) return TQ_EINVAL;
  switch (dtype) {
    case TQ_F32: return launch_store<TQ_F32>(a, write, units * a.parts, st);
    case TQ_F16: return launch_store<TQ_F16>(a, write, units * a.parts, st);
    case TQ_BF16: return launch_store<TQ_BF16>(a, write, units * a.parts, st);
    default: return TQ_EINVAL;
  }
}

}  // namespace tq

extern "C" int tq_fp8_write(const void* k, const void* v, int dtype, int64_t rows, int64_t ks_t, int64_t ks_h, int64_t vs_t, int64_t vs_h,
                            const int32_t* query_start_loc, int B, int Hkv, int d, void* k_cache, void* v_cache, uint8_t* k_scales, uint8_t* v_scales,
                            int64_t cs_blk, int64_t cs_t, int64_t cs_h, int64_t num_blocks, const int32_t* block_table, int bt_stride,
                            const int32_t* seq_lens, void* stream) {
  using namespace tq;
  if (!k || !v || !query_start_loc) return TQ_ENULL;
  Fp8Store a{};
  if (const int rc = step_init(&a.s, query_start_loc, rows, B, seq_lens, block_table, bt_stride, num_blocks)) return rc;
  if (const int rc = fp8_cache_init(&a.c, k_cache, v_cache, k_scales, v_scales, Hkv, d, cs_blk, cs_t, cs_h)) return rc;
  if (bt_stride < 0 && B > 1) return TQ_EINVAL;                         // (one table for several: they would write to the same blocks)
  if (dtype < TQ_F32 || dtype > TQ_BF16) return TQ_EINVAL;
  const int64_t piece = dtype == TQ_F32 ? 4 : 8;
  if (ks_t < 0 || ks_h < 0 || vs_t < 0 || vs_h < 0) return TQ_EINVAL;
  if (ks_t % piece || ks_h % piece || vs_t % piece || vs_h % piece || (((uintptr_t)k | (uintptr_t)v) & 15)) return TQ_EUNSUPPORTED;
  a.k = k; a.v = v; a.ks_t = ks_t; a.ks_h = ks_h; a.vs_t = vs_t; a.vs_h = vs_h;
  return store(a, dtype, true, (hipStream_t)stream);
}

extern "C" int tq_fp8_read(void* k_out, void* v_out, int dtype, int64_t rows, const int32_t* query_start_loc, int B, int Hkv, int d, const void* k_cache,
                           const void* v_cache, const uint8_t* k_scales, const uint8_t* v_scales, int64_t cs_blk, int64_t cs_t, int64_t cs_h,
                           int64_t num_blocks, const int32_t* block_table, int bt_stride, const int32_t* seq_lens, int fill, void* stream) {
  using namespace tq;
  if (!k_out || !v_out || !query_start_loc) return TQ_ENULL;
  Fp8Store a{};
  if (const int rc = step_init(&a.s, query_start_loc, rows, B, seq_lens, block_table, bt_stride, num_blocks)) return rc;
  if (const int rc = fp8_cache_init(&a.c, (void*)k_cache, (void*)v_cache, (void*)k_scales, (void*)v_scales, Hkv, d, cs_blk, cs_t, cs_h)) return rc;
  if (dtype < TQ_F32 || dtype > TQ_BF16) return TQ_EINVAL;
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return TQ_EUNSUPPORTED;
  a.k_out = k_out; a.v_out = v_out; a.fill = fill;
  return store(a, dtype, false, (hipStream_t)stream);
}
