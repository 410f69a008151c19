// The weight that a prompt's newest queries give to the tokens of a paged exact cache.
#pragma once

#include "tq_exact.h"

namespace tq {

struct ExactWindow {
  ExactCache c;                  // (its values are not read)
  const void* q;                 // (rows, Hq, d)
  const int32_t* starts;         // (B + 1): the rows of each sequence
  int64_t rows;
  int32_t B, Hq, G, W;           // W: newest rows of a sequence that count, at most
  int32_t row_tiles, tile_waves, row_groups;     // tiles of 16 (query, head) rows at most; wavefronts side by side on them; turns that they take
  int32_t n_split, chunk;        // as in decode
  int32_t waves;                 // of a workgroup: 4 or 8
  uint32_t per_head;             // 2^32 / G, rounded up (G > 1): r / G is the upper half of a product, r * G < 2^32
  float scale2;                  // |scale| log2 e, positive
  uint32_t flip;                 // the sign bits of the queries' elements, for a negative scale
  float2* ml;                    // (B, H, parts, row_tiles * 16): maximum (log2) and sum of a row over a part of the tokens
  float2* stat;                  // (B, H, row_tiles * 16): of all tokens: maximum and 1 / sum
  int32_t parts;
  float* weights;
  int64_t w_b, w_h;
  int32_t L;
};

template <int DT> int launch_exact_window(const ExactWindow& a, bool add, hipStream_t stream);

// row tiles that a wavefront holds as operands: d / 8 registers each, fp32 twice as many
__host__ __device__ constexpr int window_tiles(int dt, int d) {
  return dt == TQ_F32 ? (d <= 64 ? 4 : (d <= 128 ? 2 : 1)) : (d <= 256 ? 4 : (d <= 512 ? 2 : 1));
}
__host__ __device__ constexpr int window_waves_per_simd(int dt, int d, int waves) { return dt != TQ_F32 && d <= 128 ? (waves == 4 ? 3 : (d <= 64 ? 4 : 2)) : 2; }
// bytes of a block's keys (32 tokens, fp32 16) in LDS, and of all blocks that a workgroup may hold
__host__ __device__ constexpr int window_block_bytes(int d) { return 64 * d; }
constexpr int WINDOW_LDS = 96 * 1024;
// Queries go by way of LDS where eight wavefronts stand on tiles of their own and a tile for each of them fits beside the keys: read as operands, sixteen rows of 64
// bytes a load, 256 KB of them (512 rows of 256 channels) took 20000 clocks, half of a workgroup's time (nine prompts of 17 .. 4099, 16 / 2 heads of 256, 64
// queries: passes of 22.2 and 23.7 us, this way 20.3 and 19.8).  Workgroups of four have fewer rows.
__host__ __device__ constexpr int window_tile_bytes(int dt, int d) { return 16 * d * (dt == TQ_F32 ? 4 : 2); }
__host__ __device__ constexpr bool window_staged(int dt, int d, int waves) {
  return waves == 8 && d >= 128 && waves * window_tile_bytes(dt, d) <= 64 * 1024 && 2 * window_block_bytes(d) + waves * window_tile_bytes(dt, d) <= WINDOW_LDS;
}

}  // namespace tq
