// Attention over a paged EXACT cache: blocks of 16 tokens x KV heads x head_dim in fp32, fp16 or bf16, as a serving engine keeps them.
#pragma once

#include <atomic>

#include "tq_common.h"

namespace tq {

// A paged exact cache and the sequences in it.  Element strides; channels lie one behind another, rows start on 16-byte boundaries.
struct ExactCache {
  const void *k, *v;
  int64_t s_blk, s_h;      // of a block, of a KV head
  int32_t s_t;             // of a token
  int32_t H, d;
  int64_t num_blocks;
  const int32_t* table;
  const int32_t* lens;
  int64_t table_step;      // entries from one sequence's row to the next; 0: one row for all
  int32_t table_row;       // entries of a row
};

// tokens of sequence b that the cache can hold
__device__ __forceinline__ int exact_len(const ExactCache& c, int b) {
  const int64_t most = (int64_t)c.table_row * TQ_PAGE_TOKENS;
  const int n = c.lens[b];
  return n < 0 ? 0 : (n > most ? (int)most : n);
}

// Splits of a sequence: every workgroup takes `chunk` blocks of tokens, more of them only where a sequence would need more splits than there are
// (a length beyond the bound that the host planned for).
__host__ __device__ __forceinline__ int exact_blocks_per_split(int blocks, int n_split, int chunk) {
  const int least = (blocks + n_split - 1) / n_split;
  return least > chunk ? least : chunk;
}
__host__ __device__ __forceinline__ int exact_splits_used(int blocks, int n_split, int chunk) {
  const int per = exact_blocks_per_split(blocks, n_split, chunk);
  return (blocks + per - 1) / per;
}

constexpr int EXACT_HEADS = 16;                     // query heads of a workgroup: columns of a matrix instruction
template <int DT> constexpr int exact_tokens() { return DT == TQ_F32 ? 16 : 32; }      // tokens of a wavefront's block

struct ExactDecode {
  ExactCache c;
  const void* q;           // (B, Hq, d)
  void* out;               // (B, Hq, d)
  int32_t B, Hq, G, groups, n_split, chunk;
  float scale2;            // scale x log2 e: the softmax is one of powers of two
  float* acc;              // (B, Hq, n_split, d): numerators of a split; unused with one split
  float2* ml;              // (B, Hq, n_split): its maximum (log2) and its sum
  float* scores;           // (B, H, score_pages, G, 16) scaled scores (log2), for the weights; or null
  int32_t score_pages;
};

// Which part of the work a workgroup takes.  Workgroups go to the eight dies in turn: the groups of heads of one part, which read the same keys and
// values, go to one die one after another; the splits of a sequence go to different ones (with as many pairs of sequence and KV head as
// dies, or splits as dies, a long sequence would otherwise be one die's work).
__host__ __device__ __forceinline__ int64_t exact_grid(const ExactDecode& a) {
  const int64_t parts = (int64_t)a.n_split * a.c.H * a.B;
  return a.groups == 1 ? parts : (parts + 7) / 8 * 8 * a.groups;
}
__device__ __forceinline__ bool exact_place(const ExactDecode& a, int* split, int* group, int* h, int* b) {
  const unsigned pairs = (unsigned)(a.c.H * a.B);
  unsigned id = blockIdx.x, part = id;
  *group = 0;
  if (a.groups > 1) {
    const unsigned turn = id >> 3;
    *group = (int)(turn % (unsigned)a.groups);
    part = (turn / (unsigned)a.groups) * 8 + (id & 7);
    if (part >= pairs * (unsigned)a.n_split) return false;
  }
  const unsigned s = part / pairs, pair = (part - s * pairs + s) % pairs;
  *split = (int)s;
  *h = (int)(pair % (unsigned)a.c.H);
  *b = (int)(pair / (unsigned)a.c.H);
  return true;
}

struct ExactJoin {
  const int32_t* lens;
  int32_t table_row, B, Hq, H, G, d, n_split, chunk, block_tokens;
  const float* acc;
  const float2* ml;
  void* out;
  const float* scores;
  int32_t score_pages;
  float* weights;          // (B, H, L): element strides w_b, w_h
  int64_t w_b, w_h;
  int32_t L, weight_chunks, weight_tokens;
};

// what the entry points check of a cache, and its description
int exact_cache_init(ExactCache* c, const void* k, const void* v, int dtype, int H, int d, int64_t s_blk, int64_t s_t, int64_t s_h, int64_t num_blocks,
                     const int32_t* table, int bt_stride, const int32_t* lens);

template <int DT> int launch_exact_decode(const ExactDecode& a, hipStream_t stream);
template <int DT> int launch_exact_heads(const ExactDecode& a, hipStream_t stream);

// a kernel may use more than 64 KB of LDS once it is told so, on every device for itself
inline int exact_allow_lds(const void* kern, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  if (const hipError_t e = hipGetDevice(&dev)) return (int)e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (ready.load(std::memory_order_relaxed) & bit) return TQ_OK;
  if (const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return (int)e;
  ready.fetch_or(bit, std::memory_order_relaxed);
  return TQ_OK;
}

}  // namespace tq
