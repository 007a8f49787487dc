// Attention of a chunk of new tokens over a paged KV cache: how a batch is cut into tiles and
// work items. Shared by the attention kernel and the kernel that merges split items.
#pragma once

#include "common.cuh"

namespace tasft {

constexpr int kChunkBlk = 64;          // block size (tokens) of the kept lists
constexpr int kChunkMaxSplits = 128;   // most items one tile is cut into
constexpr int kChunkMinPiece = 4;      // fewest blocks an item is cut down to
constexpr int kChunkBuckets = 256;     // entries of the per-CTA prefix over sequences

// Launch-wide choices the host makes from types and sizes.
struct ChunkShape {
  int mode;       // how the 128 rows of a tile are filled, see chunk_tc.cu
  int hpt, tpt;   // query heads and tokens of a tile (mode 2: unused)
  int units;      // tiles beside one another at the same tokens (kv-heads, or pairs of query heads)
  int bound;      // most blocks a row can visit: list width, or capacity of the block table
  int capacity;   // tokens the block table can hold (max_pages * page_size)
  int slots;      // split items the workspace has room for
  int rows;       // rows of a split item's partials
  int stride;     // sequences per entry of the per-CTA prefix
};

// Workspace: plan [B] {splits, first slot}, then (m, l) and O of every split item's rows.
struct ChunkWs {
  int2* plan;
  float2* ml;   // [slots, rows] (row maximum in base-2 units, row sum)
  float* o;     // [slots, rows, D] sums not yet divided by l
};

struct ChunkSeq {
  int start, n, ctx, len;  // first row of its new tokens, how many, tokens before them, all tokens
  int tiles, cost;         // tiles per unit; most blocks one tile visits
  bool bad;
};

__device__ __forceinline__ ChunkSeq chunk_seq(const tasft_chunk_args& a, const ChunkShape& sh, int b) {
  ChunkSeq s;
  s.start = a.cu_seqlens[b];
  const int end = a.cu_seqlens[b + 1];
  s.len = a.kv_len[b];
  s.bad = s.start < 0 || end < s.start || end > a.T;
  s.n = s.bad ? 0 : end - s.start;
  if (s.n > 0 && (s.len < s.n || s.len > sh.capacity || s.n > a.max_q)) {
    s.bad = true;
    s.n = 0;
  }
  s.ctx = s.n > 0 ? s.len - s.n : 0;
  if (s.n == 0) {
    s.tiles = s.cost = 0;
  } else {
    if (sh.mode == 0) {
      s.tiles = (s.n + sh.tpt - 1) / sh.tpt;
    } else {
      // tiles stand at multiples of their token count, so none spans two rows of the lists
      // (mode 2 with one head per kv-head: two rows on purpose)
      s.tiles = (s.len - 1) / sh.tpt - s.ctx / sh.tpt + 1;
    }
    s.cost = min((s.len + kChunkBlk - 1) / kChunkBlk, sh.bound);
  }
  return s;
}

// Items a tile of this sequence is cut into, for pieces of about `target` blocks.
__device__ __forceinline__ int chunk_splits(const ChunkSeq& s, int target) {
  return s.n == 0 ? 1 : max(1, min(kChunkMaxSplits, (s.cost + target - 1) / target));
}

__device__ __forceinline__ int warp_sum_int(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int warp_scan_int(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

}  // namespace tasft
