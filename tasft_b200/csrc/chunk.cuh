// Attention of a chunk of new tokens over a paged KV cache: how a batch is cut into tiles and
// work items. Shared by the attention kernel and the kernel that merges split items.
#pragma once

#include "common.cuh"

namespace tasft {

constexpr int kChunkBlk = 64;          // block size (tokens) of the kept lists
constexpr int kChunkMaxSplits = 128;   // most items one tile is cut into
constexpr int kChunkMinPiece = 4;      // fewest blocks an item is cut down to
constexpr int kChunkMergeCost = 10;    // what a cut costs (partials, merge), in blocks
constexpr int kChunkBuckets = 256;     // entries of the per-CTA prefix over sequences

// Launch-wide choices the host makes from types and sizes.
struct ChunkShape {
  int mode;       // how the 128 rows of a tile are filled, see chunk_tc.cu
  int hpt, tpt;   // query heads and tokens of a tile (mode 2: unused)
  int units;      // tiles beside one another at the same tokens (kv-heads, or pairs of query heads)
  int tpt_log2;   // modes 1 and 2
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
  int tiles;               // per unit
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
  s.tiles = 0;
  if (s.n > 0) {
    if (sh.mode == 0) {
      s.tiles = (uint32_t)(s.n + sh.tpt - 1) / (uint32_t)sh.tpt;
    } else {
      // tiles stand at multiples of their token count, so none spans two rows of the lists
      // (mode 2 with one head per kv-head: two rows on purpose)
      s.tiles = ((s.len - 1) >> sh.tpt_log2) - (s.ctx >> sh.tpt_log2) + 1;
    }
  }
  return s;
}

// Blocks a tile of the sequence visits, for balance alone: those up to its last token, or the
// length of that token's list (first head; mode 2 walks two lists).
__device__ __forceinline__ int chunk_cost(const tasft_chunk_args& a, const ChunkShape& sh, const ChunkSeq& s, int b) {
  if (s.n == 0) return 0;
  const int last = (s.len - 1) / kChunkBlk;
  if (sh.mode == 0) return last + 1;
  const int cnt = a.kept_cnt[(int64_t)b * a.Hm * a.nb_q + (last - s.ctx / kChunkBlk)];
  return min(max(cnt, 0) * (sh.mode == 2 ? 2 : 1), last + 1);
}

// Items a tile is cut into, for pieces of about `target` blocks.
__device__ __forceinline__ int chunk_splits(int cost, int target) {
  if (cost <= target + kChunkMergeCost) return 1;
  return min(kChunkMaxSplits, (int)((uint32_t)(cost + target - 1) / (uint32_t)target));
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
