// Attention of a chunk of new tokens over a paged KV cache: how a batch is cut into tiles and
// its work shared out over the CTAs.
#pragma once

#include "common.cuh"

namespace tasft {

constexpr int kChunkBlk = 64;        // block size (tokens) of the kept lists
constexpr int kChunkMinPiece = 4;    // fewest blocks a CTA's share is cut down to
constexpr int kChunkMergeCost = 10;  // what cutting tiles costs a call (partials, merge), in blocks
constexpr int kChunkBuckets = 256;   // entries of the per-CTA table of sequences

// Launch-wide choices the host makes from types and sizes.
struct ChunkShape {
  int mode;       // how the 128 rows of a tile are filled, see chunk_tc.cu
  int hpt, tpt;   // query heads and tokens of a tile
  int tpt_log2;   // modes 1 and 2
  int units;      // tiles beside one another at the same tokens (kv-heads, or pairs of query heads)
  int capacity;   // tokens the block table can hold (max_pages * page_size)
  int rows;       // rows of a piece's partials
  int stride;     // sequences per entry of the table
  int may_cut;    // 0: cutting tiles gains nothing
  int wide;       // rows of out on 32-byte boundaries
  int zero_rest;  // rows of out that no sequence accounts for become 0
};

struct ChunkSeq {
  int start, n, ctx, len;  // first row of its new tokens, how many, tokens before them, all tokens
  int tiles;               // per unit
  int cost;                // blocks a tile visits, for balance alone (lists; the dense mode counts tokens)
  bool bad;
};

__device__ __forceinline__ int chunk_tiles(const ChunkShape& sh, int n, int ctx, int len) {
  if (n <= 0) return 0;
  if (sh.mode == 0) return (uint32_t)(n + sh.tpt - 1) / (uint32_t)sh.tpt;
  // tiles stand at multiples of their token count, so none spans two rows of the lists (mode 2
  // with one head per kv-head: two rows on purpose)
  return ((len - 1) >> sh.tpt_log2) - (ctx >> sh.tpt_log2) + 1;
}

// Whether sequence rows and lengths fit T, max_q, the block table and each other.
__device__ __forceinline__ bool chunk_fits(const tasft_chunk_args& a, const ChunkShape& sh, int start, int end, int len) {
  if (start < 0 || end < start || end > a.T) return false;
  const int n = end - start;
  return n == 0 || (len >= n && len <= sh.capacity && n <= a.max_q);
}

__device__ __forceinline__ ChunkSeq chunk_seq(const tasft_chunk_args& a, const ChunkShape& sh, int b) {
  ChunkSeq s;
  s.start = a.cu_seqlens[b];
  const int end = a.cu_seqlens[b + 1];
  s.len = a.kv_len[b];
  s.bad = !chunk_fits(a, sh, s.start, end, s.len);
  s.n = s.bad ? 0 : end - s.start;
  s.ctx = s.n > 0 ? s.len - s.n : 0;
  s.tiles = chunk_tiles(sh, s.n, s.ctx, s.len);
  s.cost = 0;
  if (sh.mode != 0 && s.n > 0) {
    // the length of the last token's list (first head; mode 2 walks two lists)
    const int last = (s.len - 1) / kChunkBlk;
    const int cnt = a.kept_cnt[(int64_t)b * a.Hm * a.nb_q + (last - s.ctx / kChunkBlk)];
    s.cost = max(1, min(cnt * (sh.mode == 2 ? 2 : 1), last + 1));
  }
  return s;
}

// Weight of a tile (64 per block) and of all tiles of a unit before it. Without lists a tile
// visits the blocks up to its last token; with lists all tiles of a sequence count alike.
__device__ __forceinline__ int64_t chunk_weight(const ChunkShape& sh, const ChunkSeq& s, int i) {
  return sh.mode == 0 ? (int64_t)s.ctx + 63 + (int64_t)(i + 1) * sh.tpt : (int64_t)s.cost * kChunkBlk;
}
__device__ __forceinline__ int64_t chunk_weight_before(const ChunkShape& sh, const ChunkSeq& s, int i) {
  return sh.mode == 0 ? (int64_t)i * (s.ctx + 63) + (int64_t)sh.tpt * ((int64_t)i * (i + 1) / 2)
                      : (int64_t)i * s.cost * kChunkBlk;
}

// A place in the sequence of all tiles (sequence, unit, tile) and the weight `rho` into the tile;
// b == B: the end.
struct ChunkCut {
  int b, unit, tile;
  int64_t rho, w;
  ChunkSeq s;
};

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int64_t warp_max64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const int64_t x = __shfl_xor_sync(0xffffffffu, v, o);
    v = x > v ? x : v;
  }
  return v;
}
__device__ __forceinline__ int64_t warp_scan64(int64_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

}  // namespace tasft
