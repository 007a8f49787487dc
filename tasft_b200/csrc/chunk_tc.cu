// Attention of a chunk of new tokens over a paged KV cache on the 5th-generation tensor cores.
//
// For token t at position p of its sequence and query head h of kv-head g,
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q.k_j,  m = max_j s_j,
// over the kept keys j <= p: one pass over the keys with the running (m, sum, o) of the
// online softmax in fp32. P is rounded to the value dtype for P.V, as the prefill does (bf16: half
// a step, 2^-8 of each p; fp16: 2^-11 of it or, where it is small, 2^-31 of the largest).
//
// Tile = 128 rows that share one kv-head, filled by mode:
//   0  every block kept: all query heads of a group times as many tokens as fit
//      (row = token * heads + head), so a single token of a group of 4 is 4 rows
//   1  lists per kv-head: the same, with a power of two of tokens that divides 64 and starts
//      at its multiples, so a tile has one list
//   2  lists per query head: two 64-token slots, two heads of a group at one 64-token block
//      (one head at two blocks where a group has one head); the tile walks the union of the
//      two lists and each entry says which slots keep it
// Persistent CTAs (2 per SM, 256 threads) share the work evenly: all tiles in a row, weighted by
// the blocks they visit, are cut into as many equal lengths as there are CTAs, through the middle
// of tiles where that gains more than the merge costs (ChunkCut). A tile cut into pieces leaves
// each piece's (m, l, O) in the workspace and chunk_merge_kernel joins them. Every CTA computes
// the same cuts from cu_seqlens and kv_len, so the host needs neither. A CTA takes its length from
// the back: the piece at its end starts at block 0 and the one at its start ends at the last, so
// CTAs that share K and V run over them side by side and find them in L2. Warps:
//   0     producer: Q of the tile, then K and V of every entry through separate rings
//         (TMA from the pages, 128B swizzle)
//   1     MMA issuer: S = Q K^T (SS, M128 N64) into a double-buffered TMEM tile, O += P V (TS:
//         P read from TMEM where it overwrote S)
//   2     lists: the next segment (at most kSeg entries) of block indices with their pages,
//         double-buffered, ahead of the producer
//   3     looks over the tiles of V that need it
//   4-7   softmax, one thread per row; epilogue
// Warps 0-3 hand registers to the second warpgroup (128 -> 88 and 168 a thread), each role at its
// start: the compiler gives the code behind a common point the smaller count and spills.
// A 0 of P must not meet what V holds behind the mask. Rows of V that no key stands for (past
// kv_len, or of a page that is not there) are zeroed in shared memory before P.V. Where a block
// holds keys that some row of the tile must not see, values that are not finite go to zero too,
// and the rows that do see them take the infinity or NaN in the epilogue. Warp 3 does both while
// the softmax of the block is under way.
// Measured on B200s (in a graph): 2048 tokens over 16384 cached ones, 32/8 heads, D 128, 493 to 576
// us = 1.18 to 1.02 PFLOP/s (the latter under the power cap), held by the chain S -> softmax -> P.V
// of the two tiles an SM has in flight (tensor pipe and MUFU half busy each); 64 single tokens with
// 26 kept blocks in 16-token pages 80 to 84 us = 5.1 to 5.4 TB/s, HBM; one token over 4000 17 us: 4
// for a launch that finds no token, 6 for a first tile, 2 for the merge's launch, 5 for four blocks
// a CTA and the merge.
// Every mbarrier phase is indexed by a global counter and every wait is arranged so the waiter
// is at most one phase behind; every wait is bounded (TASFT_DEVERR_TIMEOUT).
#include "chunk.cuh"
#include "tc.cuh"

#include <cfloat>

namespace tasft {

namespace {

constexpr int kThreads = 256;
constexpr int kMergeThreads = 1024;        // four rows a warp: the merge is a chain of latencies
constexpr int kSeg = 128;                  // entries of a list segment
constexpr uint32_t kTmemCols = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
// fp16 holds nothing below 2^-25, so many small probabilities beside a large one would come to 0
// (60000 of 2^-25.4 are 0.14 %): P is held, and l summed, 2^6 times as large, 2^14 at most
constexpr float kHalfShift = 6.0f;

// entry of a list segment: block index, which of its (up to four) pages are there, slots
constexpr int kKbBits = 20;
constexpr int kKbMask = (1 << kKbBits) - 1;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  return ((uint64_t)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ float lo_f(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_f(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// 32-byte store: a whole sector per lane, where rows lie far apart.
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// One arrival for the warp: what its lanes did before is released by lane 0. (32 lanes that
// arrive one by one on the same barrier take some 500 cycles.)
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  tc::tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// Up to 32 consecutive entries of a kept list, one a lane (INT32_MAX behind its end): whether the
// lane's stands above every entry before it, `top` being the largest of those before lane 0's, and
// whether it is an index at all. `top` moves on to the largest of the first n. Entries that ascend,
// as they should, take one comparison; the running maximum is for those that do not.
struct ListCheck {
  bool index, order;
};
__device__ __forceinline__ ListCheck check_entries(int kb, int n, int lane, int& top) {
  int before = __shfl_up_sync(0xffffffffu, kb, 1);
  if (lane == 0) before = top;
  const bool in = lane < n;
  if (__any_sync(0xffffffffu, in && (kb < 0 || kb <= before))) {
    int upto = in ? kb : -1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto = max(upto, x);
    }
    before = __shfl_up_sync(0xffffffffu, upto, 1);
    before = lane == 0 ? top : max(before, top);
    top = max(top, __shfl_sync(0xffffffffu, upto, 31));
  } else if (n > 0) {
    top = __shfl_sync(0xffffffffu, kb, n - 1);
  }
  return {in && kb >= 0, in && kb > before};
}

// One list segment and the tile it belongs to.
struct Work {
  int n;            // entries; -1: no more work
  int first, last;  // of the item's segments
  int len;          // tokens of the sequence
  int part;         // slot of the item's partials, or -1: the item is the whole tile
  int hk;
  // rows, by slot (modes 0 and 1 use slot 0 alone)
  int valid[2];     // mode 0/1: tokens of the tile in [0]; mode 2: whether the slot is used
  int head[2];      // first query head
  int pos[2];       // position of row 0 of the slot
  int row[2];       // its row in q and out (mode 2: of position pos, maybe before the sequence)
  int ctx;
  int pieces;       // in the workspace's records: how many pieces the tile is in
};

// Workspace: one record per CTA (the tile that its length starts inside of, if it is the first to
// do so; pieces 0 otherwise), then (m, l) and O of two pieces per CTA.
struct ChunkWs {
  Work* cut;
  float2* ml;   // [2 CTAs, rows] (row maximum in base-2 units, row sum)
  float* o;     // [2 CTAs, rows, D] sums not yet divided by l
};

// Which blocks of a tile warp 3 looks over.
struct Look {
  int lowest, slots;  // first position of the tile's tokens; slots in use
  __device__ __forceinline__ Look(const Work& w, const ChunkShape& sh) {
    lowest = w.pos[0];
    slots = 1;
    if (sh.mode == 2) {
      lowest = min(w.valid[0] ? max(w.pos[0], w.ctx) : INT32_MAX, w.valid[1] ? max(w.pos[1], w.ctx) : INT32_MAX);
      slots = (w.valid[0] ? 1 : 0) | (w.valid[1] ? 2 : 0);
    }
  }
  // keys that some row of the tile must not see
  __device__ __forceinline__ bool mixed(int entry, int kbase, int len) const {
    return min(kbase + kChunkBlk, len) - 1 > lowest || ((entry >> (kKbBits + 4)) & slots) != slots;
  }
  // those, or rows of V without a key
  __device__ __forceinline__ bool wanted(int entry, int kbase, int have, int all_pages, int len) const {
    return have != all_pages || kbase + kChunkBlk > len || mixed(entry, kbase, len);
  }
};

template <int D>
struct Smem {
  static constexpr int kChunks = D / 64;                  // 64-element (128 B) swizzle atoms along D
  static constexpr int kQBytes = kChunks * 128 * 128;
  static constexpr int kKVTileBytes = kChunks * 64 * 128;
  static constexpr int kRing = D == 64 ? 4 : 2;            // stages of K and of V (64 KB together)
  static constexpr int kKOff = 0;
  static constexpr int kVOff = kRing * kKVTileBytes;
  static constexpr int kQOff = 0;
  static constexpr int kStageOff = kQOff + kQBytes;
  static constexpr int kListOff = kStageOff + 2 * kRing * kKVTileBytes;  // [2][kSeg] entries
  static constexpr int kPageOff = kListOff + 2 * kSeg * 4;       // [2][kSeg][4] pages
  static constexpr int kSumOff = kPageOff + 2 * kSeg * 16;        // [kChunkBuckets] int64, weight before
  static constexpr int kSeqOff = kSumOff + kChunkBuckets * 8;     // [kChunkBuckets] int4
  static constexpr int kBitmapOff = kSeqOff + kChunkBuckets * 16;  // [2][kSeg / 32]
  static constexpr int kCodeOff = kBitmapOff + 2 * (kSeg / 32) * 4;  // [D / 16][128 rows]
  static constexpr int kMarkOff = kCodeOff + (D / 16) * 128 * 4;  // tile << 3 | softmax warps that still have to read them
  static constexpr int kWorkOff = (kMarkOff + 8 + 7) / 8 * 8;
  static constexpr int kBarOff = (kWorkOff + 2 * (int)sizeof(Work) + 7) / 8 * 8;
  static constexpr int kNumBars = 14 + 5 * kRing;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kBytes = kMiscOff + 16;
  static constexpr int kAlloc = kBytes + 1024;  // slack for 1024-byte alignment
};

// Whether any of eight 16-bit values is not finite: exponents of all ones carry into the sign bits.
template <bool kF16>
__device__ __forceinline__ bool any_nonfinite(const uint4& u) {
  constexpr uint32_t mask = kF16 ? 0x7c007c00u : 0x7f807f80u, one = kF16 ? 0x04000400u : 0x00800080u;
  return ((((u.x & mask) + one) | ((u.y & mask) + one) | ((u.z & mask) + one) | ((u.w & mask) + one)) & 0x80008000u) != 0;
}
template <bool kF16>
__device__ __forceinline__ bool nonfinite16(uint32_t v) {
  constexpr uint32_t mask = kF16 ? 0x7c00u : 0x7f80u;
  return (v & mask) == mask;
}

// 2-bit code of what values that are not finite make of a sum: 1 = +inf, 2 = -inf, 3 = NaN.
__device__ __forceinline__ float nonfinite_of(uint32_t code, float v) {
  return code == 0 ? v : code == 1 ? INFINITY : code == 2 ? -INFINITY : NAN;
}

struct PagedGeo {
  int nsub;       // pages of a block (page_size < 64)
  int sub_rows;   // rows of a page's share of a block
};

template <int D, bool kF16>
__global__ void __launch_bounds__(kThreads, 2)
    bsa_chunk_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                        const __grid_constant__ CUtensorMap tmv, const tasft_chunk_args a, const ChunkShape sh,
                        const ChunkWs ws) {
  using L = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem + L::kQOff;
  int32_t* lists = reinterpret_cast<int32_t*>(smem + L::kListOff);
  int4* pages = reinterpret_cast<int4*>(smem + L::kPageOff);
  Work* works = reinterpret_cast<Work*>(smem + L::kWorkOff);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* q_full = bars + 0;       // per tile: Q landed
  uint64_t* q_empty = bars + 1;      // per tile: every S of the tile has run (Q reusable)
  uint64_t* o_final = bars + 2;      // per tile: O complete
  uint64_t* o_free = bars + 3;       // per tile: epilogue has read O (one arrival per warp)
  uint64_t* s_full = bars + 4;       // [2] per block
  uint64_t* p_ready = bars + 6;      // [2] per block (one arrival per softmax warp)
  uint64_t* pv_done = bars + 8;      // [2] per block: P.V(g) has run
  uint64_t* list_full = bars + 10;   // [2] per segment
  uint64_t* list_empty = bars + 12;  // [2] per segment (arrivals: four softmax warps, warps 0 and 3)
  uint64_t* k_full = bars + 14;              // [kRing] per block
  uint64_t* k_empty = k_full + L::kRing;     // [kRing] per block: S(g) has run
  uint64_t* v_full = k_empty + L::kRing;     // [kRing] per block (by the copy, or by warp 3 where it looks over it)
  uint64_t* v_empty = v_full + L::kRing;     // [kRing] per block: P.V(g) has run
  uint64_t* v_look = v_empty + L::kRing;     // [kRing] per block whose V warp 3 looks over: it has landed
  uint32_t* codes = reinterpret_cast<uint32_t*>(smem + L::kCodeOff);
  volatile int32_t* mark = reinterpret_cast<volatile int32_t*>(smem + L::kMarkOff);
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = a.Hq / a.Hk;

  if (warp == 0 && lane == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < L::kRing; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_look[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&list_full[i], 1);
      mbar_init(&list_empty[i], 6);
    }
    mbar_init(o_final, 1);
    mbar_init(o_free, 4);
    *mark = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(&misc[0], kTmemCols);
    tc::tmem_relinquish();
  }
  if (warp == 3) {
    // tables and lists, a share per CTA, on their way to L2 while warp 2 counts: it reads them in
    // a chain (a prefetch of what the kernel before is still writing does no harm, L2 holds it)
    auto fetch = [&](const void* p, int64_t bytes) {
      const int64_t lines = (bytes + 127) / 128, stride = (int64_t)gridDim.x * 32;
      for (int64_t i = (int64_t)blockIdx.x * 32 + lane, k = 0; i < lines && k < 4; i += stride, ++k)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p) + i * 128));
    };
    fetch(a.block_table, (int64_t)a.B * a.max_pages * 4);
    if (a.kept_idx) {
      fetch(a.kept_cnt, (int64_t)a.B * a.Hm * a.nb_q * 4);
      fetch(a.kept_idx, (int64_t)a.B * a.Hm * a.nb_q * a.nb_w * 4);
    }
    if (sh.zero_rest) {  // beside warp 2's count, a share of the rows per CTA
      asm volatile("griddepcontrol.wait;" ::: "memory");
      auto zero = [&](int from, int to) {
        constexpr int kPieces = D / 8;  // of 16 bytes, of a head's row
        for (int64_t r = (int64_t)from + blockIdx.x; r < to; r += gridDim.x)
          for (int i = lane; i < a.Hq * kPieces; i += 32)
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + r * a.o_stride[0] +
                                      (i / kPieces) * a.o_stride[1] + (i % kPieces) * 8) = make_uint4(0, 0, 0, 0);
      };
      auto within = [&](int r) { return max(0, min(r, a.T)); };
      // before the first sequence, behind the last one, and those that do not fit
      zero(0, within(a.cu_seqlens[0]));
      zero(within(a.cu_seqlens[a.B]), a.T);
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + lane;
        unsigned left_out = __ballot_sync(
            0xffffffffu, b < a.B && !chunk_fits(a, sh, a.cu_seqlens[b], a.cu_seqlens[b + 1], a.kv_len[b]));
        for (; left_out; left_out &= left_out - 1) {
          const int bad = b0 + __ffs(left_out) - 1;
          zero(within(a.cu_seqlens[bad]), within(a.cu_seqlens[bad + 1]));
        }
      }
      __syncwarp();
    }
  }
  int64_t* before = reinterpret_cast<int64_t*>(smem + L::kSumOff);  // weight before a bucket's first sequence
  int4* seqs = reinterpret_cast<int4*>(smem + L::kSeqOff);          // start, n, len, cost (stride 1)
  int64_t total = 0, step = 1;
  bool cutting = false;
  if (warp == 2) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- the weight of all tiles, and each CTA's length of it ----
    int64_t widest = 0, count = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + lane;
      int64_t w = 0;
      if (b < a.B) {
        const ChunkSeq s = chunk_seq(a, sh, b);
        if (s.bad && blockIdx.x == 0) set_err(a.err, TASFT_DEVERR_INDEX);
        w = chunk_weight_before(sh, s, s.tiles) * sh.units;
        if (s.tiles > 0) widest = max(widest, chunk_weight(sh, s, s.tiles - 1));
        count += s.tiles;
        if (sh.stride == 1) seqs[b] = make_int4(s.start, s.n, s.len, s.cost);
      }
      const int64_t upto = warp_scan64(w, lane);
      if (b < a.B && (sh.stride == 1 || b % sh.stride == 0)) before[sh.stride == 1 ? b : b / sh.stride] = total + upto - w;
      total += __shfl_sync(0xffffffffu, upto, 31);
    }
    widest = warp_max64(widest);
    count = warp_sum64(count) * sh.units;
    const int64_t G = gridDim.x;
    step = total + G < (1ll << 32) ? (uint32_t)(total + G - 1) / (uint32_t)G : (total + G - 1) / G;
    step = max(step, (int64_t)kChunkMinPiece * kChunkBlk);
    // whole tiles would take rounds * widest; cut ones take `step`
    const int64_t rounds = (uint32_t)(count + G - 1) / (uint32_t)G;
    cutting = sh.may_cut && rounds * widest - step > (int64_t)kChunkMergeCost * kChunkBlk;
    if (!cutting) {  // whole tiles: each CTA takes as many, one more here and there (weight 64 each)
      total = 0;
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + lane;
        int64_t w = 0;
        if (b < a.B) {
          int tiles;
          if (sh.stride == 1) {
            const int4 q4 = seqs[b];
            tiles = chunk_tiles(sh, q4.y, q4.z - q4.y, q4.z);
          } else {
            tiles = chunk_seq(a, sh, b).tiles;
          }
          w = (int64_t)tiles * sh.units * kChunkBlk;
        }
        const int64_t upto = warp_scan64(w, lane);
        if (b < a.B && (sh.stride == 1 || b % sh.stride == 0)) before[sh.stride == 1 ? b : b / sh.stride] = total + upto - w;
        total += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  // nothing above touched memory that the kernel before this one may still use (warp 2 waited)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the merge kernel behind this one waits for this grid before it reads anything
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = misc[0];
  const uint32_t tS0 = tmem;       // S buffers: columns [0,64) and [64,128)
  const uint32_t tO = tmem + 128;  // O: columns [128, 128 + D)

  if (warp == 2) {
    // ================= lists =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    uint32_t* bitmap = reinterpret_cast<uint32_t*>(smem + L::kBitmapOff);
    const int buckets = (a.B + sh.stride - 1) / sh.stride;
    const int page_log2 = 31 - __clz(a.page_size);
    const PagedGeo geo = {max(1, kChunkBlk >> page_log2), min(kChunkBlk, a.page_size)};
    auto get_seq = [&](int b) -> ChunkSeq {
      if (sh.stride != 1) return chunk_seq(a, sh, b);
      const int4 q4 = seqs[b];
      ChunkSeq s;
      s.start = q4.x;
      s.n = q4.y;
      s.len = q4.z;
      s.cost = q4.w;
      s.ctx = s.n > 0 ? s.len - s.n : 0;
      s.tiles = chunk_tiles(sh, s.n, s.ctx, s.len);
      s.bad = false;
      return s;
    };
    auto weight = [&](const ChunkSeq& s, int i) -> int64_t { return cutting ? chunk_weight(sh, s, i) : kChunkBlk; };
    auto weight_before = [&](const ChunkSeq& s, int i) -> int64_t {
      return cutting ? chunk_weight_before(sh, s, i) : (int64_t)i * kChunkBlk;
    };
    // The place at weight x, in Int arithmetic. Cuts within two blocks of a tile's end go there.
    auto find = [&](auto zero, int64_t x64) -> ChunkCut {
      using Int = decltype(zero);
      ChunkCut c;
      c.b = a.B;
      c.unit = c.tile = 0;
      c.rho = 0;
      c.w = 1;
      if (x64 >= total) return c;
      int bl = 0, bh = buckets - 1;
      while (bl < bh) {  // the last bucket that starts at or before x
        const int mid = (bl + bh + 1) >> 1;
        if (before[mid] <= x64) bl = mid;
        else bh = mid - 1;
      }
      Int x = (Int)(x64 - before[bl]);
      c.b = bl * sh.stride;
      c.s = get_seq(c.b);
      Int per = (Int)weight_before(c.s, c.s.tiles);
      while (x >= per * (Int)sh.units) {  // sequences without new tokens have no weight
        x -= per * (Int)sh.units;
        c.s = get_seq(++c.b);
        per = (Int)weight_before(c.s, c.s.tiles);
      }
      c.unit = (int)(x / per);
      x -= (Int)c.unit * per;
      if (sh.mode != 0 || !cutting) {
        c.tile = (int)(x / (Int)weight(c.s, 0));
      } else {  // the weights before tiles grow as t i^2 / 2 + (ctx + 63 + t / 2) i
        const float t = (float)sh.tpt, h = (float)(c.s.ctx + 63) + 0.5f * t;
        int i = (int)((sqrtf(h * h + 2.f * t * (float)x) - h) / t);
        i = max(0, min(i, c.s.tiles - 1));
        while (i > 0 && (Int)weight_before(c.s, i) > x) --i;
        while (i + 1 < c.s.tiles && (Int)weight_before(c.s, i + 1) <= x) ++i;
        c.tile = i;
      }
      c.rho = (int64_t)(x - (Int)weight_before(c.s, c.tile));
      c.w = weight(c.s, c.tile);
      constexpr int kEdge = 2 * kChunkBlk;
      if (c.rho < kEdge) {  // (always, where tiles stay whole)
        c.rho = 0;
      } else if (c.w - c.rho < kEdge) {  // the start of the next tile
        c.rho = 0;
        if (++c.tile == c.s.tiles) {
          c.tile = 0;
          if (++c.unit == sh.units) {
            c.unit = 0;
            do {
              if (++c.b == a.B) break;
              c.s = get_seq(c.b);
            } while (c.s.tiles == 0);
          }
        }
      }
      return c;
    };
    // both ends at once, in the even and the odd lanes
    const int64_t nth = blockIdx.x + (lane & 1);
    const int64_t end_x = cutting ? nth * step : nth * (total / kChunkBlk) / (int64_t)gridDim.x * kChunkBlk;
    const ChunkCut end = total < (1ll << 31) ? find(0u, end_x) : find((int64_t)0, end_x);
    auto take = [&](int from_lane) -> ChunkCut {
      ChunkCut c;
      c.b = __shfl_sync(0xffffffffu, end.b, from_lane);
      c.unit = __shfl_sync(0xffffffffu, end.unit, from_lane);
      c.tile = __shfl_sync(0xffffffffu, end.tile, from_lane);
      c.rho = __shfl_sync(0xffffffffu, end.rho, from_lane);
      c.w = __shfl_sync(0xffffffffu, end.w, from_lane);
      return c;
    };
    const ChunkCut from = take(0);
    ChunkCut cur = take(1);
    if (cur.b < a.B) cur.s = get_seq(cur.b);
    bool more = !(from.b == cur.b && from.unit == cur.unit && from.tile == cur.tile && from.rho == cur.rho);
    bool partial_end = cur.rho > 0;  // the piece at hand stops inside its tile
    // whether the CTA before this one starts inside the same tile: then that one records it
    bool recorded = from.rho == 0;
    if (from.rho > 0) {
      const int64_t edge = 2 * kChunkBlk, back = from.rho - step;
      recorded = back >= edge && blockIdx.x > 0;
    }
    // (a CTA that gives up leaves no record: the merge then does nothing for it)
    if (lane == 0) ws.cut[blockIdx.x].pieces = 0;
    __syncwarp();

    int u = 0;  // segment counter
    bool ok = true;
    while (ok) {
      Work w;
      int lo = 0, hi = 0;                 // range of the piece: list positions, or blocks
      const int32_t* idx[2] = {nullptr, nullptr};
      int cnt[2] = {0, 0}, qb[2] = {0, 0};
      int b = 0;
      const bool done = !more;
      if (!done) {
        if (!partial_end) {  // step back to the tile before
          if (--cur.tile < 0) {
            if (--cur.unit < 0) {
              do {
                cur.s = get_seq(--cur.b);
              } while (cur.s.tiles == 0);
              cur.unit = sh.units - 1;
            }
            cur.tile = cur.s.tiles - 1;
          }
        }
        const ChunkSeq& s = cur.s;
        b = cur.b;
        const int unit = cur.unit, tile = cur.tile;
        const bool at_start = b == from.b && unit == from.unit && tile == from.tile;
        const bool partial_start = at_start && from.rho > 0;
        w.len = s.len;
        w.ctx = s.ctx;
        w.part = partial_start ? 2 * (int)blockIdx.x : partial_end ? 2 * (int)blockIdx.x + 1 : -1;
        w.pieces = 0;
        int diag;  // last block the tile may visit
        if (sh.mode == 2) {
          const int base = ((s.ctx >> sh.tpt_log2) + tile) << sh.tpt_log2;
          if (grp >= 2) {
            const int pairs = (grp + 1) / 2, p = unit % pairs;
            w.hk = unit / pairs;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              w.head[x] = w.hk * grp + 2 * p + x;
              w.valid[x] = 2 * p + x < grp;
              w.pos[x] = base;
            }
          } else {
            w.hk = unit;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              w.head[x] = unit;
              w.pos[x] = base + x * kChunkBlk;
              w.valid[x] = w.pos[x] < s.len && w.pos[x] + kChunkBlk > s.ctx;
            }
          }
          diag = 0;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            w.row[x] = s.start + w.pos[x] - s.ctx;
            qb[x] = w.pos[x] / kChunkBlk;
            if (!w.valid[x]) continue;
            diag = max(diag, qb[x]);
            const int64_t lrow =
                ((int64_t)b * a.Hm + w.head[x] / (a.Hq / a.Hm)) * a.nb_q + (qb[x] - s.ctx / kChunkBlk);
            cnt[x] = min(max(a.kept_cnt[lrow], 0), a.nb_w);
            idx[x] = a.kept_idx + lrow * a.nb_w;
          }
          // (its pieces are ranges of block indices)
          hi = diag + 1;
        } else {
          w.hk = unit;
          w.head[0] = w.head[1] = unit * grp;
          int p0, p1;
          if (sh.mode == 0) {
            p0 = s.ctx + tile * sh.tpt;
            p1 = min(p0 + sh.tpt, s.len);
          } else {
            p0 = ((s.ctx >> sh.tpt_log2) + tile) << sh.tpt_log2;
            p1 = min(p0 + sh.tpt, s.len);
            p0 = max(p0, s.ctx);
          }
          w.valid[0] = p1 - p0;
          w.valid[1] = 0;
          w.pos[0] = w.pos[1] = p0;
          w.row[0] = w.row[1] = s.start + p0 - s.ctx;
          diag = (p1 - 1) / kChunkBlk;
          qb[0] = diag;
          cnt[0] = diag + 1;
          if (sh.mode == 1) {
            const int64_t lrow = ((int64_t)b * a.Hm + unit) * a.nb_q + (diag - s.ctx / kChunkBlk);
            cnt[0] = min(max(a.kept_cnt[lrow], 0), a.nb_w);
            idx[0] = a.kept_idx + lrow * a.nb_w;
          }
          hi = cnt[0];
        }
        // the cuts' places in the tile: both CTAs beside a cut compute the same one
        const int all = hi;
        auto part_of = [&](int64_t rho, int64_t wt) -> int {
          const uint64_t x = (uint64_t)(rho * all);
          return (x >> 32) == 0 ? (int)((uint32_t)x / (uint32_t)wt) : (int)(x / (uint64_t)wt);
        };
        if (partial_end) hi = part_of(cur.rho, cur.w);
        if (partial_start) lo = part_of(from.rho, from.w);
        if (partial_start && !recorded) {
          // pieces: the CTA before, this one, and those that start further on in the tile
          if (lane == 0) {
            w.pieces = 2 + (int)((from.w - 2 * kChunkBlk - from.rho) / step);
            ws.cut[blockIdx.x] = w;
            w.pieces = 0;
          }
        }
        partial_end = false;
        more = !at_start;
      }
      // ---- the piece's segments ----
      int at = lo;                       // next list position or block
      int pt[2] = {0, 0};                // mode 2: next position of each list
      int top[2] = {-1, -1};             // largest entry so far of each list
      if (!done && sh.mode == 1 && lo > 0) {  // of the pieces before this one
        for (int i = lane; i < lo; i += 32) top[0] = max(top[0], idx[0][i]);
        top[0] = __reduce_max_sync(0xffffffffu, top[0]);
      }
      bool first = true;
      while (ok) {
        const int lb = u & 1;
        if (u >= 2 && !warp_wait(&list_empty[lb], ((u >> 1) - 1) & 1)) {
          set_err(a.err, TASFT_DEVERR_TIMEOUT | (1 << 9));
          ok = false;
          break;
        }
        int32_t* list = lists + lb * kSeg;
        int4* pgs = pages + lb * kSeg;
        if (done) {
          if (lane == 0) {
            works[lb].n = -1;
            mbar_arrive(&list_full[lb]);
          }
          break;
        }
        int n = 0;
        // ---- block indices (with slots in mode 2) ----
        if (sh.mode == 2) {
          const int wend = min(at + kSeg, hi);
          if (lane < 2 * (kSeg / 32)) bitmap[lane] = 0;
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            while (pt[x] < cnt[x]) {
              const int i = pt[x] + lane;
              const int kb = i < cnt[x] ? idx[x][i] : INT32_MAX;
              const bool mine = kb < wend;  // this window's (a list ascends, so a prefix)
              const unsigned out = __ballot_sync(0xffffffffu, !mine);
              const int take = out ? __ffs(out) - 1 : 32;
              const ListCheck good = check_entries(kb, take, lane, top[x]);
              if (lane < take) {
                if (!good.index) set_err(a.err, TASFT_DEVERR_INDEX);
                else if (!good.order) set_err(a.err, TASFT_DEVERR_ORDER);
                else if (kb >= at && kb <= qb[x])
                  atomicOr(&bitmap[x * (kSeg / 32) + ((kb - at) >> 5)], 1u << ((kb - at) & 31));
              }
              pt[x] += take;
              if (take < 32) break;
            }
          }
          __syncwarp();
          for (int wd = 0; wd < kSeg / 32; ++wd) {
            const uint32_t m0 = bitmap[wd], m1 = bitmap[kSeg / 32 + wd], bit = 1u << lane;
            const bool any = ((m0 | m1) & bit) != 0;
            const unsigned bal = __ballot_sync(0xffffffffu, any);
            if (any)
              list[n + __popc(bal & (bit - 1u))] =
                  (at + wd * 32 + lane) | (((m0 & bit) ? 1 : 0) << (kKbBits + 4)) | (((m1 & bit) ? 1 : 0) << (kKbBits + 5));
            n += __popc(bal);
          }
          at = wend;
        } else {
          const int end = min(at + kSeg, hi);
          for (int i0 = at; i0 < end; i0 += 32) {
            const int i = i0 + lane;
            int kb = i;
            bool good = i < end;
            if (sh.mode == 1) {
              kb = good ? idx[0][i] : INT32_MAX;
              const ListCheck c = check_entries(kb, min(32, end - i0), lane, top[0]);
              if (good && !c.index) set_err(a.err, TASFT_DEVERR_INDEX);
              else if (good && !c.order) set_err(a.err, TASFT_DEVERR_ORDER);
              good = c.index && c.order && kb <= qb[0];
            }
            const unsigned bal = __ballot_sync(0xffffffffu, good);
            if (good) list[n + __popc(bal & ((1u << lane) - 1u))] = kb | (1 << (kKbBits + 4));
            n += __popc(bal);
          }
          at = end;
        }
        __syncwarp();
        // ---- their pages ----
        for (int i = lane; i < n; i += 32) {
          const int e = list[i], kb = e & kKbMask;
          // kv_len is within the table's capacity, so the pages of its tokens have entries
          const int32_t* row = a.block_table + (int64_t)b * a.max_pages + (kb * kChunkBlk >> page_log2);
          int pg[4] = {0, 0, 0, 0}, have = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (x < geo.nsub && kb * kChunkBlk + x * geo.sub_rows < w.len) pg[x] = row[x];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (x >= geo.nsub || kb * kChunkBlk + x * geo.sub_rows >= w.len) continue;
            if (pg[x] >= 0 && pg[x] < a.num_pages) have |= 1 << x;
            else set_err(a.err, TASFT_DEVERR_INDEX);
          }
          list[i] = e | (have << kKbBits);
          pgs[i] = make_int4(pg[0], pg[1], pg[2], pg[3]);
        }
        __syncwarp();
        const bool last = at >= hi;
        // nothing kept here: on to the next (the MMA issuer could fall two empty segments behind)
        if (n == 0 && !last) continue;
        if (lane == 0) {
          w.n = n;
          w.first = first;
          w.last = last;
          works[lb] = w;
          mbar_arrive(&list_full[lb]);  // release: the entries, their pages and the record
        }
        first = false;
        ++u;
        if (last) break;
      }
      if (done) break;
    }
  } else if (warp == 0) {
    // ================= producer =================
    // The lanes share the copies of a tile, one each: eight for pages of 16 tokens at D 128.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (lane == 0) {
      tc::prefetch_tmap(&tmq);
      tc::prefetch_tmap(&tmk);
      tc::prefetch_tmap(&tmv);
    }
    const int nsub = max(1, kChunkBlk / a.page_size), sub_rows = min(kChunkBlk, a.page_size);
    const uint32_t q_bytes = sh.mode == 2 ? 0 : (uint32_t)(L::kChunks * sh.hpt * sh.tpt * 128);
    const int all_pages = (1 << nsub) - 1;
    const int my_c = lane % L::kChunks, my_x = lane / L::kChunks;  // the lane's column chunk and page (or slot of Q)
    int gk = 0, gv = 0, tile = 0, looks = 0;  // K and V tiles asked for, tiles, V tiles for warp 3
    bool ok = true;
    for (int u = 0; ok; ++u) {
      const int lb = u & 1;
      if (!warp_wait(&list_full[lb], (u >> 1) & 1)) { ok = false; break; }
      const Work& w = works[lb];
      const int n = w.n;
      if (n < 0) break;
      if (w.first) {
        if (tile >= 1 && !warp_wait(q_empty, (tile - 1) & 1)) { ok = false; break; }
        if (lane == 0)
          mbar_arrive_expect_tx(q_full, sh.mode == 2 ? ((w.valid[0] ? 1 : 0) + (w.valid[1] ? 1 : 0)) * L::kChunks * 64 * 128
                                                     : q_bytes);
        __syncwarp();
        if (sh.mode == 2) {
          if (my_x < 2 && w.valid[my_x])
            tc::tma_load_4d(sQ + my_c * 128 * 128 + my_x * 64 * 128, &tmq, my_c * 64, w.head[my_x], w.row[my_x], 0, q_full);
        } else if (my_x == 0) {
          tc::tma_load_4d(sQ + my_c * 128 * 128, &tmq, my_c * 64, w.head[0], w.row[0], 0, q_full);
        }
        ++tile;
      }
      const int32_t* list = lists + lb * kSeg;
      const int32_t* pgs = reinterpret_cast<const int32_t*>(pages + lb * kSeg);
      const Look look(w, sh);
      const int hk = w.hk, len = w.len;
      // one entry's K or V: the share of each page it has, into the stage's rows
      auto load = [&](int gi, int j, const CUtensorMap* map, uint64_t* full, uint64_t* empty, int off) -> bool {
        const int st = gi % L::kRing;
        const int e = list[j], have = (e >> kKbBits) & 15, kbase = (e & kKbMask) * kChunkBlk;
        const int page = pgs[4 * j + (my_x & 3)];
        const int in_page = a.page_size > kChunkBlk ? ((e & kKbMask) & 1) * kChunkBlk : 0;
        uint8_t* dst = smem + L::kStageOff + off + st * L::kKVTileBytes;
        uint64_t* bar = &full[st];
        if (full == v_full && look.wanted(e, kbase, have, all_pages, len)) bar = &v_look[looks++ % L::kRing];
        if (gi >= L::kRing && !warp_wait(&empty[st], (gi / L::kRing - 1) & 1)) return false;
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(__popc(have) * L::kChunks * sub_rows * 128));
        __syncwarp();
        if (my_x < nsub && ((have >> my_x) & 1))
          tc::tma_load_4d(dst + my_c * 64 * 128 + my_x * sub_rows * 128, map, my_c * 64, hk, in_page, page, bar);
        return true;
      };
      // K(j) then V(j-1): the order the MMA warp consumes them
      for (int j = 0; ok && j <= n && n > 0; ++j) {
        if (j < n) {
          ok = load(gk, j, &tmk, k_full, k_empty, L::kKOff);
          if (ok) ++gk;
        }
        if (ok && j >= 1) {
          ok = load(gv, j - 1, &tmv, v_full, v_empty, L::kVOff);
          if (ok) ++gv;
        }
      }
      // the softmax warps may be through with the segment while its last V is not on its way yet
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(&list_empty[lb]);
    }
    if (!ok) set_err(a.err, TASFT_DEVERR_TIMEOUT | (1 << 10));
    // do not leave while copies into shared memory are in flight, after a timeout either (a look that
    // was counted but not asked for then only runs out its wait)
    if (tile > 0) warp_wait(q_full, (tile - 1) & 1);
    for (int i = max(0, gk - L::kRing); i < gk; ++i) warp_wait(&k_full[i % L::kRing], (i / L::kRing) & 1);
    for (int i = max(0, looks - L::kRing); i < looks; ++i) warp_wait(&v_look[i % L::kRing], (i / L::kRing) & 1);
    for (int i = max(0, gv - L::kRing); i < gv; ++i) warp_wait(&v_full[i % L::kRing], (i / L::kRing) & 1);
  } else if (warp == 1) {
    // ================= MMA issuer =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (lane == 0) {
      constexpr uint32_t fmt = kF16 ? 0u : 1u;
      constexpr uint32_t idesc_s = tc::make_idesc(128, 64, fmt, false);
      constexpr uint32_t idesc_o = tc::make_idesc(128, D, fmt, true);
      // descriptors once; the address field counts 16-byte units and does not overflow
      const uint64_t q_desc = tc::make_sdesc(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = tc::make_sdesc(smem_u32(smem + L::kStageOff + L::kKOff), 16, 1024);
      const uint64_t v_desc = tc::make_sdesc(smem_u32(smem + L::kStageOff + L::kVOff), 64 * 128, 1024);
      int g = 0, tile = -1;
      bool ok = true, started = false;
      auto issue_s = [&](int gi) -> bool {
        const int st = gi & 1, kst = gi % L::kRing;
        if (!mbar_wait(&k_full[kst], (gi / L::kRing) & 1)) return false;
        // S(gi) overwrites P(gi - 2) in TMEM: P.V(gi - 2) was issued earlier by this thread, and
        // the MMAs of one thread run through the tensor pipe in issue order
        tc::tc_fence_after();
        const uint64_t kd = k_desc + (uint32_t)(kst * (L::kKVTileBytes >> 4));
        const uint32_t dst = tS0 + st * 64;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_ss(dst, q_desc + (uint32_t)(((kk >> 2) * 128 * 128 + (kk & 3) * 32) >> 4),
                     kd + (uint32_t)(((kk >> 2) * 64 * 128 + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
        tc::mma_commit(&s_full[st]);
        tc::mma_commit(&k_empty[kst]);
        return true;
      };
      for (int u = 0; ok; ++u) {
        const int lb = u & 1;
        if (!mbar_wait(&list_full[lb], (u >> 1) & 1)) { ok = false; break; }
        const int n = works[lb].n, first = works[lb].first, last = works[lb].last;
        if (n < 0) break;
        if (first) {
          ++tile;
          started = false;
          if (!mbar_wait(q_full, tile & 1)) { ok = false; break; }
          tc::tc_fence_after();
        }
        if (n > 0) ok = issue_s(g);
        if (ok && last && n <= 1) tc::mma_commit(q_empty);  // no further S of this tile reads Q
        for (int j = 0; ok && j < n; ++j) {
          const int gi = g + j;
          if (j + 1 < n) {
            ok = issue_s(gi + 1);
            if (!ok) break;
            if (last && j + 2 == n) tc::mma_commit(q_empty);
          }
          if (!mbar_wait(&p_ready[gi & 1], (gi >> 1) & 1)) { ok = false; break; }
          // O is reused: the previous tile's epilogue must have read it
          if (!started && tile >= 1 && !mbar_wait(o_free, (tile - 1) & 1)) { ok = false; break; }
          const int vst = gi % L::kRing;
          if (!mbar_wait(&v_full[vst], (gi / L::kRing) & 1)) { ok = false; break; }
          tc::tc_fence_after();
          const uint64_t vd = v_desc + (uint32_t)(vst * (L::kKVTileBytes >> 4));
          const uint32_t p_tmem = tS0 + (gi & 1) * 64;
#pragma unroll
          for (int kk = 0; kk < kChunkBlk / 16; ++kk)
            tc::mma_ts(tO, p_tmem + kk * 8, vd + (uint32_t)(kk * 16 * 128 >> 4), idesc_o, (started || kk > 0) ? 1u : 0u);
          started = true;
          tc::mma_commit(&v_empty[vst]);
          tc::mma_commit(&pv_done[gi & 1]);
        }
        if (!ok) break;
        if (last) {
          if (!started && tile >= 1 && !mbar_wait(o_free, (tile - 1) & 1)) { ok = false; break; }
          tc::mma_commit(o_final);
        }
        g += n;
      }
      if (!ok) set_err(a.err, TASFT_DEVERR_TIMEOUT | (1 << 11));
    }
  } else if (warp >= 4) {
    // ================= softmax + epilogue (warps 4..7) =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int quarter = warp & 3;       // TMEM lanes [32*quarter, 32*quarter + 32)
    const int r = quarter * 32 + lane;  // tile row
    const int slot = sh.mode == 2 ? r >> 6 : 0;
    const int tok = sh.mode == 2 ? r & 63 : r / sh.hpt;   // token of the row within its slot
    const int hd = sh.mode == 2 ? 0 : r % sh.hpt;
    const int sub_rows = min(kChunkBlk, a.page_size);
    const int all_pages = (1 << max(1, kChunkBlk / a.page_size)) - 1;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const float sl2 = a.scale * kLog2e;
    using T = typename std::conditional<kF16, __half, __nv_bfloat16>::type;
    int g = 0, tile = -1;
    bool ok = true, started = false;
    float m = -INFINITY, l = 0.f;
    for (int u = 0; ok; ++u) {
      const int lb = u & 1;
      if (!warp_wait(&list_full[lb], (u >> 1) & 1)) { ok = false; break; }
      const Work* w = &works[lb];
      const int n = w->n, last = w->last, len = w->len;
      if (n < 0) break;
      const int32_t* list = lists + lb * kSeg;
      const int qpos = w->pos[slot] + tok;
      const bool live = sh.mode == 2 ? w->valid[slot] && qpos >= w->ctx && qpos < len : tok < w->valid[0];
      // a warp whose rows hold no token only keeps the barriers going: what P and O hold in its
      // rows meets nothing else
      const bool any_live = __any_sync(0xffffffffu, live);
      if (w->first) {
        ++tile;
        started = false;
        m = -INFINITY;
        l = 0.f;
      }
      for (int j = 0; j < n; ++j) {
        const int gi = g + j;
        if (!warp_wait(&s_full[gi & 1], (gi >> 1) & 1)) { ok = false; break; }
        tc::tc_fence_after();
        const int entry = list[j];
        const int kbase = (entry & kKbMask) * kChunkBlk;
        const int have = (entry >> kKbBits) & 15;
        // keys this row may see: up to its own position
        int lim = qpos - kbase + 1;
        if (!live || !((entry >> (kKbBits + 4 + slot)) & 1)) lim = 0;
        lim = max(0, min(lim, kChunkBlk));
        if (!__any_sync(0xffffffffu, lim > 0)) {
          if (any_live) {  // no row of the warp sees a key of this block: p = 0
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) pk[c] = 0u;
            tc::tmem_st32(tS0 + (gi & 1) * 64 + lane_off, pk);
            tc::tmem_wait_st();
          }
        } else {
          uint32_t sraw[64];
          tc::tmem_ld64_sync(tS0 + (gi & 1) * 64 + lane_off, sraw);
          float sv[64];
#pragma unroll
          for (int c = 0; c < 64; ++c) sv[c] = __uint_as_float(sraw[c]);
          if (__any_sync(0xffffffffu, lim < kChunkBlk) || have != all_pages) {
            uint64_t seen = lim == kChunkBlk ? ~0ull : (1ull << lim) - 1;
            if (have != all_pages) {  // keys of a page that is not there
              uint64_t keys = 0;
              for (int x = 0; x * sub_rows < kChunkBlk; ++x)
                if ((have >> x) & 1) keys |= (sub_rows == 64 ? ~0ull : (1ull << sub_rows) - 1) << (x * sub_rows & 63);
              seen &= keys;
            }
            const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (!((s0 >> c) & 1)) sv[c] = -INFINITY;
              if (!((s1 >> c) & 1)) sv[32 + c] = -INFINITY;
            }
          }
          float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 64; c += 8) {
#pragma unroll
            for (int qd = 0; qd < 4; ++qd) mq[qd] = max3(mq[qd], sv[c + 2 * qd], sv[c + 2 * qd + 1]);
          }
          const float mb = max3(mq[0], mq[1], fmaxf(mq[2], mq[3]));
          const float m_new = fmaxf(m, mb * sl2);
          const bool need = (m != -INFINITY) && (m_new > m + kRescaleThreshold);
          if (m == -INFINITY) m = m_new;  // O row is still exactly zero: no rescale
          if (__any_sync(0xffffffffu, need)) {
            // O must hold every earlier P.V of this tile before it is rescaled
            if (!warp_wait(&pv_done[(gi - 1) & 1], ((gi - 1) >> 1) & 1)) { ok = false; break; }
            tc::tc_fence_after();
            const float alpha = need ? ex2(m - m_new) : 1.0f;
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t o[32];
              tc::tmem_ld32_sync(tO + c0 + lane_off, o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
              tc::tmem_st32(tO + c0 + lane_off, o);
            }
            tc::tmem_wait_st();
            if (need) {
              l *= alpha;
              m = m_new;
            }
          }
          uint32_t pk[32];
          float rs = 0.f;
          if (m == -INFINITY) {  // nothing to see yet, or only scores that are NaN
#pragma unroll
            for (int c = 0; c < 32; ++c) pk[c] = 0u;
            if (lim > 0) {
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (sv[c] != sv[c]) rs = sv[c];
            }
          } else {
            const float nm = kF16 ? kHalfShift - m : -m;
            const uint64_t sc2 = f2(sl2, sl2), nm2 = f2(nm, nm);
            uint64_t rs2 = 0;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const uint64_t x2 = fma2(f2(sv[2 * c], sv[2 * c + 1]), sc2, nm2);  // s * scale - m
              const uint64_t p2 = f2(ex2(lo_f(x2)), ex2(hi_f(x2)));
              rs2 = add2(rs2, p2);
              pk[c] = kF16 ? tc::pack_f16x2(lo_f(p2), hi_f(p2)) : tc::pack_bf16x2(lo_f(p2), hi_f(p2));
            }
            rs = lo_f(rs2) + hi_f(rs2);
          }
          l += rs;
          tc::tmem_st32(tS0 + (gi & 1) * 64 + lane_off, pk);
          tc::tmem_wait_st();
        }
        warp_arrive(&p_ready[gi & 1], lane);
        started = true;
      }
      if (!ok) break;
      g += n;
      if (last) {
        if (!warp_wait(o_final, tile & 1)) { ok = false; break; }
        tc::tc_fence_after();
        const int tag = *mark;  // warp 3 may be at the next tile already
        const bool marked = (tag >> 3) == tile && (tag & 7) != 0;
        const uint32_t* code = codes + r;
        if (!any_live) {
        } else if (w->part < 0) {
          T* orow = reinterpret_cast<T*>(a.out) + (int64_t)(w->row[slot] + tok) * a.o_stride[0] +
                    (int64_t)(w->head[slot] + hd) * a.o_stride[1];
          const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that kept nothing gives 0
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            if (started) {
              tc::tmem_ld32_sync(tO + c0 + lane_off, o);
            } else {
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = 0u;
            }
            if (live) {
              uint32_t pk[16];
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                float v0 = __uint_as_float(o[2 * c]) * inv, v1 = __uint_as_float(o[2 * c + 1]) * inv;
                if (marked) {
                  const uint32_t cd = code[((c0 + 2 * c) >> 4) * 128] >> (((c0 + 2 * c) & 15) * 2);
                  v0 = nonfinite_of(cd & 3, v0);
                  v1 = nonfinite_of((cd >> 2) & 3, v1);
                }
                pk[c] = kF16 ? tc::pack_f16x2(v0, v1) : tc::pack_bf16x2(v0, v1);
              }
              if (sh.wide) {
                store32(orow + c0, pk);
                store32(orow + c0 + 16, pk + 8);
              } else {
                uint4* dst = reinterpret_cast<uint4*>(orow + c0);
#pragma unroll
                for (int v = 0; v < 4; ++v) dst[v] = make_uint4(pk[4 * v], pk[4 * v + 1], pk[4 * v + 2], pk[4 * v + 3]);
              }
            }
          }
        } else {
          const int64_t prow = (int64_t)w->part * sh.rows + r;
          if (live) ws.ml[prow] = make_float2(m, l);
          if (started) {
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t o[32];
              tc::tmem_ld32_sync(tO + c0 + lane_off, o);
              if (marked) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  o[c] = __float_as_uint(nonfinite_of((code[((c0 + c) >> 4) * 128] >> (((c0 + c) & 15) * 2)) & 3, __uint_as_float(o[c])));
              }
              if (live) {
#pragma unroll
                for (int v = 0; v < 4; ++v) store32(ws.o + prow * D + c0 + 8 * v, o + 8 * v);
              }
            }
          }
        }
        if (marked) {
          __syncwarp();
          if (lane == 0) atomicSub(const_cast<int32_t*>(mark), 1);
        }
        warp_arrive(o_free, lane);
      }
      warp_arrive(&list_empty[lb], lane);
    }
    if (!ok) set_err(a.err, TASFT_DEVERR_TIMEOUT | (1 << 12));
  } else {
    // ================= looking over V (warp 3) =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int sub_rows = min(kChunkBlk, a.page_size);
    const int all_pages = (1 << max(1, kChunkBlk / a.page_size)) - 1;
    int g = 0, tile = -1, looks = 0, open = -1;  // open: the tile whose codes are being collected
    bool ok = true;
    for (int u = 0; ok; ++u) {
      const int lb = u & 1;
      if (!warp_wait(&list_full[lb], (u >> 1) & 1)) { ok = false; break; }
      const Work* w = &works[lb];
      const int n = w->n, len = w->len;
      if (n < 0) break;
      if (w->first) ++tile;
      const Look look(*w, sh);
      for (int j = 0; j < n; ++j) {
        const int gi = g + j, entry = lists[lb * kSeg + j];
        const int kbase = (entry & kKbMask) * kChunkBlk, have = (entry >> kKbBits) & 15;
        if (!look.wanted(entry, kbase, have, all_pages, len)) continue;
        if (!warp_wait(&v_look[looks % L::kRing], (looks / L::kRing) & 1)) { ok = false; break; }
        ++looks;
        const bool mixed = look.mixed(entry, kbase, len);
        uint4* vt = reinterpret_cast<uint4*>(smem + L::kStageOff + L::kVOff + (gi % L::kRing) * L::kKVTileBytes);
        uint64_t keys = 0;  // rows of the tile that stand for a key
        for (int x = 0; x * sub_rows < kChunkBlk; ++x)
          if ((have >> x) & 1) keys |= (sub_rows == 64 ? ~0ull : (1ull << sub_rows) - 1) << (x * sub_rows & 63);
        if (kbase + kChunkBlk > len) keys &= (1ull << (len - kbase)) - 1;
        bool bad = false;
        if (keys == ~0ull) {  // (so it is looked over for its values; eight loads in flight)
#pragma unroll
          for (int i0 = 0; i0 < 64 * L::kChunks * 8; i0 += 256) {
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = vt[i0 + i * 32 + lane];
#pragma unroll
            for (int i = 0; i < 8; ++i) bad |= any_nonfinite<kF16>(v[i]);
          }
        } else for (int i = lane; i < 64 * L::kChunks * 8; i += 32) {  // 16-byte pieces
          if (!((keys >> ((i >> 3) & 63)) & 1)) vt[i] = make_uint4(0, 0, 0, 0);
          else if (mixed) bad |= any_nonfinite<kF16>(vt[i]);
        }
        if (__any_sync(0xffffffffu, bad)) {
          if (open != tile) {  // once an earlier tile's codes have been read
            const uint64_t t0 = globaltimer_ns();
            while ((*mark & 7) != 0 && globaltimer_ns() - t0 < kWaitLimitNs) {}
            if ((*mark & 7) != 0) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            for (int i = lane; i < (D / 16) * 128; i += 32) codes[i] = 0;
            __syncwarp();
            if (lane == 0) *mark = (tile << 3) | 4;
            open = tile;
          }
          for (int q = 0; q < 4; ++q) {
            const int r = q * 32 + lane, slot = sh.mode == 2 ? r >> 6 : 0;
            const int tok = sh.mode == 2 ? r & 63 : r / sh.hpt;
            const bool use = sh.mode == 2 ? ((entry >> (kKbBits + 4 + slot)) & 1) != 0 : tok < w->valid[0];
            const int lim = max(0, min(w->pos[slot] + tok - kbase + 1, kChunkBlk));
            const uint64_t seen = !use || lim == 0 ? 0 : keys & (lim == 64 ? ~0ull : (1ull << lim) - 1);
            for (int c = 0; c < 64; ++c) {
              if (!((seen >> c) & 1)) continue;
              for (int i = 0; i < D / 8; ++i) {
                const uint4 v = vt[(i >> 3) * 512 + c * 8 + (i & 7)];
                if (!any_nonfinite<kF16>(v)) continue;
                for (int e = 0; e < 8; ++e) {
                  const uint32_t v2 = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
                  const uint32_t x = (v2 >> ((e & 1) * 16)) & 0xffffu;
                  if (!nonfinite16<kF16>(x)) continue;
                  const int d = (i >> 3) * 64 + (((i & 7) ^ (c & 7)) << 3) + e;  // 128B swizzle
                  const uint32_t kind = (x & (kF16 ? 0x3ffu : 0x7fu)) ? 3u : (x & 0x8000u) ? 2u : 1u;
                  codes[(d >> 4) * 128 + r] |= kind << ((d & 15) * 2);
                }
              }
            }
          }
          __syncwarp();  // every row has its codes: the values go
          for (int i = lane; i < 64 * L::kChunks * 8; i += 32) {
            uint4 v = vt[i];
            if (!any_nonfinite<kF16>(v)) continue;
            uint32_t* x = &v.x;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (nonfinite16<kF16>((x[e >> 1] >> ((e & 1) * 16)) & 0xffffu)) x[e >> 1] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
            vt[i] = v;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[gi % L::kRing]);
      }
      g += n;
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_empty[lb]);
    }
    if (!ok) set_err(a.err, TASFT_DEVERR_TIMEOUT | (1 << 13));
  }
  // ---------------- teardown ----------------
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

// Tiles in pieces: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, pieces in order. CTA c
// joins the tile that work CTA c was the first to start inside of: its pieces are the second
// partial of CTA c - 1 and the first ones of CTAs c, c + 1, ... A warp takes a row at a time; lane
// x holds piece x's weight; D / 32 consecutive columns per lane, eight pieces' loads in flight.
template <int D, bool kF16>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const tasft_chunk_args a, const ChunkShape sh, const ChunkWs ws) {
  using T = typename std::conditional<kF16, __half, __nv_bfloat16>::type;
  constexpr int V = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int c = blockIdx.x;
  const Work w = ws.cut[c];
  const int ns = w.pieces;
  if (ns < 2 || c + ns - 2 >= (int)gridDim.x) return;
  const int warp = threadIdx.x >> 5;
  // where a row of the tile goes, or null
  auto target = [&](int r) -> T* {
    const int slot = sh.mode == 2 ? r >> 6 : 0;
    const int tok = sh.mode == 2 ? r & 63 : r / sh.hpt;
    const int hd = sh.mode == 2 ? 0 : r % sh.hpt;
    const int qpos = (slot ? w.pos[1] : w.pos[0]) + tok;
    const bool live = sh.mode == 2 ? (slot ? w.valid[1] : w.valid[0]) && qpos >= w.ctx && qpos < w.len : tok < w.valid[0];
    if (r >= sh.rows || !live) return nullptr;
    return reinterpret_cast<T*>(a.out) + (int64_t)((slot ? w.row[1] : w.row[0]) + tok) * a.o_stride[0] +
           (int64_t)((slot ? w.head[1] : w.head[0]) + hd) * a.o_stride[1] + lane * V;
  };
  auto place = [&](int x) -> int64_t { return (int64_t)(x == 0 ? 2 * c - 1 : 2 * (c + x - 1)) * sh.rows; };
  auto store = [&](T* dst, const float* acc, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint32_t pk[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      pk[i] = kF16 ? tc::pack_f16x2(acc[2 * i] * inv, acc[2 * i + 1] * inv)
                   : tc::pack_bf16x2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
    if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pk[0], pk[1]);
    else *reinterpret_cast<uint32_t*>(dst) = pk[0];
  };
  if (ns <= 8) {
    // many rows, few pieces: a warp's four rows at once, eight lanes on the pieces of each
    const int mine = lane >> 3, x = lane & 7, r0 = warp + mine * 32;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (x < ns && r0 < sh.rows && target(r0)) ml = ws.ml[place(x) + r0];
    float M = ml.x;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float wgt = ml.y == 0.f ? 0.f : ml.x == -INFINITY ? 1.f : ex2(ml.x - M);
    float sum = wgt * ml.y;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const unsigned have = __ballot_sync(0xffffffffu, ml.y != 0.f);
    float acc[4][V];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[i][k] = 0.f;
    for (int p = 0; p < ns; ++p) {
      float v[4][V];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[i][k] = 0.f;
        if ((have >> (8 * i + p)) & 1) {
          const float* o = ws.o + (place(p) + warp + 32 * i) * D + lane * V;
          if constexpr (V == 4) *reinterpret_cast<float4*>(v[i]) = *reinterpret_cast<const float4*>(o);
          else *reinterpret_cast<float2*>(v[i]) = *reinterpret_cast<const float2*>(o);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float wp = __shfl_sync(0xffffffffu, wgt, 8 * i + p);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[i][k] += wp * v[i][k];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float total = __shfl_sync(0xffffffffu, sum, 8 * i);
      if (T* dst = target(warp + 32 * i)) store(dst, acc[i], total);
    }
    return;
  }
  for (int r = warp; r < sh.rows; r += kMergeThreads / 32) {
    T* dst = target(r);
    if (!dst) continue;
    float M = -INFINITY, acc[V], sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int x0 = 0; x0 < ns; x0 += 32) {
      const int nx = min(32, ns - x0);
      const float2 ml = lane < nx ? ws.ml[place(x0 + lane) + r] : make_float2(-INFINITY, 0.f);
      const float Mn = fmaxf(M, warp_max(ml.x));
      if (Mn != M) {  // earlier pieces (more than 32) move to the new maximum
        const float f = M == -INFINITY ? 1.f : ex2(M - Mn);
        sum *= f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= f;
        M = Mn;
      }
      // a piece with nothing to see (l = 0) wrote no O
      const float wgt = ml.y == 0.f ? 0.f : ml.x == -INFINITY ? 1.f : ex2(ml.x - M);
      const unsigned have = __ballot_sync(0xffffffffu, ml.y != 0.f);
      const float lw = wgt * ml.y;
      for (int x1 = 0; x1 < nx; x1 += 8) {
        float v[8][V];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[x][i] = 0.f;
          if ((have >> (x1 + x)) & 1) {
            const float* o = ws.o + (place(x0 + x1 + x) + r) * D + lane * V;
            if constexpr (V == 4) *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(o);
            else *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(o);
          }
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          if (x1 + x >= nx) break;
          const float wx = __shfl_sync(0xffffffffu, wgt, x1 + x);
          sum += __shfl_sync(0xffffffffu, lw, x1 + x);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] += wx * v[x][i];
        }
      }
    }
    store(dst, acc, sum);
  }
}

// How a call's tiles are laid out; false when no layout covers it.
bool chunk_shape(ChunkShape& sh, int Hq, int Hk, int Hm, int max_q) {
  const int grp = Hq / Hk;
  if (grp > 64) return false;
  if (Hm > 0 && (Hm != Hk || grp == 1)) {
    sh.mode = 2;
    sh.hpt = 1;
    sh.tpt = grp >= 2 ? 64 : 128;
    sh.units = grp >= 2 ? Hk * ((grp + 1) / 2) : Hk;
    sh.rows = 128;
  } else {
    sh.mode = Hm > 0 ? 1 : 0;
    sh.hpt = grp;
    sh.units = Hk;
    sh.tpt = 128 / grp;
    if (sh.mode == 1) {
      int t = 64;
      while (t > sh.tpt) t >>= 1;
      sh.tpt = t;
    }
    sh.rows = grp * (max_q < sh.tpt ? max_q : sh.tpt);
  }
  sh.tpt_log2 = 0;
  while ((1 << sh.tpt_log2) < sh.tpt) ++sh.tpt_log2;
  return true;
}

// Parts of the workspace for G work CTAs, in bytes from its start.
struct WsLayout {
  int64_t ml, o, bytes;
};
WsLayout ws_layout(const ChunkShape& sh, int D, int G) {
  WsLayout w;
  w.ml = ((int64_t)G * sizeof(Work) + 255) / 256 * 256;
  w.o = w.ml + (2LL * G * sh.rows * 8 + 255) / 256 * 256;
  w.bytes = w.o + 2LL * G * sh.rows * D * 4;
  return w;
}

template <int D, bool kF16>
int launch(const tasft_chunk_args& a, ChunkShape sh, int sms, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  const int box = a.page_size < kChunkBlk ? a.page_size : kChunkBlk;
  if (!make_tmap_thd(&mq, a.q, a.T, a.Hq, D, a.q_stride[0], a.q_stride[1], sh.mode == 2 ? 1 : sh.hpt,
                     sh.mode == 2 ? 64 : sh.tpt))
    return TASFT_ERR_UNSUPPORTED;
  if (!make_tmap_paged(&mk, a.k_pages, a.num_pages, a.page_size, a.Hk, D, a.k_stride, box)) return TASFT_ERR_UNSUPPORTED;
  if (!make_tmap_paged(&mv, a.v_pages, a.num_pages, a.page_size, a.Hk, D, a.v_stride, box)) return TASFT_ERR_UNSUPPORTED;
  auto kern = bsa_chunk_tc_kernel<D, kF16>;
  const int smem = Smem<D>::kAlloc;
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(kern, smem, allowed)) return TASFT_ERR_CUDA;
  const int grid = 2 * sms;  // persistent: two CTAs per SM
  const WsLayout lay = ws_layout(sh, D, grid);
  uint8_t* p = reinterpret_cast<uint8_t*>(a.workspace);
  const ChunkWs ws = {reinterpret_cast<Work*>(p), reinterpret_cast<float2*>(p + lay.ml),
                      reinterpret_cast<float*>(p + lay.o)};
  if (debug_enabled()) debug_log("chunk_tc D=%d mode=%d grid=%d smem=%d", D, sh.mode, grid, smem);
  // both launches may begin while the kernel before them ends; they wait for it on the device
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int rc = cuda_status(cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, a, sh, ws));
  count_launch();
  if (rc != TASFT_OK || !sh.may_cut) return rc;
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = 0;
  rc = cuda_status(cudaLaunchKernelEx(&cfg, chunk_merge_kernel<D, kF16>, a, sh, ws));
  count_launch();
  return rc;
}

}  // namespace
}  // namespace tasft

using namespace tasft;

extern "C" int64_t tasft_chunk_workspace_size(int32_t B, int32_t T, int32_t Hq, int32_t Hk, int32_t D, int32_t max_q,
                                              int32_t Hm) {
  if (B <= 0 || T < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || D <= 0 || max_q <= 0 || Hm < 0) return TASFT_ERR_INVALID_ARG;
  ChunkShape sh = {};
  if (!chunk_shape(sh, Hq, Hk, Hm, max_q)) return TASFT_ERR_UNSUPPORTED;
  return ws_layout(sh, D, 2 * sm_count()).bytes;
}

extern "C" int tasft_bsa_chunk_paged_fwd(const tasft_chunk_args* ap, tasft_stream_t stream) {
  return tasft_bsa_chunk_paged_fwd_opt(ap, 0, stream);
}

extern "C" int tasft_bsa_chunk_paged_fwd_opt(const tasft_chunk_args* ap, int32_t options, tasft_stream_t stream) {
  if (!ap || (options & ~TASFT_ZERO_REST)) return TASFT_ERR_INVALID_ARG;
  tasft_chunk_args a = *ap;
  // strides of axes of length one say nothing
  if (a.T == 1) a.q_stride[0] = a.o_stride[0] = a.D;
  if (a.Hq == 1) a.q_stride[1] = a.o_stride[1] = a.D;
  if (a.Hk == 1) a.k_stride[2] = a.v_stride[2] = a.D;
  if (a.num_pages == 1) a.k_stride[0] = a.v_stride[0] = a.D;
  if (a.B <= 0 || a.T < 0 || a.Hq <= 0 || a.Hk <= 0 || a.D <= 0 || a.Hq % a.Hk != 0 || a.max_q <= 0 ||
      a.max_pages <= 0 || a.num_pages <= 0 || !(a.scale > 0.f && a.scale <= FLT_MAX))
    return TASFT_ERR_INVALID_ARG;
  if (!a.cu_seqlens || !a.kv_len || !a.block_table || !a.k_pages || !a.v_pages) return TASFT_ERR_INVALID_ARG;
  if (a.k_stride[3] != 1 || a.v_stride[3] != 1) return TASFT_ERR_INVALID_ARG;
  if (a.kept_idx) {
    if (!a.kept_cnt || (a.Hm != a.Hk && a.Hm != a.Hq) || a.nb_w <= 0 || a.nb_q < ((int64_t)a.max_q + 126) / 64)
      return TASFT_ERR_INVALID_ARG;
  }
  if (a.T == 0) return TASFT_OK;
  if (!a.q || !a.out) return TASFT_ERR_INVALID_ARG;
  if (a.dtype != TASFT_BF16 && a.dtype != TASFT_F16) return TASFT_ERR_UNSUPPORTED;
  if ((a.D != 64 && a.D != 128) || a.block != kChunkBlk) return TASFT_ERR_UNSUPPORTED;
  if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size != 128) return TASFT_ERR_UNSUPPORTED;
  // block indices travel in kKbBits bits
  if ((int64_t)a.max_pages * a.page_size > (int64_t)kKbMask * kChunkBlk) return TASFT_ERR_TOO_LARGE;
  // 16-byte stores of out's rows (q and the pages are checked with their tensor maps)
  if (!aligned16(a.out) || a.o_stride[0] % 8 || a.o_stride[1] % 8) return TASFT_ERR_UNSUPPORTED;
  ChunkShape sh;
  if (!chunk_shape(sh, a.Hq, a.Hk, a.kept_idx ? a.Hm : 0, a.max_q)) return TASFT_ERR_UNSUPPORTED;
  sh.capacity = a.max_pages * a.page_size;
  // most blocks a tile visits
  int bound = (sh.capacity + kChunkBlk - 1) / kChunkBlk;
  if (a.kept_idx && (int64_t)a.nb_w * 2 < bound) bound = a.nb_w * (sh.mode == 2 ? 2 : 1);
  // 32-byte stores of out's rows
  sh.wide = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0 && a.o_stride[0] % 16 == 0 && a.o_stride[1] % 16 == 0;
  sh.zero_rest = (options & TASFT_ZERO_REST) != 0;
  sh.stride = (a.B + kChunkBuckets - 1) / kChunkBuckets;
  // One launch where cutting tiles gains nothing (the device decides the rest). Tiles with lists
  // take about as long as one another: the gain is the last round's idle share of the longest, for
  // as many tiles as the tokens fill. Without lists they may differ by all their blocks.
  const int64_t G = 2 * sm_count(), tiles = ((int64_t)a.T / sh.tpt + a.B) * sh.units;
  sh.may_cut = sh.mode == 0 ? bound > kChunkMergeCost
                            : ((tiles + G - 1) / G * G - tiles) * bound > kChunkMergeCost * G;
  if (!a.workspace || a.workspace_bytes < ws_layout(sh, a.D, (int)G).bytes) return TASFT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(a.workspace) & 31u) != 0) return TASFT_ERR_WORKSPACE;  // 32-byte stores of partials
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int sms = sm_count();
  const bool f16 = a.dtype == TASFT_F16;
  if (a.D == 128) return f16 ? launch<128, true>(a, sh, sms, st) : launch<128, false>(a, sh, sms, st);
  return f16 ? launch<64, true>(a, sh, sms, st) : launch<64, false>(a, sh, sms, st);
}
