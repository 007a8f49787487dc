// Kept blocks from gate scores: per (sequence, kv-head, row) the first blocks, the last blocks
// up to the row's own, and the best-scored of the others, `top_k` in all, as an ascending list.
//
// A block's score is the highest of its group's query heads (NaN counts as -inf; a -inf score
// is never chosen), optionally with a floor tau. Ties go to the lowest index. The k-th largest
// score is found exactly, without a sort: scores are mapped to integers of the same order, held
// in registers, and the threshold is fixed from the top. Up to 128 blocks a warp takes a row and
// counts "at least this much" bit by bit; longer rows take one CTA and eight bits at a time,
// with a histogram in shared memory, below the bits that the row's largest and smallest score
// share (gate scores lie close together). Either stops as soon as the count comes out exactly.
// Kept blocks become one bit each, and a scan over the words' population counts places them.
//
// kT threads per row, kV values per thread (value v of thread t is block v * kT + t, so loads
// are coalesced and a warp's ballot is one word of the bit rows). The scores are read once, 64 MB
// for 2064 rows of up to 1535 blocks and 7 heads: 24 us on a B200 (9.8 at the copy rate), bound by
// issue (1,067 instructions a warp, slots 61% busy) and the chain of loads and barriers; 512 short rows 5 us.
#include "common.cuh"

namespace tasft {
namespace {

// fp32 (not NaN) -> uint32 of the same order, -0 and +0 alike
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
constexpr uint32_t kNever = 0x007fffffu;  // ordered(-inf): never chosen; below every other score

// Threads of a block: kT for one row, or four warps with a row each when kT is 32.
template <int kT, int kV>
__global__ void __launch_bounds__(kT == 32 ? 128 : kT) select_blocks_kernel(const tasft_select_args a, const int log2_block) {
  constexpr int kWords = kT * kV / 32;
  constexpr int kRowsPerCta = kT == 32 ? 4 : 1;
  __shared__ uint32_t bits_[kRowsPerCta][2 * kWords];  // above the threshold, at it
  __shared__ uint2 kept_[kRowsPerCta][kWords];  // the kept bits of a word, and the place of its first
  __shared__ int32_t total_[kRowsPerCta];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = kT == 32 ? warp : 0, t = kT == 32 ? lane : threadIdx.x;
  // one CTA per row of a (row, kv-head, sequence) grid, or four consecutive rows per CTA
  int i, hk, b;
  if constexpr (kT == 32) {
    const uint32_t r = blockIdx.x * kRowsPerCta + sub, nq = a.NBq, nh = a.Hk;
    if (r >= (uint32_t)a.B * nh * nq) return;  // whole warps
    i = r % nq;
    hk = r / nq % nh;
    b = r / nq / nh;
  } else {
    i = blockIdx.x;
    hk = blockIdx.y;
    b = blockIdx.z;
  }
  const int64_t row = ((int64_t)b * a.Hk + hk) * a.NBq + i;
  uint32_t* above = bits_[sub];
  uint32_t* at = above + kWords;
  uint2* kept = kept_[sub];
  int32_t* idx = a.kept_idx + row * a.width;
  const int grp = a.Hq / a.Hk;

  const int len = a.kv_len[b];
  const int64_t n_new = (int64_t)a.cu_seqlens[b + 1] - a.cu_seqlens[b];  // (may leave 32 bits)
  const int own0 = (int)((len - n_new) >> log2_block), own_last = (len - 1) >> log2_block;
  const bool bad = n_new < 0 || (n_new > 0 && (len < n_new || own_last >= a.NBk || own_last - own0 >= a.NBq));
  const int mine = own0 + i;
  if (bad || n_new <= 0 || mine > own_last) {  // no such row
    if (bad && t == 0) set_err(a.err, TASFT_DEVERR_INDEX);
    for (int j = t; j < a.width; j += kT) idx[j] = -1;
    if (t == 0) a.kept_cnt[row] = 0;
    return;
  }
  // always kept: [0, lead) and [tail, mine]
  const int lead = min(a.first, mine + 1), tail = max(lead, mine + 1 - a.local);
  const int want = max(0, min(a.top_k - lead - (mine + 1 - tail), tail - lead));

  const float* s = a.scores + b * a.stride[0] + (int64_t)hk * grp * a.stride[1] + (int64_t)i * a.stride[2];
  uint32_t key[kV];
  {
    float x[kV];
#pragma unroll
    for (int v = 0; v < kV; ++v) x[v] = -INFINITY;
    if (want > 0) {
      for (int h = 0; h < grp; h += 4) {  // four heads' loads go out together
        float y[4][kV];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float* sh = s + min(h + g, grp - 1) * a.stride[1] + t;
#pragma unroll
          for (int v = 0; v < kV; ++v) y[g][v] = v * kT + t < tail ? __ldg(sh + v * kT) : -INFINITY;
        }
#pragma unroll
        for (int v = 0; v < kV; ++v)  // fmaxf drops NaN
          x[v] = fmaxf(x[v], fmaxf(fmaxf(y[0][v], y[1][v]), fmaxf(y[2][v], y[3][v])));
      }
    }
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const int j = v * kT + t;
      key[v] = !a.use_tau || x[v] >= a.tau ? ordered(x[v]) : 0u;
      if (key[v] <= kNever || j < lead || j >= tail) key[v] = 0;
    }
  }
  // keys from thr on are taken; where `quota` says so, only that many of those at thr itself
  uint32_t thr = 0xffffffffu;
  int quota = 0;
  if constexpr (kT == 32) {
    if (want > 0) {
      thr = 0;  // the largest value that `want` keys reach (0: fewer keys than that, all taken)
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t cand = thr | (1u << bit);
        int n = 0;
#pragma unroll
        for (int v = 0; v < kV; ++v) n += key[v] >= cand;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= want) thr = cand;
        if (n == want) break;  // exactly these: no smaller bit can part them
      }
      if (thr == 0) {
        thr = 1;
        quota = INT32_MAX;
      } else {
        int n = 0;
#pragma unroll
        for (int v = 0; v < kV; ++v) n += key[v] > thr;
        quota = want - __reduce_add_sync(0xffffffffu, n);
      }
    }
  } else {
    __shared__ uint32_t red[3][kT / 32];
    __shared__ int32_t hist[256];
    __shared__ int32_t part[8];
    __shared__ int32_t found[3];  // digit, how many of it are wanted, how many there are
    if (want > 0) {               // the same for the whole CTA
      uint32_t hi = 0, lo = 0xffffffffu, n = 0;
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        hi = max(hi, key[v]);
        lo = min(lo, key[v] ? key[v] : 0xffffffffu);
        n += key[v] != 0;
      }
      hi = __reduce_max_sync(0xffffffffu, hi);
      lo = __reduce_min_sync(0xffffffffu, lo);
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) {
        red[0][warp] = hi;
        red[1][warp] = lo;
        red[2][warp] = n;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kT / 32; ++w) {
        hi = max(hi, red[0][w]);
        lo = min(lo, red[1][w]);
        n = (w == 0 ? 0 : n) + red[2][w];
      }
      if ((int)n <= want) {
        thr = 1;
        quota = INT32_MAX;
      } else {
        int left = want;
        int top = hi == lo ? 0 : 32 - __clz(hi ^ lo);  // bits [0, top) are open
        thr = top == 32 ? 0u : hi >> top << top;
        quota = INT32_MAX;
        bool first_digit = true;
        while (true) {
          if (top == 0) {  // all open keys are thr itself
            quota = left;
            break;
          }
          const int shift = max(0, top - 8);
          for (int i = t; i < 256; i += kT) hist[i] = 0;
          __syncthreads();
          if (first_digit) {  // every key is open
#pragma unroll
            for (int v = 0; v < kV; ++v)
              if (key[v]) atomicAdd(&hist[(key[v] >> shift) & ((1u << (top - shift)) - 1u)], 1);
          } else {
#pragma unroll
            for (int v = 0; v < kV; ++v)
              if (key[v] >> top == thr >> top) atomicAdd(&hist[(key[v] >> shift) & ((1u << (top - shift)) - 1u)], 1);
          }
          first_digit = false;
          __syncthreads();
          // the digit in which the count from the top reaches `left` (256 threads or the first 128,
          // two digits each)
          constexpr int kPer = kT >= 256 ? 1 : 256 / kT;
          int mine_n[kPer], sum = 0, pre = 0;
          if (t < 256) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) sum += mine_n[i] = hist[255 - (t * kPer + i)];
            pre = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int x = __shfl_up_sync(0xffffffffu, pre, o);
              if (lane >= o) pre += x;
            }
            if (lane == 31) part[warp] = pre;
          }
          __syncthreads();
          if (t < 256) {
            for (int w = 0; w < warp; ++w) pre += part[w];
            int c = pre - sum;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              if (c < left && c + mine_n[i] >= left) {
                found[0] = 255 - (t * kPer + i);
                found[1] = left - c;
                found[2] = mine_n[i];
              }
              c += mine_n[i];
            }
          }
          __syncthreads();
          thr |= (uint32_t)found[0] << shift;
          left = found[1];
          if (left == found[2]) break;  // the whole digit is taken
          top = shift;
        }
      }
    }
  }
  // ---- bits: always kept or above the threshold; at the threshold, where not all of those are ----
  const bool all = quota == INT32_MAX;
  const uint32_t from = want == 0 ? 0xffffffffu : all ? thr : thr + 1;  // scores are below the top value
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const int j = v * kT + t;
    const unsigned wa = __ballot_sync(0xffffffffu, key[v] >= from || j < lead || (j >= tail && j <= mine));
    if (lane == 0) above[(v * kT + t) >> 5] = wa;
    if (!all) {
      const unsigned we = __ballot_sync(0xffffffffu, key[v] == thr);
      if (lane == 0) at[(v * kT + t) >> 5] = we;
    }
  }
  if constexpr (kT > 32) __syncthreads();
  else __syncwarp();
  // ---- one warp: the first `quota` at the threshold join; places of the words ----
  if (t < 32) {
    int ties = quota, out = 0;
    for (int w0 = 0; w0 < kWords; w0 += 32) {
      const int w = w0 + lane;
      uint32_t e = !all && w < kWords ? at[w] : 0u, m = w < kWords ? above[w] : 0u;
      const int ne = __popc(e);
      int pre = ne;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, pre, o);
        if (lane >= o) pre += x;
      }
      const int total = __shfl_sync(0xffffffffu, pre, 31);
      int join = min(max(ties - (pre - ne), 0), ne);
      if (join == ne) {
        m |= e;
      } else {
        for (; join > 0; --join) {  // lowest indices first
          m |= e & (0u - e);
          e &= e - 1;
        }
      }
      if (!all) ties -= total;
      const int nk = __popc(m);
      int pk = nk;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, pk, o);
        if (lane >= o) pk += x;
      }
      if (w < kWords) kept[w] = make_uint2(m, out + pk - nk);
      out += __shfl_sync(0xffffffffu, pk, 31);
    }
    if (lane == 0) {
      total_[sub] = out;
      a.kept_cnt[row] = out;
    }
  }
  if constexpr (kT > 32) __syncthreads();
  else __syncwarp();
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const int j = v * kT + t;
    const uint2 m = kept[j >> 5];
    if ((m.x >> lane) & 1) idx[m.y + __popc(m.x & ((1u << lane) - 1u))] = j;
  }
  for (int j = total_[sub] + t; j < a.width; j += kT) idx[j] = -1;
}

template <int kT, int kV>
int run(const tasft_select_args& a, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Hk * a.NBq;
  if (rows > INT32_MAX / 2 || a.B > 65535 || a.Hk > 65535) return TASFT_ERR_TOO_LARGE;
  const dim3 grid = kT == 32 ? dim3((unsigned)((rows + 3) / 4)) : dim3((unsigned)a.NBq, (unsigned)a.Hk, (unsigned)a.B);
  int log2_block = 0;
  while ((1 << log2_block) < a.block) ++log2_block;
  select_blocks_kernel<kT, kV><<<grid, kT == 32 ? 128 : kT, 0, st>>>(a, log2_block);
  count_launch();
  return launch_status();
}

}  // namespace
}  // namespace tasft

using namespace tasft;

extern "C" int tasft_select_blocks(const tasft_select_args* ap, tasft_stream_t stream) {
  if (!ap) return TASFT_ERR_INVALID_ARG;
  const tasft_select_args& a = *ap;
  if (!a.scores || !a.cu_seqlens || !a.kv_len || !a.kept_idx || !a.kept_cnt) return TASFT_ERR_INVALID_ARG;
  if (a.B <= 0 || a.Hq <= 0 || a.Hk <= 0 || a.Hq % a.Hk || a.NBq <= 0 || a.NBk <= 0 || a.block <= 0)
    return TASFT_ERR_INVALID_ARG;
  if (a.top_k <= 0 || a.first < 0 || a.local < 1 || a.width <= 0) return TASFT_ERR_INVALID_ARG;
  if (a.block & (a.block - 1)) return TASFT_ERR_UNSUPPORTED;
  // a row never keeps more than this, so a list never runs over its row
  const int64_t most = a.first + (int64_t)a.local > a.top_k ? a.first + (int64_t)a.local : a.top_k;
  if (a.width < (most < a.NBk ? most : a.NBk)) return TASFT_ERR_INVALID_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // by the width of the scores (the rows' own lengths are on the device). At 1535 blocks 64 to 512
  // threads a row took 27 to 39 us where 256 took 24 to 27; the widest spills 280 bytes (2064 rows of
  // up to 4158 blocks: 315 us)
  if (a.NBk <= 128) return run<32, 4>(a, st);
  if (a.NBk <= 512) return run<128, 4>(a, st);
  if (a.NBk <= 2048) return run<256, 8>(a, st);
  if (a.NBk <= 16384) return run<512, 32>(a, st);
  return TASFT_ERR_TOO_LARGE;
}
