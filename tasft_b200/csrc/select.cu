// Kept blocks from gate scores: per (sequence, kv-head, row) the first blocks, the last blocks
// up to the row's own, and the best-scored of the others, `top_k` in all, as an ascending list.
//
// A block's score is the highest of its group's query heads (NaN counts as -inf; a -inf score
// is never chosen), optionally with a floor tau. Ties go to the lowest index. The k-th largest
// score is found exactly, without a sort: scores are mapped to integers of the same order and
// the threshold's bits are fixed from the top, one count of "at least this much" per bit, over
// values that stay in registers. Kept blocks become one bit each, and a scan over the words'
// population counts places them.
//
// One group of kT threads per row, kV values per thread (value i of thread t is block
// i * kT + t, so loads are coalesced and a warp's ballot is one word of the bit rows).
#include "common.cuh"

namespace tasft {
namespace {

// fp32 -> uint32 of the same order (-inf lowest, NaN as -inf; -0 and +0 alike)
__device__ __forceinline__ uint32_t ordered(float x) {
  if (!(x == x)) x = -INFINITY;
  if (x == 0.f) x = 0.f;
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kNever = 0x007fffffu;  // ordered(-inf): never chosen; below every other score

template <int kT>
__device__ __forceinline__ int group_count(int n, int32_t* scratch, int parity) {
  n = __reduce_add_sync(0xffffffffu, n);
  if constexpr (kT > 32) {
    // two alternating rows of scratch: one barrier per count
    int32_t* row = scratch + parity * (kT / 32);
    if ((threadIdx.x & 31) == 0) row[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < kT / 32; ++w) n += row[w];
  }
  return n;
}

// Threads of a block: kT for one row, or four warps with a row each when kT is 32.
template <int kT, int kV>
__global__ void __launch_bounds__(kT == 32 ? 128 : kT) select_blocks_kernel(const tasft_select_args a) {
  constexpr int kWords = kT * kV / 32;
  constexpr int kRowsPerCta = kT == 32 ? 4 : 1;
  __shared__ uint32_t bits_[kRowsPerCta][2 * kWords];  // above the threshold, at it
  __shared__ int32_t place_[kRowsPerCta][kWords + 1];
  __shared__ int32_t scratch[2 * (kT / 32)];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = kT == 32 ? warp : 0, t = kT == 32 ? lane : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerCta + sub;
  if (row >= (int64_t)a.B * a.Hk * a.NBq) return;  // whole warps (kT 32) or never
  uint32_t* above = bits_[sub];
  uint32_t* at = above + kWords;
  int32_t* place = place_[sub];
  const int i = (int)(row % a.NBq), hk = (int)(row / a.NBq % a.Hk), b = (int)(row / a.NBq / a.Hk);
  int32_t* idx = a.kept_idx + row * a.width;
  const int grp = a.Hq / a.Hk;

  const int n_new = a.cu_seqlens[b + 1] - a.cu_seqlens[b], len = a.kv_len[b];
  const bool bad = n_new < 0 || (n_new > 0 && (len < n_new || (len - 1) / a.block >= a.NBk ||
                                               (len - 1) / a.block - (len - n_new) / a.block >= a.NBq));
  const int mine = n_new > 0 && !bad ? (len - n_new) / a.block + i : 0;
  if (bad || n_new <= 0 || mine > (len - 1) / a.block) {  // no such row
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
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const int j = v * kT + t;
    key[v] = 0;
    if (j >= lead && j < tail) {
      float x = -INFINITY;
      for (int h = 0; h < grp; ++h) x = fmaxf(x, __ldg(s + h * a.stride[1] + j));  // fmaxf drops NaN
      if (!a.use_tau || x >= a.tau) key[v] = ordered(x);
      if (key[v] <= kNever) key[v] = 0;
    }
  }
  // the largest threshold that `want` keys reach (0: they do not, everything above 0 is taken)
  uint32_t thr = 0;
  int parity = 0;
  if (want > 0) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = thr | (1u << bit);
      int n = 0;
#pragma unroll
      for (int v = 0; v < kV; ++v) n += key[v] >= cand;
      n = group_count<kT>(n, scratch, parity);
      parity ^= 1;
      if (n >= want) thr = cand;
      if (n == want) break;  // exactly these: no smaller bit can part them
    }
  }
  // ---- bits: always kept or above the threshold; at the threshold ----
  int n_above = 0;
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const int j = v * kT + t;
    const bool forced = j < lead || (j >= tail && j <= mine);
    const bool up = want > 0 && key[v] > thr;
    n_above += up;
    const unsigned wa = __ballot_sync(0xffffffffu, forced || up);
    const unsigned we = __ballot_sync(0xffffffffu, want > 0 && thr > 0 && key[v] == thr);
    if (lane == 0) {
      above[(v * kT + t) >> 5] = wa;
      at[(v * kT + t) >> 5] = we;
    }
  }
  n_above = group_count<kT>(n_above, scratch, parity);
  if constexpr (kT > 32) __syncthreads();
  else __syncwarp();
  // ---- one warp: the first (want - n_above) at the threshold join; places of the words ----
  if (t < 32) {
    int ties = want - n_above, out = 0;
    for (int w0 = 0; w0 < kWords; w0 += 32) {
      const int w = w0 + lane;
      uint32_t e = w < kWords ? at[w] : 0u, m = w < kWords ? above[w] : 0u;
      const int ne = __popc(e);
      int pre = ne;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, pre, o);
        if (lane >= o) pre += x;
      }
      const int total = __shfl_sync(0xffffffffu, pre, 31);
      int quota = min(max(ties - (pre - ne), 0), ne);
      if (quota == ne) {
        m |= e;
      } else {
        for (; quota > 0; --quota) {  // lowest indices first
          m |= e & (0u - e);
          e &= e - 1;
        }
      }
      ties -= total;
      const int nk = __popc(m);
      int pk = nk;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, pk, o);
        if (lane >= o) pk += x;
      }
      if (w < kWords) {
        above[w] = m;
        place[w] = out + pk - nk;
      }
      out += __shfl_sync(0xffffffffu, pk, 31);
    }
    if (lane == 0) {
      place[kWords] = out;
      a.kept_cnt[row] = out;
    }
  }
  if constexpr (kT > 32) __syncthreads();
  else __syncwarp();
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const int j = v * kT + t;
    const uint32_t m = above[j >> 5];
    if ((m >> lane) & 1) idx[place[j >> 5] + __popc(m & ((1u << lane) - 1u))] = j;
  }
  for (int j = place[kWords] + t; j < a.width; j += kT) idx[j] = -1;
}

template <int kT, int kV>
int run(const tasft_select_args& a, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Hk * a.NBq;
  const int64_t ctas = kT == 32 ? (rows + 3) / 4 : rows;
  if (ctas > INT32_MAX) return TASFT_ERR_TOO_LARGE;
  select_blocks_kernel<kT, kV><<<(unsigned)ctas, kT == 32 ? 128 : kT, 0, st>>>(a);
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
  // a row never keeps more than this, so a list never runs over its row
  const int64_t most = a.first + (int64_t)a.local > a.top_k ? a.first + (int64_t)a.local : a.top_k;
  if (a.width < (most < a.NBk ? most : a.NBk)) return TASFT_ERR_INVALID_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.NBk <= 128) return run<32, 4>(a, st);
  if (a.NBk <= 512) return run<128, 4>(a, st);
  if (a.NBk <= 2048) return run<256, 8>(a, st);
  if (a.NBk <= 16384) return run<512, 32>(a, st);
  return TASFT_ERR_TOO_LARGE;
}
