// Rotary embedding of new tokens on their way into a paged KV cache, with the gate's block
// means, in one pass over the projection outputs.
//
// A token at position p turns the pair (x, y) number i of its first rot columns by the angle
// p * f_i: (x cos - y sin, y cos + x sin) times `factor`; pairs are (i, i + rot/2), or
// (2i, 2i + 1) when interleaved. Products and sums are fp32, rounded once to the tensors' type.
// The angle is taken in turns, p * f_i / 2pi in fp64 with the whole turns dropped, since fp32
// has lost the angle's fraction by position 10^5; one fp64 sine and cosine per thread and
// segment start it and fp64 complex products step it from token to token, so cos and sin are
// those of the exact angle, rounded to fp32.
//
// Means are those AttnGate pools (zero padding counts): the sum of a 64-token block's rows as
// they are held, divided by the block. A key block begun by an earlier call is read back from
// the cache, so its mean depends only on what the cache holds. The queries of earlier calls are
// gone, so with TASFT_ROPE_MEAN_NEW a query mean is over the block's new rows alone.
//
// Bound by HBM: every row is read and written once. One CTA of 4 warps takes one 64-token block
// of one sequence and as many of its heads; a warp takes a head, lanes over (16-byte column
// pairs x rows), and holds the block sums in registers. Measured on a B200: 7695 tokens of 28/4
// heads, D 128, 32 us = 4.5 TB/s (no less without the trigonometry: loads and stores in flight); 64
// tokens 9 us, a chain of table, cached rows, cos and sin, and new rows.
#include "common.cuh"

namespace tasft {
namespace {

constexpr int kRopeThreads = 128;  // one head per warp
constexpr int kRopeBlk = 64;
constexpr int kRopeRows = 64;      // rows whose cos and sin are at hand at a time (16 and 32 were slower)

template <typename T>
__device__ __forceinline__ void pack16(uint4& u, const float* f);
template <>
__device__ __forceinline__ void pack16<float>(uint4& u, const float* f) {
  u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <>
__device__ __forceinline__ void pack16<__nv_bfloat16>(uint4& u, const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&v);
  }
  u = make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void pack16<__half>(uint4& u, const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&v);
  }
  u = make_uint4(w[0], w[1], w[2], w[3]);
}

// Rotates a 16-byte column pair. Half layout: u1 are x of V pairs, u2 their y. Interleaved: u1
// holds V/2 pairs and u2 the next V/2. c, s: the V pairs' cos and sin in order.
template <typename T, bool kMixed>
__device__ __forceinline__ void turn(uint4& u1, uint4& u2, const float* c, const float* s) {
  constexpr int V = Vec16<T>::N;
  float x[2 * V], y[2 * V];
  Vec16<T>::unpack(u1, x);
  Vec16<T>::unpack(u2, x + V);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = kMixed ? 2 * i : i, o = kMixed ? 2 * i + 1 : i + V;
    // separate products: the plain formula's roundings
    y[e] = __fsub_rn(__fmul_rn(x[e], c[i]), __fmul_rn(x[o], s[i]));
    y[o] = __fadd_rn(__fmul_rn(x[o], c[i]), __fmul_rn(x[e], s[i]));
  }
  pack16<T>(u1, y);
  pack16<T>(u2, y + V);
}

template <typename T>
__device__ __forceinline__ void add_pair(float* acc, const uint4& u1, const uint4& u2) {
  constexpr int V = Vec16<T>::N;
  float x[2 * V];
  Vec16<T>::unpack(u1, x);
  Vec16<T>::unpack(u2, x + V);
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) acc[i] += x[i];
}

template <typename T, bool kMixed>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_append_kernel(const tasft_rope_append_args a, const int options) {
  constexpr int V = Vec16<T>::N;
  // [row][float4 of cos, then of sin][column pair]: the lanes of a row read 16 bytes beside one another
  extern __shared__ __align__(16) float trig[];
  __shared__ int64_t place[kRopeBlk];  // element offset of each row in the page pools; -1: not there
  __shared__ int64_t place_v[kRopeBlk];
  const int b = blockIdx.z, qi = blockIdx.y;  // heads vary fastest: a block's rows are read together
  const int half = a.rot / 2;
  const int start = a.cu_seqlens[b], end = a.cu_seqlens[b + 1], len = a.kv_len[b];
  const int n = end - start;
  // (end < start, not n < 0: the difference may leave 32 bits)
  const bool bad = start < 0 || end < start || end > a.T ||
                   (n > 0 && (len < n || len > (int64_t)a.max_pages * a.page_size || n > a.max_q));
  const int ctx = len - n;
  const int blk = bad || n == 0 ? 0 : ctx / kRopeBlk + qi;
  const bool there = !bad && n > 0 && (int64_t)blk * kRopeBlk < len;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.Hq + 2 * a.Hk;
  const int h = blockIdx.x * (kRopeThreads / 32) + warp;
  if ((options & TASFT_ZERO_REST) && h < a.Hq) {  // rows of q_out that no sequence accounts for
    auto zero = [&](int from, int to) {
      T* row = reinterpret_cast<T*>(a.q_out) + h * a.o_stride[1];
      for (int64_t r = (int64_t)from + qi; r < to; r += gridDim.y)
        for (int d = lane * V; d < a.D; d += 32 * V)
          *reinterpret_cast<uint4*>(row + r * a.o_stride[0] + d) = make_uint4(0, 0, 0, 0);
    };
    const int lo = max(0, min(start, a.T)), hi = max(0, min(end, a.T));
    if (b == 0) zero(0, lo);
    if (b == a.B - 1) zero(hi, a.T);
    if (bad) zero(lo, hi);
  }
  if (!there) {
    if (bad && qi == 0 && blockIdx.x == 0 && threadIdx.x == 0) set_err(a.err, TASFT_DEVERR_INDEX);
    if (a.pooled_q && h < a.Hq)  // a row that no new token falls in has a mean of zero
      for (int d = lane; d < a.D; d += 32) a.pooled_q[(((int64_t)b * a.Hq + h) * a.NBq + qi) * a.D + d] = 0.f;
    return;
  }
  if (a.pooled_k && blk >= a.NBk && blockIdx.x == 0 && threadIdx.x == 0) set_err(a.err, TASFT_DEVERR_INDEX);
  const int p0 = blk * kRopeBlk;
  const int r_lo = max(ctx - p0, 0), r_hi = min(len - p0, kRopeBlk);  // rows of the block with new tokens

  // ---- where the block's rows lie ----
  if (threadIdx.x < kRopeBlk) {
    const int r = threadIdx.x, p = p0 + r;
    int64_t at = -1, atv = -1;
    if (r < r_hi) {
      const int pg = a.block_table[(int64_t)b * a.max_pages + p / a.page_size];
      if (pg >= 0 && pg < a.num_pages) {
        at = pg * a.k_stride[0] + (p % a.page_size) * a.k_stride[1];
        atv = pg * a.v_stride[0] + (p % a.page_size) * a.v_stride[1];
      } else if (blockIdx.x == 0) {
        set_err(a.err, TASFT_DEVERR_INDEX);
      }
    }
    place[r] = at;
    place_v[r] = atv;
  }
  constexpr int kQuads = 2 * V / 4;    // float4s of cos and sin that a column pair takes
  const int turned = a.rot / (2 * V);  // column pairs of a row that turn
  // ---- the warp's head: lanes over (column pair, row) ----
  const int items = a.D / (2 * V);     // 16-byte column pairs of a row, at most 32
  const int step = 32 / items;         // rows at once
  const int item = lane % items, r0 = lane / items;
  const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
  // (lanes left over where items does not divide 32, and warps behind the last head, do nothing)
  const bool active = r0 < step && h < heads;
  const int hh = is_q ? h : is_v ? h - a.Hq - a.Hk : h - a.Hq;
  const bool rotated = !is_v && item < turned;
  // columns of the pair: half layout (i, i + rot/2), otherwise neighbours
  const int c1 = !kMixed && rotated ? item * V : 2 * item * V;
  const int c2 = !kMixed && rotated ? item * V + half : (2 * item + 1) * V;
  const int64_t in_step = is_q ? a.q_stride[0] : is_v ? a.v_in_stride[0] : a.k_in_stride[0];
  const int64_t in_head = is_q ? a.q_stride[1] : is_v ? a.v_in_stride[1] : a.k_in_stride[1];
  const int64_t tok0 = (int64_t)start + p0 - ctx;  // token of the block's row 0
  const T* in = reinterpret_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + hh * in_head + tok0 * in_step;
  T* out;
  if (is_q) out = reinterpret_cast<T*>(a.q_out) + hh * a.o_stride[1] + tok0 * a.o_stride[0];
  else if (is_v) out = reinterpret_cast<T*>(a.v_pages) + hh * a.v_stride[2];
  else out = reinterpret_cast<T*>(a.k_pages) + hh * a.k_stride[2];
  const int64_t* at = is_v ? place_v : place;
  const bool sum = is_q ? a.pooled_q != nullptr : !is_v && a.pooled_k != nullptr && blk < a.NBk;
  float acc[2 * V];
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) acc[i] = 0.f;
  // rows go kBatch at a time, every load of a batch before its first store
  constexpr int kBatch = 4;
  __syncthreads();
  if (active && sum && !is_q) {  // key rows of earlier calls
    for (int rb = r0; rb < r_lo; rb += kBatch * step) {
      uint4 u1[kBatch], u2[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = rb + i * step;
        u1[i] = u2[i] = make_uint4(0, 0, 0, 0);
        if (r < r_lo && at[r] >= 0) {
          u1[i] = *reinterpret_cast<const uint4*>(out + at[r] + c1);
          u2[i] = *reinterpret_cast<const uint4*>(out + at[r] + c2);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) add_pair<T>(acc, u1[i], u2[i]);
    }
  }
  const bool any_turn = half > 0 && blockIdx.x * (kRopeThreads / 32) < a.Hq + a.Hk;
  for (int lo = r_lo; lo < r_hi; lo = (lo / kRopeRows + 1) * kRopeRows) {
    const int hi = min((lo / kRopeRows + 1) * kRopeRows, r_hi);
    // ---- cos and sin of the rows: a thread steps one pair through a segment of them ----
    if (any_turn) {
      if (lo > r_lo) __syncthreads();  // the rows before are done with theirs
      const int segs = max(1, kRopeThreads / half), per = (hi - lo + segs - 1) / segs;
      for (int w = threadIdx.x; w < segs * half; w += kRopeThreads) {
        const int i = w % half, seg = w / half, e = i % V;
        const int first = seg * per, lastr = min(first + per, hi - lo);
        if (first >= lastr) continue;
        const double f = (a.freq_f64 ? reinterpret_cast<const double*>(a.inv_freq)[i]
                                     : (double)reinterpret_cast<const float*>(a.inv_freq)[i]) *
                         0.15915494309189533577;  // turns per position
        double turns = (double)(p0 + lo + first) * f;
        turns -= rint(turns);
        double s, c, ds, dc;
        sincospi(2.0 * turns, &s, &c);
        if (lastr - first > 1) sincospi(2.0 * (f - rint(f)), &ds, &dc);
        c *= a.factor;
        s *= a.factor;
        for (int r = first; r < lastr; ++r) {
          trig[((r * kQuads + e / 4) * turned + i / V) * 4 + e % 4] = (float)c;
          trig[((r * kQuads + V / 4 + e / 4) * turned + i / V) * 4 + e % 4] = (float)s;
          if (r + 1 < lastr) {
            const double c2 = c * dc - s * ds;
            s = s * dc + c * ds;
            c = c2;
          }
        }
      }
      __syncthreads();
    }
    if (!active) continue;
    for (int rb = lo + r0; rb < hi; rb += kBatch * step) {
      uint4 u1[kBatch], u2[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = rb + i * step;
        if (r < hi) {
          u1[i] = *reinterpret_cast<const uint4*>(in + r * in_step + c1);
          u2[i] = *reinterpret_cast<const uint4*>(in + r * in_step + c2);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = rb + i * step;
        if (r >= hi) break;
        if (rotated) {
          float4 cs[kQuads];
#pragma unroll
          for (int q = 0; q < kQuads; ++q)
            cs[q] = reinterpret_cast<const float4*>(trig)[((r - lo) * kQuads + q) * turned + item];
          turn<T, kMixed>(u1[i], u2[i], reinterpret_cast<const float*>(cs),
                          reinterpret_cast<const float*>(cs + kQuads / 2));
        }
        const int64_t off = is_q ? r * a.o_stride[0] : at[r];
        if (!is_q && off < 0) continue;  // its page is not there: it is not held, and in no mean
        if (sum) add_pair<T>(acc, u1[i], u2[i]);
        *reinterpret_cast<uint4*>(out + off + c1) = u1[i];
        *reinterpret_cast<uint4*>(out + off + c2) = u2[i];
      }
    }
  }
  if (sum && h < heads) {
    for (int o = items; o < 32; o <<= 1) {  // the other lanes' rows, into those with r0 = 0
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) {
        const float x = __shfl_down_sync(0xffffffffu, acc[i], o);
        if (lane + o < 32) acc[i] += x;
      }
    }
    if (r0 == 0) {
      // (1 / 64 is exact: the same bits as a division)
      const float inv = is_q && (options & TASFT_ROPE_MEAN_NEW) ? 1.f / (r_hi - r_lo) : 1.f / kRopeBlk;
      float* dst = is_q ? a.pooled_q + (((int64_t)b * a.Hq + hh) * a.NBq + qi) * a.D
                        : a.pooled_k + (((int64_t)b * a.Hk + hh) * a.NBk + blk) * a.D;
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        *reinterpret_cast<float4*>(dst + c1 + i) =
            make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
        *reinterpret_cast<float4*>(dst + c2 + i) =
            make_float4(acc[V + i] * inv, acc[V + i + 1] * inv, acc[V + i + 2] * inv, acc[V + i + 3] * inv);
      }
    }
  }
}

template <typename T, bool kMixed>
int run(const tasft_rope_append_args& a, int options, cudaStream_t st) {
  auto kern = rope_append_kernel<T, kMixed>;
  const int smem = kRopeRows * a.rot * (int)sizeof(float);  // cos and sin, rot / 2 each
  constexpr int kPlaces = 2 * kRopeBlk * (int)sizeof(int64_t);  // static, and counted against the limit too
  static std::atomic<uint64_t> allowed{0};
  if (smem + kPlaces > 48 * 1024 && !allow_smem(kern, kRopeRows * 256 * (int)sizeof(float), allowed)) return TASFT_ERR_CUDA;
  const int z = (a.Hq + 2 * a.Hk + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
  if (a.B > 65535) return TASFT_ERR_TOO_LARGE;
  kern<<<dim3((unsigned)z, (unsigned)a.NBq, (unsigned)a.B), kRopeThreads, smem, st>>>(a, options);
  count_launch();
  return launch_status();
}

bool rows_ok(const void* p, const int64_t* st, int n, int per16) {
  if (!aligned16(p)) return false;
  for (int i = 0; i < n; ++i)
    if (st[i] % per16 || st[i] < 0) return false;
  return true;
}

}  // namespace
}  // namespace tasft

using namespace tasft;

extern "C" int tasft_rope_append_paged(const tasft_rope_append_args* ap, tasft_stream_t stream) {
  return tasft_rope_append_paged_opt(ap, 0, stream);
}

extern "C" int tasft_rope_append_paged_opt(const tasft_rope_append_args* ap, int32_t options, tasft_stream_t stream) {
  if (!ap || (options & ~(TASFT_ROPE_MEAN_NEW | TASFT_ZERO_REST))) return TASFT_ERR_INVALID_ARG;
  tasft_rope_append_args a = *ap;
  // strides of axes of length one say nothing
  if (a.T <= 1) a.q_stride[0] = a.k_in_stride[0] = a.v_in_stride[0] = a.o_stride[0] = 0;
  if (a.Hq == 1) a.q_stride[1] = a.o_stride[1] = 0;
  if (a.Hk == 1) a.k_in_stride[1] = a.v_in_stride[1] = a.k_stride[2] = a.v_stride[2] = 0;
  if (a.num_pages == 1) a.k_stride[0] = a.v_stride[0] = 0;
  if (a.page_size == 1) a.k_stride[1] = a.v_stride[1] = 0;
  if (a.B <= 0 || a.T < 0 || a.Hq <= 0 || a.Hk <= 0 || a.Hq % a.Hk || a.D <= 0 || a.max_q <= 0 || a.max_pages <= 0 ||
      a.num_pages <= 0 || a.page_size <= 0)
    return TASFT_ERR_INVALID_ARG;
  if (!a.cu_seqlens || !a.kv_len || !a.block_table || !a.k_pages || !a.v_pages) return TASFT_ERR_INVALID_ARG;
  if (a.NBq < ((int64_t)a.max_q + 126) / 64 || a.NBq > 65535) return TASFT_ERR_INVALID_ARG;
  if (a.pooled_k && a.NBk <= 0) return TASFT_ERR_INVALID_ARG;
  if (a.rot < 0 || a.rot > a.D || (a.rot > 0 && !a.inv_freq)) return TASFT_ERR_INVALID_ARG;
  if (a.k_stride[3] != 1 || a.v_stride[3] != 1) return TASFT_ERR_INVALID_ARG;
  if ((int64_t)a.max_pages * a.page_size > INT32_MAX) return TASFT_ERR_TOO_LARGE;
  if (a.block != kRopeBlk) return TASFT_ERR_UNSUPPORTED;
  if (a.dtype != TASFT_F32 && a.dtype != TASFT_BF16 && a.dtype != TASFT_F16) return TASFT_ERR_UNSUPPORTED;
  const int per16 = 16 / elem_size(a.dtype);
  // 16-byte column pairs: whole heads and the rotated part are multiples of two of them
  if (a.D % (2 * per16) || a.rot % (2 * per16) || a.D > 256) return TASFT_ERR_UNSUPPORTED;
  if (a.T == 0 && !a.pooled_q) return TASFT_OK;
  if (a.T > 0 && (!a.q || !a.k || !a.v || !a.q_out)) return TASFT_ERR_INVALID_ARG;
  if (!aligned16(a.pooled_q) || !aligned16(a.pooled_k)) return TASFT_ERR_UNSUPPORTED;
  if (!rows_ok(a.q, a.q_stride, 2, per16) || !rows_ok(a.k, a.k_in_stride, 2, per16) ||
      !rows_ok(a.v, a.v_in_stride, 2, per16) || !rows_ok(a.q_out, a.o_stride, 2, per16) ||
      !rows_ok(a.k_pages, a.k_stride, 3, per16) || !rows_ok(a.v_pages, a.v_stride, 3, per16))
    return TASFT_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool mixed = a.interleaved != 0;
  if (a.dtype == TASFT_F32) return mixed ? run<float, true>(a, options, st) : run<float, false>(a, options, st);
  if (a.dtype == TASFT_F16) return mixed ? run<__half, true>(a, options, st) : run<__half, false>(a, options, st);
  return mixed ? run<__nv_bfloat16, true>(a, options, st) : run<__nv_bfloat16, false>(a, options, st);
}
