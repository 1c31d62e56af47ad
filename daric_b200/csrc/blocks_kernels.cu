// Block selection for sparse attention over the paged KV cache.
//
// page_bounds: mn[d], mx[d] = smallest and largest key value of dimension d
// over the tokens of a page, per KV head. Bound: the K bytes read (16 prompts
// of 2047 to 8192 tokens: 36 us, 5.0 TB/s of K and bounds). One warp
// per (page, head): a row of a key is D / 8 lanes of 16 bytes, the page's
// rows are loaded before any is reduced, and the two-lane minimum and maximum
// instructions of the 16-bit types (NaN propagates) keep it at a few
// instructions per 16 bytes.
//
// select_pages: for query row n, KV head h and page g
//   u = max over the heads of h's group of  sum_d max(q_d mn_d, q_d mx_d),
// an upper bound of q . k over the page's keys. For finite bounds this is a
// matrix product of (max(q, 0), min(q, 0)) with the stored (mx, mn) rows (where
// some are infinite or NaN all pages are scored in 64 bits, as below), so the bounds go from
// global memory straight into matrix fragments (16 bytes a thread; the order
// of the summed dimension is the same for both operands, so any order is
// right) and no shared memory, unpacking or shuffle stands beside the loads.
// Bound: the bytes of the bounds (8 rows over 8192 pages each, 8 KV heads: 49
// us, 4.8 TB/s), then the selection's barriers (12 to 17 us).
//
// The k pages of highest u are those of sums in 64 bits, ties to the lower page:
// |fp32 result - exact| <= E = 2^-14 * max over pages of
// sum |q_d| |bound_d| (256 * 2 products of one sum, each addition off by at
// most 2^-23 of the largest partial sum; the products are exact in fp32). A page whose
// fp32 score is over 2E above the k-th is in, one 2E below it is out, and the
// few between are scored again in 64 bits (products of 16-bit values are
// exact there).
#include "attend_common.cuh"

#include <algorithm>

namespace daric {
namespace {
using namespace att;

// ------------------------------------------------------------- bounds --
template <class T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static __device__ __forceinline__ uint32_t mn(uint32_t a, uint32_t b) {
    V r = __hmin2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t mx(uint32_t a, uint32_t b) {
    V r = __hmax2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static constexpr uint32_t kPosInf = 0x7f807f80u, kNegInf = 0xff80ff80u;
};
template <>
struct Pair<__half> {
  using V = __half2;
  static __device__ __forceinline__ uint32_t mn(uint32_t a, uint32_t b) {
    V r = __hmin2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t mx(uint32_t a, uint32_t b) {
    V r = __hmax2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static constexpr uint32_t kPosInf = 0x7c007c00u, kNegInf = 0xfc00fc00u;
};

constexpr int kBoundWarps = 8;

template <class T, int D>
__global__ void __launch_bounds__(kBoundWarps * 32) bounds_kernel(const __grid_constant__ BoundsLaunch p) {
  constexpr int CH = D / 8;
  constexpr int TPI = 32 / CH;  // tokens a warp reads at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y, H = p.kv.heads, bs = p.kv.page_size;
  Seq s;
  s.rows = 0;
  s.len = __ldg(&p.sq.seq_lens[b]);
  clamp_len(p.sq, bs, s);
  const int start = p.start ? max(__ldg(&p.start[b]), 0) : 0;
  const int p0 = (int)fdiv((uint32_t)start, p.kv.page_div);
  const int pages = start < s.len ? (s.len + bs - 1) / bs - p0 : 0;
  const int c = lane % CH, t0 = lane / CH;
  const int32_t* trow = p.sq.table + (int64_t)b * p.sq.table_ld + p0;
  const int64_t items = (int64_t)pages * H, stride = (int64_t)gridDim.x * kBoundWarps;
  int nxt = 0;
  if ((int64_t)blockIdx.x * kBoundWarps + warp < items)
    nxt = ld_ahead(&trow[((int64_t)blockIdx.x * kBoundWarps + warp) / H]);
  for (int64_t w = (int64_t)blockIdx.x * kBoundWarps + warp; w < items; w += stride) {
    const int pg = p0 + (int)(w / H), h = (int)(w % H);
    const int blk = nxt;
    if (w + stride < items) nxt = ld_ahead(&trow[(w + stride) / H]);
    if (blk < 0 || blk >= p.kv.num_pages) {
      if (lane == 0) atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
      continue;
    }
    const uint8_t* src = p.kv.base + (int64_t)blk * p.kv.page_stride + (int64_t)h * p.kv.head_stride + c * 16;
    const int n = min(bs, s.len - pg * bs);
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = Pair<T>::kPosInf;
      hi[e] = Pair<T>::kNegInf;
    }
    for (int t = t0; t < n; t += 8 * TPI) {
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {  // a token past the end repeats one that is in
        const int tt = t + u * TPI < n ? t + u * TPI : t;
        v[u] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)tt * p.kv.tok_stride));
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(&v[u]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = Pair<T>::mn(lo[e], x[e]);
          hi[e] = Pair<T>::mx(hi[e], x[e]);
        }
      }
    }
#pragma unroll
    for (int o = CH; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = Pair<T>::mn(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
        hi[e] = Pair<T>::mx(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
      }
    if (lane < CH) {
      uint4* dst = reinterpret_cast<uint4*>(p.bounds + ((int64_t)blk * H + h) * (4 * D)) + lane;
      dst[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      dst[CH] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    }
  }
}

// ------------------------------------------------------------- scores --
// Order-preserving key of a score; every NaN is the largest key.
__device__ __forceinline__ uint32_t key_of(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  if (k == 0xffffffffu) return __int_as_float(0x7fffffff);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long key64_of(double f) {
  if (f != f) return ~0ull;
  if (f == 0.0) f = 0.0;  // -0 and 0 are one value
  const unsigned long long u = (unsigned long long)__double_as_longlong(f);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}

// Query row n against its sequence: pages it can see (0: no sequence).
struct RowView {
  int seq, pages;
};
__device__ __forceinline__ RowView row_view(const SeqBatch& sq, int page_size, int n) {
  RowView v{find_seq(sq, n), 0};
  if (v.seq < 0) return v;
  Seq s = load_seq(sq, v.seq);
  clamp_len(sq, page_size, s);
  if (n - s.row0 >= s.rows) return RowView{-1, 0};  // behind its last row, or its offsets are bad
  const int pos = s.ctx + (n - s.row0);
  v.pages = pos < 0 || pos >= s.len ? 0 : pos / page_size + 1;
  return v;
}

// The part of q that meets the stored minima (sign bit set) or maxima.
__device__ __forceinline__ uint32_t q_part(uint32_t w, bool maxima) {
  const uint32_t lo = w & 0xffffu, hi = w >> 16;
  const uint32_t a = ((lo >> 15) != 0) != maxima ? lo : 0u, b = ((hi >> 15) != 0) != maxima ? hi : 0u;
  return a | (b << 16);
}

constexpr int kScoreWarps = 4;
constexpr int kScoreStages = 3;

// N pieces of 16 bytes, 64 bytes apart, to slots STEP bytes apart.
template <int N, int STEP, int I = 0>
__device__ __forceinline__ void copy_row(uint32_t dst, const uint8_t* src, int n) {
  if constexpr (I < N) {
    cp16_at<I * STEP, I * 64>(dst, src, n);
    copy_row<N, STEP, I + 1>(dst, src, n);
  }
}

// A warp scores 16 pages at a time, the minima and then the maxima, each a
// stage of its threads' own ring slots (a thread copies the fragment pieces
// that it multiplies). Four CTAs of four warps an SM keep the loads going.
template <class T, int D>
__global__ void __launch_bounds__(kScoreWarps * 32, D > 128 ? 2 : 4) page_score_kernel(const __grid_constant__ SelectPagesLaunch p) {
  constexpr int KB = D / 32;  // 64-byte pieces of the minima (or maxima) of a page
  constexpr int TH = kScoreWarps * 32, S = kScoreStages;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_mag[kScoreWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = blockIdx.x, h = blockIdx.z, chunk = blockIdx.y;
  const int g = lane >> 2, t = lane & 3;
  grid_next();
  const RowView rv = row_view(p.sq, p.page_size, n);
  if (rv.pages <= p.k || chunk * p.chunk >= rv.pages) return;  // every page is taken, or none is here
  const int group = p.sq.group;
  const int32_t* trow = p.sq.table + (int64_t)rv.seq * p.sq.table_ld;
  uint32_t* keys = p.keys + ((int64_t)n * p.heads + h) * p.keys_row;
  const int first = chunk * p.chunk + warp * 16;
  const int tiles = first >= rv.pages ? 0
                                      : min(p.chunk / (kScoreWarps * 16),
                                            (rv.pages - first + kScoreWarps * 16 - 1) / (kScoreWarps * 16));
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;  // [stage][row][piece][thread]
  int blk[2];  // pages g and g + 8 of the tile that is copied next
  auto lookup = [&](int it) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int pg = first + it * kScoreWarps * 16 + g + 8 * r;
      blk[r] = it < tiles && pg < rv.pages ? ld_ahead(&trow[pg]) : -1;
    }
  };
  const uint8_t* src[2];
  bool in[2];
  auto issue = [&](int half, int st) {  // half 2 it: minima of tile it, half 2 it + 1: its maxima
    if (half < 2 * tiles) {
      if (!(half & 1)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          in[r] = blk[r] >= 0 && blk[r] < p.num_pages;
          if (!in[r] && first + (half >> 1) * kScoreWarps * 16 + g + 8 * r < rv.pages) atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
          src[r] = p.bounds + ((int64_t)(in[r] ? blk[r] : 0) * p.heads + h) * (4 * D) + t * 16;
        }
        lookup((half >> 1) + 1);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
        copy_row<KB, TH * 16>(smem_u32(ring + (st * 2 + r) * KB * TH), src[r] + (half & 1) * 2 * D, in[r] ? 16 : 0);
    }
    cp_commit();
  };
  lookup(0);
#pragma unroll
  for (int k = 0; k < S - 1; ++k) issue(k, k);
  // the parts of the first eight query heads that meet minima and maxima
  uint4 w[2][KB];
  auto query = [&](int q0) {
    const bool real = q0 + g < group;
    const uint4* qp = reinterpret_cast<const uint4*>(
        p.q + (int64_t)n * p.q_row + (int64_t)(h * group + (real ? q0 + g : 0)) * p.q_head) + t;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const uint4 v = real ? __ldg(qp + 4 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < 2; ++m) w[m][k] = make_uint4(q_part(v.x, m), q_part(v.y, m), q_part(v.z, m), q_part(v.w, m));
    }
  };
  query(0);
  float mag = 0.f;
  int st = 0;
  for (int it = 0; it < tiles; ++it) {
    uint32_t best[2] = {0u, 0u};
    // heads eight at a time; all of a page's bytes stay in the ring meanwhile
    // only for the first eight, so more heads read them again from global
    for (int q0 = 0; q0 < group; q0 += 8) {
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
      if (group > 8) query(q0);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (q0 == 0) {
          issue(2 * it + m + S - 1, st == 0 ? S - 1 : st - 1);
          cp_wait<S - 1>();
        }
        const uint4* a = ring + st * 2 * KB * TH;
        const uint8_t* again[2] = {nullptr, nullptr};
        if (q0 > 0) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int pg = first + it * kScoreWarps * 16 + g + 8 * r;
            const int bk = pg < rv.pages ? __ldg(&trow[pg]) : -1;
            if (bk >= 0 && bk < p.num_pages)
              again[r] = p.bounds + ((int64_t)bk * p.heads + h) * (4 * D) + m * 2 * D + t * 16;
          }
        }
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          uint4 u, v;
          if (q0 == 0) {
            u = a[k * TH];
            v = a[(KB + k) * TH];
          } else {
            u = again[0] ? __ldg(reinterpret_cast<const uint4*>(again[0] + k * 64)) : make_uint4(0, 0, 0, 0);
            v = again[1] ? __ldg(reinterpret_cast<const uint4*>(again[1] + k * 64)) : make_uint4(0, 0, 0, 0);
          }
          const uint4 z = w[m][k];
          constexpr uint32_t M = 0x7fff7fffu;
          { uint32_t f[4] = {u.x, v.x, u.y, v.y}; Mma<T>::run(x, f, z.x, z.y); }
          { uint32_t f[4] = {u.z, v.z, u.w, v.w}; Mma<T>::run(x, f, z.z, z.w); }
          { uint32_t f[4] = {u.x & M, v.x & M, u.y & M, v.y & M}; Mma<T>::run(y, f, z.x & M, z.y & M); }
          { uint32_t f[4] = {u.z & M, v.z & M, u.w & M, v.w & M}; Mma<T>::run(y, f, z.z & M, z.w & M); }
        }
        if (q0 == 0) st = st + 1 == S ? 0 : st + 1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (q0 + 2 * t + (e & 1) < group) {
          best[e >> 1] = max(best[e >> 1], key_of(x[e]));
          // a NaN or infinite magnitude stays the largest
          mag = (y[e] <= mag) ? mag : (y[e] == y[e] ? y[e] : __int_as_float(0x7f800000));
        }
    }
    if (group > 8) query(0);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      best[r] = max(best[r], __shfl_xor_sync(0xffffffffu, best[r], 1));
      best[r] = max(best[r], __shfl_xor_sync(0xffffffffu, best[r], 2));
      const int pg = first + it * kScoreWarps * 16 + g + 8 * r;
      if (t == 0 && pg < rv.pages) keys[pg] = best[r];
    }
  }
  cp_wait<0>();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, o));
  if (lane == 0) s_mag[warp] = mag;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kScoreWarps; ++i) mag = fmaxf(mag, s_mag[i]);
    p.mags[((int64_t)n * p.heads + h) * gridDim.y + chunk] = mag;
  }
}

// ------------------------------------------------------------- select --
constexpr int kBins = 2048;
constexpr int kNear = 256;  // candidates ranked against each other at once

// Block-wide exclusive prefix sum; *total gets the sum. All threads call it.
__device__ __forceinline__ int block_prefix(int v, int* total, int* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < nw ? sm[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    if (lane < nw) sm[lane] = w;
  }
  __syncthreads();
  *total = sm[nw - 1];
  return x - v + (warp > 0 ? sm[warp - 1] : 0);
}

// Digit of the rem-th largest entry of hist[0, bins), and the entries above it.
__device__ __forceinline__ void find_digit(const uint32_t* hist, int bins, int rem, int* s_digit, int* s_above, int* sm) {
  const int per = (bins + blockDim.x - 1) / blockDim.x;
  int mine = 0;
  for (int i = 0; i < per; ++i) {  // thread 0 owns the highest digits
    const int d = bins - 1 - ((int)threadIdx.x * per + i);
    if (d >= 0) mine += (int)hist[d];
  }
  int total;
  int above = block_prefix(mine, &total, sm);
  if (above < rem && rem <= above + mine) {
    for (int i = 0; i < per; ++i) {
      const int d = bins - 1 - ((int)threadIdx.x * per + i);
      if (d < 0) break;
      if (above < rem && rem <= above + (int)hist[d]) {
        *s_digit = d;
        *s_above = above;
      }
      above += (int)hist[d];
    }
  }
  __syncthreads();
}

// Score of a page in 64 bits (all lanes of a warp call it with one page):
// four heads at a time, so that their sums go side by side.
template <class T, int D>
__device__ __forceinline__ unsigned long long exact_key(const SelectPagesLaunch& p, int n, int h, int blk) {
  const int lane = threadIdx.x & 31, group = p.sq.group;
  const uint16_t* bd = reinterpret_cast<const uint16_t*>(p.bounds + ((int64_t)max(blk, 0) * p.heads + h) * (4 * D));
  uint16_t lo[D / 32], hi[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    lo[k] = blk >= 0 ? __ldg(&bd[lane + 32 * k]) : 0;
    hi[k] = blk >= 0 ? __ldg(&bd[D + lane + 32 * k]) : 0;
  }
  unsigned long long best = 0;
  for (int e0 = 0; e0 < group; e0 += 4) {
    uint16_t qw[4][D / 32];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
        qw[e][k] = e0 + e < group ? __ldg(reinterpret_cast<const uint16_t*>(p.q + (int64_t)n * p.q_row +
                                                                             (int64_t)(h * group + e0 + e) * p.q_head) +
                                          lane + 32 * k)
                                  : 0;
    double u[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      const double l = (double)Mma<T>::widen(lo[k]), m = (double)Mma<T>::widen(hi[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double qv = (double)Mma<T>::widen(qw[e][k]);
        // max(q mn, q mx), NaN where either is: an infinite bound that the
        // sign of q does not meet says nothing
        const double a = qv * l, b = qv * m;
        u[e] += a != a || b != b ? a + b : fmax(a, b);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] += __shfl_xor_sync(0xffffffffu, u[e], o);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e0 + e < group) {
        const unsigned long long k = key64_of(u[e]);
        best = k > best ? k : best;
      }
  }
  return best;
}

template <class T, int D>
__global__ void __launch_bounds__(1024) page_select_kernel(const __grid_constant__ SelectPagesLaunch p) {
  extern __shared__ uint32_t dyn[];  // [bitmap words | staged keys]
  __shared__ uint32_t hist[kBins];
  __shared__ int sm[32];
  __shared__ int s_digit, s_above, s_near, s_in, s_count;
  __shared__ uint32_t s_kth;
  __shared__ float s_e, s_lo[32], s_hi[32];
  __shared__ int near_page[kNear];
  __shared__ unsigned long long near_key[kNear];
  const int n = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  grid_wait();
  const RowView rv = row_view(p.sq, p.page_size, n);
  if (rv.seq < 0) return;  // a row behind the last sequence
  int32_t* out = p.out + ((int64_t)n * p.heads + h) * p.k;
  const int P = rv.pages;
  if (P <= p.k) {
    for (int i = tid; i < p.k; i += blockDim.x) out[i] = i < P ? i : -1;
    return;
  }
  const int64_t item = (int64_t)n * p.heads + h;
  const uint32_t* gkeys = p.keys + item * p.keys_row;
  const int words = (P + 31) / 32;
  uint32_t* taken = dyn;
  uint32_t* skeys = dyn + ((p.sq.table_cols + 31) / 32 + 3) / 4 * 4;
  const int32_t* trow = p.sq.table + (int64_t)rv.seq * p.sq.table_ld;
  // eligible pages [e0, e1); the ones before and after are always taken
  const int e0 = p.first, e1 = P - p.last;
  const int kk = p.k - p.first - p.last;
  if (tid == 0) s_near = s_in = 0;
  float mag = 0.f;
  for (int i = tid; i < (P + p.chunk - 1) / p.chunk; i += blockDim.x) mag = fmaxf(mag, p.mags[item * p.chunks + i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, o));
  if (lane == 0) sm[warp] = __float_as_int(mag);
  if (p.staged)  // rows of keys are whole 16-byte vectors
    for (int i = tid; i < (P + 3) / 4; i += blockDim.x)
      reinterpret_cast<uint4*>(skeys)[i] = __ldcg(reinterpret_cast<const uint4*>(gkeys) + i);
  for (int i = tid; i < words; i += blockDim.x) taken[i] = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < nw; ++w) mag = fmaxf(mag, __int_as_float(sm[w]));
    s_e = mag * 6.103515625e-05f;  // E = 2^-14 of the largest magnitude
  }
  __syncthreads();
  auto key_at = [&](int i) { return p.staged ? skeys[i] : gkeys[i]; };
  const float E = s_e;

  if (kk > 0) {
    uint32_t prefix = 0, mask = 0;
    int rem = kk;
    // The k-th largest fp32 key. Scores of one row lie close together (their
    // leading bits are the same), so they are first spread over bins of equal
    // width between the smallest and the largest; the keys of the bin that
    // holds the k-th are few and are ranked against each other.
    bool found = false;
    if (E < 1e38f) {  // all scores are finite then
      float lo = __int_as_float(0x7f800000), hi = DARIC_NEG_INF;
      for (int i = e0 + tid; i < e1; i += blockDim.x) {
        const float v = value_of(key_at(i));
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      for (int i = tid; i < kBins; i += blockDim.x) hist[i] = 0;
      if (lane == 0) {
        s_lo[warp] = lo;
        s_hi[warp] = hi;
      }
      if (tid == 0) s_count = 0;
      __syncthreads();
      for (int w = 0; w < nw; ++w) {
        lo = fminf(lo, s_lo[w]);
        hi = fmaxf(hi, s_hi[w]);
      }
      // monotone in v: each step of it is
      const float scale = (float)(kBins - 1) / fmaxf(hi - lo, 1e-30f);
      auto bin_of = [&](float v) { return min(max((int)((v - lo) * scale), 0), kBins - 1); };
      for (int i = e0 + tid; i < e1; i += blockDim.x) atomicAdd(&hist[bin_of(value_of(key_at(i)))], 1u);
      __syncthreads();
      find_digit(hist, kBins, rem, &s_digit, &s_above, sm);
      const int bin = s_digit, left = rem - s_above;
      const uint32_t in_bin = hist[bin];
      // every thread has read the bin's count before the digits below clear
      // the histogram: the threads take one way together
      __syncthreads();
      if (in_bin <= (uint32_t)kNear) {
        for (int i = e0 + tid; i < e1; i += blockDim.x) {
          const uint32_t k = key_at(i);
          if (bin_of(value_of(k)) != bin) continue;
          const int at = atomicAdd(&s_count, 1);
          if (at < kNear) near_key[at] = k;
        }
        __syncthreads();
        const int n = min(s_count, kNear);
        for (int i = tid; i < n; i += blockDim.x) {  // ties do not matter: one value is wanted
          int above = 0, same = 0;
          for (int j = 0; j < n; ++j) {
            above += near_key[j] > near_key[i];
            same += near_key[j] == near_key[i];
          }
          if (above < left && left <= above + same) s_kth = (uint32_t)near_key[i];
        }
        __syncthreads();
        prefix = s_kth;
        found = true;
      }
    }
    // otherwise digits of 11, 11 and 10 bits
    for (int pass = 0; pass < 3 && !found; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < kBins; i += blockDim.x) hist[i] = 0;
      __syncthreads();
      for (int i = e0 + tid; i < e1; i += blockDim.x) {
        const uint32_t k = key_at(i);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (uint32_t)(bins - 1)], 1u);
      }
      __syncthreads();
      find_digit(hist, bins, rem, &s_digit, &s_above, sm);
      prefix |= (uint32_t)s_digit << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      rem -= s_above;
      __syncthreads();
    }
    // pages certainly in, and those whose order against the k-th fp32 cannot tell
    const float t = value_of(prefix);
    const bool wide = !(E < 1e38f) || !(fabsf(t) < 1e38f);  // infinities or NaN about: settle all in 64 bits
    const float hi = t + 2.f * E, lo = t - 2.f * E;
    for (int i0 = 0; i0 < words * 32; i0 += blockDim.x) {  // a warp: one word of the bitmap
      const int i = i0 + tid;
      bool sure = false, maybe = false;
      if (i >= e0 && i < e1) {
        const float v = value_of(key_at(i));
        sure = !wide && v > hi;
        maybe = wide || (v >= lo && v <= hi);
      }
      const unsigned m = __ballot_sync(0xffffffffu, sure);
      if (lane == 0 && i < words * 32) {
        taken[i >> 5] = m;
        if (m) atomicAdd(&s_in, __popc(m));
      }
      if (maybe) {
        const int at = atomicAdd(&s_near, 1);
        if (at < kNear) near_page[at] = i;
      }
    }
    __syncthreads();
    const int n_in = s_in, n_near = s_near;
    const int need = kk - n_in;  // of the candidates
    if (n_near <= need) {
      for (int i = tid; i < n_near && i < kNear; i += blockDim.x) atomicOr(&taken[near_page[i] >> 5], 1u << (near_page[i] & 31));
      if (n_near > kNear)
        for (int i = e0 + tid; i < e1; i += blockDim.x) {
          const float v = value_of(key_at(i));
          if (wide || (v >= lo && v <= hi)) atomicOr(&taken[i >> 5], 1u << (i & 31));
        }
    } else if (n_near <= kNear) {
      for (int i = warp; i < n_near; i += nw) {
        const int blk = __ldg(&trow[near_page[i]]);
        const unsigned long long k = exact_key<T, D>(p, n, h, blk >= 0 && blk < p.num_pages ? blk : -1);
        if (lane == 0) near_key[i] = k;
      }
      __syncthreads();
      for (int i = tid; i < n_near; i += blockDim.x) {
        int better = 0;
        for (int j = 0; j < n_near; ++j)
          better += near_key[j] > near_key[i] || (near_key[j] == near_key[i] && near_page[j] < near_page[i]);
        if (better < need) atomicOr(&taken[near_page[i] >> 5], 1u << (near_page[i] & 31));
      }
    } else {
      // many candidates (pages alike, or an infinite or NaN bound, which makes
      // all pages candidates): radix selection over their 64-bit keys, scored
      // anew in every pass so that nothing has to be stored. Nine passes of
      // 8192 pages, 4 query heads of 128: 8.8 ms where the usual way takes 27 us.
      unsigned long long pre = 0, msk = 0;
      int left = need;
      for (int pass = 0; pass < 8; ++pass) {
        const int shift = 56 - 8 * pass;
        for (int i = tid; i < 256; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        for (int i = e0 + warp; i < e1; i += nw) {
          const float v = value_of(key_at(i));
          if (!(wide || (v >= lo && v <= hi))) continue;
          const int blk = __ldg(&trow[i]);
          const unsigned long long k = exact_key<T, D>(p, n, h, blk >= 0 && blk < p.num_pages ? blk : -1);
          if (lane == 0 && (k & msk) == pre) atomicAdd(&hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        find_digit(hist, 256, left, &s_digit, &s_above, sm);
        pre |= (unsigned long long)s_digit << shift;
        msk |= 255ull << shift;
        left -= s_above;
        __syncthreads();
      }
      // keys above the k-th are in; of the equal ones the `left` lowest pages:
      // their places are found in page order by one warp per 32 pages
      uint32_t* equal = hist;  // bitmap of a span of pages
      for (int s0 = e0; s0 < e1; s0 += kBins * 32) {
        const int s1 = min(e1, s0 + kBins * 32);
        for (int i = tid; i < kBins; i += blockDim.x) equal[i] = 0;
        __syncthreads();
        for (int i = s0 + warp; i < s1; i += nw) {
          const float v = value_of(key_at(i));
          if (!(wide || (v >= lo && v <= hi))) continue;
          const int blk = __ldg(&trow[i]);
          const unsigned long long k = exact_key<T, D>(p, n, h, blk >= 0 && blk < p.num_pages ? blk : -1);
          if (lane == 0) {
            if (k > pre) atomicOr(&taken[i >> 5], 1u << (i & 31));
            if (k == pre) atomicOr(&equal[(i - s0) >> 5], 1u << ((i - s0) & 31));
          }
        }
        __syncthreads();
        if (tid == 0) {
          for (int w = 0; w < kBins && left > 0; ++w)
            for (uint32_t m = equal[w]; m && left > 0; m &= m - 1, --left) {
              const int i = s0 + w * 32 + (__ffs((int)m) - 1);
              atomicOr(&taken[i >> 5], 1u << (i & 31));
            }
          s_near = left;
        }
        __syncthreads();
        left = s_near;
        __syncthreads();
      }
    }
  }
  __syncthreads();
  // the pages that are always taken, then the list in ascending order
  for (int i = tid; i < p.first + p.last; i += blockDim.x) {
    const int pg = i < p.first ? i : P - p.last + (i - p.first);
    atomicOr(&taken[pg >> 5], 1u << (pg & 31));
  }
  __syncthreads();
  const int per = (words + blockDim.x - 1) / blockDim.x;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w < words) mine += __popc(taken[w]);
  }
  int total;
  int at = block_prefix(mine, &total, sm);
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w >= words) break;
    for (uint32_t m = taken[w]; m; m &= m - 1) {
      if (at < p.k) out[at] = w * 32 + (__ffs((int)m) - 1);
      ++at;
    }
  }
  for (int i = total + tid; i < p.k; i += blockDim.x) out[i] = -1;
}

template <class T, int D>
void bounds_d(const BoundsLaunch& p, int sm_count, cudaStream_t s) {
  const int64_t items = (int64_t)p.sq.table_cols * p.kv.heads;
  int64_t x = (items + kBoundWarps - 1) / kBoundWarps;
  // about sixteen CTAs per SM over all sequences; the warps stride over the rest
  x = std::min<int64_t>(x, std::max<int64_t>(1, (int64_t)sm_count * 16 / p.sq.num_seqs));
  bounds_kernel<T, D><<<dim3((unsigned)x, (unsigned)p.sq.num_seqs), kBoundWarps * 32, 0, s>>>(p);
  DARIC_CUDA(cudaGetLastError());
}

template <class T, int D>
void select_d(const SelectPagesLaunch& p0, cudaStream_t s) {
  SelectPagesLaunch p = p0;
  // pages of a CTA: 512, fewer while that leaves less than four CTAs an SM
  p.chunk = 512;
  while (p.chunk > kScoreChunk &&
         (int64_t)(p.sq.table_cols + p.chunk - 1) / p.chunk * p.sq.num_rows * p.heads < 4 * (int64_t)p.sm_count)
    p.chunk /= 2;
  p.chunks = (p.sq.table_cols + p.chunk - 1) / p.chunk;
  if (p.sq.table_cols > p.k) {
    constexpr int bytes = kScoreStages * 2 * (D / 32) * kScoreWarps * 32 * 16;
    static std::atomic<uint64_t> ready{0};
    allow_smem(page_score_kernel<T, D>, bytes, ready);
    page_score_kernel<T, D>
        <<<dim3((unsigned)p.sq.num_rows, (unsigned)p.chunks, (unsigned)p.heads), kScoreWarps * 32, bytes, s>>>(p);
    DARIC_CUDA(cudaGetLastError());
  }
  // keys are staged in shared memory while they fit
  const int words = ((p.sq.table_cols + 31) / 32 + 3) / 4 * 4;
  p.staged = p.sq.table_cols <= 40960;
  const int bytes = (words + (p.staged ? p.keys_row : 0)) * 4;
  // a thread per eight keys, so that short tables keep many CTAs on an SM
  const int threads = std::min(1024, std::max(128, (p.sq.table_cols / 8 + 31) / 32 * 32));
  static std::atomic<uint64_t> done{0};
  allow_smem(page_select_kernel<T, D>, 190 * 1024, done);
  launch_after(page_select_kernel<T, D>, dim3((unsigned)p.sq.num_rows, (unsigned)p.heads), threads, s, p, bytes);
}

}  // namespace

#define DARIC_BY_DIM(F, T, ...)                        \
  switch (dim) {                                       \
    case 64: F<T, 64>(__VA_ARGS__); return;            \
    case 128: F<T, 128>(__VA_ARGS__); return;          \
    case 256: F<T, 256>(__VA_ARGS__); return;          \
  }

void launch_page_bounds(const BoundsLaunch& p, int dtype, int sm_count, cudaStream_t s) {
  const int dim = p.kv.head_dim;
  if (dtype == DARIC_DTYPE_BF16) { DARIC_BY_DIM(bounds_d, __nv_bfloat16, p, sm_count, s) }
  if (dtype == DARIC_DTYPE_F16) { DARIC_BY_DIM(bounds_d, __half, p, sm_count, s) }
  throw Error(DARIC_ERR_INVALID, "page_bounds: bfloat16 or float16 keys of 64, 128 or 256");
}

void launch_select_pages(const SelectPagesLaunch& p, int dtype, cudaStream_t s) {
  const int dim = p.head_dim;
  if (dtype == DARIC_DTYPE_BF16) { DARIC_BY_DIM(select_d, __nv_bfloat16, p, s) }
  if (dtype == DARIC_DTYPE_F16) { DARIC_BY_DIM(select_d, __half, p, s) }
  throw Error(DARIC_ERR_INVALID, "select_pages: bfloat16 or float16 keys of 64, 128 or 256");
}

}  // namespace daric
