// Attention weight that each cached token receives, for eviction:
// scores[h, p] (+)= sum over the sequence's query rows j and the heads e of
// h's group of  exp(scale q_je . k_p - lse_je)  where j sees p.
//
// Keys are the rows of the matrix fragments and query rows their columns, so a
// key's sum stays in the four threads that hold its row: no atomics, one fixed
// order of additions. Both operands take the head dimension in the same
// permuted order (16 bytes of a row per thread and step), which leaves the
// products alone and lets a thread hold exactly the bytes it loads: nothing is
// shared between threads, no ldmatrix, no barrier.
//
// The heads of a token lie together in the cache, so the CTAs of its heads are
// neighbours in the grid and open its DRAM pages once.
//
// Few rows (16 (row, head) pairs or fewer): weight_stream_kernel. Bound: the K
// bytes (32 sequences up to 32K, 8 KV heads: 213 us, 5.8 TB/s). Every thread copies its own fragment pieces, and the scores it will
// add to, into its own slots of a ring of three stages.
// Many rows: weight_block_kernel. A warp keeps 32 keys in registers and all
// query rows pass by them from shared memory. Bound: the latency of a warp's
// chain at prompt sizes (32 rows x 4 heads over 8192 keys, 8 KV heads: 20 us),
// the matrix and exp2 rates for long ones.
// Without an lse, lse_kernel first runs the same products and keeps the
// maximum and the sum of each query row over the 256 keys of a CTA, and
// lse_join_kernel joins them; K is read twice then (the second time from the
// L2 cache for prompts up to about 100 MB of keys).
#include "attend_common.cuh"

#include <algorithm>

namespace daric {
namespace {
using namespace att;

// Byte offset of a key's row in the layer, -1 where there is none.
__device__ __forceinline__ int64_t key_offset(const ScoresLaunch& p, const Seq& s, int b, int h, int pos) {
  if (pos >= s.len) return -1;
  const int pg = (int)fdiv((uint32_t)pos, p.kv.page_div);
  const int blk = __ldg(&p.sq.table[(int64_t)b * p.sq.table_ld + pg]);
  if (blk < 0 || blk >= p.kv.num_pages) {
    atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
    return -1;
  }
  return (int64_t)blk * p.kv.page_stride + (int64_t)(pos - pg * p.kv.page_size) * p.kv.tok_stride +
         (int64_t)h * p.kv.head_stride;
}

// Products of 16 keys (u: row g, v: row g + 8) and 8 query rows (w) over 32
// elements of the head dimension.
template <class T>
__device__ __forceinline__ void products(float (&x)[4], uint4 u, uint4 v, uint4 w) {
  { uint32_t f[4] = {u.x, v.x, u.y, v.y}; Mma<T>::run(x, f, w.x, w.y); }
  { uint32_t f[4] = {u.z, v.z, u.w, v.w}; Mma<T>::run(x, f, w.z, w.w); }
}

// N pieces of 16 bytes, 64 bytes apart in the row, to slots STEP bytes apart.
template <int N, int STEP, int I>
__device__ __forceinline__ void copy_pieces(uint32_t dst, const uint8_t* src, int n) {
  if constexpr (I < N) {
    cp16_at<I * STEP, I * 64>(dst, src, n);
    copy_pieces<N, STEP, I + 1>(dst, src, n);
  }
}

__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// exp(x * scale - z): weights are at most about 1
__device__ __forceinline__ float weight_of(float x, float scale, float z) {
  return exp2_fast(__fmaf_rn(x, scale, -z) * kLog2e);
}

// ------------------------------------------------------------- stream --
constexpr int kStreamWarps = 4;

template <int D>
struct StreamGeom {
  static constexpr int KB = D / 32;                      // 64-byte pieces of a row
  static constexpr int THREADS = kStreamWarps * 32;
  static constexpr int STAGE = THREADS * (2 * KB * 16 + 8);  // fragment pieces and two old scores
  static constexpr int S = 3;
  static constexpr int SMEM = S * STAGE;
};

// NT: eights of (row, head) pairs. A CTA takes `iters` rounds of 64 keys.
template <class T, int D, int NT>
__global__ void __launch_bounds__(kStreamWarps * 32, D > 128 ? 2 : 4) weight_stream_kernel(const __grid_constant__ ScoresLaunch p, int iters) {
  using G = StreamGeom<D>;
  constexpr int KB = G::KB, S = G::S, TH = G::THREADS;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, h = blockIdx.x, group = p.sq.group;
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, p.kv.page_size, s);
  const int64_t col = __ldg(&p.col_off[b]);
  if (col < 0 || col > p.scores_cols - s.len) {
    if (threadIdx.x == 0) atomicOr(p.sq.err, DEV_ERR_INDEX_RANGE);
    return;
  }
  const int first = (int)blockIdx.y * iters * kStreamWarps * 16 + warp * 16;
  if (first >= s.len) return;
  const int n = min(iters, (s.len - first + kStreamWarps * 16 - 1) / (kStreamWarps * 16));
  const int pairs = s.rows * group;
  float* out = p.scores + (int64_t)h * p.scores_row + col;
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;                          // [stage][vector][thread]
  float* old = reinterpret_cast<float*>(smem + S * 2 * KB * TH * 16) + threadIdx.x;  // [stage][2][thread]

  // A round's 16 keys lie in one page when 16 divides the page size: one
  // lookup serves the warp and a thread's rows are at fixed distances. Else
  // every thread looks its two rows up.
  const bool one = p.kv.page_size % 16 == 0;
  unsigned valid = 0;  // bits 2 * stage + r: the thread's row g + 8 r of the stage exists
  const uint8_t* const keys = p.kv.base + (int64_t)h * p.kv.head_stride + t * 16;
  const int64_t row0 = g * p.kv.tok_stride, row1 = (g + 8) * p.kv.tok_stride;
  int64_t nxt[2];      // rows g and g + 8 of the round that is copied next
  int blk = -1;        // one: its block and first token
  int tok = 0;
  auto lookup = [&](int it) {
    const int key0 = first + it * kStreamWarps * 16;
    if (one) {
      blk = -1;
      if (it < n) {
        const int pg = (int)fdiv((uint32_t)key0, p.kv.page_div);
        tok = key0 - pg * p.kv.page_size;
        blk = ld_ahead(&p.sq.table[(int64_t)b * p.sq.table_ld + pg]);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 2; ++r) nxt[r] = it < n ? key_offset(p, s, b, 0, key0 + g + 8 * r) : -1;
    }
  };
  auto issue = [&](int it, int st) {
    if (it < n) {
      const int pos = first + it * kStreamWarps * 16 + g;
      bool in[2];
      const uint8_t* src[2];
      if (one) {
        const bool ok = (unsigned)blk < (unsigned)p.kv.num_pages;
        if (!ok) atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
        const uint8_t* page = keys + (ok ? blk : 0) * p.kv.page_stride + tok * p.kv.tok_stride;
        src[0] = page + row0;
        src[1] = page + row1;
        in[0] = ok && pos < s.len;
        in[1] = ok && pos + 8 < s.len;
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          in[r] = nxt[r] >= 0;
          src[r] = keys + (in[r] ? nxt[r] : 0);
        }
      }
      valid = (valid & ~(3u << (2 * st))) | ((unsigned)in[0] << (2 * st)) | ((unsigned)in[1] << (2 * st + 1));
      const uint32_t dst = smem_u32(ring + st * 2 * KB * TH);
      copy_pieces<KB, TH * 16, 0>(dst, src[0], in[0] ? 16 : 0);
      copy_pieces<KB, TH * 16, 0>(dst + KB * TH * 16, src[1], in[1] ? 16 : 0);
      if (p.accumulate && t == 0) {
        if (pos < s.len) cp4(smem_u32(old + (st * 2) * TH), out + pos);
        if (pos + 8 < s.len) cp4(smem_u32(old + (st * 2 + 1) * TH), out + pos + 8);
      }
    }
    cp_commit();
  };
  lookup(0);
#pragma unroll
  for (int k = 0; k < S - 1; ++k) {
    issue(k, k);
    lookup(k + 1);
  }
  // query rows and their lse: of the first 8 NT pairs for the whole round, of
  // the others (a sequence of more rows than the mean) in every iteration
  struct Eight {
    uint4 w[KB];
    float z[2];
    int row[2];
  };
  auto eight = [&](int q0, Eight& a) {
    const int i = q0 + g, j = (int)fdiv((uint32_t)i, p.sq.group_div);
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(s.row0 + j) * p.q_row +
                                                      (int64_t)(h * group + i - j * group) * p.q_head) + t;
#pragma unroll
    for (int k = 0; k < KB; ++k) a.w[k] = i < pairs ? __ldg(src + 4 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int ci = q0 + 2 * t + e, cj = (int)fdiv((uint32_t)ci, p.sq.group_div);
      a.row[e] = s.row0 + cj;
      a.z[e] = ci < pairs ? __ldg(&p.lse[(int64_t)a.row[e] * p.lse_row + h * group + ci - cj * group]) : DARIC_NEG_INF;
    }
  };
  Eight qs[NT];
#pragma unroll
  for (int q = 0; q < NT; ++q) eight(q * 8, qs[q]);
  int st = 0;
  for (int it = 0; it < n; ++it) {
    issue(it + S - 1, st == 0 ? S - 1 : st - 1);
    lookup(it + S);
    cp_wait<S - 1>();
    const int key0 = first + it * kStreamWarps * 16;
    const bool draft = key0 + 16 > s.ctx;
    float sum[2] = {0.f, 0.f};
    auto add_weights = [&](const float (&x)[4], const Eight& a) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (a.z[e] == DARIC_NEG_INF) continue;  // no such pair, or a row that sees nothing
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float y = weight_of(x[2 * r + e], p.scale, a.z[e]);
          const int d = key0 + g + 8 * r - s.ctx;
          if (!draft || d < 0 || sees_draft(p.sq, a.row[e], a.row[e] - s.row0, d)) sum[r] += y;
        }
      }
    };
    const uint4* u = ring + st * 2 * KB * TH;
    {
      float x[NT][4];
#pragma unroll
      for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[q][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const uint4 lo = u[k * TH], hi = u[(KB + k) * TH];
#pragma unroll
        for (int q = 0; q < NT; ++q) products<T>(x[q], lo, hi, qs[q].w[k]);
      }
#pragma unroll
      for (int q = 0; q < NT; ++q) add_weights(x[q], qs[q]);
    }
    for (int q0 = 8 * NT; q0 < pairs; q0 += 8) {
      Eight a;
      eight(q0, a);
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KB; ++k) products<T>(x, u[k * TH], u[(KB + k) * TH], a.w[k]);
      add_weights(x, a);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      const int pos = key0 + g + 8 * r;
      if (t == 0 && pos < s.len) {
        const float add = (valid >> (2 * st + r)) & 1u ? sum[r] : 0.f;
        out[pos] = p.accumulate ? old[(st * 2 + r) * TH] + add : add;
      }
    }
    st = st + 1 == S ? 0 : st + 1;
  }
  cp_wait<0>();
}

// -------------------------------------------------------------- block --
constexpr int kBlockWarps = 8;
constexpr int kBlockRows = 64;  // pairs in shared memory at a time

// 16 M keys of a warp in fragment order: rows g, g + 8 (, g + 16, g + 24).
template <int D, int M>
struct KeyTile {
  static constexpr int KB = D / 32;
  uint4 a[2 * M][KB];
  unsigned valid;  // bit r: this thread's row g + 8 r exists

  __device__ __forceinline__ void load(const ScoresLaunch& p, const Seq& s, int b, int h, int key0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    valid = 0;
#pragma unroll
    for (int r = 0; r < 2 * M; ++r) {
      const int64_t o = key_offset(p, s, b, h, key0 + g + 8 * r);
      if (o >= 0) valid |= 1u << r;
#pragma unroll
      for (int k = 0; k < KB; ++k)
        a[r][k] = o >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.kv.base + o) + 4 * k + t) : make_uint4(0, 0, 0, 0);
    }
  }
};

// kBlockRows query rows in shared memory; rows 64 bytes longer than they are,
// so that eight rows of a fragment read fall into different banks.
template <int D>
struct QueryBlock {
  static constexpr int CH = D / 8, PITCH = D * 2 + 64;
  uint8_t rows[kBlockRows * PITCH];
  float z[kBlockRows];
  int row[kBlockRows];

  // pairs [i0, i0 + kBlockRows) of the sequence; the CTA's threads meet around it
  __device__ __forceinline__ void load(const ScoresLaunch& p, const Seq& s, int h, int i0, int pairs) {
    const int group = p.sq.group;
    __syncthreads();
    for (int v = threadIdx.x; v < kBlockRows * CH; v += kBlockWarps * 32) {
      const int i = v / CH, c = v % CH, pi = i0 + i, j = (int)fdiv((uint32_t)pi, p.sq.group_div);
      uint4 w = make_uint4(0, 0, 0, 0);
      if (pi < pairs)
        w = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)(s.row0 + j) * p.q_row +
                                                 (int64_t)(h * group + pi - j * group) * p.q_head) + c);
      *reinterpret_cast<uint4*>(rows + i * PITCH + c * 16) = w;
    }
    if (threadIdx.x < kBlockRows) {
      const int pi = i0 + threadIdx.x, j = (int)fdiv((uint32_t)pi, p.sq.group_div);
      row[threadIdx.x] = s.row0 + j;
      z[threadIdx.x] = pi < pairs && p.lse ? __ldcg(&p.lse[(int64_t)(s.row0 + j) * p.lse_row + h * group + pi - j * group])
                                           : DARIC_NEG_INF;
    }
    __syncthreads();
  }
};

// Products of a key tile with the eight query rows from `i` of the block on.
template <class T, int D, int M>
__device__ __forceinline__ void block_products(const KeyTile<D, M>& kt, const QueryBlock<D>& qb, int i, float (&x)[M][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[m][e] = 0.f;
  const uint8_t* q = qb.rows + (i + g) * QueryBlock<D>::PITCH + t * 16;
  float y[M][4];  // every other piece: two shorter chains of products
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) y[m][e] = 0.f;
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    const uint4 w = *reinterpret_cast<const uint4*>(q + k * 64);
#pragma unroll
    for (int m = 0; m < M; ++m) products<T>(k & 1 ? y[m] : x[m], kt.a[2 * m][k], kt.a[2 * m + 1][k], w);
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[m][e] += y[m][e];
}

template <class T, int D, int M>
__global__ void __launch_bounds__(kBlockWarps * 32, D > 128 ? 1 : 2) weight_block_kernel(const __grid_constant__ ScoresLaunch p) {
  constexpr int KEYS = 16 * M;
  __shared__ __align__(16) QueryBlock<D> qb;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  // heads and tiles share grid x (y ends at 65535): the heads of a tile are neighbours
  const int b = blockIdx.z, tile = (int)(blockIdx.x / (unsigned)p.kv.heads), h = (int)blockIdx.x - tile * p.kv.heads;
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, p.kv.page_size, s);
  const int64_t col = __ldg(&p.col_off[b]);
  const bool outside = col < 0 || col > p.scores_cols - s.len;
  if (outside && threadIdx.x == 0) atomicOr(p.sq.err, DEV_ERR_INDEX_RANGE);
  const int pairs = s.rows * p.sq.group;
  const int key0 = (tile * kBlockWarps + warp) * KEYS;
  if (outside || tile * kBlockWarps * KEYS >= s.len) {
    grid_wait();  // none of a grid that was launched ahead ends before the one that it follows
    return;
  }
  KeyTile<D, M> kt;
  kt.load(p, s, b, h, key0);  // beside the log-sums, where those are computed here
  grid_wait();
  const bool draft = key0 + KEYS > s.ctx;
  float sum[2 * M];  // keys g, g + 8, ...
#pragma unroll
  for (int r = 0; r < 2 * M; ++r) sum[r] = 0.f;
  for (int i0 = 0; i0 < pairs; i0 += kBlockRows) {
    qb.load(p, s, h, i0, pairs);
    const int n = min(kBlockRows, pairs - i0);
#pragma unroll 2
    for (int i = 0; i < n; i += 8) {
      float x[M][4];
      block_products<T, D, M>(kt, qb, i, x);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float z = qb.z[i + 2 * t + e];
        const int row = qb.row[i + 2 * t + e];
#pragma unroll
        for (int r = 0; r < 2 * M; ++r) {
          const float a = weight_of(x[r >> 1][(r & 1) * 2 + e], p.scale, z);
          const int d = key0 + g + 8 * r - s.ctx;
          // z = -inf: no such pair, or a row that sees nothing
          if (z != DARIC_NEG_INF && (!draft || d < 0 || sees_draft(p.sq, row, row - s.row0, d))) sum[r] += a;
        }
      }
    }
  }
  float* out = p.scores + (int64_t)h * p.scores_row + col;
#pragma unroll
  for (int r = 0; r < 2 * M; ++r) {
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    const int pos = key0 + g + 8 * r;
    if (t == 0 && pos < s.len) {
      const float add = (kt.valid >> r) & 1u ? sum[r] : 0.f;
      out[pos] = p.accumulate ? out[pos] + add : add;
    }
  }
}

// ---------------------------------------------------------------- lse --
// Maximum and sum of each query row over the kLseKeys keys of a CTA (a split).
// Here query rows are the rows of the fragments, so a thread keeps the
// maximum and sum of its own columns to the end. The keys lie in shared
// memory; eight warps take (16 rows) x (a share of the keys) each, shares as
// the rows leave warps over.
template <int D>
constexpr int lse_smem() {
  return kLseKeys * (D * 2 + 16);
}

template <class T, int D>
__global__ void __launch_bounds__(kBlockWarps * 32, D > 128 ? 1 : 2) lse_kernel(const __grid_constant__ ScoresLaunch p) {
  constexpr int PITCH = D * 2 + 16, CH = D / 8, RPI = 32 / CH, CHUNK = 32;
  extern __shared__ __align__(128) uint8_t ktile[];
  __shared__ float2 s_ml[kBlockWarps][16];
  __shared__ uint32_t s_valid[kBlockWarps];  // 32 keys each
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, h = blockIdx.x, group = p.sq.group, split = blockIdx.y;
  grid_next();
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, p.kv.page_size, s);
  const int pairs = s.rows * group;
  const float cexp = p.scale * kLog2e;
  auto at = [&](int i) {  // part of pair i
    const int j = (int)fdiv((uint32_t)i, p.sq.group_div);
    return ((int64_t)(s.row0 + j) * (p.kv.heads * group) + h * group + i - j * group) * p.splits + split;
  };
  const int key0 = split * kLseKeys;
  if (key0 >= s.len) {  // behind the end: empty parts
    for (int i = threadIdx.x; i < pairs; i += kBlockWarps * 32) p.part[at(i)] = make_float2(DARIC_NEG_INF, 0.f);
    return;
  }
  {  // a warp brings 32 keys, a lane looks one up
    const int64_t off = key_offset(p, s, b, h, key0 + warp * 32 + lane);
    const unsigned ok = __ballot_sync(0xffffffffu, off >= 0);
    if (lane == 0) s_valid[warp] = ok;
    const uint32_t dst = smem_u32(ktile) + (warp * 32 + lane / CH) * PITCH + (lane % CH) * 16;
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int64_t o = __shfl_sync(0xffffffffu, off, i * RPI + lane / CH);
      cp16(dst + i * RPI * PITCH, p.kv.base + (o >= 0 ? o + (lane % CH) * 16 : 0), o >= 0);
    }
    cp_commit();
  }
  const int row_groups = (pairs + 15) / 16;
  int shares = 1;  // of the keys per row group: 1, 2, 4 or 8
  while (shares < kBlockWarps && row_groups * shares * 2 <= kBlockWarps) shares *= 2;
  const int share = warp % shares, lanes_rg = kBlockWarps / shares;
  const int k_first = share * (kLseKeys / shares);
  for (int r0 = 0; r0 < row_groups; r0 += lanes_rg) {
    const int pi = (r0 + warp / shares) * 16;  // first pair of this warp's rows
    float m[2] = {DARIC_NEG_INF, DARIC_NEG_INF}, l[2] = {0.f, 0.f};
    int row[2] = {0, 0};
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = pi + g + 8 * r, j = (int)fdiv((uint32_t)i, p.sq.group_div);
      row[r] = s.row0 + j;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q + (int64_t)(s.row0 + j) * p.q_row +
                                                            (int64_t)(h * group + i - j * group) * p.q_head) + t;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][r] = i < pairs ? __ldg(q + 8 * k) : 0u;
        qf[k][2 + r] = i < pairs ? __ldg(q + 8 * k + 4) : 0u;
      }
    }
    if (r0 == 0) {
      cp_wait<0>();
      __syncthreads();
    }
    if (pi < pairs) {
      for (int c = k_first; c < k_first + kLseKeys / shares && key0 + c < s.len; c += CHUNK) {
        float x[CHUNK / 8][4];
#pragma unroll
        for (int n = 0; n < CHUNK / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][e] = 0.f;
        const uint32_t ka = smem_u32(ktile) + (c + (lane >> 4) * 8 + (lane & 7)) * PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int n = 0; n < CHUNK / 16; ++n) {
            uint32_t kf[4];
            ldsm4(ka + n * 16 * PITCH + k * 32, kf);
            Mma<T>::run(x[2 * n], qf[k], kf[0], kf[1]);
            Mma<T>::run(x[2 * n + 1], qf[k], kf[2], kf[3]);
          }
        const uint32_t valid = s_valid[c / 32];
        const bool draft = key0 + c + CHUNK > s.ctx;
        if (valid != 0xffffffffu || draft) {
#pragma unroll
          for (int n = 0; n < CHUNK / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = n * 8 + 2 * t + (e & 1), d = key0 + c + key - s.ctx, i = pi + g + 8 * (e >> 1);
              const bool ok = ((valid >> key) & 1u) &&
                              (d < 0 || (i < pairs && sees_draft(p.sq, row[e >> 1], row[e >> 1] - s.row0, d)));
              if (!ok) x[n][e] = DARIC_NEG_INF;
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float mx = m[r];
#pragma unroll
          for (int n = 0; n < CHUNK / 8; ++n) mx = fmaxf(mx, fmaxf(x[n][2 * r], x[n][2 * r + 1]));
          const float bs = mx == DARIC_NEG_INF ? 0.f : mx;
          float sum = l[r] * exp2_fast((m[r] - bs) * cexp);
#pragma unroll
          for (int n = 0; n < CHUNK / 8; ++n)
            sum += exp2_fast((x[n][2 * r] - bs) * cexp) + exp2_fast((x[n][2 * r + 1] - bs) * cexp);
          l[r] = sum;
          m[r] = mx;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m[r], o), ol = __shfl_xor_sync(0xffffffffu, l[r], o);
        const float mx = fmaxf(m[r], om), bs = mx == DARIC_NEG_INF ? 0.f : mx;
        l[r] = l[r] * exp2_fast((m[r] - bs) * cexp) + ol * exp2_fast((om - bs) * cexp);
        m[r] = mx;
      }
    if (r0) __syncthreads();  // the shares of the rows before are joined
    if (t == 0) {
      s_ml[warp][g] = make_float2(m[0], l[0]);
      s_ml[warp][g + 8] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    const int rg = threadIdx.x / 16, i = (r0 + rg) * 16 + (threadIdx.x & 15);
    if (rg < lanes_rg && i < pairs) {
      float mx = DARIC_NEG_INF, ll = 0.f;
      for (int w = 0; w < shares; ++w) mx = fmaxf(mx, s_ml[rg * shares + w][threadIdx.x & 15].x);
      const float bs = mx == DARIC_NEG_INF ? 0.f : mx;
      for (int w = 0; w < shares; ++w) {
        const float2 v = s_ml[rg * shares + w][threadIdx.x & 15];
        ll += v.y * exp2_fast((v.x - bs) * cexp);
      }
      p.part[at(i)] = make_float2(mx, ll);
    }
  }
}

// lse of each query row and head from its parts (one warp each).
__global__ void __launch_bounds__(256) lse_join_kernel(const __grid_constant__ ScoresLaunch p) {
  const int64_t items = (int64_t)p.sq.num_rows * p.kv.heads * p.sq.group;
  grid_next();
  grid_wait();
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= items) return;
  const float cexp = p.scale * kLog2e;
  float m = DARIC_NEG_INF, l = 0.f;
  for (int i = lane; i < p.splits; i += 32) {
    const float2 v = p.part[at * p.splits + i];
    const float mx = fmaxf(m, v.x), bs = mx == DARIC_NEG_INF ? 0.f : mx;
    l = l * exp2_fast((m - bs) * cexp) + v.y * exp2_fast((v.x - bs) * cexp);
    m = mx;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), ol = __shfl_xor_sync(0xffffffffu, l, o);
    const float mx = fmaxf(m, om), bs = mx == DARIC_NEG_INF ? 0.f : mx;
    l = l * exp2_fast((m - bs) * cexp) + ol * exp2_fast((om - bs) * cexp);
    m = mx;
  }
  if (lane == 0) p.lse_work[at] = l == 0.f ? DARIC_NEG_INF : __fmaf_rn(m, p.scale, logf(l));
}

template <class T, int D, int NT>
void stream_n(const ScoresLaunch& p, cudaStream_t s) {
  const int64_t cap = (int64_t)p.sq.table_cols * p.kv.page_size;
  // long rounds (the ring fills once) that still leave the SMs several CTAs
  int iters = 64;
  auto ctas = [&](int n) { return (cap + 16 * kStreamWarps * n - 1) / (16 * kStreamWarps * n) * p.sq.num_seqs * p.kv.heads; };
  while (iters > 1 && ctas(iters) < 6 * (int64_t)p.sm_count) iters /= 2;
  const unsigned tiles = (unsigned)((cap + 16 * kStreamWarps * iters - 1) / (16 * kStreamWarps * iters));
  static std::atomic<uint64_t> done{0};
  allow_smem(weight_stream_kernel<T, D, NT>, StreamGeom<D>::SMEM, done);
  weight_stream_kernel<T, D, NT>
      <<<dim3((unsigned)p.kv.heads, tiles, (unsigned)p.sq.num_seqs), kStreamWarps * 32, StreamGeom<D>::SMEM, s>>>(p, iters);
  DARIC_CUDA(cudaGetLastError());
}

template <class T, int D>
void scores_d(const ScoresLaunch& p0, cudaStream_t s) {
  ScoresLaunch p = p0;
  const int64_t cap = (int64_t)p.sq.table_cols * p.kv.page_size;
  if (!p.lse) {
    const int64_t items = (int64_t)p.sq.num_rows * p.kv.heads * p.sq.group;
    static std::atomic<uint64_t> done{0};
    allow_smem(lse_kernel<T, D>, lse_smem<D>(), done);
    lse_kernel<T, D><<<dim3((unsigned)p.kv.heads, (unsigned)p.splits, (unsigned)p.sq.num_seqs), kBlockWarps * 32,
                       lse_smem<D>(), s>>>(p);
    DARIC_CUDA(cudaGetLastError());
    launch_after(lse_join_kernel, dim3((unsigned)((items + 7) / 8)), 256, s, p);
    p.lse = p.lse_work;
    p.lse_row = (int64_t)p.kv.heads * p.sq.group;
  }
  // by the mean rows of a sequence (the real ones are on the device); a
  // sequence of more rows is right in either form
  const int64_t pairs = (int64_t)(p.sq.num_rows + p.sq.num_seqs - 1) / p.sq.num_seqs * p.sq.group;
  if (pairs <= 8) return stream_n<T, D, 1>(p, s);
  if (pairs <= 16) return stream_n<T, D, 2>(p, s);
  constexpr int M = D > 128 ? 1 : 2;
  const int64_t tiles = (cap + kBlockWarps * 16 * M - 1) / (kBlockWarps * 16 * M);  // 2^17 at most: times 4095 heads, 2^29
  const dim3 grid((unsigned)(tiles * p.kv.heads), 1, (unsigned)p.sq.num_seqs);
  if (!p0.lse) return launch_after(weight_block_kernel<T, D, M>, grid, kBlockWarps * 32, s, p);
  weight_block_kernel<T, D, M><<<grid, kBlockWarps * 32, 0, s>>>(p);
  DARIC_CUDA(cudaGetLastError());
}

}  // namespace

void launch_scores(const ScoresLaunch& p, int dtype, cudaStream_t s) {
  switch (dtype == DARIC_DTYPE_BF16 ? p.kv.head_dim : (dtype == DARIC_DTYPE_F16 ? -p.kv.head_dim : 0)) {
    case 64: return scores_d<__nv_bfloat16, 64>(p, s);
    case 128: return scores_d<__nv_bfloat16, 128>(p, s);
    case 256: return scores_d<__nv_bfloat16, 256>(p, s);
    case -64: return scores_d<__half, 64>(p, s);
    case -128: return scores_d<__half, 128>(p, s);
    case -256: return scores_d<__half, 256>(p, s);
  }
  throw Error(DARIC_ERR_INVALID, "attention_scores: bfloat16 or float16 keys of 64, 128 or 256");
}

}  // namespace daric
