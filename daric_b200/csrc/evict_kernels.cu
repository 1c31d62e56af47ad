// Eviction from the paged KV cache: the attention weight each cached token
// received, and the move of the kept tokens to the front of their blocks.
//
// weight_kernel: scores[h, p] (+)= sum over the sequence's query rows j and the
// group's heads e of  exp(scale q_je . k_p - lse_je)  where j sees p. Keys are
// the rows of the matrix fragments and query rows their columns, so a key's
// sum stays in the four threads that hold its row: no atomics, one fixed order
// of additions. A warp holds 32 keys in registers (16 bytes a thread straight
// from the cache: both operands take the head dimension in the same permuted
// order, which leaves the products alone) and passes all query rows by them.
// Bound: the K bytes for a few rows, the matrix and exp2 rates for many.
//
// Without an lse, lse_kernel first runs the same products and keeps the
// maximum and the sum of each query row over the 512 keys of a CTA;
// lse_join_kernel joins them. K is read twice then (the second time from the
// L2 cache for prompts up to about 100 MB of keys).
//
// compact_kernel: kept token n of a list, position i_n (ascending), moves to
// position dst + n. Since i_n >= dst + n, a destination is never behind the
// source of a later token, so one CTA that goes through the tokens in order
// and loads each batch before it stores it moves them in place; the
// parallelism is over layers, segments, heads, the K and V planes and slices
// of the row. Keys turn by (new - old): C = nc oc + ns os, S = ns oc - nc os
// from the table rows of both positions, in fp32 without rounding between,
// and the turned key is rounded once.
// Bound: the bytes of the tokens that move, read and written once.
#include "attend_common.cuh"
#include "device_common.cuh"

#include <algorithm>

namespace daric {
namespace {
using namespace att;

constexpr int kSW = 8;  // warps of a score CTA
constexpr int kKeysWarp = 32;
static_assert(kScoreKeys % (kSW * kKeysWarp) == 0, "whole rounds");

// 32 keys of a warp: pages, then the rows in fragment order.
template <int D>
struct KeyTile {
  static constexpr int KB = D / 32;  // 64-byte pieces of a row
  uint4 a[4][KB];                    // rows g, g + 8, g + 16, g + 24
  unsigned valid;                    // bit r: this thread's row g + 8 r exists
};

template <int D>
__device__ __forceinline__ void load_keys(const ScoresLaunch& p, const Seq& s, int b, int h, int key0, KeyTile<D>& kt) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pos = key0 + lane;
  int64_t off = -1;
  if (pos < s.len) {
    const int pg = (int)fdiv((uint32_t)pos, p.kv.page_div);
    const int blk = __ldg(&p.sq.table[(int64_t)b * p.sq.table_ld + pg]);
    if (blk >= 0 && blk < p.kv.num_pages)
      off = (int64_t)blk * p.kv.page_stride + (int64_t)(pos - pg * p.kv.page_size) * p.kv.tok_stride +
            (int64_t)h * p.kv.head_stride;
    else
      atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
  }
  kt.valid = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t o = __shfl_sync(0xffffffffu, off, g + 8 * r);
    if (o >= 0) kt.valid |= 1u << r;
#pragma unroll
    for (int k = 0; k < KeyTile<D>::KB; ++k)
      kt.a[r][k] = o >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.kv.base + o) + 4 * k + t) : make_uint4(0, 0, 0, 0);
  }
}

// Products of 32 keys and 8 query rows: x[m][e], m = 16-key half.
template <class T, int D>
__device__ __forceinline__ void key_products(const KeyTile<D>& kt, const uint8_t* qrow, bool real, float (&x)[2][4]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[m][e] = 0.f;
#pragma unroll
  for (int k = 0; k < KeyTile<D>::KB; ++k) {
    const uint4 w = real ? __ldg(reinterpret_cast<const uint4*>(qrow) + 4 * k + t) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint4 u = kt.a[2 * m][k], v = kt.a[2 * m + 1][k];
      { uint32_t f[4] = {u.x, v.x, u.y, v.y}; Mma<T>::run(x[m], f, w.x, w.y); }
      { uint32_t f[4] = {u.z, v.z, u.w, v.w}; Mma<T>::run(x[m], f, w.z, w.w); }
    }
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kSW * 32) weight_kernel(const __grid_constant__ ScoresLaunch p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.x, h = blockIdx.z, group = p.sq.group;
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, p.kv.page_size, s);
  const int64_t col = __ldg(&p.col_off[b]);
  if (col < 0 || col + s.len > p.scores_cols) {
    if (threadIdx.x == 0) atomicOr(p.sq.err, DEV_ERR_INDEX_RANGE);
    return;
  }
  const int pairs = s.rows * group;
  for (int it = 0; it < kScoreKeys / (kSW * kKeysWarp); ++it) {
    const int key0 = blockIdx.y * kScoreKeys + (it * kSW + warp) * kKeysWarp;
    if (key0 >= s.len) return;
    KeyTile<D> kt;
    load_keys<D>(p, s, b, h, key0, kt);
    const bool draft = key0 + kKeysWarp > s.ctx;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};  // keys g, g + 8, g + 16, g + 24
    for (int i0 = 0; i0 < pairs; i0 += 8) {
      const bool real = i0 + g < pairs;
      const int i = real ? i0 + g : 0;
      const uint8_t* qrow = p.q + (int64_t)(s.row0 + i / group) * p.q_row + (int64_t)(h * group + i % group) * p.q_head;
      float x[2][4];
      key_products<T, D>(kt, qrow, real, x);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int ci = i0 + 2 * t + e;  // this column's (row, head) pair
        if (ci >= pairs) continue;
        const int j = ci / group, row = s.row0 + j;
        const float z = __ldg(&p.lse[(int64_t)row * p.lse_row + h * group + ci % group]);
        if (z == DARIC_NEG_INF) continue;  // a row that sees nothing
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = exp2f(__fmaf_rn(x[r >> 1][(r & 1) * 2 + e], p.scale, -z) * kLog2e);
          bool ok = true;
          if (draft) {
            const int d = key0 + g + 8 * r - s.ctx;
            ok = d < 0 || sees_draft(p.sq, row, j, d);
          }
          if (ok) sum[r] += w;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      const int pos = key0 + g + 8 * r;
      if (t == 0 && pos < s.len) {
        float* dst = p.scores + (int64_t)h * p.scores_row + col + pos;
        const float add = (kt.valid >> r) & 1u ? sum[r] : 0.f;
        *dst = p.accumulate ? *dst + add : add;
      }
    }
  }
}

// Maximum and sum of each query row over this CTA's keys.
template <class T, int D>
__global__ void __launch_bounds__(kSW * 32) lse_kernel(const __grid_constant__ ScoresLaunch p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.x, h = blockIdx.z, group = p.sq.group, split = blockIdx.y;
  __shared__ float2 s_ml[kSW][8];
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, p.kv.page_size, s);
  const int pairs = s.rows * group;
  const float cexp = p.scale * kLog2e;
  constexpr int IT = kScoreKeys / (kSW * kKeysWarp);
  for (int i0 = 0; i0 < pairs; i0 += 8) {
    const bool real = i0 + g < pairs;
    const int i = real ? i0 + g : 0;
    const uint8_t* qrow = p.q + (int64_t)(s.row0 + i / group) * p.q_row + (int64_t)(h * group + i % group) * p.q_head;
    float m[2] = {DARIC_NEG_INF, DARIC_NEG_INF}, l[2] = {0.f, 0.f};
    for (int base = split * kScoreKeys; base < s.len; base += p.splits * kScoreKeys) {
#pragma unroll 1
      for (int it = 0; it < IT; ++it) {
        const int key0 = base + (it * kSW + warp) * kKeysWarp;
        if (key0 >= s.len) break;
        KeyTile<D> kt;
        load_keys<D>(p, s, b, h, key0, kt);
        float x[2][4];
        key_products<T, D>(kt, qrow, real, x);
        const bool draft = key0 + kKeysWarp > s.ctx;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int ci = i0 + 2 * t + e;
          const int j = ci / group;
          float y[4];
          float mx = m[e];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            y[r] = x[r >> 1][(r & 1) * 2 + e];
            bool ok = ((kt.valid >> r) & 1u) && ci < pairs;
            if (ok && draft) {
              const int d = key0 + g + 8 * r - s.ctx;
              ok = d < 0 || sees_draft(p.sq, s.row0 + j, j, d);
            }
            if (!ok) y[r] = DARIC_NEG_INF;
            mx = fmaxf(mx, y[r]);
          }
          const float bs = mx == DARIC_NEG_INF ? 0.f : mx;
          l[e] *= exp2f((m[e] - bs) * cexp);
#pragma unroll
          for (int r = 0; r < 4; ++r) l[e] += exp2f((y[r] - bs) * cexp);
          m[e] = mx;
        }
      }
    }
    // over the eight threads of a column, then the warps
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m[e], o), ol = __shfl_xor_sync(0xffffffffu, l[e], o);
        const float mx = fmaxf(m[e], om), bs = mx == DARIC_NEG_INF ? 0.f : mx;
        l[e] = l[e] * exp2f((m[e] - bs) * cexp) + ol * exp2f((om - bs) * cexp);
        m[e] = mx;
      }
    __syncthreads();
    if (g == 0) {
      s_ml[warp][2 * t] = make_float2(m[0], l[0]);
      s_ml[warp][2 * t + 1] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    if (threadIdx.x < 8 && i0 + (int)threadIdx.x < pairs) {
      const int ci = i0 + threadIdx.x;
      float mx = DARIC_NEG_INF;
      for (int w = 0; w < kSW; ++w) mx = fmaxf(mx, s_ml[w][threadIdx.x].x);
      const float bs = mx == DARIC_NEG_INF ? 0.f : mx;
      float ll = 0.f;
      for (int w = 0; w < kSW; ++w) ll += s_ml[w][threadIdx.x].y * exp2f((s_ml[w][threadIdx.x].x - bs) * cexp);
      const int64_t at = (int64_t)(s.row0 + ci / group) * (p.kv.heads * group) + h * group + ci % group;
      p.part[at * p.splits + split] = make_float2(mx, ll);
    }
  }
}

// lse of each query row and head from its parts (one warp each).
__global__ void __launch_bounds__(256) lse_join_kernel(const __grid_constant__ ScoresLaunch p, int64_t items) {
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= items) return;
  const float cexp = p.scale * kLog2e;
  float m = DARIC_NEG_INF, l = 0.f;
  for (int i = lane; i < p.splits; i += 32) {
    const float2 v = p.part[at * p.splits + i];
    const float mx = fmaxf(m, v.x), bs = mx == DARIC_NEG_INF ? 0.f : mx;
    l = l * exp2f((m - bs) * cexp) + v.y * exp2f((v.x - bs) * cexp);
    m = mx;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), ol = __shfl_xor_sync(0xffffffffu, l, o);
    const float mx = fmaxf(m, om), bs = mx == DARIC_NEG_INF ? 0.f : mx;
    l = l * exp2f((m - bs) * cexp) + ol * exp2f((om - bs) * cexp);
    m = mx;
  }
  if (lane == 0) p.lse_work[at] = l == 0.f ? DARIC_NEG_INF : __fmaf_rn(m, p.scale, logf(l));
}

// ------------------------------------------------------------ compact --
constexpr int kMoveThreads = 256;
constexpr int kMoveTokens = 256;  // tokens whose places a CTA keeps at a time

// E: cache element, TE: rotary table element. A thread moves one 16-byte
// vector of a V row, or of a K row that is not turned; of a turned K row one
// task: the two vectors that pair up (NeoX), one vector (GPT-J).
template <class E, class TE>
__global__ void __launch_bounds__(kMoveThreads) compact_kernel(const __grid_constant__ CompactLaunch p) {
  constexpr int EPV = E::kPerVec;
  __shared__ int64_t s_src[kMoveTokens], s_dst[kMoveTokens];
  __shared__ int2 s_pos[kMoveTokens];
  const int slice = blockIdx.x % p.slices;
  const int x = blockIdx.x / p.slices;
  const int plane = x & 1, h = x >> 1;
  const CompactSeg sg = p.segs[blockIdx.y];
  const int l = blockIdx.z;
  const CompactLayer L = p.layers[l];
  const int64_t list = p.shared ? (p.per_head ? h : 0)
                                : (int64_t)(p.layer0 + l) * (p.per_head ? p.heads : 1) + (p.per_head ? h : 0);
  const int count = min(max(__ldg(&p.count[list * p.count_row + sg.seg]), 0), sg.cap);
  const int32_t* idx = p.idx + list * p.idx_row + sg.out_off;
  uint8_t* base = L.base + (int64_t)h * L.head_stride + (plane ? L.v_off : 0);
  const int vecs = p.head_dim / EPV;
  const bool turn = p.rotate && plane == 0;
  const int rot_vecs = turn ? (p.neox ? p.half_rot / EPV : 2 * p.half_rot / EPV) : 0;  // turning tasks of a row
  const int tail0 = turn ? 2 * p.half_rot / EPV : 0;                                   // first vector that only moves
  const int tasks = rot_vecs + vecs - tail0;
  const int c0 = tasks * slice / p.slices, c1 = tasks * (slice + 1) / p.slices;
  const int per = c1 - c0;
  if (per <= 0) return;
  for (int n0 = 0; n0 < count; n0 += kMoveTokens) {
    const int nt = min(kMoveTokens, count - n0);
    __syncthreads();
    for (int i = threadIdx.x; i < nt; i += kMoveThreads) {
      const int from = __ldg(&idx[n0 + i]), to = sg.dst + n0 + i;
      int64_t so = -1, dof = -1;
      // a list that does not ascend, or would move a token up, is not moved in place
      if (from < to || (n0 + i > 0 && __ldg(&idx[n0 + i - 1]) >= from)) {
        atomicOr(p.err, DEV_ERR_INDEX_RANGE);
      } else if (from != to) {
        int64_t off[2] = {-1, -1};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = e ? to : from;
          const int pg = pos < 0 ? -1 : (int)fdiv((uint32_t)pos, p.page_div);
          if (pg < 0 || sg.blk_off + pg >= p.table_numel) {
            atomicOr(p.err, DEV_ERR_INDEX_RANGE);
            continue;
          }
          const int blk = __ldg(&p.block_table[sg.blk_off + pg]);
          if (blk < 0 || blk >= p.num_pages) {
            atomicOr(p.err, DEV_ERR_BLOCK_RANGE);
            continue;
          }
          off[e] = (int64_t)blk * L.page_stride + (int64_t)(pos - pg * p.page_size) * L.tok_stride;
        }
        const bool in = !turn || (from < p.max_pos && to < p.max_pos);
        if (!in) atomicOr(p.err, DEV_ERR_TABLE_RANGE);
        if (off[0] >= 0 && off[1] >= 0 && in) {
          so = off[0];
          dof = off[1];
        }
      }
      s_src[i] = so;
      s_dst[i] = dof;
      s_pos[i] = make_int2(from, to);
    }
    __syncthreads();
    constexpr int U = 4;
    for (int w0 = 0; w0 < nt * per; w0 += U * kMoveThreads) {
      uint4 a[U], b[U];
      int tok[U], c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int w = w0 + u * kMoveThreads + threadIdx.x;
        tok[u] = -1;
        if (w < nt * per) {
          const int i = w / per;
          c[u] = c0 + w % per;
          if (s_src[i] >= 0) {
            tok[u] = i;
            const uint8_t* src = base + s_src[i];
            if (c[u] >= rot_vecs) {
              a[u] = dev::ld_vec(src + (int64_t)(tail0 + c[u] - rot_vecs) * 16);
            } else {
              a[u] = dev::ld_vec(src + (int64_t)c[u] * 16);
              if (p.neox) b[u] = dev::ld_vec(src + (int64_t)(c[u] + rot_vecs) * 16);
            }
          }
        }
      }
      if (turn) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (tok[u] < 0 || c[u] >= rot_vecs) continue;
          const int2 ps = s_pos[tok[u]];
          constexpr int TS = (int)sizeof(typename TE::raw);
          const uint8_t* orow = L.table + (int64_t)ps.x * p.table_row;
          const uint8_t* nrow = L.table + (int64_t)ps.y * p.table_row;
          const int nf = p.neox ? EPV : EPV / 2;  // frequencies of a task
          float v[EPV], y[EPV];
          dev::unpack<E>(a[u], v);
          if (p.neox) dev::unpack<E>(b[u], y);
#pragma unroll
          for (int f = 0; f < EPV; ++f) {
            if (f >= nf) break;
            const int d = c[u] * nf + f;
            const float oc = TE::to_f(*reinterpret_cast<const typename TE::raw*>(orow + d * TS));
            const float os = TE::to_f(*reinterpret_cast<const typename TE::raw*>(orow + (p.half_rot + d) * TS));
            const float nc = TE::to_f(*reinterpret_cast<const typename TE::raw*>(nrow + d * TS));
            const float ns = TE::to_f(*reinterpret_cast<const typename TE::raw*>(nrow + (p.half_rot + d) * TS));
            const float C = nc * oc + ns * os, S = ns * oc - nc * os;
            if (p.neox) {
              const float x1 = v[f], x2 = y[f];
              v[f] = x1 * C - x2 * S;
              y[f] = x2 * C + x1 * S;
            } else if (2 * f + 1 < EPV) {
              const float x1 = v[2 * f], x2 = v[2 * f + 1];
              v[2 * f] = x1 * C - x2 * S;
              v[2 * f + 1] = x2 * C + x1 * S;
            }
          }
          a[u] = dev::pack_vec<E>(v);
          if (p.neox) b[u] = dev::pack_vec<E>(y);
        }
      }
      __syncthreads();  // every load of the batch is done before its stores
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (tok[u] < 0) continue;
        uint8_t* dst = base + s_dst[tok[u]];
        if (c[u] >= rot_vecs) {
          dev::st_vec(dst + (int64_t)(tail0 + c[u] - rot_vecs) * 16, a[u]);
        } else {
          dev::st_vec(dst + (int64_t)c[u] * 16, a[u]);
          if (p.neox) dev::st_vec(dst + (int64_t)(c[u] + rot_vecs) * 16, b[u]);
        }
      }
      // the next batch's loads may start before these stores have landed: its
      // sources are behind every destination of this batch
    }
  }
}

template <class T, int D>
void scores_d(const ScoresLaunch& p0, cudaStream_t s) {
  ScoresLaunch p = p0;
  const int64_t cap = (int64_t)p.sq.table_cols * p.kv.page_size;
  const unsigned tiles = (unsigned)((cap + kScoreKeys - 1) / kScoreKeys);
  if (!p.lse) {
    const int64_t items = (int64_t)p.sq.num_rows * p.kv.heads * p.sq.group;
    lse_kernel<T, D><<<dim3((unsigned)p.sq.num_seqs, (unsigned)p.splits, (unsigned)p.kv.heads), kSW * 32, 0, s>>>(p);
    DARIC_CUDA(cudaGetLastError());
    lse_join_kernel<<<(unsigned)((items + 7) / 8), 256, 0, s>>>(p, items);
    DARIC_CUDA(cudaGetLastError());
    p.lse = p.lse_work;
    p.lse_row = (int64_t)p.kv.heads * p.sq.group;
  }
  weight_kernel<T, D><<<dim3((unsigned)p.sq.num_seqs, tiles, (unsigned)p.kv.heads), kSW * 32, 0, s>>>(p);
  DARIC_CUDA(cudaGetLastError());
}

template <class E>
void compact_e(const CompactLaunch& p, int tab, dim3 grid, cudaStream_t s) {
  using namespace dev;
  if (!p.rotate || tab == DARIC_DTYPE_F32) compact_kernel<E, Elem<DARIC_DTYPE_F32>><<<grid, kMoveThreads, 0, s>>>(p);
  else if (tab == DARIC_DTYPE_BF16) compact_kernel<E, Elem<DARIC_DTYPE_BF16>><<<grid, kMoveThreads, 0, s>>>(p);
  else compact_kernel<E, Elem<DARIC_DTYPE_F16>><<<grid, kMoveThreads, 0, s>>>(p);
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

void launch_compact(const CompactLaunch& p, int kv_dtype, int tab_dtype, cudaStream_t s) {
  const dim3 grid((unsigned)(p.heads * 2 * p.slices), (unsigned)p.num_segs, (unsigned)p.num_layers);
  switch (kv_dtype) {
    case DARIC_DTYPE_BF16: return compact_e<dev::Elem<DARIC_DTYPE_BF16>>(p, tab_dtype, grid, s);
    case DARIC_DTYPE_F16: return compact_e<dev::Elem<DARIC_DTYPE_F16>>(p, tab_dtype, grid, s);
    case DARIC_DTYPE_F32: return compact_e<dev::Elem<DARIC_DTYPE_F32>>(p, tab_dtype, grid, s);
    case DARIC_DTYPE_FP8_E4M3: return compact_e<dev::Elem<DARIC_DTYPE_FP8_E4M3>>(p, tab_dtype, grid, s);
  }
  throw Error(DARIC_ERR_INVALID, "compact: unknown KV dtype");
}

}  // namespace daric
