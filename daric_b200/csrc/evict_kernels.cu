// Eviction from the paged KV cache: the attention weight each cached token
// received, and the move of the kept tokens to the front of their blocks.
//
// weight_kernel: scores[h, p] (+)= sum over the sequence's query rows j and the
// group's heads e of  exp(scale q_je . k_p - lse_je)  where j sees p. Keys are
// the rows of the matrix fragments and query rows their columns, so a key's
// sum stays in the four threads that hold its row: no atomics, one fixed order
// of additions. A warp holds 32 keys in registers (16 bytes a thread straight
// from the cache: both operands take the head dimension in the same permuted
// order, which leaves the products alone) and passes all query rows by them
// (16 keys where the rows are few).
// Bound: the K bytes for a few rows, the matrix and exp2 rates for many.
//
// Without an lse, lse_kernel first runs the same products and keeps the
// maximum and the sum of each query row over the 256 keys of a CTA;
// lse_join_kernel joins them. K is read twice then (the second time from the
// L2 cache for prompts up to about 100 MB of keys).
//
// compact_kernel: kept token n of a list, position i_n (ascending), moves to
// position dst + n. Since i_n >= dst + n, a destination is never behind the
// source of a later token, so one CTA that goes through the tokens in order
// and loads each batch before it stores it moves them in place; the
// parallelism is over layers, segments, heads, the K and V planes and slices
// of the row. Keys turn by (new - old): C = nc oc + ns os, S = ns oc - nc os
// from the table rows of both positions, in fp32 (a product and a fused
// multiply-add each), and the turned key is rounded once to the cache's type.
// Bound: the bytes of the tokens that move, read and written once.
#include "attend_common.cuh"
#include "device_common.cuh"

#include <algorithm>
#include <type_traits>

namespace daric {
namespace {
using namespace att;

constexpr int kSW = 8;  // warps of a score CTA

// Address of the keys of a tile: M * 16 keys of a warp, lane i looks key i up.
template <int M>
__device__ __forceinline__ int64_t key_offset(const ScoresLaunch& p, const Seq& s, int b, int h, int key0) {
  const int pos = key0 + (int)(threadIdx.x & (16 * M - 1));
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

// M * 16 keys in fragment order: rows g, g + 8 (, g + 16, g + 24).
template <int D, int M>
struct KeyTile {
  static constexpr int KB = D / 32;  // 64-byte pieces of a row
  uint4 a[2 * M][KB];
  unsigned valid;                    // bit r: this thread's row g + 8 r exists

  __device__ __forceinline__ void load(const ScoresLaunch& p, int64_t off) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    valid = 0;
#pragma unroll
    for (int r = 0; r < 2 * M; ++r) {
      const int64_t o = __shfl_sync(0xffffffffu, off, g + 8 * r);
      if (o >= 0) valid |= 1u << r;
#pragma unroll
      for (int k = 0; k < KB; ++k)
        a[r][k] = o >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.kv.base + o) + 4 * k + t) : make_uint4(0, 0, 0, 0);
    }
  }
};

// Eight query rows in fragment order: pair i0 + g of the sequence.
template <int D>
struct QueryTile {
  static constexpr int KB = D / 32;
  uint4 w[KB];
  __device__ __forceinline__ void load(const ScoresLaunch& p, const Seq& s, int h, int i0, int pairs) {
    const int lane = threadIdx.x & 31, i = i0 + (lane >> 2), t = lane & 3;
    const bool real = i < pairs;
    const int j = (int)fdiv((uint32_t)i, p.sq.group_div);
    const uint4* q = reinterpret_cast<const uint4*>(p.q + (int64_t)(s.row0 + j) * p.q_row +
                                                    (int64_t)(h * p.sq.group + i - j * p.sq.group) * p.q_head) + t;
#pragma unroll
    for (int k = 0; k < KB; ++k) w[k] = real ? __ldg(q + 4 * k) : make_uint4(0, 0, 0, 0);
  }
};

template <class T, int D, int M>
__device__ __forceinline__ void key_products(const KeyTile<D, M>& kt, const QueryTile<D>& qt, float (&x)[M][4]) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[m][e] = 0.f;
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    const uint4 w = qt.w[k];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint4 u = kt.a[2 * m][k], v = kt.a[2 * m + 1][k];
      { uint32_t f[4] = {u.x, v.x, u.y, v.y}; Mma<T>::run(x[m], f, w.x, w.y); }
      { uint32_t f[4] = {u.z, v.z, u.w, v.w}; Mma<T>::run(x[m], f, w.z, w.w); }
    }
  }
}

// A CTA takes `iters` rounds of kSW tiles of M * 16 keys. With M = 1 (few
// query rows) the next round's keys are on their way while a round is worked
// on; with M = 2 (many) the next eight query rows are.
template <class T, int D, int M>
__global__ void __launch_bounds__(kSW * 32, D > 128 ? 1 : (M == 1 ? 2 : 1)) weight_kernel(const __grid_constant__ ScoresLaunch p, int iters) {
  constexpr int KEYS = 16 * M;
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
  int key0 = (int)blockIdx.y * iters * kSW * KEYS + warp * KEYS;
  if (key0 >= s.len) return;
  KeyTile<D, M> kt, nx;
  kt.load(p, key_offset<M>(p, s, b, h, key0));
  int64_t off = iters > 1 ? key_offset<M>(p, s, b, h, key0 + kSW * KEYS) : -1;
  QueryTile<D> qt;
  qt.load(p, s, h, 0, pairs);
  for (int it = 0; it < iters && key0 < s.len; ++it, key0 += kSW * KEYS) {
    if (M == 1 && it + 1 < iters) {
      nx.load(p, off);
      off = it + 2 < iters ? key_offset<M>(p, s, b, h, key0 + 2 * kSW * KEYS) : -1;
    }
    const bool draft = key0 + KEYS > s.ctx;
    float sum[2 * M];  // keys g, g + 8, ...
#pragma unroll
    for (int r = 0; r < 2 * M; ++r) sum[r] = 0.f;
    for (int i0 = 0; i0 < pairs; i0 += 8) {
      QueryTile<D> qn;
      if (M == 2 && pairs > 8) qn.load(p, s, h, i0 + 8 < pairs ? i0 + 8 : 0, pairs);
      float x[M][4];
      key_products<T, D, M>(kt, qt, x);
      if (M == 1 && pairs > 8) qt.load(p, s, h, i0 + 8 < pairs ? i0 + 8 : 0, pairs);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int ci = i0 + 2 * t + e;  // this column's (row, head) pair
        if (ci >= pairs) continue;
        const int j = (int)fdiv((uint32_t)ci, p.sq.group_div), row = s.row0 + j;
        const float z = __ldg(&p.lse[(int64_t)row * p.lse_row + h * group + ci - j * group]);
        if (z == DARIC_NEG_INF) continue;  // a row that sees nothing
#pragma unroll
        for (int r = 0; r < 2 * M; ++r) {
          const float w = exp2f(__fmaf_rn(x[r >> 1][(r & 1) * 2 + e], p.scale, -z) * kLog2e);
          bool ok = true;
          if (draft) {
            const int d = key0 + g + 8 * r - s.ctx;
            ok = d < 0 || sees_draft(p.sq, row, j, d);
          }
          if (ok) sum[r] += w;
        }
      }
      if (M == 2 && pairs > 8) qt = qn;
    }
#pragma unroll
    for (int r = 0; r < 2 * M; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      const int pos = key0 + g + 8 * r;
      if (t == 0 && pos < s.len) {
        float* dst = p.scores + (int64_t)h * p.scores_row + col + pos;
        const float add = (kt.valid >> r) & 1u ? sum[r] : 0.f;
        *dst = p.accumulate ? *dst + add : add;
      }
    }
    if (M == 1) kt = nx;
    else if (it + 1 < iters) {
      kt.load(p, off);
      off = it + 2 < iters ? key_offset<M>(p, s, b, h, key0 + 2 * kSW * KEYS) : -1;
    }
  }
}

// Maximum and sum of each query row over the kLseKeys keys of a CTA (a split).
template <class T, int D>
__global__ void __launch_bounds__(kSW * 32) lse_kernel(const __grid_constant__ ScoresLaunch p) {
  constexpr int M = 2, KEYS = 16 * M, COLS = 32;  // pairs between two meetings of the warps
  static_assert(kSW * KEYS == kLseKeys, "one tile per warp");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.x, h = blockIdx.z, group = p.sq.group, split = blockIdx.y;
  __shared__ float2 s_ml[2][kSW][COLS];
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, p.kv.page_size, s);
  const int pairs = s.rows * group;
  const float cexp = p.scale * kLog2e;
  const int heads = p.kv.heads * group;
  auto at = [&](int i) {  // part of pair i
    const int j = (int)fdiv((uint32_t)i, p.sq.group_div);
    return ((int64_t)(s.row0 + j) * heads + h * group + i - j * group) * p.splits + split;
  };
  if (split * kLseKeys >= s.len) {  // behind the end: empty parts
    for (int i = threadIdx.x; i < pairs; i += kSW * 32) p.part[at(i)] = make_float2(DARIC_NEG_INF, 0.f);
    return;
  }
  const int key0 = split * kLseKeys + warp * KEYS;
  KeyTile<D, M> kt;
  kt.load(p, key_offset<M>(p, s, b, h, key0));
  const bool draft = key0 + KEYS > s.ctx;
  QueryTile<D> qt;
  qt.load(p, s, h, 0, pairs);
  for (int c0 = 0, par = 0; c0 < pairs; c0 += COLS, par ^= 1) {
    for (int i0 = c0; i0 < c0 + COLS && i0 < pairs; i0 += 8) {
      QueryTile<D> qn;
      if (i0 + 8 < pairs) qn.load(p, s, h, i0 + 8, pairs);
      float x[M][4];
      key_products<T, D, M>(kt, qt, x);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int ci = i0 + 2 * t + e;
        const int j = (int)fdiv((uint32_t)ci, p.sq.group_div);
        float y[2 * M], mx = DARIC_NEG_INF, l = 0.f;
#pragma unroll
        for (int r = 0; r < 2 * M; ++r) {
          y[r] = x[r >> 1][(r & 1) * 2 + e];
          bool ok = ((kt.valid >> r) & 1u) && ci < pairs;
          if (ok && draft) {
            const int d = key0 + g + 8 * r - s.ctx;
            ok = d < 0 || sees_draft(p.sq, s.row0 + j, j, d);
          }
          if (!ok) y[r] = DARIC_NEG_INF;
          mx = fmaxf(mx, y[r]);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float bs = mx == DARIC_NEG_INF ? 0.f : mx;
#pragma unroll
        for (int r = 0; r < 2 * M; ++r) l += exp2f((y[r] - bs) * cexp);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (g == 0) s_ml[par][warp][i0 - c0 + 2 * t + e] = make_float2(mx, l);
      }
      if (i0 + 8 < pairs) qt = qn;
    }
    __syncthreads();  // the other half of s_ml is free until the meeting after this one
    const int i = c0 + (int)threadIdx.x;
    if (threadIdx.x < COLS && i < pairs) {
      float mx = DARIC_NEG_INF, l = 0.f;
#pragma unroll
      for (int w = 0; w < kSW; ++w) mx = fmaxf(mx, s_ml[par][w][threadIdx.x].x);
      const float bs = mx == DARIC_NEG_INF ? 0.f : mx;
#pragma unroll
      for (int w = 0; w < kSW; ++w) l += s_ml[par][w][threadIdx.x].y * exp2f((s_ml[par][w][threadIdx.x].x - bs) * cexp);
      p.part[at(i)] = make_float2(mx, l);
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
constexpr int kMoveThreads = 512;
constexpr int kMoveTokens = 2048;  // tokens whose places a CTA keeps: two chunks
constexpr int kMoveBatch = 256;    // most tokens of a batch
constexpr int kMoveStages = 3;     // batches of loads under way
constexpr int kMoveVecs = 8;       // vectors of a thread in a batch
constexpr int kMoveRing = kMoveStages * kMoveVecs * kMoveThreads * 16;
constexpr int kMoveSmem = kMoveRing + kMoveTokens * 12;

// The places of a batch that is being stored (or was, one barrier ago) and of
// the batches ahead of it fit beside the chunk that is being written.
static_assert((kMoveStages + 1) * kMoveBatch <= kMoveTokens / 2, "places stay until their batch is stored");

constexpr uint32_t kStays = 0xffffffffu;  // source of a token that is not moved

// Table entries of NF frequencies from d0 on at the old and the new position,
// and the factors of the turn between them, in fp32.
template <class TE, int NF>
struct TurnEntries {
  float oc[NF], os[NF], nc[NF], ns[NF];
  __device__ __forceinline__ void load(const uint8_t* table, int64_t row, int half, int from, int to, int d0) {
    constexpr int TS = (int)sizeof(typename TE::raw);
    const uint8_t* orow = table + (int64_t)from * row + d0 * TS;
    const uint8_t* nrow = table + (int64_t)to * row + d0 * TS;
    dev::load_entries<TE, NF>(orow, oc);
    dev::load_entries<TE, NF>(orow + half * TS, os);
    dev::load_entries<TE, NF>(nrow, nc);
    dev::load_entries<TE, NF>(nrow + half * TS, ns);
  }
  __device__ __forceinline__ void factors(float (&C)[NF], float (&S)[NF]) const {
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      C[f] = __fmaf_rn(nc[f], oc[f], ns[f] * os[f]);
      S[f] = __fmaf_rn(ns[f], oc[f], -(nc[f] * os[f]));
    }
  }
};

template <class E, int NF>
__device__ __forceinline__ void turn_neox(const float (&C)[NF], const float (&S)[NF], uint4& lo, uint4& hi) {
  float x[NF], y[NF], o1[NF], o2[NF];
  dev::unpack<E>(lo, x);
  dev::unpack<E>(hi, y);
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    o1[f] = __fmaf_rn(x[f], C[f], -(y[f] * S[f]));
    o2[f] = __fmaf_rn(y[f], C[f], x[f] * S[f]);
  }
  lo = dev::pack_vec<E>(o1);
  hi = dev::pack_vec<E>(o2);
}

template <class E, int NF>
__device__ __forceinline__ void turn_gptj(const float (&C)[NF], const float (&S)[NF], uint4& v) {
  float x[2 * NF];
  dev::unpack<E>(v, x);
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const float a = x[2 * f], b = x[2 * f + 1];
    x[2 * f] = __fmaf_rn(a, C[f], -(b * S[f]));
    x[2 * f + 1] = __fmaf_rn(b, C[f], a * S[f]);
  }
  v = dev::pack_vec<E>(x);
}

// One CTA: the tokens of one segment of one layer, in order, for one piece of
// their rows. blockIdx.x counts the pieces: first (rotate) the turning
// columns of K as turn_slices column slices x head groups, then the columns
// that only move: (plane, head, slice). A thread of a turning piece holds one
// column task (NeoX: the two vectors that pair up) of four heads of a token,
// so the factors are made once for them; with lists per head it holds four
// tokens (GPT-J: the same with one vector a task). A moving piece: eight
// tokens. Loads go to the thread's own slots of a shared-memory ring three
// batches ahead of the stores.
template <class E, class TE, bool NEOX, bool BYHEAD>
__global__ void __launch_bounds__(kMoveThreads, 1) compact_kernel(const __grid_constant__ CompactLaunch p) {
  constexpr int EPV = E::kPerVec, NF = NEOX ? EPV : EPV / 2, U = kMoveVecs / 2, ST = kMoveStages;
  extern __shared__ __align__(128) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;  // [stage][vector][thread]
  uint2* s_at = reinterpret_cast<uint2*>(smem + kMoveRing);    // source and destination, 16-byte units of the layer
  int* s_from = reinterpret_cast<int*>(smem + kMoveRing + kMoveTokens * 8);
  const CompactSeg sg = p.segs[blockIdx.y];
  const int l = blockIdx.z;
  const CompactLayer L = p.layers[l];
  int x = blockIdx.x;
  const bool turn = x < p.turn_pieces;
  int h, heads = 1, c0, c1;
  uint8_t* base = L.base;
  if (turn) {
    const int slice = x % p.turn_slices;
    h = x / p.turn_slices * p.turn_heads;
    heads = BYHEAD ? min(p.turn_heads, p.heads - h) : U;
    c0 = p.rot_vecs * slice / p.turn_slices;
    c1 = p.rot_vecs * (slice + 1) / p.turn_slices;
  } else {
    x -= p.turn_pieces;
    const int slice = x % p.slices, groups = (p.heads + p.move_heads - 1) / p.move_heads;
    x /= p.slices;
    h = x % groups * p.move_heads;
    heads = min(p.move_heads, p.heads - h);
    const bool v_plane = x / groups == 0;  // V first; then K, or its columns that do not turn
    if (v_plane) base += L.v_off;
    const int first = v_plane ? 0 : p.tail0;
    c0 = first + (p.vecs - first) * slice / p.slices;
    c1 = first + (p.vecs - first) * (slice + 1) / p.slices;
  }
  const int64_t list = (p.shared ? 0 : (int64_t)(p.layer0 + l) * (p.per_head ? p.heads : 1)) + (p.per_head ? h : 0);
  const int count = min(max(__ldg(&p.count[list * p.count_row + sg.seg]), 0), sg.cap);
  const int32_t* idx = p.idx + list * p.idx_row + sg.out_off;
  if (c1 <= c0) return;
  const int per = turn ? c1 - c0 : (c1 - c0) * heads;  // threads of a token
  const int rows = min(kMoveThreads / per, kMoveBatch);  // tokens the CTA's threads cover at once
  const int i0 = (int)threadIdx.x / per, e0 = (int)threadIdx.x % per;
  const int c = c0 + e0 % (c1 - c0);
  const bool idle = i0 >= rows;                          // per does not divide the threads
  uint8_t* col = base + (int64_t)(h + (turn ? 0 : e0 / (c1 - c0))) * L.head_stride + c * 16;
  const int pair_off = p.rot_vecs * 16;                  // NeoX: to the other half
  const int reps = turn && BYHEAD ? 1 : min(turn ? U : kMoveVecs, kMoveBatch / rows);  // tokens of a thread
  const int batch = rows * reps;                         // tokens of a batch

  // Places of the next chunk of tokens, [ready, ready + kMoveTokens / 2).
  int ready = 0;
  auto places = [&]() {
    for (int i = ready + (int)threadIdx.x; i < min(ready + kMoveTokens / 2, count); i += kMoveThreads) {
      const int from = __ldg(&idx[i]), to = sg.dst + i;
      uint2 pl = make_uint2(kStays, 0);
      // a list that does not ascend, or would move a token up, is not moved in place
      if (from < to || (i > 0 && __ldg(&idx[i - 1]) >= from)) {
        atomicOr(p.err, DEV_ERR_INDEX_RANGE);
      } else if (from != to) {
        int64_t off[2] = {-1, -1};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = e ? to : from;
          const int pg = (int)fdiv((uint32_t)pos, p.page_div);
          if (sg.blk_off + pg >= p.table_numel) {
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
        const bool in = !p.rotate || (from < p.max_pos && to < p.max_pos);
        if (!in) atomicOr(p.err, DEV_ERR_TABLE_RANGE);
        if (off[0] >= 0 && off[1] >= 0 && in)  // both planes or neither
          pl = make_uint2((uint32_t)(off[0] >> 4), (uint32_t)(off[1] >> 4));
      }
      s_at[i % kMoveTokens] = pl;
      s_from[i % kMoveTokens] = from;
    }
    ready += kMoveTokens / 2;
    __syncthreads();
  };
  // place of the token of vector u in batch w
  auto place = [&](int w, int u) {
    const int i = w + i0 + u * rows;
    return i < count && u < reps && !idle ? s_at[i % kMoveTokens] : make_uint2(kStays, 0);
  };
  auto load = [&](int w, int stage) {
    uint4* slot = ring + stage * (kMoveVecs * kMoveThreads);
    if (turn && BYHEAD) {
      const uint2 at = place(w, 0);
      if (at.x != kStays) {
        const uint8_t* src = col + (int64_t)at.x * 16;
#pragma unroll
        for (int u = 0; u < U; ++u, src += L.head_stride) {
          if (u < heads) {
            cp16(smem_u32(slot + u * kMoveThreads), src, true);
            if (NEOX) cp16(smem_u32(slot + (u + U) * kMoveThreads), src + pair_off, true);
          }
        }
      }
    } else {
      constexpr int N = kMoveVecs;
      uint2 at[N];
#pragma unroll
      for (int u = 0; u < N; ++u) at[u] = turn && u >= U ? make_uint2(kStays, 0) : place(w, u);
#pragma unroll
      for (int u = 0; u < N; ++u)
        if (at[u].x != kStays) {
          const uint8_t* src = col + (int64_t)at[u].x * 16;
          cp16(smem_u32(slot + u * kMoveThreads), src, true);
          if (NEOX && u < U && turn) cp16(smem_u32(slot + (u + U) % N * kMoveThreads), src + pair_off, true);
        }
    }
    cp_commit();
  };
  TurnEntries<TE, NF> te;
  auto entries = [&](int w) {  // of the batch's token, ahead of their use
    const int i = w + i0;
    if (turn && BYHEAD && place(w, 0).x != kStays)
      te.load(L.table, p.table_row, p.half_rot, s_from[i % kMoveTokens], sg.dst + i, c * NF);
  };
  places();
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) load(k * batch, k);
  entries(0);
  int stage = 0;
  for (int w = 0; w < count; w += batch) {
    if (w + ST * batch > ready && ready < count) places();
    load(w + (ST - 1) * batch, stage == 0 ? ST - 1 : stage - 1);
    cp_wait<ST - 1>();
    // Every load of this batch is done before its stores; the sources of
    // the batches under way are behind all its destinations.
    __syncthreads();
    const uint4* slot = ring + stage * (kMoveVecs * kMoveThreads);
    if (turn && BYHEAD) {
      const uint2 at = place(w, 0);
      float C[NF], S[NF];
      te.factors(C, S);
      entries(w + batch);
      if (at.x != kStays) {
        uint8_t* dst = col + (int64_t)at.y * 16;
#pragma unroll
        for (int u = 0; u < U; ++u, dst += L.head_stride) {
          if (u < heads) {
            uint4 a = slot[u * kMoveThreads];
            if constexpr (NEOX) {
              uint4 b = slot[(u + U) * kMoveThreads];
              turn_neox<E, NF>(C, S, a, b);
              dev::st_vec(dst + pair_off, b);
            } else {
              turn_gptj<E, NF>(C, S, a);
            }
            dev::st_vec(dst, a);
          }
        }
      }
    } else if (turn) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint2 at = place(w, u);
        if (at.x == kStays) continue;
        const int i = w + i0 + u * rows;
        float C[NF], S[NF];
        te.load(L.table, p.table_row, p.half_rot, s_from[i % kMoveTokens], sg.dst + i, c * NF);
        te.factors(C, S);
        uint8_t* dst = col + (int64_t)at.y * 16;
        uint4 a = slot[u * kMoveThreads];
        if constexpr (NEOX) {
          uint4 b = slot[(u + U) * kMoveThreads];
          turn_neox<E, NF>(C, S, a, b);
          dev::st_vec(dst + pair_off, b);
        } else {
          turn_gptj<E, NF>(C, S, a);
        }
        dev::st_vec(dst, a);
      }
    } else {
      uint2 at[kMoveVecs];
      uint4 a[kMoveVecs];
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u) {
        at[u] = place(w, u);
        a[u] = slot[u * kMoveThreads];
      }
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u)
        if (at[u].x != kStays) dev::st_vec(col + (int64_t)at[u].y * 16, a[u]);
    }
    stage = stage + 1 == ST ? 0 : stage + 1;
  }
  cp_wait<0>();
}

template <class T, int D, int M>
void weights_m(const ScoresLaunch& p, cudaStream_t s) {
  const int64_t cap = (int64_t)p.sq.table_cols * p.kv.page_size;
  // eight rounds of keys per CTA where that still leaves several CTAs per SM
  int iters = 8;
  auto ctas = [&](int n) { return (cap + 16 * M * kSW * n - 1) / (16 * M * kSW * n) * p.sq.num_seqs * p.kv.heads; };
  while (iters > 1 && ctas(iters) < 8 * (int64_t)p.sm_count) iters /= 2;
  const unsigned tiles = (unsigned)((cap + 16 * M * kSW * iters - 1) / (16 * M * kSW * iters));
  weight_kernel<T, D, M><<<dim3((unsigned)p.sq.num_seqs, tiles, (unsigned)p.kv.heads), kSW * 32, 0, s>>>(p, iters);
  DARIC_CUDA(cudaGetLastError());
}

template <class T, int D>
void scores_d(const ScoresLaunch& p0, cudaStream_t s) {
  ScoresLaunch p = p0;
  if (!p.lse) {
    const int64_t items = (int64_t)p.sq.num_rows * p.kv.heads * p.sq.group;
    lse_kernel<T, D><<<dim3((unsigned)p.sq.num_seqs, (unsigned)p.splits, (unsigned)p.kv.heads), kSW * 32, 0, s>>>(p);
    DARIC_CUDA(cudaGetLastError());
    lse_join_kernel<<<(unsigned)((items + 7) / 8), 256, 0, s>>>(p, items);
    DARIC_CUDA(cudaGetLastError());
    p.lse = p.lse_work;
    p.lse_row = (int64_t)p.kv.heads * p.sq.group;
  }
  // few query rows: small tiles, all of them key bytes in flight; many: twice
  // the keys per pass over the rows
  const int64_t pairs = (int64_t)(p.sq.num_rows + p.sq.num_seqs - 1) / p.sq.num_seqs * p.sq.group;
  if (pairs <= 16) weights_m<T, D, 1>(p, s);
  else weights_m<T, D, 2>(p, s);
}

template <class E, class TE, bool NEOX, bool BYHEAD>
void compact_one(const CompactLaunch& p, dim3 grid, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  allow_smem(compact_kernel<E, TE, NEOX, BYHEAD>, kMoveSmem, done);
  compact_kernel<E, TE, NEOX, BYHEAD><<<grid, kMoveThreads, kMoveSmem, s>>>(p);
  DARIC_CUDA(cudaGetLastError());
}

template <class E, class TE>
void compact_et(const CompactLaunch& p, dim3 grid, cudaStream_t s) {
  if (p.neox) return p.per_head ? compact_one<E, TE, true, false>(p, grid, s) : compact_one<E, TE, true, true>(p, grid, s);
  p.per_head ? compact_one<E, TE, false, false>(p, grid, s) : compact_one<E, TE, false, true>(p, grid, s);
}

template <class E>
void compact_e(const CompactLaunch& p, int tab, dim3 grid, cudaStream_t s) {
  using namespace dev;
  if (tab == DARIC_DTYPE_F32) return compact_et<E, Elem<DARIC_DTYPE_F32>>(p, grid, s);
  if (tab == DARIC_DTYPE_BF16) return compact_et<E, Elem<DARIC_DTYPE_BF16>>(p, grid, s);
  compact_et<E, Elem<DARIC_DTYPE_F16>>(p, grid, s);
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

void launch_compact(CompactLaunch& p, int kv_dtype, int tab_dtype, int elem, int sm_count, cudaStream_t s) {
  // Pieces of the rows. A CTA (one to an SM) keeps one piece, up to four whole
  // heads. What counts first is (waves of CTAs) x (size of a piece), then that
  // pieces are large: the rows of a token's heads lie together, and their
  // DRAM pages are opened once. Column slices of 64 bytes or more (whole
  // sectors) are for launches of few lists.
  const int64_t lists = (int64_t)p.num_segs * p.num_layers;
  const int row = p.head_dim * elem, half = p.half_rot * elem;
  const bool tail = p.rotate && 2 * p.half_rot < p.head_dim;
  const int planes = p.rotate ? (tail ? 2 : 1) : 2;
  double best = 1e30;
  for (int heads = p.per_head ? 1 : 4; heads >= 1; heads /= 2)
    for (int slices = 1; slices <= 4; slices *= 2) {
      if (slices > 1 && row / slices < 64) break;
      if (row / 16 / slices * heads > kMoveThreads) continue;
      const int groups = (p.heads + heads - 1) / heads;
      const int turn = p.rotate ? groups * slices : 0;
      const int64_t ctas = (turn + (int64_t)planes * groups * slices) * lists;
      const double cost = (double)((ctas + sm_count - 1) / sm_count) * heads / slices;
      if (cost < 0.8 * best) {
        best = cost;
        p.turn_heads = p.move_heads = heads;
        p.turn_slices = p.slices = slices;
        p.turn_pieces = turn;
      }
    }
  const int groups = (p.heads + p.move_heads - 1) / p.move_heads;
  p.vecs = row / 16;
  p.rot_vecs = p.rotate ? half / 16 * (p.neox ? 1 : 2) : 0;
  p.tail0 = p.rotate ? 2 * half / 16 : 0;
  const dim3 grid((unsigned)(p.turn_pieces + planes * groups * p.slices), (unsigned)p.num_segs, (unsigned)p.num_layers);
  if (!p.rotate) {  // bytes only: one kernel for every dtype
    return compact_one<dev::Elem<DARIC_DTYPE_BF16>, dev::Elem<DARIC_DTYPE_F32>, true, true>(p, grid, s);
  }
  switch (kv_dtype) {
    case DARIC_DTYPE_BF16: return compact_e<dev::Elem<DARIC_DTYPE_BF16>>(p, tab_dtype, grid, s);
    case DARIC_DTYPE_F16: return compact_e<dev::Elem<DARIC_DTYPE_F16>>(p, tab_dtype, grid, s);
    case DARIC_DTYPE_F32: return compact_e<dev::Elem<DARIC_DTYPE_F32>>(p, tab_dtype, grid, s);
    case DARIC_DTYPE_FP8_E4M3: return compact_e<dev::Elem<DARIC_DTYPE_FP8_E4M3>>(p, tab_dtype, grid, s);
  }
  throw Error(DARIC_ERR_INVALID, "compact: unknown KV dtype");
}

}  // namespace daric
