// Eviction from the paged KV cache: the move of the kept tokens to the front of
// their blocks.
//
// Kept token n of a list, position i_n (ascending), moves to position dst + n.
// Since i_n >= dst + n, a destination is never behind the source of a later
// token, so one CTA that goes through the tokens in order and loads each batch
// before it stores it moves them in place; the parallelism is over layers,
// segments, heads, the K and V planes and slices of the row. Keys turn by
// (new - old): C = nc oc + ns os, S = ns oc - nc os from the table rows of both
// positions, in fp32 (a product and a fused multiply-add each), and the turned
// key is rounded once to the cache's type.
// Bound: the bytes of the tokens that move, read and written once (32 layers,
// 8 KV heads of 128, bf16, 40 % of 8192 tokens, keys turned: 175 us, 5.0 TB/s;
// few short lists: the chain of a segment's batches, one layer of 6001 tokens
// in 27 us).
#include "attend_common.cuh"
#include "device_common.cuh"

#include <algorithm>
#include <type_traits>

namespace daric {
namespace {
using namespace att;

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

  // Places of the next chunk of tokens, [ready, ready + kMoveTokens / 2), in
  // three steps, each a batch after the one before, so that no load is waited
  // for: list entries, block ids, places.
  constexpr int CT = kMoveTokens / 2 / kMoveThreads;  // tokens of a thread in a chunk
  constexpr int kNoTable = -0x7fffffff - 1;           // a block id of no table entry
  const int64_t table_len = p.table_numel - sg.blk_off;  // entries of this segment's table: the offset may be any
  int ready = 0, step = 0;
  int from_of[CT], prev_of[CT], blk_of[CT][2];
  auto entries_of = [&]() {
#pragma unroll
    for (int k = 0; k < CT; ++k) {
      const int i = ready + (int)threadIdx.x + k * kMoveThreads;
      from_of[k] = i < count ? ld_ahead(&idx[i]) : 0;
      prev_of[k] = i < count && i > 0 ? ld_ahead(&idx[i - 1]) : -1;
    }
  };
  auto blocks_of = [&]() {
#pragma unroll
    for (int k = 0; k < CT; ++k) {
      const int i = ready + (int)threadIdx.x + k * kMoveThreads, to = sg.dst + i;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int pos = e ? to : from_of[k];
        const int pg = (int)fdiv((uint32_t)pos, p.page_div);
        blk_of[k][e] = i < count && from_of[k] > to && pg < table_len ? ld_ahead(&p.block_table[sg.blk_off + pg]) : kNoTable;
      }
    }
  };
  auto places = [&]() {
#pragma unroll
    for (int k = 0; k < CT; ++k) {
      const int i = ready + (int)threadIdx.x + k * kMoveThreads;
      if (i >= count) break;
      const int from = from_of[k], to = sg.dst + i;
      uint2 pl = make_uint2(kStays, 0);
      // a list that does not ascend, or would move a token up, is not moved in place
      if (from < to || prev_of[k] >= from) {
        atomicOr(p.err, DEV_ERR_INDEX_RANGE);
      } else if (from != to) {
        int64_t off[2] = {-1, -1};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = e ? to : from;
          const int pg = (int)fdiv((uint32_t)pos, p.page_div);
          const int blk = blk_of[k][e];
          if (blk == kNoTable && pg >= table_len) {
            atomicOr(p.err, DEV_ERR_INDEX_RANGE);
            continue;
          }
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
  entries_of();
  blocks_of();
  places();
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) load(k * batch, k);
  entries(0);
  int stage = 0;
  for (int w = 0; w < count; w += batch) {
    if (ready < count) {
      if (step == 0 && w + (ST + 2) * batch > ready) {
        entries_of();
        step = 1;
      } else if (step == 1) {
        blocks_of();
        step = 2;
      }
      if (w + ST * batch > ready) {  // a short way, where the first batches already reach here
        if (step == 1) blocks_of();
        places();
        step = 0;
      }
    }
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
  // NeoX pairs the two halves (whole vectors each); GPT-J neighbours, so there
  // the halves together are whole vectors
  p.rot_vecs = !p.rotate ? 0 : (p.neox ? half / 16 : 2 * half / 16);
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
