// Attention of many query rows over the paged KV cache on the tensor cores.
//
// The mathematics and the split of the work are those of attend_kernels.cu;
// here a CTA holds MT = 1 or 2 tiles of 128 (query row, query head) pairs of
// one KV head and passes tiles of 128 keys by them:
//   S = Q K^T   tcgen05.mma, Q and K from shared memory, S in tensor memory
//   P = 2^((S - m) c) by one thread per row, rounded to the cache's type and
//       written over S in tensor memory (half a step: relative 2^-8 bf16, 2^-11
//       fp16 per weight; l sums the unrounded values; fp16 weights carry a
//       factor of 2^7, which cancels at the end, so that they keep their
//       precision down to 2^-21 and vanish below 2^-32)
//   O += P V    tcgen05.mma, P from tensor memory, V from shared memory in the
//       layout it was copied in (its rows are the summed dimension)
// m is the maximum when it was last moved: it moves, and O and l are rescaled,
// only when the running maximum is over 2^8 times ahead, so that O is rarely
// read back (weights are 2^8 at most, times the factor 2^15). m, l, S and O are fp32.
//
// Two streams of (scores, weights, output) take turns, so that one is
// multiplied while the other is exponentiated: with MT = 2 the two row tiles,
// with MT = 1 the even and the odd key tiles, whose two outputs are joined at
// the end of a segment. Warps: four of softmax per stream, one thread a row;
// four that copy; one that issues the matrix instructions. A copy slot is a K
// or a V tile (16-byte cp.async, a page table lookup per key, into the
// 128-byte swizzle); each copying thread reports a slot when its own copies of
// it have landed, some slots behind the newest.
//
// Bound: the K and V bytes, their copies and latency with one tile (16
// sequences x 16 drafted rows x 4 heads at 8K: 115 us, 4.1 TB/s of K and V; 512
// rows that list 64 of 512 pages each, from L2: 166 us); with two, per stream
// the chain of product, exponentials, product (8 sequences of 512 pairs at 32K:
// 92 us, 0.57 PFLOP/s; 2048 appended rows of a prompt of 8192, 8 heads of 4: 403
// us, 0.60). One group copies all slots in order and one warp
// issues all products in order, so that every wait is for the phase next to
// the one its barrier is in, which is all that parity can tell. Why tcgen05 and not the warp matrix
// instructions here: from 33 pairs on those need more time per key than its
// bytes do.
#include "attend_common.cuh"
#include "tensor_common.cuh"

#include <algorithm>
#include <type_traits>

namespace daric {
namespace {
using namespace att;
using bulk::fence_proxy_async;
using bulk::mbar_arrive;
using bulk::mbar_init;
using bulk::mbar_init_fence;
using bulk::mbar_try_wait;
using bulk::mbar_wait;

constexpr int kKeys = 128;      // keys of a tile
constexpr int kMaskRing = 8;    // tiles whose key masks are kept
constexpr int kCopyThreads = 128;
// A wait gives up after five seconds, not the copy kernels' 200 ms: the other
// roles wait while the softmax warps put values back that are not finite, which
// takes as long as there are such values.
constexpr uint64_t kLongWaitNs = 5000000000ull;
static_assert(kLongWaitNs >= bulk::kWaitNs, "mbar_wait polls as often as it does for its default limit");

template <int D, int MT, bool SPARSE>
struct Wide {
  static constexpr int ROWS = 128 * MT;
  static constexpr int SLOT = kKeys * D * 2;
  static constexpr int QB = ROWS * D * 2;
  static constexpr int NS = D == 64 ? 10 : (MT == 2 || SPARSE ? 5 : 6);
  static constexpr int BEHIND = NS > 5 ? 3 : 2;  // slots copied but not reported yet
  static constexpr int THREADS = 512;  // the last three warps only lend their registers
  static constexpr int COPY_WARP = 8;
  static constexpr int MMA_WARP = 12;
  static constexpr int TILES = QB + NS * SLOT;
};

struct WideShared {
  uint64_t full[10], empty[10];
  uint64_t s_full[2], p_full[2], pv_done[2], o_empty[2];
  uint64_t q_full, q_empty, ml_full;
  uint64_t drained;        // every product that was issued has completed
  float2 ml[128];          // MT = 1: maximum and sum of the odd key tiles
  uint32_t vmask[kMaskRing][4];
  uint32_t off[3][kKeys];  // row offsets of three key tiles, 16-byte units of the layer
  uint32_t tmem;
  int abort;               // a wait gave up: everyone leaves
  int poison[4];           // by count modulo 4: the segment if its drafted V rows hold infinities or NaN
};
// SPARSE: which of a tile's (up to) 32 query rows see each of its keys.
struct SparseShared {
  uint32_t vis[kMaskRing][32][4];
};
template <int D, int MT, bool SPARSE>
constexpr int wide_smem() {
  return Wide<D, MT, SPARSE>::TILES + (int)sizeof(WideShared) + (SPARSE ? (int)sizeof(SparseShared) : 0);
}

// Weights may be 2^kLag: how far a row's maximum may run ahead of m.
constexpr float kLag = 8.f;
template <class T>
constexpr int kWideLift = Mma<T>::kLift ? Mma<T>::kLift - (int)kLag : 0;

// The part of a segment that a CTA works on.
struct Part {
  int b, h, rt, tile0, n, ntiles;
  Seq s;
  int row_base, my_rows;  // first pair of the row tile, and pairs that exist
  int listed;             // SPARSE: pages of the tile's list
  const uint4* list;      // SPARSE: page, rows of the tile that see it, block
};

template <class T, int D, int MT, bool SPARSE>
__global__ void __launch_bounds__(512, 1) wide_kernel(const __grid_constant__ AttendLaunch p) {
  using W = Wide<D, MT, SPARSE>;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr int HB = D / 64;          // 64-element halves of a row
  constexpr int HALF = kKeys * 128;   // bytes of such a half of a tile
  constexpr int LIFT = kWideLift<T>;
  extern __shared__ __align__(1024) uint8_t base[];  // the only shared memory: it starts on 1024 bytes
  WideShared& sh = *reinterpret_cast<WideShared*>(base + W::TILES);
  SparseShared& sp = *reinterpret_cast<SparseShared*>(base + W::TILES + sizeof(WideShared));
  uint8_t* q_tile = base;
  uint8_t* slots = base + W::QB;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.sq.group;
  grid_next();

  // ---- the line of tiles and this CTA's part of it (as in attend_kernels.cu)
  uint32_t* sums = reinterpret_cast<uint32_t*>(slots);  // before any copy
  // units of the line: sequences, or (SPARSE) the lists of a row tile and head
  const int units = SPARSE ? p.lists : p.sq.num_seqs;
  const int per = (units + W::THREADS - 1) / W::THREADS;
  auto tiles_of = [&](const Seq& s) { return max((s.len + kKeys - 1) / kKeys, 1); };
  auto list_tiles = [&](int i) {  // 0: no such row tile
    const int n = p.list_count[i];
    return n < 0 ? 0 : max((int)(((int64_t)n * p.kv.page_size + kKeys - 1) / kKeys), 1);
  };
  auto tiles_seq = [&](const Seq& s) {
    return ((uint32_t)(s.rows * group) + W::ROWS - 1) / W::ROWS * (uint32_t)p.kv.heads * (uint32_t)tiles_of(s);
  };
  {
    uint32_t mine = 0;
    if (SPARSE) grid_wait();  // the lists are there
    for (int i = tid * per; i < min((tid + 1) * per, units); ++i) {
      if (SPARSE) {
        mine += (uint32_t)list_tiles(i);
      } else {
        Seq s = load_seq(p.sq, i);
        clamp_len(p.sq, p.kv.page_size, s);
        mine += tiles_seq(s);
      }
    }
    sums[tid] = mine;
    __syncthreads();
    for (int o = 1; o < W::THREADS; o <<= 1) {
      const uint32_t v = tid >= o ? sums[tid - o] : 0;
      __syncthreads();
      sums[tid] += v;
      __syncthreads();
    }
  }
  const uint32_t total = sums[W::THREADS - 1];
  uint32_t t0, t1;
  split_range(total, gridDim.x, blockIdx.x, t0, t1);
  int b = 0;
  uint32_t seg_at = 0;
  if (t0 < t1) {
    int lo = 0, hi = W::THREADS - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] > t0) hi = mid; else lo = mid + 1;
    }
    b = lo * per;
    seg_at = lo ? sums[lo - 1] : 0;
  }
  if (tid == 0) {
    p.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (smem_u32(base) & 1023) atomicOr(p.sq.err, DEV_ERR_TIMEOUT);
    for (int i = 0; i < W::NS; ++i) {
      mbar_init(&sh.full[i], kCopyThreads);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 128);
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.o_empty[i], 128);
    }
    mbar_init(&sh.q_full, kCopyThreads);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.ml_full, 128);
    mbar_init(&sh.drained, 1);
    mbar_init_fence();
    sh.abort = 0;
    for (int i = 0; i < 4; ++i) sh.poison[i] = -1;
  }
  __syncthreads();  // sums are read, barriers are ready
  if (t0 >= t1 || (smem_u32(base) & 1023)) return;
  if (warp == W::MMA_WARP) tc::alloc512(&sh.tmem);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sh.tmem;

  volatile int* abort = &sh.abort;
  // A wait that is out of time ends the kernel: its error bit is set and every role leaves its loop.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (mbar_wait(bar, parity, kLongWaitNs)) return true;
    *abort = 1;
    atomicOr(p.sq.err, DEV_ERR_TIMEOUT);
    return false;
  };
  // Part of the line at tile t; false: none (lengths changed while the kernel ran).
  auto part_at = [&](uint32_t t, Part& g) {
    if constexpr (SPARSE) {
      for (;; ++b) {
        if (b >= units) return false;
        const uint32_t n = (uint32_t)list_tiles(b);
        if (t < seg_at + n) break;
        seg_at += (uint32_t)list_tiles(b);
      }
      const int2 where = p.list_tile[b / p.kv.heads];
      g.b = where.x;
      g.rt = where.y;
      g.h = b % p.kv.heads;
      g.s = load_seq(p.sq, g.b);
      clamp_len(p.sq, p.kv.page_size, g.s);
      g.ntiles = list_tiles(b);
      g.listed = p.list_count[b];
      g.list = p.list + (int64_t)b * p.list_row;
      g.tile0 = (int)(t - seg_at);
    } else {
      for (;; ++b) {
        if (b >= p.sq.num_seqs) return false;
        g.s = load_seq(p.sq, b);
        clamp_len(p.sq, p.kv.page_size, g.s);
        const uint32_t n = tiles_seq(g.s);
        if (t < seg_at + n) break;
        seg_at += n;
      }
      uint32_t x = t - seg_at;
      g.ntiles = tiles_of(g.s);
      g.tile0 = (int)(x % (uint32_t)g.ntiles);
      x /= (uint32_t)g.ntiles;
      const int rts = (g.s.rows * group + W::ROWS - 1) / W::ROWS;
      g.rt = (int)(x % (uint32_t)rts);
      g.h = (int)(x / (uint32_t)rts);
      g.b = b;
    }
    g.n = (int)min((uint32_t)(g.ntiles - g.tile0), t1 - t);
    g.row_base = g.rt * W::ROWS;
    g.my_rows = min(W::ROWS, g.s.rows * group - g.row_base);
    return true;
  };
  // First position of the drafted part that some row of the tile does not
  // see: tiles that end at or before it need no mask but that of their keys.
  auto all_see = [&](const Part& g) {
    if (p.sq.mask) return g.s.ctx;
    return g.s.ctx + (int)fdiv((uint32_t)g.row_base, p.sq.group_div) + 1;
  };
  // items of stream s in a part of n key tiles, and the key tile of its local item
  auto items_of = [&](int s, int n) { return MT == 2 ? n : (n + 1 - s) / 2; };

  if (warp >= W::COPY_WARP && warp < W::MMA_WARP) {
    // ------------------------------------------------------------ copies --
    // Registers: 512 threads start with 128 each, 65536 in all; 256 x 176 of
    // softmax + 128 x 80 here + 128 x 80 = 65536.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    const int ct = tid - W::COPY_WARP * 32;
    uint32_t n_slot = 0, n_seg = 0, n_tile = 0;  // slots, segments, key tiles so far
    constexpr int BH = W::BEHIND;
    constexpr int CH = D / 8, RPI = kCopyThreads / CH;  // vectors of a row, rows at a time
    uint64_t* pend[BH];                          // groups not reported yet, older first
    int pend_v[BH], pend_seg[BH];                // SPARSE: their slot if it is a V tile, and the segment
#pragma unroll
    for (int i = 0; i < BH; ++i) pend[i] = nullptr;
    // V rows that some rows must not see: values without a finite size would
    // reach them through 0 * inf. They are taken out here and added where
    // they are seen, at the end of the segment.
    auto take_out = [&](int st, uint32_t seg) {
      const int c = ct % CH, r0 = ct / CH;
      uint8_t* tile = slots + st * W::SLOT + (c >> 3) * HALF;
      auto vec = [&](int k) {
        const int r = r0 + k * RPI;
        return reinterpret_cast<uint4*>(tile + r * 128 + (((c & 7) ^ (r & 7)) << 4));
      };
      // x * 0 summed up: 0, or NaN where some x is not finite
      uint32_t sum = 0;
#pragma unroll
      for (int k0 = 0; k0 < kKeys / RPI; k0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = *vec(k0 + k);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          sum = Mma<T>::zero_sum(x[k].x, Mma<T>::zero_sum(x[k].y, Mma<T>::zero_sum(x[k].z, Mma<T>::zero_sum(x[k].w, sum))));
      }
      if ((sum & 0x7fff7fffu) == 0) return;
      for (int k = 0; k < kKeys / RPI; ++k) {
        uint16_t* v = reinterpret_cast<uint16_t*>(vec(k));
        for (int e = 0; e < 8; ++e)
          if ((v[e] & Mma<T>::kExpMask) == Mma<T>::kExpMask) v[e] = 0;
      }
      *(volatile int*)&sh.poison[seg & 3] = (int)seg;
    };
    auto report = [&](uint64_t* bar, int v_slot_of, int seg) {
      if (!bar) return;
      if (SPARSE && v_slot_of >= 0) take_out(v_slot_of, (uint32_t)seg);
      fence_proxy_async();
      mbar_arrive(bar);
    };
    auto flush = [&]() {
      cp_wait<0>();
#pragma unroll
      for (int i = 0; i < BH; ++i) {
        report(pend[i], pend_v[i], pend_seg[i]);
        pend[i] = nullptr;
      }
    };
    auto push = [&](uint64_t* bar, int v) {  // a group was issued: reports the one BH before it
      cp_commit();
      cp_wait<BH>();
      report(pend[0], pend_v[0], pend_seg[0]);
#pragma unroll
      for (int i = 0; i + 1 < BH; ++i) {
        pend[i] = pend[i + 1];
        pend_v[i] = pend_v[i + 1];
        pend_seg[i] = pend_seg[i + 1];
      }
      pend[BH - 1] = bar;
      pend_v[BH - 1] = v;
      pend_seg[BH - 1] = (int)n_seg;
    };
    auto take = [&](uint64_t* bar, uint32_t parity) {  // what is reported late must not be waited for
      if (tc::mbar_test(bar, parity)) return true;
      flush();
      return wait(bar, parity);
    };
    // The copying threads go on or stop together: what each found, for all.
    auto together = [&](bool mine) {
      uint32_t all;
      __syncwarp();
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
          : "=r"(all)
          : "r"((uint32_t)mine), "n"(kCopyThreads)
          : "memory");
      return all != 0;
    };
    uint32_t t = t0;
    bool ok = true;
    while (ok && t < t1) {
      Part g;
      if (!together(part_at(t, g))) break;  // the same for all: they read the same lengths
      const int32_t* trow = p.sq.table + (int64_t)g.b * p.sq.table_ld;
      const uint8_t* kv = p.kv.base + (int64_t)g.h * p.kv.head_stride;
      const int see = all_see(g);
      // query rows
      if (n_seg) ok = together(take(&sh.q_empty, (n_seg - 1) & 1));
      if (!ok) break;
      {
        for (int v = ct; v < W::ROWS * CH; v += kCopyThreads) {
          const int r = v / CH, c = v % CH, i = g.row_base + r;
          const bool in = r < g.my_rows;
          const int j = (int)fdiv((uint32_t)i, p.sq.group_div);
          const uint8_t* src = in ? p.q + (int64_t)(g.s.row0 + j) * p.q_row +
                                        (int64_t)(g.h * group + i - j * group) * p.q_head + c * 16
                                  : p.q;
          const uint32_t dst = smem_u32(q_tile) + (r >> 7) * (HB * HALF) + (c >> 3) * HALF + (r & 127) * 128 +
                               (((c & 7) ^ (r & 7)) << 4);
          cp16(dst, src, in);
        }
        push(&sh.q_full, -1);
      }
      // this thread's key of the next tile: block (-1: none), position, and
      // (SPARSE) the rows of the tile that list its page
      int blk = -1, pos = 0;
      uint32_t rows_see = 0;
      const int j_first = SPARSE ? (int)fdiv((uint32_t)g.row_base, p.sq.group_div) : 0;
      auto lookup = [&](int i) {
        const int k = (g.tile0 + i) * kKeys + ct;
        blk = -1;
        pos = 0x7fffffff;
        if (i >= g.n) return;
        if (SPARSE) {
          const int e = (int)fdiv((uint32_t)k, p.kv.page_div);
          rows_see = 0;
          if (e < g.listed) {
            const int4 x = ld_ahead(reinterpret_cast<const int4*>(g.list + e));
            pos = x.x * p.kv.page_size + k - e * p.kv.page_size;
            rows_see = (uint32_t)x.y;
            blk = x.z;
          }
        } else {
          pos = k;
          if (k < g.s.len) blk = ld_ahead(&trow[fdiv((uint32_t)k, p.kv.page_div)]);
        }
      };
      lookup(0);
      auto place = [&](int i) {  // offsets and masks of tile i; looks the next one up
        bool in = pos < g.s.len;
        if (in && (blk < 0 || blk >= p.kv.num_pages)) {
          atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
          in = false;
        }
        int64_t off = 0;
        if (in) {
          const int pg = (int)fdiv((uint32_t)pos, p.kv.page_div);
          off = (int64_t)blk * p.kv.page_stride + (int64_t)(pos - pg * p.kv.page_size) * p.kv.tok_stride;
        }
        if (SPARSE) {
          // rows at or behind the position see it; then turned over: a word of
          // 32 keys for each row
          const int before = pos - g.s.ctx - j_first;  // rows of the tile that stand before it
          const uint32_t m = !in || before >= 32 ? 0u : (before <= 0 ? rows_see : rows_see & (0xffffffffu << before));
          uint32_t mine = m;  // lane: key, bit: row; then lane: row, bit: key
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const uint32_t lo = o == 16 ? 0x0000ffffu : o == 8 ? 0x00ff00ffu : o == 4 ? 0x0f0f0f0fu : o == 2 ? 0x33333333u : 0x55555555u;
            const uint32_t y = __shfl_xor_sync(0xffffffffu, mine, o);
            mine = (lane & o) ? (mine & ~lo) | ((y >> o) & lo) : (mine & lo) | ((y << o) & ~lo);
          }
          sp.vis[(n_tile + i) % kMaskRing][lane][ct >> 5] = mine;
        } else {
          const unsigned m = __ballot_sync(0xffffffffu, in);
          if (lane == 0) sh.vmask[(n_tile + i) % kMaskRing][ct >> 5] = m;
        }
        sh.off[i % 3][ct] = in ? (uint32_t)(off >> 4) : 0xffffffffu;
        lookup(i + 1);
        // The offsets of the tile three before this one are read by now: its
        // last copies were issued before the meeting of the tile in between.
        ok = together(ok);
      };
      auto copy = [&](int i, bool v_tile) {
        const uint32_t st = n_slot % W::NS, use = n_slot / W::NS;
        if (!ok) return;
        if (use) ok = take(&sh.empty[st], (use - 1) & 1);
        if (!ok) return;  // all stop at the next meeting
        const int c = ct % CH;
        const uint8_t* src = kv + (v_tile ? p.kv.v_off : 0) + c * 16;
        const uint32_t dst = smem_u32(slots) + st * W::SLOT + (c >> 3) * HALF;
        const uint32_t* off = sh.off[i % 3];
        uint32_t o[kKeys / RPI];  // read ahead of the copies, which nothing is moved across
#pragma unroll
        for (int k = 0; k < kKeys / RPI; ++k) o[k] = off[ct / CH + k * RPI];
        const uint32_t d0 = dst + (ct / CH) * 128;
#pragma unroll
        for (int k = 0; k < kKeys / RPI; ++k) {
          const bool in = o[k] != 0xffffffffu;
          const int r7 = (ct / CH + k * RPI) & 7;
          cp16(d0 + k * RPI * 128 + (((c & 7) ^ r7) << 4), src + (in ? (int64_t)o[k] * 16 : 0), in);
        }
        if (!SPARSE && v_tile && (g.tile0 + i + 1) * kKeys > see) {
          cp_commit();
          cp_wait<0>();
          take_out((int)st, n_seg);
        }
        push(&sh.full[st], v_tile ? (int)st : -1);
        ++n_slot;
      };
      // Order of the slots: K0 V0 K1 V1 ..., with one row tile K0 K1 V0 K2 V1
      // ... (the next scores are under way while a tile is exponentiated).
      if (MT == 2) {
        for (int i = 0; i < g.n; ++i) {
          place(i);
          if (!ok) break;
          copy(i, false);
          copy(i, true);
        }
      } else {
        place(0);
        copy(0, false);
        for (int i = 1; i < g.n; ++i) {
          place(i);
          if (!ok) break;
          copy(i, false);
          copy(i - 1, true);
        }
        copy(g.n - 1, true);
      }
      ok = together(ok);
      n_tile += (uint32_t)g.n;
      ++n_seg;
      t += (uint32_t)g.n;
    }
    flush();
    cp_wait<0>();
  } else if (warp >= W::MMA_WARP) {
    // ---------------------------------------------------------- products --
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == W::MMA_WARP) {
      constexpr uint32_t id_qk = tc::instr_desc(BF, false, 128, kKeys), id_pv = tc::instr_desc(BF, true, 128, D);
      // The tensor pipe runs dry while this warp does anything else, so the
      // loop is kept short: ring places move by addition, a slot is waited
      // for once.
      uint32_t at = 0, at_par = 0;  // slot of the segment's first tile and its parity
      uint32_t n_seg = 0;
      uint32_t p_par[2] = {0, 0}, o_par[2] = {0, 0}, o_used = 0;
      const uint64_t q_desc = tc::smem_desc(smem_u32(q_tile), 16), k_desc = tc::smem_desc(smem_u32(slots), 16),
                     v_desc = tc::smem_desc(smem_u32(slots), HALF);
      const uint32_t tm = tc::uniform(tmem);
      auto commit = [&](uint64_t* bar) {
        if (tc::elect()) tc::commit(bar);
      };
      uint32_t t = t0;
      bool ok = true;
      while (ok && t < t1) {
        Part g;
        if (!part_at(t, g)) break;
        const int n = (int)tc::uniform((uint32_t)g.n);
        // a place of the ring: slot and the parity of its use
        struct Place {
          uint32_t st, par;
        };
        auto step = [&](Place& x, uint32_t by) {
          x.st += by;
          if (x.st >= (uint32_t)W::NS) {
            x.st -= W::NS;
            x.par ^= 1;
          }
        };
        Place first{at, at_par};
        auto full = [&](const Place& x) { return __all_sync(0xffffffffu, wait(&sh.full[x.st], x.par)) != 0; };
        auto qk = [&](uint32_t s, const Place& k) {  // scores of stream s with the K tile of a place
          const uint64_t qa = q_desc + (MT == 2 ? s * (uint32_t)(HB * HALF >> 4) : 0u);
          const uint64_t ka = k_desc + tc::uniform(k.st) * (uint32_t)(W::SLOT >> 4);
          if (tc::elect()) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const int o = (i >> 2) * (HALF >> 4) + (i & 3) * (32 >> 4);
              tc::mma_ss(tm + s * kKeys, qa + o, ka + o, id_qk, i > 0);
            }
            tc::commit(&sh.s_full[s]);
          }
        };
        auto pv = [&](uint32_t s, const Place& v, bool add) {
          const uint64_t va = v_desc + tc::uniform(v.st) * (uint32_t)(W::SLOT >> 4);
          if (tc::elect()) {
#pragma unroll
            for (int i = 0; i < kKeys / 16; ++i)
              tc::mma_ts(tm + 2 * kKeys + s * D, tm + s * kKeys + i * 8, va + i * (2048 >> 4), id_pv, add || i > 0);
            tc::commit(&sh.pv_done[s]);
          }
        };
        // weights of a stream are there, and before a segment's first product
        // its output has been read
        auto weights = [&](uint32_t s, bool first_item) {
          if (first_item && ((o_used >> s) & 1)) {
            if (!__all_sync(0xffffffffu, wait(&sh.o_empty[s], o_par[s]))) return false;
            o_par[s] ^= 1;
          }
          if (!__all_sync(0xffffffffu, wait(&sh.p_full[s], p_par[s]))) return false;
          p_par[s] ^= 1;
          tc::fence_after();
          return true;
        };
        ok = __all_sync(0xffffffffu, wait(&sh.q_full, n_seg & 1)) && full(first);
        if (!ok) break;
        tc::fence_after();
        if (MT == 2) {
          Place k = first, v = first;
          step(v, 1);
          qk(0, k);
          qk(1, k);
          commit(&sh.empty[k.st]);
          if (n == 1) commit(&sh.q_empty);
          for (int i = 0; i < n; ++i) {
            const bool more = i + 1 < n;
            step(k, 2);
            ok = full(v) && weights(0, i == 0);
            if (!ok) break;
            pv(0, v, i > 0);
            if (more) {
              ok = full(k);
              if (!ok) break;
              qk(0, k);
            }
            ok = weights(1, i == 0);
            if (!ok) break;
            pv(1, v, i > 0);
            commit(&sh.empty[v.st]);
            if (more) {
              qk(1, k);
              commit(&sh.empty[k.st]);
              if (i + 2 == n) commit(&sh.q_empty);
            }
            step(v, 2);
          }
        } else {
          // K0 K1 V0 K2 V1 ... V(n-1)
          Place k = first, v = first;
          qk(0, k);
          commit(&sh.empty[k.st]);
          if (n > 1) {
            step(k, 1);
            ok = full(k);
            if (!ok) break;
            qk(1, k);
            commit(&sh.empty[k.st]);
          }
          if (n <= 2) commit(&sh.q_empty);
          step(v, n > 1 ? 2 : 1);
          for (int i = 0; i < n; ++i) {
            const uint32_t s = i & 1;
            ok = full(v) && weights(s, i < 2);
            if (!ok) break;
            pv(s, v, i > 1);
            commit(&sh.empty[v.st]);
            if (i + 2 < n) {
              step(k, 2);
              ok = full(k);
              if (!ok) break;
              qk(s, k);
              commit(&sh.empty[k.st]);
              if (i + 3 == n) commit(&sh.q_empty);
            }
            step(v, i + 2 < n ? 2 : 1);
          }
        }
        o_used |= MT == 2 || n > 1 ? 3u : 1u;
        Place nx{at, at_par};
        for (uint32_t left = 2 * (uint32_t)n; left > 0;) {  // 2 n places on
          const uint32_t by = min(left, (uint32_t)W::NS);
          step(nx, by);
          left -= by;
        }
        at = nx.st;
        at_par = nx.par;
        ++n_seg;
        t += (uint32_t)n;
      }
      // Where a wait gave up the softmax leaves without having waited for the
      // last products: they read shared memory and write tensor memory, so
      // this warp stays for them (for a bounded time, too).
      commit(&sh.drained);
      if (!mbar_wait(&sh.drained, 0, kLongWaitNs)) atomicOr(p.sq.err, DEV_ERR_TIMEOUT);
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------- softmax --
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int st = warp >> 2;                              // stream
    const int tile = MT == 2 ? st : 0;                     // row tile of the CTA
    const int r = (warp & 3) * 32 + lane;                  // row of it
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + st * kKeys, o_col = tmem + lanes + 2 * kKeys + st * D;
    const float cexp = p.scale * kLog2e;
    uint32_t done = 0, other = 0;                          // items of this stream, of the other one (MT = 1)
    uint32_t n_seg = 0, n_tile = 0, n_ml = 0;
    uint32_t t = t0;
    bool ok = true;
    while (ok && t < t1) {
      Part g;
      if (!part_at(t, g)) break;
      const int i_pair = tile * 128 + r;
      const bool real = i_pair < g.my_rows;
      const int pi = g.row_base + i_pair;
      const int j = real ? (int)fdiv((uint32_t)pi, p.sq.group_div) : 0;  // row of the sequence
      const int row = g.s.row0 + j, head = g.h * group + pi - j * group;
      const int see = all_see(g);
      const int items = items_of(st, g.n);
      // a row that does not exist has no maximum to wait for
      float m = real ? DARIC_NEG_INF : 0.f, l0 = 0.f, l1 = 0.f;
      const int jl = SPARSE ? j - (int)fdiv((uint32_t)g.row_base, p.sq.group_div) : 0;  // row of the tile
      for (int li = 0; li < items; ++li) {
        const uint32_t c = done + (uint32_t)li;
        const int i = MT == 2 ? li : 2 * li + st;  // key tile
        ok = wait(&sh.s_full[st], c & 1);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc::fence_after();
        const int key0 = (g.tile0 + i) * kKeys;
        const uint32_t* vm = SPARSE ? sp.vis[(n_tile + (uint32_t)i) % kMaskRing][real ? jl : 0]
                                    : sh.vmask[(n_tile + (uint32_t)i) % kMaskRing];
        const bool draft = !SPARSE && key0 + kKeys > see;
        const bool masked = SPARSE || draft || (vm[0] & vm[1] & vm[2] & vm[3]) != 0xffffffffu;
        float mb = m * cexp - (float)LIFT;
        bool careful = (masked && !SPARSE) || __any_sync(0xffffffffu, m == DARIC_NEG_INF);
        if (!careful) {
          // one pass: weights by the maximum so far, kept in registers until
          // the maximum of this tile is known to be near enough
          uint32_t y[64];
          float mx = DARIC_NEG_INF, a0 = 0.f, a1 = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t x[32];
            const uint32_t see_w = SPARSE ? vm[w] : 0;
            tc::ld32(s_col + w * 32, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float u = __uint_as_float(x[2 * e]), v = __uint_as_float(x[2 * e + 1]);
              if (SPARSE) {
                u = see_w & (1u << (2 * e)) ? u : DARIC_NEG_INF;
                v = see_w & (2u << (2 * e)) ? v : DARIC_NEG_INF;
              }
              mx = fmaxf(mx, fmaxf(u, v));
              const float a = exp2_fast(__fmaf_rn(u, cexp, -mb)), d = exp2_fast(__fmaf_rn(v, cexp, -mb));
              a0 += a;
              a1 += d;
              y[w * 16 + e] = Mma<T>::pack(a, d);
            }
          }
          careful = __any_sync(0xffffffffu, (mx - m) * cexp > kLag);
          if (!careful) {
            l0 += a0;
            l1 += a1;
#pragma unroll
            for (int w = 0; w < 2; ++w) tc::st32(s_col + w * 32, *reinterpret_cast<const uint32_t(*)[32]>(&y[w * 32]));
          }
        }
        if (careful) {
          uint32_t vis[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            vis[w] = vm[w];
            if (!draft) continue;
            const int d0 = key0 + 32 * w - g.s.ctx;  // drafted token of bit 0
            uint32_t bits;
            if (d0 <= -32) {
              bits = 0xffffffffu;
            } else if (!real) {
              bits = 0;
            } else if (!p.sq.mask) {
              const int up = j - d0 + 1;  // bits [0, up)
              bits = up <= 0 ? 0u : (up >= 32 ? 0xffffffffu : (1u << up) - 1u);
            } else {
              const int at = max(d0, 0), word = at >> 6, sft = at & 63;
              const uint64_t* mr = p.sq.mask + (int64_t)row * p.sq.mask_words;
              uint64_t x = word < p.sq.mask_words ? __ldg(&mr[word]) >> sft : 0;
              if (sft > 32 && word + 1 < p.sq.mask_words) x |= __ldg(&mr[word + 1]) << (64 - sft);
              bits = (uint32_t)x;
              if (d0 < 0) bits = (bits << -d0) | ((1u << -d0) - 1u);
            }
            vis[w] &= bits;
          }
          __syncwarp();
          float mx = DARIC_NEG_INF;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t x[32];
            tc::ld32(s_col + w * 32, x);
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, (vis[w] >> e) & 1u ? __uint_as_float(x[e]) : DARIC_NEG_INF);
          }
          // the maximum moves when it is over 2^8 ahead (or was none)
          const bool move = mx > m && (m == DARIC_NEG_INF || (mx - m) * cexp > kLag);
          const bool scale_o = move && m != DARIC_NEG_INF;
          if (__any_sync(0xffffffffu, scale_o)) {
            ok = wait(&sh.pv_done[st], (c - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after();
            const float a = scale_o ? exp2_fast((m - mx) * cexp) : 1.f;
            l0 *= a;
            l1 *= a;
#pragma unroll 1
            for (int w = 0; w < D / 32; ++w) {
              uint32_t x[32];
              tc::ld32(o_col + w * 32, x);
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * a);
              tc::st32(o_col + w * 32, x);
            }
            tc::wait_st();
          }
          if (move) m = mx;
          mb = m == DARIC_NEG_INF ? 0.f : m * cexp - (float)LIFT;
          // weights, over the scores they came from (64 scores become 32 columns)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t x[32], y[16];
            tc::ld32(s_col + w * 32, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float u = (vis[w] >> (2 * e)) & 1u ? __uint_as_float(x[2 * e]) : DARIC_NEG_INF;
              const float v = (vis[w] >> (2 * e + 1)) & 1u ? __uint_as_float(x[2 * e + 1]) : DARIC_NEG_INF;
              const float a = exp2_fast(__fmaf_rn(u, cexp, -mb)), d = exp2_fast(__fmaf_rn(v, cexp, -mb));
              l0 += a;
              l1 += d;
              y[e] = Mma<T>::pack(a, d);
            }
            tc::st16(s_col + w * 16, y);
          }
        }
        tc::wait_st();
        tc::fence_before();
        mbar_arrive(&sh.p_full[st]);
      }
      if (!ok) break;
      // ---- the segment's rows
      if (items > 0) ok = wait(&sh.pv_done[st], (done + (uint32_t)items - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      const bool pair = MT == 1 && g.n > 1;  // the odd key tiles have an output of their own
      bool writes = true;
      float a1 = 0.f, l = l0 + l1, a0 = 1.f;
      if (MT == 1) {
        writes = st == 0;
        if (pair && st == 1) {
          sh.ml[r] = make_float2(m, l);
          mbar_arrive(&sh.ml_full);
        }
        if (pair && st == 0) {
          ok = wait(&sh.ml_full, n_ml & 1) && wait(&sh.pv_done[1], (other + (uint32_t)items_of(1, g.n) - 1) & 1);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          const float2 ml = sh.ml[r];
          const float mm = fmaxf(m, ml.x), mz = mm == DARIC_NEG_INF ? 0.f : mm;
          a0 = exp2_fast((m - mz) * cexp);
          a1 = exp2_fast((ml.x - mz) * cexp);
          l = l * a0 + ml.y * a1;
          m = mm;
        }
        n_ml += pair;
        other += (uint32_t)items_of(1 - st, g.n);
      }
      if (writes) {
        tc::fence_after();
        const bool starts = g.tile0 == 0, ends = g.tile0 + g.n == g.ntiles;
        const float inv = starts && ends ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const int slot = blockIdx.x * 2 + (starts ? 1 : 0);
        const bool poison = *(volatile int*)&sh.poison[n_seg & 3] == (int)n_seg;
        uint8_t* out = p.out + (int64_t)row * p.out_row + (int64_t)head * p.out_head;
        // partial outputs lie [4 columns][row]: neighbouring rows are neighbours
        float4* part = reinterpret_cast<float4*>(p.part) + (int64_t)slot * (D / 4) * W::ROWS + i_pair;
#pragma unroll 1
        for (int w = 0; w < D / 32; ++w) {
          uint32_t x[32];
          __syncwarp();
          tc::ld32(o_col + w * 32, x);
          if (pair) {
            uint32_t z[32];
            tc::ld32(o_col + D + w * 32, z);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              x[e] = __float_as_uint(__fmaf_rn(__uint_as_float(z[e]), a1, __uint_as_float(x[e]) * a0));
          }
          if (poison) {
            // positions of the tiles that values were taken out of: whole
            // tiles, with context in front of the drafted tokens. Each lane
            // looks at one of 32; what is not finite is then added by the rows
            // that see it, position by position.
            const int k0 = SPARSE ? g.tile0 * kKeys : max(g.tile0 * kKeys, max(see, 0) / kKeys * kKeys);
            const int k1 = SPARSE ? min((g.tile0 + g.n) * kKeys, g.listed * p.kv.page_size)
                                  : min((g.tile0 + g.n) * kKeys, g.s.len);
            for (int kk = k0; kk < k1; kk += 32) {
              int pos = kk + lane, tok = 0, blk = -1;
              uint32_t rows_see = 0xffffffffu;
              if (pos < k1) {
                const int pg = (int)fdiv((uint32_t)pos, p.kv.page_div);
                tok = pos - pg * p.kv.page_size;
                if (SPARSE) {
                  const uint4 e = g.list[pg];
                  pos = (int)e.x * p.kv.page_size + tok;
                  rows_see = e.y;
                  if (pos < g.s.len) blk = (int)e.z;
                } else {
                  blk = __ldg(&p.sq.table[(int64_t)g.b * p.sq.table_ld + pg]);
                }
              }
              auto row_of = [&](int block, int token) {  // its 32 columns of V
                return reinterpret_cast<const uint16_t*>(p.kv.base + (int64_t)block * p.kv.page_stride +
                                                         (int64_t)token * p.kv.tok_stride +
                                                         (int64_t)g.h * p.kv.head_stride + p.kv.v_off) + w * 32;
              };
              bool bad = false;
              if (blk >= 0 && blk < p.kv.num_pages) {
                const uint4* v = reinterpret_cast<const uint4*>(row_of(blk, tok));
                uint32_t sum = 0;  // x * 0 summed up, as in take_out
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint4 u = v[e];
                  sum = Mma<T>::zero_sum(u.x, Mma<T>::zero_sum(u.y, Mma<T>::zero_sum(u.z, Mma<T>::zero_sum(u.w, sum))));
                }
                bad = (sum & 0x7fff7fffu) != 0;
              }
              for (unsigned left = __ballot_sync(0xffffffffu, bad); left; left &= left - 1) {
                const int from = __ffs((int)left) - 1;
                const int at = __shfl_sync(0xffffffffu, pos, from);
                const uint32_t who = __shfl_sync(0xffffffffu, rows_see, from);
                const uint16_t* v = row_of(__shfl_sync(0xffffffffu, blk, from), __shfl_sync(0xffffffffu, tok, from));
                const bool seen = real && (SPARSE ? ((who >> jl) & 1u) && at <= g.s.ctx + j
                                                  : at < g.s.ctx || sees_draft(p.sq, row, j, at - g.s.ctx));
                if (seen) {
#pragma unroll
                  for (int e = 0; e < 32; ++e) {
                    const uint16_t u = v[e];
                    if ((u & Mma<T>::kExpMask) == Mma<T>::kExpMask)
                      x[e] = __float_as_uint(__uint_as_float(x[e]) + Mma<T>::widen(u));
                  }
                }
                __syncwarp();
              }
            }
          }
          if (real && starts && ends) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t y[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                y[k] = Mma<T>::pack(__uint_as_float(x[8 * e + 2 * k]) * inv, __uint_as_float(x[8 * e + 2 * k + 1]) * inv);
              *reinterpret_cast<uint4*>(out + w * 64 + e * 16) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          } else if (real) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              part[(int64_t)(w * 8 + e) * W::ROWS] =
                  make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]),
                              __uint_as_float(x[4 * e + 3]));
          }
        }
        __syncwarp();
        tc::fence_before();
        mbar_arrive(&sh.o_empty[st]);
        if (pair) mbar_arrive(&sh.o_empty[1]);
        if (real) {
          if (starts && ends) {
            if (p.lse) p.lse[(int64_t)row * p.lse_row + head] = l == 0.f ? DARIC_NEG_INF : lse_of<LIFT>(m, p.scale, l);
          } else {
            p.part_ml[(int64_t)slot * W::ROWS + i_pair] = make_float2(m, l);
          }
        }
        if (tid == 0 && starts && !ends)
          p.desc[blockIdx.x] = make_int4(g.s.row0, g.h | g.rt << 12, g.my_rows,
                                         (int)split_owner(total, gridDim.x, t + (uint32_t)(g.ntiles - g.tile0) - 1));
      }
      done += (uint32_t)items;
      n_tile += (uint32_t)g.n;
      ++n_seg;
      t += (uint32_t)g.n;
    }
  }
  // Nothing of this CTA is under way any more: every product was waited for
  // by the warp that issued it, every copy by its thread.
  __syncthreads();
  if (warp == W::MMA_WARP) {
    __syncwarp();
    tc::dealloc512(tmem);
  }
}

// Joins the parts of the segment that starts in CTA blockIdx.x and ends in a
// later one, in the order of the CTAs. A lane is a row, a warp four columns.
template <class T, int D, int MT>
__global__ void __launch_bounds__(256) wide_join_kernel(const __grid_constant__ AttendLaunch p) {
  constexpr int ROWS = 128 * MT, AHEAD = 8;  // parts loaded at a time
  grid_wait();
  const int4 ds = p.desc[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = blockIdx.z * 8 + (threadIdx.x >> 5);
  const int i = blockIdx.y * 32 + lane;
  if (ds.x < 0 || blockIdx.y * 32 >= ds.z) return;
  const int c0 = blockIdx.x, c1 = ds.w;
  const float cexp = p.scale * kLog2e;
  float mm = DARIC_NEG_INF, ll = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* part = reinterpret_cast<const float4*>(p.part);
  for (int c = c0; c <= c1; c += AHEAD) {
    float2 ml[AHEAD];
    float4 x[AHEAD];
    float top = mm;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t s = (c + k) * 2 + (c + k == c0);
      ml[k] = c + k <= c1 ? p.part_ml[s * ROWS + i] : make_float2(DARIC_NEG_INF, 0.f);
      x[k] = c + k <= c1 ? part[(s * (D / 4) + warp) * ROWS + i] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) top = fmaxf(top, ml[k].x);
    const float base = top == DARIC_NEG_INF ? 0.f : top, a = exp2_fast((mm - base) * cexp);
    ll *= a;
    o.x *= a;
    o.y *= a;
    o.z *= a;
    o.w *= a;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float w = exp2_fast((ml[k].x - base) * cexp);
      ll = __fmaf_rn(ml[k].y, w, ll);
      o.x = __fmaf_rn(x[k].x, w, o.x);
      o.y = __fmaf_rn(x[k].y, w, o.y);
      o.z = __fmaf_rn(x[k].z, w, o.z);
      o.w = __fmaf_rn(x[k].w, w, o.w);
    }
    mm = top;
  }
  if (i >= ds.z) return;
  const int rt = ds.y >> 12, h = ds.y & 4095;
  const int pi = rt * ROWS + i;
  const int64_t row = ds.x + pi / p.sq.group;
  const int head = h * p.sq.group + pi % p.sq.group;
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  *reinterpret_cast<uint2*>(p.out + row * p.out_row + (int64_t)head * p.out_head + warp * 8) =
      make_uint2(Mma<T>::pack(o.x * inv, o.y * inv), Mma<T>::pack(o.z * inv, o.w * inv));
  if (warp == 0 && p.lse) p.lse[row * p.lse_row + head] = ll == 0.f ? DARIC_NEG_INF : lse_of<kWideLift<T>>(mm, p.scale, ll);
}

// Lists of the SPARSE form, one per row tile (blockIdx.x) and KV head: the
// pages that any of its rows lists, ascending, with the rows (bits) that do
// and the page's block. A row's page behind its own position is left out.
constexpr int kUnionThreads = 256;
__global__ void __launch_bounds__(kUnionThreads) union_kernel(const __grid_constant__ AttendLaunch p) {
  extern __shared__ uint32_t table[];  // rows that list each page of the sequence
  __shared__ int s_where[2];
  __shared__ int s_sum[kUnionThreads / 32];
  grid_next();
  const int tile = blockIdx.x, h = blockIdx.y, H = p.kv.heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = p.sq.group, bs = p.kv.page_size;
  if (warp == 0) {  // the sequence of the row tile
    int at = 0, found = -1, rt = 0;
    for (int b0 = 0; b0 < p.sq.num_seqs && found < 0; b0 += 32) {
      int n = 0;
      if (b0 + lane < p.sq.num_seqs) n = (load_seq(p.sq, b0 + lane).rows * group + 127) / 128;
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned m = __ballot_sync(0xffffffffu, tile < at + x);
      if (m) {
        const int l = __ffs((int)m) - 1;
        found = b0 + l;
        rt = tile - at - __shfl_sync(0xffffffffu, x - n, l);
      }
      at += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      s_where[0] = found;
      s_where[1] = rt;
    }
  }
  for (int i = threadIdx.x; i < p.sq.table_cols; i += kUnionThreads) table[i] = 0;
  __syncthreads();
  const int b = s_where[0], rt = s_where[1], item = tile * H + h;
  if (b < 0) {
    if (threadIdx.x == 0) p.list_count[item] = -1;
    return;
  }
  Seq s = load_seq(p.sq, b);
  clamp_len(p.sq, bs, s);
  const int j0 = rt * 128 / group, j1 = min(s.rows, (rt * 128 + 127) / group + 1);
  for (int v = threadIdx.x; v < (j1 - j0) * p.k; v += kUnionThreads) {
    const int jl = v / p.k, e = v - jl * p.k, j = j0 + jl;
    const int pg = __ldg(&p.pages[(int64_t)(s.row0 + j) * p.pages_row + (int64_t)h * p.pages_head + e]);
    if (pg >= p.sq.table_cols) {
      atomicOr(p.sq.err, DEV_ERR_INDEX_RANGE);
    } else if (pg >= 0 && (int64_t)pg * bs <= s.ctx + j) {
      atomicOr(&table[pg], 1u << jl);
    }
  }
  __syncthreads();
  // in order of the pages: a thread's run of them, then the runs before it
  const int per = (p.sq.table_cols + kUnionThreads - 1) / kUnionThreads, first = threadIdx.x * per;
  int n = 0;
  for (int i = first; i < min(first + per, p.sq.table_cols); ++i) n += table[i] != 0;
  int x = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_sum[warp] = x;
  __syncthreads();
  int at = x - n, total = 0;
  for (int w = 0; w < kUnionThreads / 32; ++w) {
    if (w < warp) at += s_sum[w];
    total += s_sum[w];
  }
  uint4* list = p.list + (int64_t)item * p.list_row;
  const int32_t* trow = p.sq.table + (int64_t)b * p.sq.table_ld;
  for (int i = first; i < min(first + per, p.sq.table_cols); ++i)
    if (table[i]) list[at++] = make_uint4((uint32_t)i, table[i], (uint32_t)__ldg(&trow[i]), 0);
  if (threadIdx.x == 0) {
    p.list_count[item] = total;
    if (h == 0) p.list_tile[tile] = make_int2(b, rt);
  }
}

template <class T, int D, int MT, bool SPARSE>
void wide_one(const AttendLaunch& p, int grid, cudaStream_t s) {
  using W = Wide<D, MT, SPARSE>;
  constexpr int bytes = wide_smem<D, MT, SPARSE>();
  static_assert(bytes <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  allow_smem(wide_kernel<T, D, MT, SPARSE>, bytes, done);
  if (SPARSE) {
    static std::atomic<uint64_t> ready{0};
    allow_smem(union_kernel, kUnionPages * 4, ready);
    union_kernel<<<dim3((unsigned)(p.lists / p.kv.heads), (unsigned)p.kv.heads), kUnionThreads, p.sq.table_cols * 4, s>>>(p);
    DARIC_CUDA(cudaGetLastError());
    launch_after(wide_kernel<T, D, MT, SPARSE>, dim3((unsigned)grid), W::THREADS, s, p, bytes);
  } else {
    wide_kernel<T, D, MT, SPARSE><<<grid, W::THREADS, bytes, s>>>(p);
    DARIC_CUDA(cudaGetLastError());
  }
  launch_after(wide_join_kernel<T, D, MT>, dim3((unsigned)grid, 4 * MT, D / 32), 256, s, p);
}

template <class T, int D>
void wide_d(const AttendLaunch& p, int mt, int grid, cudaStream_t s) {
  if (p.pages) return wide_one<T, D, 1, true>(p, grid, s);
  mt == 2 ? wide_one<T, D, 2, false>(p, grid, s) : wide_one<T, D, 1, false>(p, grid, s);
}

template <class T>
void wide_t(const AttendLaunch& p, int mt, int grid, cudaStream_t s) {
  p.kv.head_dim == 64 ? wide_d<T, 64>(p, mt, grid, s) : wide_d<T, 128>(p, mt, grid, s);
}

}  // namespace

void launch_wide(const AttendLaunch& p, int dtype, int mt, int grid, cudaStream_t s) {
  if (dtype == DARIC_DTYPE_BF16) return wide_t<__nv_bfloat16>(p, mt, grid, s);
  wide_t<__half>(p, mt, grid, s);
}

}  // namespace daric
