// Attention of a batch of query rows over the paged KV cache.
//
// Mathematics: one pass over the keys of a (sequence, KV head) with the
// running maximum m and sum l of the softmax: for a chunk of keys
//   x = q . k,  m' = max(m, x),  a = 2^((m - m') c),  p = 2^((x - m') c),
//   l = a l + sum p,  O = a O + p V,       c = scale * log2(e),
// and O / l at the end; parts of one row over different keys join the same
// way. m, l, O and x are fp32; p is rounded to the cache's type for the
// second product, which takes both operands in 16 bits (half a step: relative
// 2^-8 bf16, 2^-11 fp16 per weight, of either sign; a second product with what
// the rounding left would double that work), while l sums the unrounded p. With
// fp16 all weights carry a factor of 2^15, which cancels in O / l: they keep
// their precision down to 2^-29 of the largest and vanish below 2^-40.
//
// Bound: the K and V bytes of the cache while group * rows stays small (64
// sequences of 131 to 8192 tokens, 4 KV heads of 7, fp16: 99 us of kernel, 5.5
// TB/s; 64 rows with 128 pages each of 32K: 95 us, 5.7 TB/s).
// All query heads of a KV head and all rows of a sequence share one read of
// K and V. Work is split over the long axis: the (sequence, head, row tile)
// segments, cut in tiles of keys, form one line of tiles that is divided
// evenly over a persistent grid, so a batch of mixed lengths and a single
// long sequence both fill the SMs. A segment that one CTA covers is written
// by it; of the others at most two parts per CTA go to the workspace and
// join_kernel joins them.
//
// A CTA has four warps: RG row groups of 16 rows x 4 / RG key groups. A key
// group streams its own chunks of keys through its own ring of shared-memory
// stages (16-byte cp.async, one row of the cache at a time, rows padded by 16
// bytes so that ldmatrix is free of bank conflicts), so with RG = 1 no two
// warps ever wait for each other before the end of a segment.
#include "attend_common.cuh"

#include <algorithm>

namespace daric {
namespace {
using namespace att;

constexpr int kThreads = 128;

template <int D, int RG>
struct Geom {
  static constexpr int KG = 4 / RG;                                     // key groups
  static constexpr int KT = RG == 1 ? 16 : 32;                          // keys of a chunk
  static constexpr int KPW = KT / RG;                                   // keys a warp loads of a chunk
  static constexpr int TILE = KT * KG;                                  // keys of a tile
  static constexpr int PITCH = D * 2 + 16;
  static constexpr int STAGE = 2 * KT * PITCH;
  // stages of a ring: where four warps can be three CTAs on an SM, more warps
  // count for more than more stages (64 ragged decodes: 98 us against 105)
  static constexpr int S = RG == 1 && D <= 128 ? 2 : (D > 128 && RG == 4 ? 4 : 3);
  static constexpr int ROWS = 16 * RG;
  static constexpr int RING = KG * S * STAGE;
  static constexpr int QB = ROWS * PITCH;
  static constexpr int MERGE = KG * ROWS * (D + 2) * 4;
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + QB;
  static_assert(SMEM <= 226 * 1024, "shared memory of a CTA");
};

// One segment: keys of one KV head for up to ROWS query rows.
struct Segment {
  int b, h, rt;     // sequence (sparse: query row), KV head, row tile
  int ntiles;
  Seq s;
};

template <int D, int RG, bool SPARSE>
__device__ __forceinline__ int tiles_of(const AttendLaunch& p, const Seq& s) {
  using G = Geom<D, RG>;
  if (SPARSE) return (int)(((int64_t)p.k * p.kv.page_size + G::TILE - 1) / G::TILE);
  return (s.len + G::TILE - 1) / G::TILE;
}

template <class T, int D, int RG, bool SPARSE>
__global__ void __launch_bounds__(kThreads, D > 128 ? 1 : (RG == 1 ? 3 : 2)) attend_kernel(const __grid_constant__ AttendLaunch p) {
  using G = Geom<D, RG>;
  constexpr int CH = D / 8;  // 16-byte vectors of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_sum[kThreads];
  __shared__ uint32_t s_valid[4][4][4];  // [key group][stage][warp of the group]: keys that exist
  __shared__ int s_bad[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rg = warp % RG, kg = warp / RG;
  uint8_t* ring = smem + kg * G::S * G::STAGE;
  uint8_t* qs = smem + (G::RING > G::MERGE ? G::RING : G::MERGE);
  const int group = p.sq.group;
  grid_next();

  // ---- the line of tiles and this CTA's part of it
  uint32_t total, t0, t1;
  uint32_t seg_at = 0;  // tiles before the sequence
  int b = 0;
  uint32_t per_seq = 0;  // sparse: tiles of a query row
  if (SPARSE) {
    Seq none{};
    const int rts = (group + G::ROWS - 1) / G::ROWS;
    per_seq = (uint32_t)(tiles_of<D, RG, SPARSE>(p, none) * rts * p.kv.heads);
    total = per_seq * (uint32_t)p.sq.num_rows;
    split_range(total, gridDim.x, blockIdx.x, t0, t1);
    if (t0 < t1) {
      b = (int)(t0 / per_seq);
      seg_at = (uint32_t)b * per_seq;
    }
  } else {
    const int per = (p.sq.num_seqs + kThreads - 1) / kThreads;
    uint32_t mine = 0;
    for (int i = tid * per; i < min((tid + 1) * per, p.sq.num_seqs); ++i) {
      Seq s = load_seq(p.sq, i);
      clamp_len(p.sq, p.kv.page_size, s);
      const uint32_t rts = ((uint32_t)(s.rows * group) + G::ROWS - 1) / G::ROWS;
      mine += rts * (uint32_t)p.kv.heads * (uint32_t)max(tiles_of<D, RG, SPARSE>(p, s), 1);
    }
    s_sum[tid] = mine;
    __syncthreads();
    for (int o = 1; o < kThreads; o <<= 1) {
      const uint32_t v = tid >= o ? s_sum[tid - o] : 0;
      __syncthreads();
      s_sum[tid] += v;
      __syncthreads();
    }
    total = s_sum[kThreads - 1];
    split_range(total, gridDim.x, blockIdx.x, t0, t1);
    if (t0 < t1) {  // the thread range, then the sequence that holds tile t0
      int lo = 0, hi = kThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_sum[mid] > t0) hi = mid; else lo = mid + 1;
      }
      b = lo * per;
      seg_at = lo ? s_sum[lo - 1] : 0;
    }
  }
  if (tid == 0) p.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (t0 >= t1) return;

  uint32_t t = t0;
  while (t < t1) {
    // ---- the segment that holds tile t
    Segment sg;
    uint32_t seq_tiles;
    int seq_id;  // sequence in the block table
    int qpos = 0;
    if (SPARSE) {
      b = (int)(t / per_seq);
      seg_at = (uint32_t)b * per_seq;
      seq_id = find_seq(p.sq, b);
      if (seq_id >= 0) {
        sg.s = load_seq(p.sq, seq_id);
        clamp_len(p.sq, p.kv.page_size, sg.s);
        qpos = sg.s.ctx + (b - sg.s.row0);
        if (b - sg.s.row0 >= sg.s.rows) seq_id = -1;  // behind its last row, or its offsets are bad
      } else {
        sg.s = Seq{};
      }
      sg.ntiles = tiles_of<D, RG, SPARSE>(p, sg.s);
      seq_tiles = per_seq;
    } else {
      for (;; ++b) {
        if (b >= p.sq.num_seqs) return;  // lengths that changed while the kernel ran
        sg.s = load_seq(p.sq, b);
        clamp_len(p.sq, p.kv.page_size, sg.s);
        const uint32_t rts = ((uint32_t)(sg.s.rows * group) + G::ROWS - 1) / G::ROWS;
        sg.ntiles = max(tiles_of<D, RG, SPARSE>(p, sg.s), 1);
        seq_tiles = rts * (uint32_t)p.kv.heads * (uint32_t)sg.ntiles;
        if (t < seg_at + seq_tiles) break;
        seg_at += seq_tiles;
      }
      seq_id = b;
    }
    uint32_t x = t - seg_at;
    const int tile0 = (int)(x % (uint32_t)sg.ntiles);
    x /= (uint32_t)sg.ntiles;
    const int rts = ((SPARSE ? group : sg.s.rows * group) + G::ROWS - 1) / G::ROWS;
    sg.rt = (int)(x % (uint32_t)rts);
    sg.h = (int)(x / (uint32_t)rts);
    sg.b = b;
    const int n = (int)min((uint32_t)(sg.ntiles - tile0), t1 - t);
    const int nrows = SPARSE ? (seq_id < 0 ? 0 : group) : sg.s.rows * group;
    const int row_base = sg.rt * G::ROWS;       // first of the segment's (row, head) pairs
    const int my_rows = min(G::ROWS, nrows - row_base);  // pairs that exist (<= 0: none)

    // pair i of the segment: query row and query head
    auto pair_row = [&](int i) { return SPARSE ? sg.b : sg.s.row0 + (row_base + i) / group; };
    auto pair_head = [&](int i) { return sg.h * group + (row_base + i) % group; };

    // ---- query rows to shared memory (rows that do not exist are zero)
    __syncthreads();
    for (int v = tid; v < G::ROWS * CH; v += kThreads) {
      const int i = v / CH, c = v % CH;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (i < my_rows)
        w = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)pair_row(i) * p.q_row + (int64_t)pair_head(i) * p.q_head) + c);
      *reinterpret_cast<uint4*>(qs + i * G::PITCH + c * 16) = w;
    }
    __syncthreads();
    const uint32_t q_at = smem_u32(qs) + (rg * 16 + (lane & 15)) * G::PITCH + (lane >> 4) * 16;
    uint32_t qf[D <= 128 ? D / 16 : 1][4];
    if (D <= 128) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) ldsm4(q_at + ks * 32, qf[D <= 128 ? ks : 0]);
    }

    // ---- key stream of this key group
    const int32_t* trow = p.sq.table + (int64_t)seq_id * p.sq.table_ld;
    const int32_t* prow = SPARSE ? p.pages + (int64_t)sg.b * p.pages_row + (int64_t)sg.h * p.pages_head : nullptr;
    const int64_t head_off = (int64_t)sg.h * p.kv.head_stride;
    // A warp's share of a chunk lies in one page when the page size is a
    // multiple of it: one lookup and one address serve all its rows. Else
    // lane i looks key i up and the rows' addresses go round by shuffles.
    const bool one = p.kv.page_size % G::KPW == 0;
    int nxt_blk = -1, nxt_in = 0, nxt_n = 0;  // block, first row in it, rows (one) or 1 / 0 (else)
    auto lookup = [&](int c) {                // of this warp's share of chunk c
      nxt_n = 0;
      nxt_blk = -1;
      if (c < n && (one || lane < G::KPW)) {
        const int i = (tile0 + c) * G::TILE + kg * G::KT + rg * G::KPW + (one ? 0 : lane);
        const int e = (int)fdiv((uint32_t)i, p.kv.page_div);
        nxt_in = i - e * p.kv.page_size;
        int pg = e, left = sg.s.len - i;
        if (SPARSE) {
          pg = e < p.k && seq_id >= 0 ? ld_ahead(&prow[e]) : -1;
          if (pg >= 0 && e > 0 && ld_ahead(&prow[e - 1]) == pg) pg = -1;  // a repeated page counts once
          if (pg >= p.sq.table_cols) {
            atomicOr(p.sq.err, DEV_ERR_INDEX_RANGE);
            pg = -1;
          }
          left = pg < 0 ? 0 : qpos + 1 - pg * p.kv.page_size - nxt_in;
        }
        if (left > 0) {
          nxt_blk = ld_ahead(&trow[pg]);
          nxt_n = one ? min(left, G::KPW) : 1;
        }
      }
    };
    auto issue = [&](int stage) {  // copies of the chunk that lookup() saw last
      const uint32_t dst = smem_u32(ring) + stage * G::STAGE + rg * G::KPW * G::PITCH;
      bool ok = nxt_n > 0;
      if (ok && (nxt_blk < 0 || nxt_blk >= p.kv.num_pages)) {
        atomicOr(p.sq.err, DEV_ERR_BLOCK_RANGE);
        ok = false;
      }
      const int64_t off = ok ? (int64_t)nxt_blk * p.kv.page_stride + (int64_t)nxt_in * p.kv.tok_stride + head_off : 0;
      constexpr int RPI = 32 / CH;  // rows a warp copies at a time
      const int r0 = lane / CH, c16 = (lane % CH) * 16;
      const uint32_t d0 = dst + r0 * G::PITCH + c16;
      if (one) {
        const int rows = ok ? nxt_n : 0;
        if (lane == 0) s_valid[kg][stage][rg] = (uint32_t)((1ull << rows) - 1);
        // rows past the valid ones are in the page all the same: nothing of
        // them is read, and zeros are written
        const uint8_t* k = p.kv.base + off + r0 * p.kv.tok_stride + c16;
        const int64_t step = RPI * p.kv.tok_stride;
        int left = rows - r0;
#pragma unroll
        for (int i = 0; i < G::KPW / RPI; ++i) {
          cp16(d0 + i * RPI * G::PITCH, k, left > 0);
          cp16(d0 + (G::KT + i * RPI) * G::PITCH, k + p.kv.v_off, left > 0);
          k += step;
          left -= RPI;
        }
      } else {
        const unsigned valid = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) s_valid[kg][stage][rg] = valid;
#pragma unroll 2
        for (int i = 0; i < G::KPW / RPI; ++i) {
          const int r = r0 + i * RPI;
          const int64_t o = __shfl_sync(0xffffffffu, off, r);
          const bool in = (valid >> r) & 1;
          const uint8_t* k = p.kv.base + o + (in ? c16 : 0);
          cp16(d0 + i * RPI * G::PITCH, k, in);
          cp16(d0 + (G::KT + i * RPI) * G::PITCH, in ? k + p.kv.v_off : k, in);
        }
      }
    };
    auto group_sync = [&]() {
      if (RG == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "r"(RG * 32) : "memory");
    };

    float acc[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    float m[2] = {DARIC_NEG_INF, DARIC_NEG_INF}, l[2] = {0.f, 0.f};
    const float cexp = p.scale * kLog2e;
    const int pi0 = rg * 16 + (lane >> 2);  // this thread's pairs: pi0 and pi0 + 8

    lookup(0);
#pragma unroll
    for (int c = 0; c < G::S - 1; ++c) {
      if (c < n) issue(c);
      lookup(c + 1);
      cp_commit();
    }
    for (int c = 0; c < n; ++c) {
      cp_wait<G::S - 2>();
      group_sync();
      const int st = c % G::S;
      if (c + G::S - 1 < n) issue((c + G::S - 1) % G::S);
      lookup(c + G::S);
      cp_commit();

      bool all = true, any = false;
#pragma unroll
      for (int w = 0; w < RG; ++w) {
        const uint32_t v = s_valid[kg][st][w];
        all = all && v == (G::KPW == 32 ? 0xffffffffu : (1u << (G::KPW & 31)) - 1u);
        any = any || v;
      }
      if (!any) continue;
      const int key0 = (tile0 + c) * G::TILE + kg * G::KT;  // first position (dense)
      const bool draft = !SPARSE && key0 + G::KT > sg.s.ctx;
      const uint32_t k_at = smem_u32(ring) + st * G::STAGE;
      const uint32_t v_at = k_at + G::KT * G::PITCH;

      // x = q . k
      float x[G::KT / 8][4];
#pragma unroll
      for (int j = 0; j < G::KT / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[4];
        if (D <= 128) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = qf[D <= 128 ? ks : 0][e];
        } else {
          ldsm4(q_at + ks * 32, a);
        }
#pragma unroll
        for (int j = 0; j < G::KT / 16; ++j) {
          uint32_t kf[4];
          ldsm4(k_at + (j * 16 + (lane >> 4) * 8 + (lane & 7)) * G::PITCH + ks * 32 + ((lane >> 3) & 1) * 16, kf);
          Mma<T>::run(x[2 * j], a, kf[0], kf[1]);
          Mma<T>::run(x[2 * j + 1], a, kf[2], kf[3]);
        }
      }
      // which keys a row sees
      auto key_ok = [&](int k) { return (s_valid[kg][st][k / G::KPW] >> (k % G::KPW)) & 1u; };
      auto sees = [&](int pi, int k) {
        if (!key_ok(k)) return false;
        const int i = key0 + k - sg.s.ctx;
        if (SPARSE || i < 0) return true;
        if (pi >= my_rows) return false;
        const int row = pair_row(pi);
        return sees_draft(p.sq, row, row - sg.s.row0, i);
      };
      if (!all || draft) {
#pragma unroll
        for (int j = 0; j < G::KT / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(pi0 + (e >> 1) * 8, j * 8 + (lane & 3) * 2 + (e & 1))) x[j][e] = DARIC_NEG_INF;
      }
      // running maximum
      float mx[2] = {DARIC_NEG_INF, DARIC_NEG_INF};
#pragma unroll
      for (int j = 0; j < G::KT / 8; ++j) {
        mx[0] = fmaxf(mx[0], fmaxf(x[j][0], x[j][1]));
        mx[1] = fmaxf(mx[1], fmaxf(x[j][2], x[j][3]));
      }
      float base[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float mn = fmaxf(m[r], mx[r]);
        base[r] = mn == DARIC_NEG_INF ? 0.f : mn;
        const float a = exp2_fast((m[r] - base[r]) * cexp);
        m[r] = mn;
        l[r] *= a;
        if (__any_sync(0xffffffffu, a != 1.f)) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            acc[i][2 * r] *= a;
            acc[i][2 * r + 1] *= a;
          }
        }
      }
      if (draft) {
        // V rows that some rows must not see: an infinity or NaN in them would
        // reach every row through 0 * inf, so such values are taken out of the
        // product and added to the rows that do see them.
        bool bad = false;
        for (int v = lane + 32 * rg; v < G::KT * CH; v += 32 * RG) {
          const uint4 w = *reinterpret_cast<const uint4*>(ring + st * G::STAGE + (G::KT + v / CH) * G::PITCH + (v % CH) * 16);
          const uint16_t* u = reinterpret_cast<const uint16_t*>(&w);
#pragma unroll
          for (int e = 0; e < 8; ++e) bad = bad || (u[e] & Mma<T>::kExpMask) == Mma<T>::kExpMask;
        }
        bad = __any_sync(0xffffffffu, bad);
        if (RG > 1) {
          if (lane == 0) s_bad[warp] = bad;
          group_sync();
#pragma unroll
          for (int w = 0; w < RG; ++w) bad = bad || s_bad[kg * RG + w];
        }
        if (bad) {
          for (int k = 0; k < G::KT; ++k) {
            const uint16_t* vr = reinterpret_cast<const uint16_t*>(ring + st * G::STAGE + (G::KT + k) * G::PITCH);
            const bool s0 = sees(pi0, k), s1 = sees(pi0 + 8, k);
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint16_t u = vr[i * 8 + (lane & 3) * 2 + (e & 1)];
                if ((u & Mma<T>::kExpMask) == Mma<T>::kExpMask && (e < 2 ? s0 : s1)) acc[i][e] += Mma<T>::widen(u);
              }
          }
          group_sync();
          for (int v = lane + 32 * rg; v < G::KT * D; v += 32 * RG) {
            uint16_t* u = reinterpret_cast<uint16_t*>(ring + st * G::STAGE + (G::KT + v / D) * G::PITCH) + v % D;
            if ((*u & Mma<T>::kExpMask) == Mma<T>::kExpMask) *u = 0;
          }
          group_sync();
        }
      }
      // p = 2^((x - m) c), then O += p V
#pragma unroll
      for (int j = 0; j < G::KT / 16; ++j) {
        uint32_t a[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float(&y)[4] = x[2 * j + u];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = exp2_fast(lifted<T>(y[e] - base[e >> 1], cexp));
          l[0] += y[0] + y[1];
          l[1] += y[2] + y[3];
          a[2 * u] = Mma<T>::pack(y[0], y[1]);
          a[2 * u + 1] = Mma<T>::pack(y[2], y[3]);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t vf[4];
          ldsm4_t(v_at + (j * 16 + (lane & 15)) * G::PITCH + i * 32 + (lane >> 4) * 16, vf);
          Mma<T>::run(acc[2 * i], a, vf[0], vf[1]);
          Mma<T>::run(acc[2 * i + 1], a, vf[2], vf[3]);
        }
      }
    }
    cp_wait<0>();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }

    // ---- the key groups' parts meet in shared memory
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem);                 // [KG][ROWS][D]
    float2* mml = reinterpret_cast<float2*>(mo + G::KG * G::ROWS * D);  // [KG][ROWS]
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<float2*>(mo + (kg * G::ROWS + pi0 + 8 * r) * D + i * 8 + (lane & 3) * 2) =
            make_float2(acc[i][2 * r], acc[i][2 * r + 1]);
    if ((lane & 3) == 0) {
      mml[kg * G::ROWS + pi0] = make_float2(m[0], l[0]);
      mml[kg * G::ROWS + pi0 + 8] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    const bool starts = tile0 == 0, ends = tile0 + n == sg.ntiles;
    const int slot = blockIdx.x * 2 + (starts ? 1 : 0);
    for (int i = warp; i < my_rows; i += 4) {
      float mm = DARIC_NEG_INF;
#pragma unroll
      for (int g = 0; g < G::KG; ++g) mm = fmaxf(mm, mml[g * G::ROWS + i].x);
      const float base = mm == DARIC_NEG_INF ? 0.f : mm;
      float w[G::KG], ll = 0.f;
#pragma unroll
      for (int g = 0; g < G::KG; ++g) {
        w[g] = exp2_fast((mml[g * G::ROWS + i].x - base) * cexp);
        ll += mml[g * G::ROWS + i].y * w[g];
      }
      const float inv = starts && ends ? (ll == 0.f ? 0.f : 1.f / ll) : 1.f;
      for (int d = lane * 2; d < D; d += 64) {
        float2 o = make_float2(0.f, 0.f);
#pragma unroll
        for (int g = 0; g < G::KG; ++g) {
          const float2 v = *reinterpret_cast<const float2*>(mo + (g * G::ROWS + i) * D + d);
          o.x += v.x * w[g];
          o.y += v.y * w[g];
        }
        if (starts && ends)
          *reinterpret_cast<uint32_t*>(p.out + (int64_t)pair_row(i) * p.out_row + (int64_t)pair_head(i) * p.out_head + d * 2) =
              Mma<T>::pack(o.x * inv, o.y * inv);
        else
          *reinterpret_cast<float2*>(p.part + ((int64_t)slot * G::ROWS + i) * D + d) = o;
      }
      if (lane == 0) {
        if (starts && ends) {
          if (p.lse)
            p.lse[(int64_t)pair_row(i) * p.lse_row + pair_head(i)] =
                ll == 0.f ? DARIC_NEG_INF : lse_of<Mma<T>::kLift>(mm, p.scale, ll);
        } else {
          p.part_ml[(int64_t)slot * G::ROWS + i] = make_float2(mm, ll);
        }
      }
    }
    if (tid == 0 && starts && !ends)
      p.desc[blockIdx.x] = make_int4(SPARSE ? sg.b : sg.s.row0, sg.h | sg.rt << 12, my_rows,
                                     (int)split_owner(total, gridDim.x, t + (uint32_t)(sg.ntiles - tile0) - 1));
    t += (uint32_t)n;
  }
}

// Joins the parts of the segment that starts in CTA blockIdx.x of the
// attention and ends in a later one: slot 1 of that CTA, then slot 0 of the
// following ones, always in this order, so a result does not depend on timing.
// One warp per row.
template <class T, int D, int RG>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ AttendLaunch p) {
  constexpr int ROWS = 16 * RG;
  grid_wait();
  const int4 ds = p.desc[blockIdx.x];
  const int i = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (ds.x < 0 || i >= ds.z) return;
  const int c0 = blockIdx.x, c1 = ds.w;
  const float cexp = p.scale * kLog2e;
  float mm = DARIC_NEG_INF;
  for (int c = c0 + lane; c <= c1; c += 32) mm = fmaxf(mm, p.part_ml[(int64_t)(c * 2 + (c == c0)) * ROWS + i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  const float base = mm == DARIC_NEG_INF ? 0.f : mm;
  float ll = 0.f;
  constexpr int V = D / 64;  // float2 a lane
  float2 o[V > 0 ? V : 1];
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = make_float2(0.f, 0.f);
  for (int c = c0; c <= c1; ++c) {
    const int64_t s = (int64_t)(c * 2 + (c == c0)) * ROWS + i;
    const float2 ml = p.part_ml[s];
    const float w = exp2_fast((ml.x - base) * cexp);
    ll += ml.y * w;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 x = *reinterpret_cast<const float2*>(p.part + s * D + v * 64 + lane * 2);
      o[v].x += x.x * w;
      o[v].y += x.y * w;
    }
  }
  const int rt = ds.y >> 12, h = ds.y & 4095;
  const int pi = rt * ROWS + i;
  const int64_t row = ds.x + pi / p.sq.group;
  const int head = h * p.sq.group + pi % p.sq.group;
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
  for (int v = 0; v < V; ++v)
    *reinterpret_cast<uint32_t*>(p.out + row * p.out_row + (int64_t)head * p.out_head + (v * 64 + lane * 2) * 2) =
        Mma<T>::pack(o[v].x * inv, o[v].y * inv);
  if (lane == 0 && p.lse)
    p.lse[row * p.lse_row + head] = ll == 0.f ? DARIC_NEG_INF : lse_of<Mma<T>::kLift>(mm, p.scale, ll);
}

template <class T, int D, int RG, bool SPARSE>
void launch_one(const AttendLaunch& p, int grid, cudaStream_t s) {
  auto kern = attend_kernel<T, D, RG, SPARSE>;
  constexpr int bytes = Geom<D, RG>::SMEM;
  static std::atomic<uint64_t> done{0};
  allow_smem(kern, bytes, done);
  kern<<<grid, kThreads, bytes, s>>>(p);
  DARIC_CUDA(cudaGetLastError());
  launch_after(join_kernel<T, D, RG>, dim3((unsigned)grid, 4 * RG), 128, s, p);
}

template <class T, int D>
void launch_d(const AttendLaunch& p, int rg, int grid, cudaStream_t s) {
  if (p.pages) return rg == 1 ? launch_one<T, D, 1, true>(p, grid, s) : launch_one<T, D, 2, true>(p, grid, s);
  if (rg == 1) return launch_one<T, D, 1, false>(p, grid, s);
  if (rg == 2) return launch_one<T, D, 2, false>(p, grid, s);
  launch_one<T, D, 4, false>(p, grid, s);
}

template <class T>
void launch_t(const AttendLaunch& p, int rg, int grid, cudaStream_t s) {
  switch (p.kv.head_dim) {
    case 64: return launch_d<T, 64>(p, rg, grid, s);
    case 128: return launch_d<T, 128>(p, rg, grid, s);
    case 256: return launch_d<T, 256>(p, rg, grid, s);
  }
  throw Error(DARIC_ERR_INVALID, "attention: head dimension must be 64, 128 or 256, got " +
                                     std::to_string(p.kv.head_dim));
}

}  // namespace

void launch_attend(const AttendLaunch& p, int dtype, int rg, int grid, cudaStream_t s) {
  if (dtype == DARIC_DTYPE_BF16) return launch_t<__nv_bfloat16>(p, rg, grid, s);
  if (dtype == DARIC_DTYPE_F16) return launch_t<__half>(p, rg, grid, s);
  throw Error(DARIC_ERR_INVALID, "attention: the KV cache must be bfloat16 or float16");
}

}  // namespace daric
