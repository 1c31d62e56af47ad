// Device helpers of the attention kernels: 16-byte asynchronous copies,
// matrix fragments, and the lookup of sequences and cache rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attend.h"

#include <atomic>

namespace daric {
namespace att {

// Raises a kernel's dynamic shared memory limit once per device (the current
// one); `done` is the caller's static mask of devices.
template <class K>
void allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  DARIC_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return;
  DARIC_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
}

// A second kernel that needs the first one's results is launched while the
// first runs (programmatic dependent launch) and waits on the GPU: its launch
// costs no time of its own.
__device__ __forceinline__ void grid_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class K, class P>
void launch_after(K kern, dim3 grid, int threads, cudaStream_t s, const P& p, int smem = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = s;
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DARIC_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
#define DARIC_NEG_INF __int_as_float(0xff800000)

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes global -> shared; ok = false writes zeros and reads nothing.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// The same with constant offsets from both addresses.
template <int DST, int SRC>
__device__ __forceinline__ void cp16_at(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(DST), "n"(SRC)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A load that stays where it is written: what is read ahead of its use must
// not be moved down to it.
__device__ __forceinline__ int32_t ld_ahead(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ int4 ld_ahead(const int4* p) {
  int4 v;
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}

// 2^x (about 2 ulp; results below 2^-126 are 0)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ __forceinline__ static float widen(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  // both halves: a * 0 + b
  __device__ __forceinline__ static uint32_t zero_sum(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&a), __nv_bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0)),
                                     *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static constexpr uint16_t kExpMask = 0x7f80;  // all ones: infinity or NaN
  static constexpr int kLift = 0;
};
template <>
struct Mma<__half> {
  __device__ __forceinline__ static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ __forceinline__ static float widen(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  __device__ __forceinline__ static uint32_t zero_sum(uint32_t a, uint32_t b) {
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), __half2(__ushort_as_half(0), __ushort_as_half(0)),
                              *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static constexpr uint16_t kExpMask = 0x7c00;
  // The largest weight of a row is stored as 2^kLift (bf16: 1): fp16 has full
  // precision down to 2^-14 only, and many keys of small weights count together.
  static constexpr int kLift = 15;
};

// Exponent of a weight, x c, with the type's factor.
template <class T>
__device__ __forceinline__ float lifted(float x, float c) {
  if constexpr (Mma<T>::kLift == 0) return x * c;
  else return __fmaf_rn(x, c, (float)Mma<T>::kLift);
}
// Log-sum of a row: its maximum m before the scale, its sum l of weights that
// carry a factor of 2^LIFT.
template <int LIFT>
__device__ __forceinline__ float lse_of(float m, float scale, float l) {
  return __fmaf_rn(m, scale, logf(l * (1.f / (float)(1 << LIFT))));
}

// ------------------------------------------------------------ sequences --
struct Seq {
  int row0, rows;  // query rows [row0, row0 + rows)
  int len;         // cache positions
  int ctx;         // len - rows: positions before the first query row (may be negative)
};

// Sequence b with its fields brought into range: rows outside q and lengths
// past the block table set the device error bit and are cut off.
__device__ __forceinline__ Seq load_seq(const SeqBatch& sq, int b) {
  Seq s;
  if (sq.cu_q) {
    const int a = __ldg(&sq.cu_q[b]), e = __ldg(&sq.cu_q[b + 1]);
    s.row0 = a;
    s.rows = e - a;
    if (a < 0 || e < a || e > sq.num_rows) {
      atomicOr(sq.err, DEV_ERR_INDEX_RANGE);
      s.row0 = 0;
      s.rows = 0;
    }
  } else {
    s.row0 = b * sq.rows_each;
    s.rows = sq.rows_each;
  }
  s.len = __ldg(&sq.seq_lens[b]);
  s.ctx = 0;
  return s;
}
__device__ __forceinline__ void clamp_len(const SeqBatch& sq, int page_size, Seq& s) {
  const int64_t cap = (int64_t)sq.table_cols * page_size;
  if (s.len < 0) s.len = 0;
  if (s.len > cap) {
    atomicOr(sq.err, DEV_ERR_INDEX_RANGE);
    s.len = (int)cap;
  }
  s.ctx = s.len - s.rows;
}

// Whether drafted-token bits (or causal order) let row j see position ctx + i, i >= 0.
__device__ __forceinline__ bool sees_draft(const SeqBatch& sq, int row, int j, int i) {
  if (!sq.mask) return i <= j;
  if ((i >> 6) >= sq.mask_words) return false;
  return (__ldg(&sq.mask[(int64_t)row * sq.mask_words + (i >> 6)]) >> (i & 63)) & 1;
}

// The sequence that starts last at or before `row` (warp-wide search over cu_q, all lanes call
// it), -1 if none; whether its rows hold the row is the caller's to see.
__device__ __forceinline__ int find_seq(const SeqBatch& sq, int row) {
  if (!sq.cu_q) return row / sq.rows_each;
  const int lane = threadIdx.x & 31;
  int lo = 0, n = sq.num_seqs;  // the answer is in [lo, lo + n)
  if (row < __ldg(&sq.cu_q[0])) return -1;
  while (n > 1) {  // the last sequence that starts at or before the row
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool le = lane * step < n && __ldg(&sq.cu_q[at]) <= row;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int w = 31 - __clz(m | 1u);
    n = min(step, n - w * step);
    lo += w * step;
  }
  return lo;
}

// Contiguous split of `total` units over the CTAs of the grid.
__device__ __forceinline__ void split_range(uint32_t total, uint32_t grid, uint32_t c, uint32_t& begin, uint32_t& end) {
  const uint32_t q = total / grid, r = total % grid;
  begin = c * q + min(c, r);
  end = begin + q + (c < r ? 1u : 0u);
}
__device__ __forceinline__ uint32_t split_owner(uint32_t total, uint32_t grid, uint32_t t) {
  const uint32_t q = total / grid, r = total % grid;
  return t < r * (q + 1) ? t / (q + 1) : r + (t - r * (q + 1)) / q;
}

}  // namespace att
}  // namespace daric
