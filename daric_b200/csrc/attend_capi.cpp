// C entries of the operators over the paged KV cache: attention, block
// selection and eviction. Arguments are checked here; nothing waits for the
// GPU, allocates device memory or uploads a descriptor, so every call can be
// captured into a graph (after the first call on a device).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>
#include <vector>

#include "attend.h"

using namespace daric;

namespace {

template <class F>
int guard(F&& f) {
  try {
    f();
    clear_error();
    return DARIC_OK;
  } catch (const Error& e) {
    record_error(e.code, e.what());
    return e.code;
  } catch (const std::exception& e) {
    record_error(DARIC_ERR_STATE, e.what());
    return DARIC_ERR_STATE;
  } catch (...) {
    record_error(DARIC_ERR_STATE, "unknown error");
    return DARIC_ERR_STATE;
  }
}

struct OnDevice {
  int prev = -1;
  explicit OnDevice(int dev) {
    DARIC_CUDA(cudaGetDevice(&prev));
    if (prev == dev) prev = -1;
    else DARIC_CUDA(cudaSetDevice(dev));
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool aligned(const void* p, int64_t a, int64_t b, int64_t n) {
  return (uintptr_t)p % n == 0 && a % n == 0 && b % n == 0;
}

// The arguments that every call over a batch of query rows shares.
SeqBatch seq_batch(const int32_t* table, int64_t table_ld, int64_t num_seqs, int64_t table_cols,
                   const int32_t* seq_lens, const int32_t* cu_q, int64_t num_rows, int64_t q_heads, int64_t kv_heads,
                   int64_t page_size) {
  SeqBatch b{};
  DARIC_CHECK(num_seqs >= 1 && num_rows >= 0 && table_cols >= 1, "batch sizes must be positive");
  DARIC_CHECK(num_seqs <= 65535, "at most 65535 sequences per call");
  // (a tile of up to 1024 keys past the end is still counted in 32 bits)
  DARIC_CHECK(table_cols <= (INT32_MAX - 1024) / page_size, "block table reaches past int32 positions");
  DARIC_CHECK(table && seq_lens, "NULL block table or lengths");
  DARIC_CHECK(table_ld >= table_cols || num_seqs == 1, "block table rows overlap");
  DARIC_CHECK(q_heads >= kv_heads && q_heads % kv_heads == 0,
              "query heads (" + std::to_string(q_heads) + ") must be a multiple of KV heads (" +
                  std::to_string(kv_heads) + ")");
  DARIC_CHECK(num_rows <= INT32_MAX / q_heads, "too many query rows");
  DARIC_CHECK(cu_q || num_rows % num_seqs == 0, "query rows must divide evenly over the sequences without cu_q");
  b.table = table;
  b.table_ld = table_ld;
  b.table_cols = (int32_t)table_cols;
  b.seq_lens = seq_lens;
  b.cu_q = cu_q;
  b.num_seqs = (int32_t)num_seqs;
  b.num_rows = (int32_t)num_rows;
  b.rows_each = (int32_t)(num_rows / num_seqs);
  b.group = (int32_t)(q_heads / kv_heads);
  b.group_div = make_fastdiv((uint32_t)b.group);
  return b;
}

int check_layer(const LayerRef& L, int kv_dtype, int64_t head_dim, int device, const char* what) {
  DARIC_CHECK(L.device == device, std::string(what) + ": the tensors must be on the KV cache's device");
  DARIC_CHECK(kv_dtype == DARIC_DTYPE_BF16 || kv_dtype == DARIC_DTYPE_F16,
              std::string(what) + ": the KV cache must be bfloat16 or float16");
  DARIC_CHECK(L.elem_size == 2, std::string(what) + ": kv_dtype does not match the registered element size");
  DARIC_CHECK(L.kv.head_dim == head_dim, std::string(what) + ": query head dimension " + std::to_string(head_dim) +
                                             " differs from the KV cache's " + std::to_string(L.kv.head_dim));
  return kv_dtype;
}

void check_scale(float scale) {
  DARIC_CHECK(scale > 0.f && std::isfinite(scale), "scale must be positive and finite");
}

// How the query heads of one KV head times the rows of a sequence (their
// mean: the lengths are on the device) are tiled: up to 16 and 32 pairs as row
// groups of 16 (attend_kernels.cu, memory-bound there); from 33 on as 128 or
// 256 rows on the tensor cores (wide_kernels.cu). That form's tiles of 128 keys
// leave no room for 256-wide heads (tiles of 64 would, and are not built), which
// take four row groups (8 sequences of 8192 keys, 8 KV heads of 4, bf16, 256
// wide: 16 rows 223 us, 64 rows 770 us, 178 TFLOP/s; 128 wide: 84 and 104). (us
// for 16 sequences of 8192 keys, 8 KV heads of 128, bf16, by pairs: 16: one row
// group 104, two 105, tensor cores 120; 20: 186, 107, 120; 32: 188, 111, 121;
// 36: two row groups 184, one tile of 128 124, two 156; 128: 362, 133, 164; 132:
// 445, 216, 166.)
struct Variant {
  int rg;    // row groups of 16, or 0
  int mt;    // tiles of 128 rows, or 0
  int rows;  // of a CTA
  int ctas;  // resident per SM: rings of 70 KB with one row group, 104 KB or less with more, else all of it
};
Variant variant_rg(int rg, int64_t dim) { return {rg, 0, attend_rows(rg), dim > 128 ? 1 : (rg == 1 ? 3 : 2)}; }
Variant variant_mt(int mt) { return {0, mt, 128 * mt, 1}; }

// k: pages listed per row (0: all of the sequence).
Variant attend_variant(int64_t num_rows, int64_t num_seqs, int64_t group, int64_t head_dim, double layer_bytes, int64_t k,
                       int64_t table_cols) {
  const int64_t rows = k ? group : (num_rows + num_seqs - 1) / num_seqs * group;
  // the wide form keeps offsets in 32 bits of 16 bytes
  const bool wide = head_dim <= 128 && layer_bytes < 60.0 * (1ll << 30);
  // Listed pages: where a sequence fills a tile of pairs, and the tile has no
  // more than 32 rows (a bit each: four or more query heads per KV head), the
  // rows of a tile share one pass over the pages that any of them lists; that
  // many rows one by one read each page many times. (us for 64 of 512 pages, 8 KV heads of 4; shared where all
  // rows list the same pages, shared where no two lists are alike, row by row:
  // 1 x 16 rows 27, 39, 23; 1 x 128 rows 33, 77, 82; 1 x 512 rows 62, 185, 274;
  // 16 x 16 rows 60, 173, 163; 16 x 32 rows 67, 204, 309. Lists of 16 pages,
  // 16 x 32 rows: 30, 182, 116. How alike the lists are only the GPU knows: short
  // lists with little in common lose by the rule, long ones win.) The merge takes
  // repeats and padding as they come, so lists may be longer than the table.
  if (k && wide && group >= 4 && num_rows * group >= 128 * num_seqs && table_cols <= kUnionPages && k <= kUnionPages)
    return variant_mt(1);
  if (rows <= 16) return variant_rg(1, head_dim);
  if (rows <= 32 || k) return variant_rg(2, head_dim);
  if (!wide) return variant_rg(4, head_dim);
  return variant_mt(rows <= 128 ? 1 : 2);
}

double layer_bytes(const KvView& kv) { return (double)kv.num_pages * (double)kv.page_stride; }

// Lists of a wide call over listed pages.
struct Lists {
  int64_t lists, row;
  int64_t bytes() const { return lists * row * 16 + (lists * 4 + 15) / 16 * 16 + (lists + 1) * 8; }
};
Lists list_room(int64_t num_rows, int64_t num_seqs, int64_t q_heads, int64_t kv_heads, int64_t k, int64_t table_cols) {
  return {(num_rows * (q_heads / kv_heads) / 128 + num_seqs) * kv_heads, std::min<int64_t>(table_cols, 32 * k)};
}

size_t attend_bytes(int grid, int rows, int head_dim) {
  return (size_t)grid * (2 * (size_t)rows * head_dim * 4 + 2 * (size_t)rows * 8 + 16);
}

// Lays the attention's workspace out: descriptors, maxima and sums, outputs.
void attend_workspace(AttendLaunch& p, int grid, int rows, void* ws, int64_t ws_bytes) {
  DARIC_CHECK(ws && (uintptr_t)ws % 16 == 0, "workspace must be a 16-byte aligned device buffer");
  DARIC_CHECK((int64_t)attend_bytes(grid, rows, p.kv.head_dim) <= ws_bytes, "workspace is too small");
  uint8_t* w = (uint8_t*)ws;
  p.desc = reinterpret_cast<int4*>(w);
  p.part_ml = reinterpret_cast<float2*>(w + (size_t)grid * 16);
  p.part = reinterpret_cast<float*>(w + (size_t)grid * 16 + (size_t)grid * 2 * rows * 8);
}

}  // namespace

extern "C" {

int daric_attend_workspace(int device, int64_t head_dim, int64_t* out_bytes) {
  return guard([&] {
    DARIC_CHECK(out_bytes, "out_bytes is NULL");
    DARIC_CHECK(head_dim > 0 && head_dim <= 256, "head dimension must be at most 256");
    const int sms = device_info(device).sm_count;
    size_t most = 0;
    for (const Variant& v : {variant_rg(1, head_dim), variant_rg(2, head_dim), variant_rg(4, head_dim), variant_mt(2)})
      if (v.mt == 0 || head_dim <= 128) most = std::max(most, attend_bytes(sms * v.ctas, v.rows, (int)head_dim));
    *out_bytes = (int64_t)most;
  });
}

int daric_sparse_workspace(int device, int64_t head_dim, int64_t num_rows, int64_t num_seqs, int64_t q_heads,
                           int64_t kv_heads, int64_t k, int64_t table_cols, int64_t* out_bytes) {
  return guard([&] {
    DARIC_CHECK(out_bytes, "out_bytes is NULL");
    DARIC_CHECK(head_dim > 0 && head_dim <= 256, "head dimension must be at most 256");
    DARIC_CHECK(num_rows >= 0 && num_seqs >= 1 && kv_heads >= 1 && q_heads >= kv_heads && k >= 1 && table_cols >= 1,
                "sizes must be positive");
    const Variant v = attend_variant(num_rows, num_seqs, q_heads / kv_heads, head_dim, 0.0, k, table_cols);
    int64_t most = (int64_t)attend_bytes(device_info(device).sm_count * v.ctas, v.rows, (int)head_dim);
    for (int rg : {1, 2}) {  // a layer too large for the wide form
      const Variant u = variant_rg(rg, head_dim);
      most = std::max(most, (int64_t)attend_bytes(device_info(device).sm_count * u.ctas, u.rows, (int)head_dim));
    }
    if (v.mt) most = (most + 15) / 16 * 16 + list_room(num_rows, num_seqs, q_heads, kv_heads, k, table_cols).bytes();
    *out_bytes = most;
  });
}

int daric_copier_tree_attention(daric_copier* copier, const char* layer_name, int kv_dtype, const void* q,
                                int64_t q_row, int64_t q_head, int64_t num_rows, int64_t q_heads, int64_t head_dim,
                                const int32_t* block_table, int64_t table_ld, int64_t num_seqs, int64_t table_cols,
                                const int32_t* seq_lens, const int32_t* cu_q, const int64_t* tree_mask,
                                int64_t mask_words, float scale, void* out, int64_t out_row, int64_t out_head,
                                float* lse, int64_t lse_row, void* workspace, int64_t workspace_bytes, int device,
                                void* stream) {
  return guard([&] {
    const LayerRef L = layer_ref(copier, layer_name);
    check_layer(L, kv_dtype, head_dim, device, "tree_attention");
    check_scale(scale);
    AttendLaunch p{};
    p.kv = L.kv;
    p.sq = seq_batch(block_table, table_ld, num_seqs, table_cols, seq_lens, cu_q, num_rows, q_heads, L.kv.heads,
                     L.kv.page_size);
    if (num_rows == 0) return;
    DARIC_CHECK(q && out, "NULL query or output");
    DARIC_CHECK(!tree_mask || (mask_words >= 1 && mask_words <= (1 << 25)), "tree mask needs 1 to 2^25 words per row");
    DARIC_CHECK(aligned(q, q_row * 2, q_head * 2, 16), "query rows must be 16-byte aligned");
    DARIC_CHECK(aligned(out, out_row * 2, out_head * 2, 16), "output rows must be 16-byte aligned");
    const DeviceInfo di = device_info(device);
    p.sq.mask = reinterpret_cast<const uint64_t*>(tree_mask);
    p.sq.mask_words = (int32_t)mask_words;
    p.sq.err = di.err;
    p.q = (const uint8_t*)q;
    p.q_row = q_row * 2;
    p.q_head = q_head * 2;
    p.out = (uint8_t*)out;
    p.out_row = out_row * 2;
    p.out_head = out_head * 2;
    p.lse = lse;
    p.lse_row = lse_row;
    p.scale = scale;
    // tiles of the whole batch are counted in 32 bits
    const Variant var = attend_variant(num_rows, num_seqs, p.sq.group, head_dim, layer_bytes(L.kv), 0, table_cols);
    const int rows = var.rows;
    const double tiles = (double)L.kv.heads * ((double)num_rows * p.sq.group / rows + (double)num_seqs) *
                         ((double)table_cols * L.kv.page_size / 16.0 + 1.0);
    DARIC_CHECK(tiles < 4.0e9, "tree_attention: the batch has too many tiles for one call");
    DARIC_CHECK((int64_t)num_rows * p.sq.group / rows < (1 << 18), "tree_attention: too many query rows");
    const int grid = di.sm_count * var.ctas;
    attend_workspace(p, grid, rows, workspace, workspace_bytes);
    OnDevice on(device);
    if (var.mt) launch_wide(p, kv_dtype, var.mt, grid, (cudaStream_t)stream);
    else launch_attend(p, kv_dtype, var.rg, grid, (cudaStream_t)stream);
  });
}

int daric_copier_sparse_attention(daric_copier* copier, const char* layer_name, int kv_dtype, const void* q,
                                  int64_t q_row, int64_t q_head, int64_t num_rows, int64_t q_heads, int64_t head_dim,
                                  const int32_t* pages, int64_t pages_row, int64_t pages_head, int64_t k,
                                  const int32_t* block_table, int64_t table_ld, int64_t num_seqs, int64_t table_cols,
                                  const int32_t* seq_lens, const int32_t* cu_q, float scale, void* out,
                                  int64_t out_row, int64_t out_head, float* lse, int64_t lse_row, void* workspace,
                                  int64_t workspace_bytes, int device, void* stream) {
  return guard([&] {
    const LayerRef L = layer_ref(copier, layer_name);
    check_layer(L, kv_dtype, head_dim, device, "sparse_attention");
    check_scale(scale);
    AttendLaunch p{};
    p.kv = L.kv;
    p.sq = seq_batch(block_table, table_ld, num_seqs, table_cols, seq_lens, cu_q, num_rows, q_heads, L.kv.heads,
                     L.kv.page_size);
    if (num_rows == 0) return;
    DARIC_CHECK(q && out && pages, "NULL query, output or page list");
    DARIC_CHECK(k >= 1 && k <= (INT32_MAX - 1024) / L.kv.page_size,
                "sparse_attention: page lists must have at least one entry, and less than 2^31 - 1024 positions");
    DARIC_CHECK(aligned(q, q_row * 2, q_head * 2, 16), "query rows must be 16-byte aligned");
    DARIC_CHECK(aligned(out, out_row * 2, out_head * 2, 16), "output rows must be 16-byte aligned");
    const DeviceInfo di = device_info(device);
    p.sq.err = di.err;
    p.q = (const uint8_t*)q;
    p.q_row = q_row * 2;
    p.q_head = q_head * 2;
    p.out = (uint8_t*)out;
    p.out_row = out_row * 2;
    p.out_head = out_head * 2;
    p.lse = lse;
    p.lse_row = lse_row;
    p.pages = pages;
    p.pages_row = pages_row;
    p.pages_head = pages_head;
    p.k = (int32_t)k;
    p.scale = scale;
    Variant var = attend_variant(num_rows, num_seqs, p.sq.group, head_dim, layer_bytes(L.kv), k, table_cols);
    const Lists room = list_room(num_rows, num_seqs, q_heads, L.kv.heads, k, table_cols);
    const double per_list = (double)std::max(k, room.row) * L.kv.page_size / 16.0 + 1.0;
    const double tiles = (double)L.kv.heads * (double)num_rows * ((double)p.sq.group / 16 + 1.0) * per_list;
    DARIC_CHECK(tiles < 4.0e9, "sparse_attention: the batch has too many tiles for one call");
    DARIC_CHECK(!var.mt || num_rows * p.sq.group / var.rows < (1 << 18), "sparse_attention: too many query rows");
    const int grid = di.sm_count * var.ctas;
    attend_workspace(p, grid, var.rows, workspace, workspace_bytes);
    OnDevice on(device);
    if (var.mt) {
      const int64_t at = ((int64_t)attend_bytes(grid, var.rows, (int)head_dim) + 15) / 16 * 16;
      DARIC_CHECK(at + room.bytes() <= workspace_bytes, "workspace is too small");
      uint8_t* w = (uint8_t*)workspace + at;
      p.lists = (int32_t)room.lists;
      p.list_row = (int32_t)room.row;
      p.list = (uint4*)w;
      p.list_count = (int32_t*)(w + room.lists * room.row * 16);
      p.list_tile = (int2*)(w + room.lists * room.row * 16 + (room.lists * 4 + 15) / 16 * 16);
      launch_wide(p, kv_dtype, 1, grid, (cudaStream_t)stream);
    } else {
      launch_attend(p, kv_dtype, var.rg, grid, (cudaStream_t)stream);
    }
  });
}

int daric_copier_page_bounds(daric_copier* copier, const char* layer_name, int kv_dtype, const int32_t* block_table,
                             int64_t table_ld, int64_t num_seqs, int64_t table_cols, const int32_t* seq_lens,
                             const int32_t* start, void* bounds, int device, void* stream) {
  return guard([&] {
    const LayerRef L = layer_ref(copier, layer_name);
    check_layer(L, kv_dtype, L.kv.head_dim, device, "page_bounds");
    BoundsLaunch p{};
    p.kv = L.kv;
    p.sq = seq_batch(block_table, table_ld, num_seqs, table_cols, seq_lens, nullptr, 0, L.kv.heads, L.kv.heads,
                     L.kv.page_size);
    DARIC_CHECK(bounds && (uintptr_t)bounds % 16 == 0, "bounds must be a 16-byte aligned device buffer");
    const DeviceInfo di = device_info(device);
    p.sq.err = di.err;
    p.start = start;
    p.bounds = (uint8_t*)bounds;
    OnDevice on(device);
    launch_page_bounds(p, kv_dtype, di.sm_count, (cudaStream_t)stream);
  });
}

int daric_select_pages_workspace(int64_t num_rows, int64_t kv_heads, int64_t table_cols, int64_t* out_bytes) {
  return guard([&] {
    DARIC_CHECK(out_bytes, "out_bytes is NULL");
    DARIC_CHECK(num_rows >= 0 && kv_heads >= 1 && table_cols >= 1 && table_cols <= (1 << 20), "select_pages: sizes out of range");
    const int64_t items = num_rows * kv_heads;
    *out_bytes = items * 4 * ((table_cols + 3) / 4 * 4 + (table_cols + kScoreChunk - 1) / kScoreChunk);
  });
}

int daric_select_pages(const void* q, int kv_dtype, int64_t q_row, int64_t q_head, int64_t num_rows, int64_t q_heads,
                       int64_t head_dim, const void* bounds, int64_t num_pages, int64_t kv_heads,
                       const int32_t* block_table, int64_t table_ld, int64_t num_seqs, int64_t table_cols,
                       const int32_t* seq_lens, const int32_t* cu_q, int64_t block_size, int64_t k, int64_t first,
                       int64_t last, int32_t* out, void* workspace, int64_t workspace_bytes, int device,
                       void* stream) {
  return guard([&] {
    DARIC_CHECK(kv_dtype == DARIC_DTYPE_BF16 || kv_dtype == DARIC_DTYPE_F16,
                "select_pages: the bounds must be bfloat16 or float16");
    DARIC_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256,
                "select_pages: head dimension must be 64, 128 or 256, got " + std::to_string(head_dim));
    DARIC_CHECK(kv_heads >= 1 && kv_heads < 4096 && num_pages >= 1 && num_pages <= INT32_MAX, "bounds sizes out of range");
    DARIC_CHECK(block_size >= 1 && block_size <= 1024, "block size must be in [1, 1024]");
    DARIC_CHECK(first >= 0 && last >= 1 && k >= 1 && first <= k - last && k <= INT32_MAX,
                "select_pages: k must hold the first and last pages that are always taken (last >= 1)");
    DARIC_CHECK(table_cols <= (1 << 20), "select_pages: at most 1048576 pages per sequence");
    SelectPagesLaunch p{};
    p.sq = seq_batch(block_table, table_ld, num_seqs, table_cols, seq_lens, cu_q, num_rows, q_heads, kv_heads,
                     block_size);
    if (num_rows == 0) return;
    DARIC_CHECK(q && bounds && out, "NULL query, bounds or output");
    DARIC_CHECK(aligned(q, q_row * 2, q_head * 2, 16), "query rows must be 16-byte aligned");
    DARIC_CHECK((uintptr_t)bounds % 16 == 0, "bounds must be 16-byte aligned");
    DARIC_CHECK(workspace && (uintptr_t)workspace % 16 == 0, "workspace must be a 16-byte aligned device buffer");
    const int64_t items = num_rows * kv_heads;
    const int64_t chunks = (table_cols + kScoreChunk - 1) / kScoreChunk;
    const int64_t keys_row = (table_cols + 3) / 4 * 4;
    DARIC_CHECK(items * 4 * (keys_row + chunks) <= workspace_bytes, "workspace is too small");
    const DeviceInfo di = device_info(device);
    p.sq.err = di.err;
    p.q = (const uint8_t*)q;
    p.q_row = q_row * 2;
    p.q_head = q_head * 2;
    p.bounds = (const uint8_t*)bounds;
    p.num_pages = (int32_t)num_pages;
    p.heads = (int32_t)kv_heads;
    p.head_dim = (int32_t)head_dim;
    p.page_size = (int32_t)block_size;
    p.sm_count = di.sm_count;
    p.k = (int32_t)k;
    p.first = (int32_t)first;
    p.last = (int32_t)last;
    p.keys = (uint32_t*)workspace;
    p.keys_row = (int32_t)keys_row;
    p.mags = (float*)workspace + items * keys_row;
    p.out = out;
    OnDevice on(device);
    launch_select_pages(p, kv_dtype, (cudaStream_t)stream);
  });
}

int daric_scores_workspace(int64_t num_rows, int64_t q_heads, int64_t table_cols, int64_t block_size,
                           int64_t* out_bytes) {
  return guard([&] {
    DARIC_CHECK(out_bytes, "out_bytes is NULL");
    DARIC_CHECK(num_rows >= 0 && q_heads >= 1 && table_cols >= 1 && block_size >= 1, "sizes out of range");
    const int64_t splits = (table_cols * block_size + kLseKeys - 1) / kLseKeys;
    *out_bytes = num_rows * q_heads * (splits * 8 + 4) + 16;
  });
}

int daric_copier_attention_scores(daric_copier* copier, const char* layer_name, int kv_dtype, const void* q,
                                  int64_t q_row, int64_t q_head, int64_t num_rows, int64_t q_heads, int64_t head_dim,
                                  const int32_t* block_table, int64_t table_ld, int64_t num_seqs, int64_t table_cols,
                                  const int32_t* seq_lens, const int32_t* cu_q, const int64_t* tree_mask,
                                  int64_t mask_words, const float* lse, int64_t lse_row, float scale, float* scores,
                                  int64_t scores_row, int64_t scores_cols, const int64_t* col_off, int accumulate,
                                  void* workspace, int64_t workspace_bytes, int device, void* stream) {
  return guard([&] {
    const LayerRef L = layer_ref(copier, layer_name);
    check_layer(L, kv_dtype, head_dim, device, "attention_scores");
    check_scale(scale);
    ScoresLaunch p{};
    p.kv = L.kv;
    p.sq = seq_batch(block_table, table_ld, num_seqs, table_cols, seq_lens, cu_q, num_rows, q_heads, L.kv.heads,
                     L.kv.page_size);
    DARIC_CHECK(scores && col_off && (q || num_rows == 0), "NULL query, scores or column offsets");
    DARIC_CHECK(!tree_mask || (mask_words >= 1 && mask_words <= (1 << 25)), "tree mask needs 1 to 2^25 words per row");
    DARIC_CHECK(num_rows == 0 || aligned(q, q_row * 2, q_head * 2, 16), "query rows must be 16-byte aligned");
    DARIC_CHECK(scores_cols >= 0 && (scores_row >= scores_cols || L.kv.heads == 1), "score rows overlap");
    const int64_t splits = (table_cols * L.kv.page_size + kLseKeys - 1) / kLseKeys;
    DARIC_CHECK(splits <= 65535, "attention_scores: sequences of at most 16.7M positions");
    const DeviceInfo di = device_info(device);
    p.sq.err = di.err;
    p.sq.mask = reinterpret_cast<const uint64_t*>(tree_mask);
    p.sq.mask_words = (int32_t)mask_words;
    p.q = (const uint8_t*)q;
    p.q_row = q_row * 2;
    p.q_head = q_head * 2;
    p.lse = lse;
    p.lse_row = lse_row;
    p.scores = scores;
    p.scores_row = scores_row;
    p.scores_cols = scores_cols;
    p.col_off = col_off;
    p.accumulate = accumulate ? 1 : 0;
    p.scale = scale;
    p.splits = (int32_t)splits;
    p.sm_count = di.sm_count;
    if (num_rows == 0) p.lse = scores;  // no rows: never read, and nothing to join
    if (!p.lse) {
      DARIC_CHECK(workspace && (uintptr_t)workspace % 8 == 0, "workspace must be an 8-byte aligned device buffer");
      DARIC_CHECK(num_rows * q_heads * ((int64_t)p.splits * 8 + 4) <= workspace_bytes, "workspace is too small");
      p.part = (float2*)workspace;
      p.lse_work = (float*)workspace + num_rows * q_heads * p.splits * 2;
    }
    OnDevice on(device);
    launch_scores(p, kv_dtype, (cudaStream_t)stream);
  });
}

int daric_copier_compact(daric_copier* copier, int64_t num_layers, const char* const* layer_names, int kv_dtype,
                         int mode, int64_t lists, int per_head, const int32_t* idx, int64_t idx_row,
                         const int32_t* count,
                         int64_t count_row, int64_t num_segs, const int64_t* out_off, const int64_t* seg_cap,
                         const int64_t* seg_blk_off, const int64_t* dst_start, const int32_t* block_table,
                         int64_t block_table_numel, int device, void* stream) {
  return guard([&] {
    DARIC_CHECK(copier, "copier is NULL");
    DARIC_CHECK(mode == DARIC_ROPE_NONE || mode == DARIC_ROPE_FLEXIBLE, "compact: mode must be NONE or FLEXIBLE");
    if (num_layers <= 0 || num_segs <= 0) return;
    DARIC_CHECK(layer_names && idx && count && out_off && seg_cap, "NULL argument");
    DARIC_CHECK(block_table != nullptr, "block_table is NULL");
    std::vector<LayerRef> all;
    for (int64_t l = 0; l < num_layers; ++l) all.push_back(layer_ref(copier, layer_names[l]));
    const LayerRef& A = all[0];
    const bool rotate = mode == DARIC_ROPE_FLEXIBLE;
    int es = 0;
    switch (kv_dtype) {
      case DARIC_DTYPE_F32: es = 4; break;
      case DARIC_DTYPE_F16:
      case DARIC_DTYPE_BF16: es = 2; break;
      case DARIC_DTYPE_FP8_E4M3: es = 1; break;
      default: throw Error(DARIC_ERR_INVALID, "compact: unknown KV dtype");
    }
    for (int64_t l = 0; l < num_layers; ++l) {
      const LayerRef& L = all[l];
      DARIC_CHECK(L.device == device, "compact: the tensors must be on the KV cache's device");
      DARIC_CHECK(L.elem_size == es, "compact: kv_dtype does not match the registered element size");
      DARIC_CHECK(L.kv.page_size == A.kv.page_size && L.kv.heads == A.kv.heads && L.kv.head_dim == A.kv.head_dim &&
                      L.kv.num_pages == A.kv.num_pages,
                  "compact: layers of one call must share block size, blocks, heads and head dimension");
      // places of tokens are kept in 32 bits of 16 bytes
      DARIC_CHECK((double)L.kv.num_pages * (double)L.kv.page_stride < 60.0 * (1ll << 30),
                  "compact: layers of less than 60 GiB");
      if (rotate) {
        DARIC_CHECK(L.table, std::string("layer has no rotary table (register_rotary): ") + layer_names[l]);
        DARIC_CHECK(L.tab_dtype == A.tab_dtype && L.neox == A.neox && L.half_rot == A.half_rot &&
                        L.max_pos == A.max_pos && L.kv_dtype == kv_dtype,
                    "compact: layers of one call must share the rotary style and table shape");
      }
      for (int64_t m = 0; m < l; ++m)
        DARIC_CHECK(all[m].kv.base != L.kv.base, "compact: a layer is named twice");
    }
    const int64_t H = A.kv.heads, per_layer = per_head ? H : 1;
    DARIC_CHECK(lists == per_layer || lists == num_layers * per_layer,
                "compact: the selection must have one row per layer, or one for all layers (times the KV heads with "
                "per_head); got " + std::to_string(lists) + " rows for " + std::to_string(num_layers) + " layers and " +
                    std::to_string(H) + " heads");
    const bool shared = lists == per_layer;
    CompactLaunch p{};
    p.idx = idx;
    p.idx_row = idx_row;
    p.count = count;
    p.count_row = count_row;
    p.block_table = block_table;
    p.table_numel = block_table_numel;
    DARIC_CHECK((int64_t)A.kv.head_dim * es <= 4096, "compact: rows of at most 4096 bytes");
    p.num_pages = A.kv.num_pages;
    p.page_size = A.kv.page_size;
    p.heads = A.kv.heads;
    p.head_dim = A.kv.head_dim;
    p.page_div = A.kv.page_div;
    p.per_head = per_head ? 1 : 0;
    p.shared = shared;
    p.rotate = rotate;
    p.neox = rotate ? A.neox : 1;
    p.half_rot = rotate ? A.half_rot : 0;
    p.table_row = A.table_row;
    p.max_pos = A.max_pos;
    for (int64_t s = 0; s < num_segs; ++s) {
      DARIC_CHECK(out_off[s] >= 0 && seg_cap[s] >= 0 && (!seg_blk_off || seg_blk_off[s] >= 0) && (!dst_start || dst_start[s] >= 0),
                  "negative segment field at segment " + std::to_string(s));
      // (differences of what is not negative: no sum that could pass 64 bits)
      DARIC_CHECK(out_off[s] <= idx_row - seg_cap[s] || lists == 1, "segment " + std::to_string(s) + " exceeds the selection's row");
      DARIC_CHECK(seg_cap[s] <= INT32_MAX - (dst_start ? dst_start[s] : 0), "positions exceed int32");
    }
    const DeviceInfo di = device_info(device);
    p.err = di.err;
    OnDevice on(device);
    for (int64_t l0 = 0; l0 < num_layers; l0 += kCompactLayers) {
      p.layer0 = (int32_t)l0;
      p.num_layers = (int32_t)std::min<int64_t>(kCompactLayers, num_layers - l0);
      for (int l = 0; l < p.num_layers; ++l) {
        const LayerRef& L = all[l0 + l];
        p.layers[l] = CompactLayer{L.kv.base, L.table, L.kv.page_stride, L.kv.tok_stride, L.kv.head_stride, L.kv.v_off};
      }
      for (int64_t s0 = 0; s0 < num_segs; s0 += kCompactSegs) {
        p.num_segs = (int32_t)std::min<int64_t>(kCompactSegs, num_segs - s0);
        for (int s = 0; s < p.num_segs; ++s)
          p.segs[s] = CompactSeg{seg_blk_off ? seg_blk_off[s0 + s] : 0, out_off[s0 + s], (int32_t)seg_cap[s0 + s],
                                 (int32_t)(dst_start ? dst_start[s0 + s] : 0), (int32_t)(s0 + s)};
        launch_compact(p, kv_dtype, A.tab_dtype, es, di.sm_count, (cudaStream_t)stream);
      }
    }
  });
}

}  // extern "C"
