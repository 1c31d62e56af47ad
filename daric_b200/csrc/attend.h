// Launch structures of the operators that read the paged KV cache by
// attention (attend_kernels.cu), select blocks of it (blocks_kernels.cu) and
// shrink it (evict_kernels.cu); their C entries are in attend_capi.cpp.
#pragma once

#include "internal.h"

struct daric_copier;

namespace daric {

// K and V rows of one registered layer: row (block, token, head) of K is at
// base + block * page_stride + token * tok_stride + head * head_stride, its V
// row v_off bytes further. All strides are multiples of 16 bytes.
struct KvView {
  uint8_t* base;
  int64_t page_stride, tok_stride, head_stride, v_off;
  int32_t num_pages, page_size;
  int32_t heads, head_dim;
  FastDiv page_div;  // position -> page
};

// A registered layer as the operators need it (capi.cpp).
struct LayerRef {
  KvView kv;
  int device;
  int kv_dtype;              // dtype given by register_rotary, -1 without one
  int64_t elem_size;
  const uint8_t* table;      // rotary table (nullptr without register_rotary)
  int64_t table_row, max_pos;
  int tab_dtype, neox, half_rot;
};
LayerRef layer_ref(daric_copier* c, const char* name);

struct DeviceInfo {
  int sm_count;
  int* err;
};
DeviceInfo device_info(int device);

// The batch of query rows against the cache: sequence b has rows
// [cu_q[b], cu_q[b + 1]) of q (N / B each when cu_q is null), its last query
// row is cache position seq_lens[b] - 1.
struct SeqBatch {
  const int32_t* table;   // [B, table_cols], row stride table_ld
  int64_t table_ld;
  int32_t table_cols;
  const int32_t* seq_lens;
  const int32_t* cu_q;    // null: rows_each rows per sequence
  int32_t num_seqs, num_rows, rows_each;
  const uint64_t* mask;   // [N, mask_words] drafted-token bits, null: causal
  int32_t mask_words;
  int32_t group;          // query heads per KV head
  FastDiv group_div;
  int32_t* err;
};

struct AttendLaunch {
  KvView kv;
  SeqBatch sq;
  const uint8_t* q;
  int64_t q_row, q_head;      // bytes
  uint8_t* out;
  int64_t out_row, out_head;  // bytes
  float* lse;                 // [N, Hq], row stride lse_row (elements); may be null
  int64_t lse_row;
  const int32_t* pages;       // sparse: [N, Hkv, k] listed pages
  int64_t pages_row, pages_head;
  int32_t k;
  float scale;
  float* part;                // workspace: partial outputs
  float2* part_ml;            // workspace: their maxima and sums
  int4* desc;                 // workspace: what the join of a CTA does
  // listed pages on the tensor cores (workspace): per row tile of 128 pairs
  // and KV head the pages that any of its rows lists
  uint4* list;                // [lists, list_row]: page, rows that list it, block
  int32_t* list_count;        // [lists], -1: no such row tile
  int2* list_tile;            // [lists / heads]: sequence and its row tile
  int32_t lists, list_row;
};
constexpr int kUnionPages = 48 * 1024;  // most pages of a sequence for that

// Rows of query heads a CTA of the row-tile variant rg (1, 2, 4) holds.
constexpr int attend_rows(int rg) { return 16 * rg; }

void launch_attend(const AttendLaunch& p, int dtype, int rg, int grid, cudaStream_t s);
// Many rows: tiles of 128 * mt pairs, head_dim 64 or 128 (wide_kernels.cu).
void launch_wide(const AttendLaunch& p, int dtype, int mt, int grid, cudaStream_t s);

// Smallest and largest key value of each dimension over the tokens of a page,
// per KV head: bounds[block][head][0 = min, 1 = max][dim], contiguous.
struct BoundsLaunch {
  KvView kv;
  SeqBatch sq;           // table and lengths only
  const int32_t* start;  // first changed position per sequence, null: 0
  uint8_t* bounds;
};
void launch_page_bounds(const BoundsLaunch& p, int dtype, int sm_count, cudaStream_t s);

struct SelectPagesLaunch {
  SeqBatch sq;
  const uint8_t* q;
  int64_t q_row, q_head;  // bytes
  const uint8_t* bounds;  // [num_pages, heads, 2, head_dim]
  int32_t num_pages, heads, head_dim, page_size;
  int32_t k, first, last;
  int32_t chunk, sm_count;  // pages a CTA scores
  int32_t chunks, staged;   // such CTAs of an item; whether its keys fit shared memory when it selects
  uint32_t* keys;         // workspace: [N, heads, keys_row] ordered scores
  int32_t keys_row;       // table_cols, whole 16-byte vectors
  float* mags;            // workspace: [N, heads, chunks] largest sum of |q||bound| of a chunk of pages
  int32_t* out;           // [N, heads, k] contiguous
};
constexpr int kScoreChunk = 64;  // least pages a CTA scores
void launch_select_pages(const SelectPagesLaunch& p, int dtype, cudaStream_t s);

struct ScoresLaunch {
  KvView kv;
  SeqBatch sq;
  const uint8_t* q;
  int64_t q_row, q_head;   // bytes
  const float* lse;        // [N, Hq], row stride lse_row
  int64_t lse_row;
  float* scores;           // [heads, cols], row stride scores_row
  int64_t scores_row, scores_cols;
  const int64_t* col_off;  // [B]
  int32_t accumulate;
  float scale;
  // without an lse: per (row, query head, split) maximum and sum, and the joined lse
  float2* part;
  float* lse_work;
  int32_t splits;
  int32_t sm_count;
};
constexpr int kLseKeys = 256;  // keys of a split
void launch_scores(const ScoresLaunch& p, int dtype, cudaStream_t s);

// Kept tokens of up to kCompactSegs segments move to the front of their
// block tables, in up to kCompactLayers layers per launch.
constexpr int kCompactSegs = 256;
constexpr int kCompactLayers = 96;
struct CompactSeg {
  int64_t blk_off, out_off;
  int32_t cap;       // entries of the list
  int32_t dst;       // position of the first kept token
  int32_t seg;       // column of counts
};
struct CompactLayer {
  uint8_t* base;
  const uint8_t* table;  // rotary table or null
  int64_t page_stride, tok_stride, head_stride, v_off;
};
struct CompactLaunch {
  const int32_t* idx;      // [lists, idx_row]
  int64_t idx_row;
  const int32_t* count;    // [lists, num_segs]
  int64_t count_row;
  const int32_t* block_table;
  int64_t table_numel;
  int32_t* err;
  int32_t num_pages, page_size, heads, head_dim;
  FastDiv page_div;
  int32_t num_segs, num_layers, layer0;
  int32_t per_head;        // lists per layer: heads, else one (or one for all layers)
  int32_t shared;          // one list for all layers
  int32_t rotate, neox, half_rot;
  int64_t table_row, max_pos;
  // pieces of the rows (launch_compact): turning columns, then those that move
  int32_t turn_pieces, turn_heads, turn_slices, move_heads, slices;
  int32_t vecs, rot_vecs, tail0;  // 16-byte vectors of a row, turning tasks, first K vector that only moves
  CompactSeg segs[kCompactSegs];
  CompactLayer layers[kCompactLayers];
};
void launch_compact(CompactLaunch& p, int kv_dtype, int tab_dtype, int elem, int sm_count, cudaStream_t s);

}  // namespace daric
