// The paged cache in 8 bits: what its kernels share, and the C entry points (cache8.hip).
// Every call launches on `stream` and returns 0, a negative DN_ERR_* code (nothing was launched) or a positive hipError_t.
//
// Keys are e4m3 numbers [n_pages, Hkv, page_size, dh], values [n_pages, Hkv, dh, page_size]; k_scale and v_scale are 32-bit
// [n_pages, Hkv], powers of two: what a number of a page and head stands for is the number times its scale.  A power of two,
// because a scale that grows then moves a number's exponent and leaves its digits (a page may grow as often as it likes and a
// number is rounded anew only where it falls among the format's smallest), and because number times scale is then exact in
// bfloat16 (4 digits of 8, any exponent): the matrix instructions multiply exactly what the cache stands for.
#pragma once
#include "common.h"

extern "C" {

// A step's rows into the pages.  src [T, ld], dtype DN_F32 or DN_BF16; a row's keys stand at columns k_col .. k_col + Hkv dh, its values
// at v_col ..; slot_map[t] = page * page_size + place (negative, or a page outside the pools: the row's keys and values go nowhere).
// freq: 32-bit [dims / 2], or dims = 0: keys are turned by positions[t] * freq[i], pairs (2i, 2i + 1), or (i, i + dims / 2) with
// halves; cos and sin times mag.  n_heads > 0: queries at columns q_col .. q_col + n_heads dh are turned the same way to q_out [T, ldq],
// of src's dtype (which may be those columns themselves).  Rows of one page stand side by side, and no slot comes twice.
int dn_kv_append8(const void* src, int ld, int k_col, int v_col, const int32_t* slot_map, void* k_pool, void* v_pool, float* k_scale,
                  float* v_scale, int n_pages, const int32_t* positions, const float* freq, int dims, int halves, float mag, int q_col,
                  int n_heads, void* q_out, int ldq, int T, int Hkv, int dh, int page_size, int dtype, hipStream_t stream);

// Causal attention over the pages: any dtype of q and out, any head size up to 256, any page size; tiles of up to 16 rows.
int dn_attention8(const void* q, int ldq, void* out, int ldo, const void* k_pool, const void* v_pool, const float* k_scale,
                  const float* v_scale, int n_pages, const int32_t* block_tables, int max_blocks, const int32_t* tile_seq,
                  const int32_t* tile_row0, const int32_t* tile_nrows, const int32_t* tile_pos0, int n_tiles, int H, int Hkv, int dh,
                  int page_size, float scale, int window, int keep, int sink, const float* sink_at, float cap, int dtype,
                  hipStream_t stream);

// The same on the matrix cores for steps of single rows (a tile a row): head sizes that are multiples of 16, pages of a power of two
// from 16 keys on, pools 16-byte aligned.  n_splits > 1: a row's keys are shared out to so many workgroups, and part holds their results,
// n_tiles * H * n_splits * (dh + 2) floats.
int dn_attention8_single(const void* q, int ldq, void* out, int ldo, const void* k_pool, const void* v_pool, const float* k_scale,
                         const float* v_scale, int n_pages, const int32_t* block_tables, int max_blocks, const int32_t* tile_seq,
                         const int32_t* tile_row0, const int32_t* tile_pos0, int n_tiles, float* part, int n_splits, int H, int Hkv,
                         int dh, int page_size, float scale, int window, int keep, int sink, const float* sink_at, float cap,
                         int dtype, hipStream_t stream);

// The same on the matrix cores over tiles of up to 128 rows: head sizes that are multiples of 16, pages of a power of two from 16 keys on, a positive
// scale, pools and rows 16-byte aligned, ldq a multiple of 8.  A workgroup takes rows (4, or 2) times 32 rows of a tile, its keys shared out to `groups`
// groups of so many waves: (4, 1), or with heads that leave the registers for it (bfloat16 up to 128, 32-bit up to 96) (4, 2) and (2, 2).
// n_splits as above; part: H * n_splits * (dh + 2) floats for every row up to the tiles' last.
int dn_attention8_portions(const void* q, int ldq, void* out, int ldo, const void* k_pool, const void* v_pool, const float* k_scale,
                           const float* v_scale, int n_pages, const int32_t* block_tables, int max_blocks, const int32_t* tile_seq,
                           const int32_t* tile_row0, const int32_t* tile_nrows, const int32_t* tile_pos0, int n_tiles, float* part, int n_splits,
                           int rows, int groups, int H, int Hkv, int dh, int page_size, float scale, int window, int keep, int sink, const float* sink_at,
                           float cap, int dtype, hipStream_t stream);
}
