// What the kernels of the attention over shared pages (attn_shared.cu) agree on.
#pragma once
#include <cuda.h>

#include "attn_prefill.h"

constexpr int kSharedGroups = 1024;  // groups of rows in a call
constexpr int kSharedTiles = 4096;   // and double tiles of them
constexpr int kOwnWarps = 4;         // of a CTA that reads rows' own pages

// What CTAs (or warps) leave for attn_join_kernel to add up: `last` is the last one that has a piece.
struct qeng_tile_job {
  int t0, tokens, h, last;  // tokens of the double tile; none: no job
};
struct qeng_own_job {
  int t, h, last, shared;  // t < 0: no job; shared: the row's shared part is in row_o
};

struct qeng_shared_attn {
  const __half* q;         // [T] rows of [Hq][128], ldq values apart
  const int32_t* table;    // [table_rows][max_pages]
  const int32_t* rows;     // [T] table row (negative: not there), or null: t
  const int32_t* lens;     // [T] keys
  const int32_t *first, *pages;  // [G + 1] rows of the groups, [G] pages that the rows of a group share
  __half* pool;
  void* out;
  int32_t* status;
  long long ldq, ldo, max_pages, table_rows;
  int out_dtype, T, Hq, Hkv, grp, tokens, G, pool_pages, window, own_warps, tile_ctas;  // tokens: of a tile, 128 / grp
  float scale, softcap;
  // Working memory: sums that are not a row's whole result, each with (m, l): the sum is of 2^(x - m) v, l of 2^(x - m).
  //
  // The shared pages of a group are worked on by double tiles: 2 * tokens rows, one kv head, all keys that any of them attends, by blocks
  // of 128.  The CTAs of attn_tile_kernel divide all blocks evenly (in the order of double tiles, kv heads,
  // keys), so that a CTA has whole ones but for the first and the last.  The pages that a row has to itself are divided the same way
  // among the warps of attn_own_kernel.
  int* tile_first;             // [double tiles + 1] blocks (of one kv head) before a double tile
  float *tile_o, *tile_ml;     // cut between CTAs: [2 tile_ctas][32 x 4 dims][256], [..][256][2]: of what a CTA begins with, of what it ends with
  float *row_o, *row_ml;       // [T][Hq][128], [..][2]: the shared part of a row that has pages to itself, whole; or, where that is cut, the row's own, whole
  long long* unit_first;       // [T + 1] units (of one kv head) of the rows before a row: own pages, and what a start costs
  qeng_tile_job* tile_jobs;    // [tile_ctas]
  qeng_own_job* own_jobs;      // [own_warps]
  float* kept_o;               // f32 results: [tile_ctas][32 x 4 dims][256], what a CTA has added up of its double tile
  int* tile_list;              // how many tile jobs there are, and whose
  float *cut_o, *cut_ml;       // cut between warps: [2 own_warps][8][128], [..][2]
};
