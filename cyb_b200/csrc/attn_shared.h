// What the kernels of the attention over shared pages (attn_shared.cu) agree on.
#pragma once
#include <cuda.h>

#include "attn_prefill.h"

constexpr int kSharedGroups = 1024;  // groups of rows in a call
constexpr int kOwnWarps = 4;         // of a CTA that reads rows' own pages, and pages of a unit of its work

struct qeng_shared_attn {
  const __half* q;         // [T] rows of [Hq][128], ldq values apart
  const int32_t* table;    // [table_rows][max_pages]
  const int32_t* rows;     // [T] table row (negative: not there), or null: t
  const int32_t* lens;     // [T] keys
  const int32_t *first, *pages;  // [G + 1] rows of the groups, [G] pages that the rows of a group share
  void* out;
  int32_t* status;
  long long ldq, ldo, max_pages, table_rows;
  int out_dtype, T, Hq, Hkv, grp, G, pool_pages, window, own_ctas;
  float scale, softcap;
  // Working memory.  Units of a row: its own pages by fours, for every kv head; the CTAs of attn_own_kernel divide all units evenly
  // (CTA c: [c W / n, (c + 1) W / n)), so that a CTA has whole (row, kv head) pairs but for its first and last.
  long long* unit_first;   // [T + 1] units (of one kv head) before a row
  float *own_o, *own_ml;   // pairs with shared pages, too: [T][Hq][128] sums of weighted values, [T][Hq][2] (log2 of the largest weight, sum)
  float *cut_o, *cut_ml;   // pairs cut between CTAs: [2 own_ctas][8][128], [..][2]: of the pair a CTA begins with, of the one it ends with
};
