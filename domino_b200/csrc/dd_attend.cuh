// dd_attend.cuh -- attention of a chunk of new tokens over the paged cache.
//
//   out_p = sum_j softmax_j(scale q_p . K_j) V_j   over the keys j that p sees
//
// in one pass over the keys with a running maximum m and sum l:
//   m' = max(m, s_j);  l' = l e^(m - m') + e^(s_j - m');  o' = o e^(m - m') + e^(s_j - m') V_j
#pragma once

#include "../../include/domino_draft.h"
#include "dd_cache_write.cuh"
#include "dd_ptx.cuh"

namespace dd {

struct AttendParams {
  const void* q;
  long long q_stride[3];     // batch, token, head
  void* out;                 // [batch, tokens, heads, dim]
  const void* pool[2];       // this layer's keys, values [pages, kv_heads, page_size, dim]
  const int* table;
  const long long* start;
  const long long* lens;     // null: all tokens
  unsigned* status;
  float scale;
  int batch, tokens, heads, kv_heads, dim, pages, page_size, page_shift, row_pages;  // page_size = 1 << page_shift
  int group;                 // query heads per key head
  int copies;                // copies of the rows in a query tile of the tensor-core kernel: 1, 2 or 4
  int tile_rows, item_rows;  // rows of a query tile (whole tokens, at most 128) and of the tiles of one item
  int q_tma;                 // the queries' layout allows TMA
  int min_tiles;             // key tiles that a CTA of that kernel takes at least
  int causal, window, sinks;
};

}  // namespace dd
