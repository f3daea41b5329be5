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

// The keys that a query at position p of a row with `total` keys sees:
// [0, sinks) and [lo, hi).
struct Visible {
  long long lo, hi;
};
__device__ __forceinline__ Visible visible(const AttendParams& a, long long p, long long total) {
  Visible v;
  v.hi = a.causal ? min(total, p + 1) : total;
  v.lo = a.window > 0 ? max(p - a.window + 1, 0ll) : 0;
  return v;
}
// Keys of row b: positions below start + lens that its table can hold.
__device__ __forceinline__ long long row_keys(const AttendParams& a, int b) {
  const long long n = a.lens ? min(max(a.lens[b], 0ll), (long long)a.tokens) : a.tokens;
  return min(max(a.start[b] + n, 0ll), (long long)a.row_pages * a.page_size);
}

// One warp per (query, head): lane j of a step scores key j of a block of 32,
// then the lanes spread over the head dimension for the weighted values.
// Right for every type and shape; every query head reads its keys again.
constexpr int kSimpleWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kSimpleWarps) attend_simple_kernel(AttendParams a) {
  __shared__ float qs[kSimpleWarps][kMaxHeadDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long u = (long long)blockIdx.x * kSimpleWarps + warp;
  pdl_wait_primary();
  if (u >= (long long)a.batch * a.tokens * a.heads) return;
  const int h = (int)(u % a.heads), t = (int)(u / a.heads % a.tokens), b = (int)(u / a.heads / a.tokens);
  const long long n = a.lens ? a.lens[b] : a.tokens;
  T* out = static_cast<T*>(a.out) + u * a.dim;
  float o[kMaxHeadDim / 32] = {};
  float m = -INFINITY, l = 0.0f;
  if (t < n) {
    const long long p = a.start[b] + t, total = row_keys(a, b);
    const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + h * a.q_stride[2];
    for (int d = lane; d < a.dim; d += 32) qs[warp][d] = io<T>::to_f(q[d]);
    __syncwarp();
    const Visible v = visible(a, p, total);
    const int kvh = h / (a.heads / a.kv_heads);
    const long long head_words = (long long)a.page_size * a.dim;
    const long long sinks = min((long long)a.sinks, v.lo);
    for (long long j0 = 0; j0 < v.hi; j0 += 32) {
      if (j0 >= sinks && j0 + 32 <= v.lo) continue;
      const long long j = j0 + lane;
      float s = -INFINITY;
      int page = -1;
      const bool see = j < v.hi && (j >= v.lo || j < sinks);
      if (see) {
        page = a.table[(long long)b * a.row_pages + j / a.page_size];
        if (page >= a.pages) page = -1;
      }
      const long long at = page < 0 ? -1 : ((long long)page * a.kv_heads + kvh) * head_words + j % a.page_size * a.dim;
      if (at >= 0) {
        const T* k = static_cast<const T*>(a.pool[0]) + at;
        s = 0.0f;
        for (int d = 0; d < a.dim; ++d) s += qs[warp][d] * io<T>::to_f(k[d]);
        s *= a.scale;
      }
      float top = s;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float m1 = fmaxf(m, top);
      const float base = m1 == -INFINITY ? 0.0f : m1;  // nothing seen so far: weights of zero, not NaN
      const float keep = expf(m - base);
      const float w = at >= 0 ? expf(s - base) : 0.0f;
      float sum = w;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      l = l * keep + sum;
      m = m1;
#pragma unroll
      for (int i = 0; i < kMaxHeadDim / 32; ++i) o[i] *= keep;
      for (int k = 0; k < 32; ++k) {
        const long long atk = __shfl_sync(0xffffffffu, at, k);
        const float wk = __shfl_sync(0xffffffffu, w, k);
        if (atk < 0) continue;  // a key that is not seen has no part, whatever it holds
        const T* vv = static_cast<const T*>(a.pool[1]) + atk;
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 32; ++i)
          if (lane + 32 * i < a.dim) o[i] += wk * io<T>::to_f(vv[lane + 32 * i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMaxHeadDim / 32; ++i)
    if (lane + 32 * i < a.dim) out[lane + 32 * i] = io<T>::from_f(l == 0.0f ? 0.0f : o[i] / l);
}

}  // namespace dd
