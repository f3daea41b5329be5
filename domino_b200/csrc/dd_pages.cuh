// dd_pages.cuh -- page bookkeeping of the paged key / value cache: reserve,
// crop, fork, compact, and the copy of whole pages.
//
// State is three arrays: table [batch, row_pages], length [batch] and refs
// [pages].  A page is free when its count is 0 and the free pages are taken
// lowest number first, so the result of a call depends on the arrays alone:
// counts change by integer atomics, whose order cannot show, and every place
// in a list comes from a prefix sum.  There is no free list to keep in order.
//
// Planning is latency (one CTA walks refs, 4 bytes a page, and the rows it is
// asked for); the bytes are in the copies.
#pragma once

#include "../../include/domino_draft.h"
#include "dd_ptx.cuh"

namespace dd {

constexpr int kPlanThreads = 1024;
constexpr int kMaxCacheBatch = 1024;  // one thread of the planning CTA per row

// Scratch, in 32-bit words: a header, the free pages found, and the moves.
struct PageScratch {
  int* n_moves;      // [0] of the header; [1] is the first page past the used ones (compact)
  int* list;         // [pages] free pages / where a page goes (compact)
  int* src;          // [pages]
  int* dst;          // [pages]
  int* old_table;    // [batch * row_pages]
  long long* old_length;  // [batch]
};

__host__ __device__ inline size_t page_scratch_bytes(int pages, int batch, int row_pages) {
  return 64 + 8 * (size_t)batch + 4 * (3 * (size_t)pages + (size_t)batch * row_pages);
}
__host__ __device__ inline PageScratch page_scratch(void* p, int pages, int batch) {
  PageScratch s;
  s.n_moves = static_cast<int*>(p);
  s.old_length = reinterpret_cast<long long*>(static_cast<char*>(p) + 64);
  s.list = reinterpret_cast<int*>(s.old_length + batch);
  s.src = s.list + pages;
  s.dst = s.src + pages;
  s.old_table = s.dst + pages;
  return s;
}

// Exclusive prefix sum of one int per thread over the planning CTA; *total
// gets the sum.  Every thread calls it.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int warp_sum[33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int s = warp_sum[lane];
    int t = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, t, d);
      if (lane >= d) t += o;
    }
    warp_sum[lane] = t - s;
    if (lane == 31) warp_sum[32] = t;
  }
  __syncthreads();
  const int r = warp_sum[warp] + inc - v;
  *total = warp_sum[32];
  __syncthreads();
  return r;
}

// For reserve, where pages behind a row's first slot are shared: which of the
// slots [first, last) of every row need a copy (old_table: 1 or 0), and their
// number per row on top of `need`.  Of the rows that reach a page the lowest
// keeps it when nobody else holds it.  Counts and lowest rows stand in src and
// dst, which the moves have not used yet.
__device__ __forceinline__ void plan_deep_copies(const int* table, const int* refs, const PageScratch& s, const int* first,
                                                 const int* last, int* need, int batch, int pages, int row_pages) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int round = 0; round < 3; ++round) {
    for (int b = warp; b < batch; b += kPlanThreads / 32) {
      int copies = 0;
      for (int i = first[b] + lane; i < last[b]; i += 32) {
        const int p = table[(size_t)b * row_pages + i];
        const bool shared = p >= 0 && p < pages && refs[p] > 1;
        if (round == 0 && shared) {
          s.src[p] = 0;
          s.dst[p] = batch;
        }
        if (round == 1 && shared) {
          atomicAdd(&s.src[p], 1);
          atomicMin(&s.dst[p], b);
        }
        if (round == 2) {
          const bool copy = shared && (refs[p] > s.src[p] || s.dst[p] < b);
          s.old_table[(size_t)b * row_pages + i] = copy;
          copies += copy;
        }
      }
      copies = __reduce_add_sync(0xffffffffu, copies);
      if (round == 2 && lane == 0) need[b] += copies;
    }
    __syncthreads();
  }
}

// reserve: slots ceil'd over [length, upto) of every row, in row order and
// within a row in position order; request i gets the i-th free page.  A request
// is a slot without a page or one whose page other rows hold too.  The latter is
// as a rule a row's first slot (the page that `length` ends in); slots behind it
// hold shared pages only where a caller has set a length back by itself, and
// then plan_deep_copies decides for all slots.
__global__ void __launch_bounds__(kPlanThreads) pages_reserve_kernel(int* table, const long long* length, int* refs,
                                                                     PageScratch s, unsigned* status,
                                                                     const long long* upto, int batch, int pages,
                                                                     int page_size, int row_pages) {
  __shared__ int first[kMaxCacheBatch], last[kMaxCacheBatch], held[kMaxCacheBatch], need[kMaxCacheBatch];
  __shared__ int n_moves, deep;  // deep: shared pages behind a row's first slot
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait_primary();
  if (tid == 0) n_moves = deep = 0;
  // what each row misses
  if (tid < batch) {
    const long long len = max(length[tid], 0ll), cap = (long long)row_pages * page_size;
    long long up = upto[tid];
    if (up > cap) {
      up = cap;
      atomicOr(status, DD_STATUS_NO_PAGE);
    }
    const bool grows = up > len;
    first[tid] = grows ? (int)(len / page_size) : 0;
    last[tid] = grows ? (int)((up + page_size - 1) / page_size) : 0;
    int p = grows ? table[(size_t)tid * row_pages + first[tid]] : -1;
    held[tid] = p >= 0 && p < pages ? p : -1;
  }
  __syncthreads();
  for (int b = warp; b < batch; b += kPlanThreads / 32) {
    int miss = 0;
    for (int i = first[b] + lane; i < last[b]; i += 32) {
      const int p = table[(size_t)b * row_pages + i];
      miss += p < 0 || p >= pages;
      if (i > first[b] && p >= 0 && p < pages && refs[p] > 1) deep = 1;
    }
    miss = __reduce_add_sync(0xffffffffu, miss);
    if (lane == 0) need[b] = miss;
  }
  __syncthreads();
  if (deep) {
    plan_deep_copies(table, refs, s, first, last, need, batch, pages, row_pages);
    if (tid < batch) held[tid] = -1;  // (its copies are among them)
  }
  __syncthreads();
  // a held page that others hold too is copied, except by the first row of
  // this call when only rows of this call hold it
  bool copies = false;
  if (tid < batch && held[tid] >= 0 && refs[held[tid]] > 1) {
    int rank = 0, same = 0;
    for (int b = 0; b < batch; ++b) {
      const bool eq = held[b] == held[tid];
      same += eq;
      rank += eq && b < tid;
    }
    copies = rank > 0 || refs[held[tid]] > same;
  }
  int total;
  const int off = block_scan(tid < batch ? need[tid] + copies : 0, &total);
  // the lowest `total` free pages
  int found = 0;
  for (int base = 0; base < pages && found < total; base += 4 * kPlanThreads) {
    int n = 0, mine[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int p = base + 4 * tid + k;
      if (p < pages && refs[p] == 0) mine[n++] = p;
    }
    int chunk;
    int r = found + block_scan(n, &chunk);
    for (int k = 0; k < n; ++k, ++r)
      if (r < total) s.list[r] = mine[k];
    found += chunk;
  }
  found = min(found, total);
  __syncthreads();
  if (total > found && tid == 0) atomicOr(status, DD_STATUS_NO_PAGE);
  if (tid < batch) {
    int at = off;
    if (copies) {
      if (at < found) {
        const int p = s.list[at], m = atomicAdd(&n_moves, 1);
        s.src[m] = held[tid];
        s.dst[m] = p;
        table[(size_t)tid * row_pages + first[tid]] = p;
        refs[p] = 1;
        atomicSub(&refs[held[tid]], 1);
      }
      ++at;
    }
    need[tid] = at;  // from here on: where the row's missing pages start in the list
  }
  __syncthreads();
  for (int b = warp; b < batch; b += kPlanThreads / 32) {
    int at = need[b];
    for (int i0 = first[b]; i0 < last[b]; i0 += 32) {
      const int i = i0 + lane;
      int* e = &table[(size_t)b * row_pages + i];
      const bool copy = deep && i < last[b] && s.old_table[(size_t)b * row_pages + i];
      const bool miss = i < last[b] && (*e < 0 || *e >= pages || copy);
      const unsigned m = __ballot_sync(0xffffffffu, miss);
      const int r = at + __popc(m & ((1u << lane) - 1));
      if (miss && r < found) {
        const int p = s.list[r];
        if (copy) {
          const int move = atomicAdd(&n_moves, 1);
          s.src[move] = *e;
          s.dst[move] = p;
          atomicSub(&refs[*e], 1);
        }
        *e = p;
        refs[p] = 1;
      }
      at += __popc(m);
    }
  }
  __syncthreads();
  if (tid == 0) *s.n_moves = n_moves;
}

// crop: one CTA per row; nothing reads what another row changes but refs.
__global__ void pages_crop_kernel(int* table, long long* length, int* refs, const long long* to, int pages,
                                  int page_size, int row_pages) {
  const int b = blockIdx.x;
  pdl_wait_primary();
  const long long now = max(length[b], 0ll), len = min(max(to[b], 0ll), now);
  __syncthreads();
  if (threadIdx.x == 0) length[b] = len;
  for (long long i = (len + page_size - 1) / page_size + threadIdx.x; i < row_pages; i += blockDim.x) {
    int* e = &table[(size_t)b * row_pages + i];
    const int p = *e;
    if (p >= 0 && p < pages) atomicSub(&refs[p], 1);
    *e = -1;
  }
}

// fork, first half: the tables and lengths as they are before the call.
__global__ void pages_snapshot_kernel(const int* table, const long long* length, PageScratch s, int batch,
                                      int row_pages) {
  pdl_wait_primary();
  const size_t n = (size_t)batch * row_pages;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
    s.old_table[i] = table[i];
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < batch; b += blockDim.x) s.old_length[b] = length[b];
}

__global__ void pages_fork_kernel(int* table, long long* length, int* refs, PageScratch s, unsigned* status,
                                  const long long* src, int batch, int pages, int page_size, int row_pages) {
  const int b = blockIdx.x;
  pdl_wait_primary();
  const long long from = src[b];
  if (from == b) return;
  if (from < -1 || from >= batch) {
    if (threadIdx.x == 0) atomicOr(status, DD_STATUS_BAD_ROW);
    return;
  }
  const long long len = from < 0 ? 0 : max(s.old_length[from], 0ll);
  for (int i = threadIdx.x; i < row_pages; i += blockDim.x) {
    int p = (long long)i * page_size < len ? s.old_table[(size_t)from * row_pages + i] : -1;
    if (p < 0 || p >= pages) p = -1;
    const int old = s.old_table[(size_t)b * row_pages + i];
    if (p >= 0) atomicAdd(&refs[p], 1);
    if (old >= 0 && old < pages) atomicSub(&refs[old], 1);
    table[(size_t)b * row_pages + i] = p;
  }
  if (threadIdx.x == 0) length[b] = len;
}

// compact: with U pages in use, the k-th used page at or above U moves to the
// k-th free page below U (there are equally many of both), so sources and
// targets never meet and the copies need no order.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_kernel(int* refs, PageScratch s, int pages) {
  const int tid = threadIdx.x;
  pdl_wait_primary();
  int n = 0, used;
  for (int p = tid; p < pages; p += kPlanThreads) n += refs[p] > 0;
  block_scan(n, &used);
  int holes = 0, movers = 0;
  for (int base = 0; base < pages; base += 4 * kPlanThreads) {
    int nh = 0, nm = 0, h[4], m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int p = base + 4 * tid + k;
      if (p >= pages) break;
      const bool busy = refs[p] > 0;
      if (p < used && !busy) h[nh++] = p;
      if (p >= used && busy) m[nm++] = p;
      if (p >= used && !busy) s.list[p] = p;
    }
    int th, tm;
    int r = holes + block_scan(nh, &th);
    for (int k = 0; k < nh; ++k) s.dst[r + k] = h[k];
    r = movers + block_scan(nm, &tm);
    for (int k = 0; k < nm; ++k) s.src[r + k] = m[k];
    holes += th;
    movers += tm;
  }
  __syncthreads();
  for (int k = tid; k < movers; k += kPlanThreads) {
    const int a = s.src[k], d = s.dst[k];
    s.list[a] = d;
    refs[d] = refs[a];
    refs[a] = 0;
  }
  if (tid == 0) {
    s.n_moves[0] = movers;
    s.n_moves[1] = used;
  }
}

// The moves' pages in every plane (layer x keys / values), 16 KB a CTA step
// with four 16-byte loads in flight per thread; for compact also the table
// entries of the moved pages.  Bound by HBM (each byte read and written once).
constexpr int kCopyThreads = 256;
constexpr int kCopyStep = kCopyThreads * 4;  // 16-byte words
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(uint4* data, PageScratch s, int planes, int pages,
                                                                  long long page_words, int* table, int entries) {
  pdl_wait_primary();
  const int moves = *s.n_moves;
  if (table) {
    const int used = s.n_moves[1];
    // (64 bits: `entries` may be as near to 2^31 as one step)
    for (long long i = blockIdx.x * kCopyThreads + threadIdx.x; i < entries; i += (long long)gridDim.x * kCopyThreads) {
      const int p = table[i];
      if (p >= used && p < pages) table[i] = s.list[p];
    }
  }
  const long long steps = (page_words + kCopyStep - 1) / kCopyStep;
  const long long total = steps * planes * moves;
  for (long long u = blockIdx.x; u < total; u += gridDim.x) {
    const long long step = u % steps, rest = u / steps;
    const int plane = (int)(rest % planes), m = (int)(rest / planes);
    const uint4* from = data + ((long long)plane * pages + s.src[m]) * page_words;
    uint4* to = data + ((long long)plane * pages + s.dst[m]) * page_words;
    const long long w = step * kCopyStep + threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w + k * kCopyThreads < page_words) v[k] = __ldcs(from + w + k * kCopyThreads);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w + k * kCopyThreads < page_words) __stcs(to + w + k * kCopyThreads, v[k]);
  }
}

}  // namespace dd
