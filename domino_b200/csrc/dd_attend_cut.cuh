// dd_attend_cut.cuh -- how paged attention's work is cut over the SMs, and how
// the pieces of an item are put together again.
//
// An item is one query tile of one row of the batch and one key head; its work
// is the tiles of 128 keys that any of its queries sees.  The cut is by key
// tiles, so long and short rows balance and one row's long cache spreads over
// all SMs.  Lengths are read on the device: no host synchronisation.
//
// A piece that is not all of its item leaves unnormalised sums, maximum and
// weight sum (O, m, l) in the workspace; the CTA that finishes last, found by a
// counter that wraps back to zero, adds them up in the order of the CTAs, so
// the result is the same every time.
#pragma once

#include <type_traits>

#include "dd_attend.cuh"

namespace dd {

constexpr int kKeyTile = 128;

struct AttendWork {
  unsigned* count;  // [kMaxAttendCtas], zero between calls: finished pieces of the item that starts in a CTA and leaves it
  float* o;         // [grid][2][rows][dim_pad]: a piece from the CTA before, and one that goes on in the next
  float2* ml;       // [grid][2][rows]
};
constexpr int kMaxAttendCtas = 320;
__host__ __device__ constexpr size_t attend_work_bytes(int ctas, int rows, int dim_pad) {
  return (size_t)ctas * 2 * rows * (sizeof(float) * dim_pad + sizeof(float2));
}

// Key tiles of one (row of the batch, query tile): n_sink from 0, then from
// `first` on.  Positions are 32-bit here: a row holds at most 2^30 tokens.
struct TileSpan {
  int n_sink, first, n;
  int rows;           // query rows of the batch row (tokens x group)
  int start, lo, hi;  // position of token 0; keys that any row of the tile sees: [lo, hi) and, below hi, the sinks
  __device__ __forceinline__ int tile(int i) const { return i < n_sink ? i : first + i - n_sink; }
};
__device__ __forceinline__ TileSpan tile_span(const AttendParams& a, int b, int qt, int tile_rows) {
  TileSpan s;
  const int n_new = a.lens ? (int)min(max(a.lens[b], 0ll), (long long)a.tokens) : a.tokens;
  s.start = (int)min(max(a.start[b], -(1ll << 30)), 1ll << 30);
  s.rows = n_new * a.group;
  s.n_sink = s.first = s.n = 0;
  s.lo = s.hi = 0;
  const int r0 = qt * tile_rows;
  if (r0 >= s.rows) return s;
  const int p0 = s.start + r0 / a.group, p1 = s.start + (min(s.rows, r0 + tile_rows) - 1) / a.group;
  const int total = min(max(s.start + n_new, 0), a.row_pages << a.page_shift);
  s.hi = max(a.causal ? min(total, p1 + 1) : total, 0);
  if (s.hi == 0) return s;
  s.lo = a.window > 0 ? max(p0 - a.window + 1, 0) : 0;
  const int t_lo = s.lo / kKeyTile, t_hi = (s.hi + kKeyTile - 1) / kKeyTile;
  const int sinks = min(min(a.sinks, s.lo), s.hi);
  s.n_sink = min((sinks + kKeyTile - 1) / kKeyTile, t_lo);
  s.first = t_lo;
  s.n = s.n_sink + max(t_hi - t_lo, 0);
  return s;
}

// A CTA's share of the work, item by item.  Many items: the CTAs take equal runs
// of units, where an item counts its tiles and, before them, kItemUnits for the
// start and the end of an item.  Few items (at most a quarter of the CTAs): each
// gets CTAs of its own in proportion to its tiles, so that nobody has two.
struct Piece {
  int e, b, qt, h, i0, i1;  // entry (b, qt), key head, tiles [i0, i1) of it
  int pos, left;            // unit of the item where the run enters it; units of the run from there on
  TileSpan span;
};
// (Start and end cost about as much as seven tiles: with 3 / 5 / 7 / 10 the calls
// of 64 rows x 1 token took 210 / 198 / 198 / 199 us, of 32 rows x 16 tokens 265
// / 262 / 254 / 253 us; with none, short rows' CTAs ran twice as long as others.)
// (Own CTAs up to a quarter of the CTAs: with a half, 5 x 16 tokens over 2560 keys,
// 40 items, took 26.2 us against 23.8, 8 x 1 token over 8000, 64 items, 67.7 against
// 52.2; with an eighth, 4 x 16 over 2560, 32 items, 23.6 against 22.7.)
constexpr int kItemUnits = 7;
__device__ __forceinline__ void piece_enter(const AttendParams& a, Piece& p, int q_tiles, int tile_rows) {
  p.b = p.e / q_tiles;
  p.qt = p.e - p.b * q_tiles;
  p.span = tile_span(a, p.b, p.qt, tile_rows);
}
__device__ __forceinline__ bool piece_next(const AttendParams& a, Piece& p, int q_tiles, int tile_rows) {
  p.left -= p.span.n + kItemUnits - p.pos;
  if (p.left <= kItemUnits) return false;  // the next item's first tile is another CTA's
  if (++p.h == a.kv_heads) {
    p.h = 0;
    do {
      ++p.e;
      piece_enter(a, p, q_tiles, tile_rows);
    } while (p.span.n == 0);
  }
  p.pos = p.i0 = 0;
  p.i1 = min(p.span.n, p.left - kItemUnits);
  return true;
}
// CTAs for an item of n tiles when there are few items.
__device__ __forceinline__ int item_ctas(const AttendParams& a, int n, long long tiles, int spare) {
  if (n == 0) return 0;
  return max(min((int)((long long)n * spare / tiles), n / a.min_tiles), 1);
}

// Where CTA c's run starts: c / grid of all tiles.
__device__ __forceinline__ long long run_start(long long total, unsigned c, unsigned grid) {
  if (total < 1 << 23 && grid < 256) return (unsigned)total * c / grid;  // 32-bit division
  return total * c / grid;
}

// The CTA that holds tile g.
__device__ __forceinline__ int run_of(long long total, long long g, unsigned grid) {
  return (int)(((g + 1) * grid - 1) / total);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void store2(T* p, float x, float y) {
  *reinterpret_cast<uint32_t*>(p) = pack2<T>(x, y);
}
template <>
__device__ __forceinline__ void store2<float>(float* p, float x, float y) {
  *reinterpret_cast<float2*>(p) = make_float2(x, y);
}

// A CTA's cut, in shared memory.
struct CutShared {
  Piece first;           // where the run starts; left = 0: the CTA has none
  long long total, unit0;
  int few;
  int c0, c1, join;      // CTAs that hold the split item; whether this CTA's piece finished last
};
struct CutScan {
  long long sum[32], x[32];
  int y[32];
};

// Over the block: `before` becomes the sum over the threads before this one and
// `total` the sum over all; x and y become their sums over all.
template <int kThreads>
__device__ __forceinline__ void block_scan2(CutScan& sh, long long& before, long long& total, long long& x,
                                            int& y, int warp, int lane) {
  long long inc = before;
  const long long own = before;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, d);
    y += __shfl_xor_sync(0xffffffffu, y, d);
  }
  __syncthreads();
  if (lane == 31) {
    sh.sum[warp] = inc;
    sh.x[warp] = x;
    sh.y[warp] = y;
  }
  __syncthreads();
  before = inc - own;
  total = x = y = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sh.sum[w];
    total += sh.sum[w];
    x += sh.x[w];
    y += sh.y[w];
  }
}

// The CTA's run.  All threads call it; they synchronise before they read sh.
template <int kThreads>
__device__ __forceinline__ void cut_work(const AttendParams& a, CutShared& sh, CutScan& scan, int q_tiles, int tid) {
  const int warp = tid >> 5, lane = tid & 31;
  const int entries = a.batch * q_tiles, per = (entries + kThreads - 1) / kThreads, grid = gridDim.x;
  Piece mine;
  if (entries <= 32) {
    // One warp, a lane per entry (the general way below costs a small call 3000
    // cycles, this one 1500, most of it the lengths' way from memory).
    if (warp > 0) return;
    mine.e = lane;
    int n = 0;
    if (lane < entries) {
      piece_enter(a, mine, q_tiles, a.item_rows);
      n = mine.span.n;
    }
    const int items = __popc(__ballot_sync(0xffffffffu, n > 0));
    const int tiles = __reduce_add_sync(0xffffffffu, n);
    const bool few = (long long)items * a.kv_heads * 4 <= grid;
    // units, or CTAs, for one key head of the entry
    const int own = few ? item_ctas(a, n, (long long)tiles * a.kv_heads, grid - items * a.kv_heads) : n ? n + kItemUnits : 0;
    int inc = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    const long long before = (long long)(inc - own) * a.kv_heads;
    const long long total = (long long)__shfl_sync(0xffffffffu, inc, 31) * a.kv_heads;
    const long long u0 = few ? blockIdx.x : run_start(total, blockIdx.x, grid);
    const long long u1 = few ? u0 + 1 : run_start(total, blockIdx.x + 1, grid);
    const bool found = u0 < u1 && u0 >= before && u0 < before + (long long)own * a.kv_heads;
    if (lane == 0) {
      sh.few = few;
      sh.total = total;
      sh.unit0 = u0;
      sh.first.left = 0;
    }
    __syncwarp();
    if (found) {
      const int rem = (int)(u0 - before);
      mine.h = rem / own;
      const int part = rem - mine.h * own;
      if (few) {
        mine.i0 = (int)((long long)n * part / own);
        mine.i1 = (int)((long long)n * (part + 1) / own);
        mine.pos = 0;
        mine.left = 1;  // one piece only
        sh.c0 = blockIdx.x - part;
        sh.c1 = sh.c0 + own - 1;
      } else {
        mine.pos = part;
        mine.left = (int)(u1 - u0);
        mine.i0 = max(mine.pos - kItemUnits, 0);
        mine.i1 = min(n, mine.pos + mine.left - kItemUnits);
        if (mine.i1 <= mine.i0) mine.left = 0;
      }
      sh.first = mine;
    }
    return;
  }
  const int e0 = tid * per, e1 = min(entries, e0 + per);
  // sums over the block: tiles and items of one key head
  long long tiles = 0;
  int items = 0;
  for (mine.e = e0; mine.e < e1; ++mine.e) {
    piece_enter(a, mine, q_tiles, a.item_rows);
    tiles += mine.span.n;
    items += mine.span.n > 0;
  }
  long long before = tiles + (long long)items * kItemUnits, total;  // units before this thread's entries, of all
  const long long own = before;
  block_scan2<kThreads>(scan, before, total, tiles, items, warp, lane);
  before *= a.kv_heads;
  total *= a.kv_heads;
  const bool few = (long long)items * a.kv_heads * 4 <= grid;  // (with many entries behind the end of their chunks)
  int c0 = 0, c1 = 0;
  bool found = false;
  if (!few) {
    const long long u0 = run_start(total, blockIdx.x, grid), u1 = run_start(total, blockIdx.x + 1, grid);
    if (u0 < u1 && u0 >= before && u0 < before + own * a.kv_heads) {
      // the run starts in this thread's entries (one entry as a rule: its span is still here)
      long long rem = u0 - before;
      int len = 0;
      for (mine.e = e0; mine.e < e1; ++mine.e) {
        if (per > 1) piece_enter(a, mine, q_tiles, a.item_rows);
        len = mine.span.n ? mine.span.n + kItemUnits : 0;
        if (rem < (long long)len * a.kv_heads) break;
        rem -= (long long)len * a.kv_heads;
      }
      mine.h = (int)rem / len;  // rem < tiles x heads of one entry
      mine.pos = (int)rem - mine.h * len;
      mine.left = (int)(u1 - u0);
      mine.i0 = max(mine.pos - kItemUnits, 0);
      mine.i1 = min(mine.span.n, mine.pos + mine.left - kItemUnits);
      if (mine.i1 <= mine.i0) mine.left = 0;
      found = true;
    }
    if (tid == 0) {
      sh.total = total;
      sh.unit0 = u0;
    }
  } else {
    const int spare = grid - items * a.kv_heads;
    tiles *= a.kv_heads;
    long long ctas = 0, all, unused0 = 0;
    int unused1 = 0;
    for (int e = e0; e < e1; ++e) {
      if (per > 1) {
        mine.e = e;
        piece_enter(a, mine, q_tiles, a.item_rows);
      }
      ctas += item_ctas(a, mine.span.n, tiles, spare);
    }
    const long long mine_ctas = ctas;
    block_scan2<kThreads>(scan, ctas, all, unused0, unused1, warp, lane);
    if ((int)blockIdx.x >= ctas * a.kv_heads && (int)blockIdx.x < (ctas + mine_ctas) * a.kv_heads) {
      int rem = blockIdx.x - (int)ctas * a.kv_heads, k = 1;
      for (mine.e = e0; mine.e < e1; ++mine.e) {
        if (per > 1) piece_enter(a, mine, q_tiles, a.item_rows);
        k = item_ctas(a, mine.span.n, tiles, spare);
        if (rem < k * a.kv_heads) break;
        rem -= k * a.kv_heads;
      }
      mine.h = rem / k;
      const int part = rem - mine.h * k;
      mine.i0 = (int)((long long)mine.span.n * part / k);
      mine.i1 = (int)((long long)mine.span.n * (part + 1) / k);
      mine.pos = 0;
      mine.left = 1;  // one piece only
      c0 = blockIdx.x - part;
      c1 = c0 + k - 1;
      found = true;
    }
  }
  if (tid == 0) sh.first.left = 0;
  __syncthreads();
  if (found) {
    sh.first = mine;
    sh.few = few;
    sh.c0 = c0;
    sh.c1 = c1;
  }
}

// A piece is in the workspace (one thread of the CTA, after all have written
// and fenced): sh.join tells whether it was the item's last.
__device__ __forceinline__ void finish_piece(const AttendWork& work, CutShared& sh, const Piece& p) {
  if (!sh.few) {
    const long long g0 = sh.unit0 + (sh.first.left - p.left) - p.pos + kItemUnits;
    sh.c0 = run_of(sh.total, g0, gridDim.x);
    sh.c1 = run_of(sh.total, g0 + p.span.n - 1, gridDim.x);
  }
  const unsigned others = sh.c1 - sh.c0;
  const unsigned done = atomicInc(&work.count[sh.c0], others);
  __threadfence();
  sh.join = done == others;
}

// A split item whose last piece this CTA brought.
struct JoinItem {
  int b, qt, h, rows;  // rows: of the batch row (tokens x group)
  int c0, c1;
};

// Its pieces, in slot 1 of CTA c0 and slot 0 of those behind it, by kWarps warps.
// A warp takes kBatch rows at a time: the lanes read the pieces' (m, l) side by
// side, then the rows are added up, kUnroll pieces at once.  All that counts here
// is how many loads are in flight: each comes from L2 and takes about 1000 cycles,
// and one SM does them all (with 8 loads a thread, 64 rows of 7 pieces took
// 17 000 cycles of a 45 000-cycle call).
template <typename T, int kDim, int kRows, int kWarps, int kBatch, int kUnroll>
__device__ __forceinline__ void join_pieces(const AttendParams& a, const AttendWork& work, const JoinItem& j, int tid) {
  constexpr int kVec = kDim / 32;  // values per lane
  const int lane = tid & 31, r0 = j.qt * a.item_rows, last = min(a.item_rows, a.tokens * a.group - r0);
  for (int row0 = tid >> 5; row0 < last; row0 += kWarps * kBatch) {
    float o[kBatch][kVec] = {}, m[kBatch], l[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
    for (int c = j.c0; c <= j.c1; c += 32) {
      const int mine = c + lane, pieces = min(32, j.c1 - c + 1);
      float2 ml[kBatch];
      float w[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int row = min(row0 + kWarps * i, last - 1);
        ml[i] = mine <= j.c1 ? __ldcg(&work.ml[(2 * (size_t)mine + (mine == j.c0)) * kRows + row])
                             : make_float2(-INFINITY, 0.0f);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        float top = ml[i].x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float m1 = fmaxf(m[i], top), base = m1 == -INFINITY ? 0.0f : m1;
        const float keep = exp2_approx(m[i] - base);
        w[i] = exp2_approx(ml[i].x - base);
        float sum = ml[i].y * w[i];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l[i] = l[i] * keep + sum;
        m[i] = m1;
#pragma unroll
        for (int v = 0; v < kVec; ++v) o[i][v] *= keep;
      }
      // (nothing is read behind the last piece: read again and given weight zero, an infinity in it would be NaN)
#pragma unroll 1
      for (int k = 0; k < pieces; k += kUnroll) {
        alignas(16) float x[kUnroll][kBatch][kVec];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (k + u >= pieces) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
              for (int v = 0; v < kVec; ++v) x[u][i][v] = 0.0f;
            continue;
          }
          const int piece = c + k + u;
          const float* part = work.o + (2 * (size_t)piece + (piece == j.c0)) * kRows * kDim + lane * kVec;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const float* from = part + min(row0 + kWarps * i, last - 1) * kDim;
            if constexpr (kVec == 2) {
              *reinterpret_cast<float2*>(x[u][i]) = __ldcg(reinterpret_cast<const float2*>(from));
            } else {
#pragma unroll
              for (int v = 0; v < kVec; v += 4)
                *reinterpret_cast<float4*>(x[u][i] + v) = __ldcg(reinterpret_cast<const float4*>(from + v));
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const float wk = __shfl_sync(0xffffffffu, w[i], (k + u) & 31);
#pragma unroll
            for (int v = 0; v < kVec; ++v) o[i][v] += x[u][i][v] * wk;
          }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int row = row0 + kWarps * i, r = r0 + row, t = r / a.group, g = r - t * a.group;
      if (row >= last || lane * kVec >= a.dim) continue;
      const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
      const bool live = r < j.rows;  // the pieces of rows behind the chunk's end hold anything
#pragma unroll
      for (int v = 0; v < kVec; ++v) o[i][v] = live ? o[i][v] * inv : 0.0f;
      T* out = static_cast<T*>(a.out) + (((long long)j.b * a.tokens + t) * a.heads + j.h * a.group + g) * a.dim + lane * kVec;
#pragma unroll
      for (int v = 0; v < kVec; v += 2) store2(out + v, o[i][v], o[i][v + 1]);
    }
  }
}

// Query tiles with nothing to see or behind the end of a short chunk: zeros.
template <typename T>
__device__ __forceinline__ void zero_blind_tiles(const AttendParams& a, int q_tiles, int thread, int threads) {
  for (int e = blockIdx.x; e < a.batch * q_tiles; e += gridDim.x) {
    const int b = e / q_tiles, qt = e - b * q_tiles;
    if (tile_span(a, b, qt, a.item_rows).n) continue;
    const int r1 = min((qt + 1) * a.item_rows, a.tokens * a.group);
    for (int r = qt * a.item_rows; r < r1; ++r) {
      const int t = r / a.group, g = r - t * a.group;
      for (int i = thread; i < a.kv_heads * (a.dim / 8); i += threads) {
        const int h = i / (a.dim / 8), d = (i - h * (a.dim / 8)) * 8;
        T* out = static_cast<T*>(a.out) + (((long long)b * a.tokens + t) * a.heads + h * a.group + g) * a.dim + d;
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(out)[k] = make_uint4(0, 0, 0, 0);
      }
    }
  }
}

}  // namespace dd
