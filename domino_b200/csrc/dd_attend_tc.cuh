// dd_attend_tc.cuh -- paged attention on the tensor cores, for 16-bit caches
// with heads of up to 128 values.
//
// The query rows of one key head (token t, head g of the group: row t G + g)
// fill the 128 rows of a tile, so a block of 16 tokens with 4 heads a group
// reads its keys once for 64 rows.  Per tile of 128 keys:
//
//   S = Q K^T       tcgen05, Q and K in shared memory, S in TMEM
//   P = e^(S - m)   one thread per row: TMEM -> registers -> TMEM (16 bits)
//   O += P V        tcgen05, P from TMEM, V in shared memory, O in TMEM
//
// Two streams, each with its own S, O and four softmax warps, keep the tensor
// cores busy while the other stream's exponentials run.  With kPair they are
// two query tiles over the same keys (long chunks: every key tile serves 256
// rows); without, they take alternate key tiles of one query tile and are
// joined at the end (few rows, bound by the bytes of the cache).
//
// Work is cut by key tiles, not by rows: the tiles of all (row of the batch,
// query tile, key head) items are numbered through and every CTA takes an
// equal run of them, so long and short rows balance and one row's long cache
// spreads over all SMs.  An item that crosses CTAs leaves its pieces
// (unnormalised O, m, l) in the workspace; the CTA that finishes last, found by
// a counter that wraps back to zero, adds them in the order of the CTAs, so the
// result is the same every time.  Lengths are read on the device, so the cut
// needs no host synchronisation.
//
// The running maximum m moves only when a row's scores pass it by more than 8
// (as powers of two): P then stays below 2^8 and the rescaling of O, a round
// trip through TMEM, is rare.  m, l, S and O are fp32; P is rounded to the
// cache's type, the one rounding besides the result's.
//
// In fp16, where weights below 2^-14 would lose bits and those below 2^-25
// vanish (from O, not from l: a long even tail under one large weight), P and l
// are 2^7 times as large: P then stays below 2^15.3, and what loses bits is
// below 2^-21.  (O is fp32 all the same: of products below 2^-25 of it the
// tensor cores add nothing.)
//
// m is a whole number, the maximum rounded up: pieces, streams and copies of a
// row that took different maxima differ by exact powers of two, so that P's
// rounding is the same wherever a row's keys are cut.  What else shares the
// batch changes a row by the order of fp32 sums, and by the few weights that lie
// on the border between two 16-bit numbers: 0.1-0.2 % of the results of 4096
// keys in bf16, 0.4-1.5 % in fp16; 42-46 % with the maximum itself as m.  The
// largest weight, which that made 1, is rounded now; it counts in l as it was
// rounded.  That leaves errors of 1.15 to 1.3 times a result's own rounding;
// without, 1.4 to 1.7 times.
//
// A masked key has weight 0, and 0 times a NaN is NaN in a matrix product.
// So the values of keys that no row of the item sees are set to zero in
// shared memory (pages behind the end, missing pages, the rest of a page).
// Keys that only some rows see are searched for infinities and NaN, which are
// set to zero too; where there was one, every row adds those that it sees to
// its result (add_part_seen).  These keys are at most two for every token of
// the item (behind its first token, and before its last one's window), so that
// takes as long for a long row of keys as for a short one.
#pragma once

#include "dd_attend_cut.cuh"

namespace dd {

constexpr int kAttThreads = 384;  // 8 softmax warps, key producer, MMA issuer, value producer, query loader
constexpr int kMaxTensorCtas = 160;
constexpr int kMaxStages = 12;
constexpr int kMergeCols = 16;  // of the two buffers of each stream's warps that join copies of rows

// The ring of key and value tiles.  Tiles are loaded in the order in which the
// tensor cores take them: with kPair K0 V0 K1 V1 .., without K0 K1 V0 K2 V1 K3
// .. (the two streams one tile apart), so producer and issuer walk it in step.
template <int kStages>
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
};
// Position of tile i's keys / values in a piece's load order; n tiles.
template <bool kPair>
__device__ __forceinline__ int load_index_k(int i) {
  return kPair ? 2 * i : i < 2 ? i : 2 * i - 1;
}
template <bool kPair>
__device__ __forceinline__ int load_index_v(int i, int n) {
  return kPair ? 2 * i + 1 : i + min(i + 2, n);
}

// A row's table entries, 32 at a time with the next 32 on their way, one per lane.
struct PageWindow {
  int w = -2, now = -1, next = -1;
  __device__ __forceinline__ int entry(const AttendParams& a, const Piece& p, int w32, int lane) const {
    const int slot = w32 * 32 + lane;
    int page = -1;
    if (slot < a.row_pages && (slot << a.page_shift) < p.span.hi) {
      page = a.table[(long long)p.b * a.row_pages + slot];
      if (page >= a.pages) page = -1;
    }
    return page;
  }
  // Page of lane's part of a key tile (lanes below 128 / page_size; -1 elsewhere and where there is none).
  __device__ __forceinline__ int get(const AttendParams& a, const Piece& p, int tile, int lane) {
    const int per = kKeyTile >> a.page_shift, slot = tile * per, w32 = slot >> 5;
    if (w32 != w) {
      now = w32 == w + 1 ? next : entry(a, p, w32, lane);
      next = entry(a, p, w32 + 1, lane);
      w = w32;
    }
    const int page = __shfl_sync(0xffffffffu, now, (slot & 31) + lane);
    return lane < per ? page : -1;
  }
};

// Page of 16-key group `lane` (0 .. 7) of a key tile.
__device__ __forceinline__ int group_page(const AttendParams& a, int b, int tile, int lane) {
  const int slot = (tile * kKeyTile + lane * 16) >> a.page_shift;
  return lane < 8 && slot < a.row_pages ? a.table[(long long)b * a.row_pages + slot] : -1;
}

// One arrival for a whole warp, after all of its lanes got here.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
// The n lowest bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
// Scores that are not seen become -infinity.
__device__ __forceinline__ void mask32(uint32_t* x, uint32_t see) {
  if (__all_sync(0xffffffffu, see == ~0u)) return;
#pragma unroll
  for (int k = 0; k < 32; ++k) x[k] = see >> k & 1 ? x[k] : 0xff800000u;
}
// Whether either half of a packed word is an infinity or a NaN.
template <typename T>
__device__ __forceinline__ bool non_finite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w >> 16 & e) == e;
}

// The word with its infinities and NaN set to zero.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0u : w & 0xffffu) | ((w >> 16 & e) == e ? 0u : w & 0xffff0000u);
}

// (Out of line: in line it cost the softmax loop its registers, and 8192 tokens
// behind 8192 took 1930 us against 1746.)
template <typename T>
__device__ __noinline__ void clean16(uint4* at) {
  const uint4 w = *at;
  *at = make_uint4(finite2<T>(w.x), finite2<T>(w.y), finite2<T>(w.z), finite2<T>(w.w));
}

// The keys that all rows of a piece's item see are [lo, hi) and, below hi, the sinks.
struct SeenByAll {
  int lo, hi;
};
__device__ __forceinline__ SeenByAll seen_by_all(const AttendParams& a, const Piece& p) {
  const int first = p.span.start + p.qt * a.item_rows / a.group;
  const int last = p.span.start + (min(p.span.rows, (p.qt + 1) * a.item_rows) - 1) / a.group;
  return {a.window > 0 ? max(last - a.window + 1, 0) : 0, a.causal ? min(p.span.hi, first + 1) : p.span.hi};
}

// Infinities and NaN among values [col, end) of the piece's keys that only some
// rows of its item see: those that `row` sees are added to its result, which
// stands in `out` (value col at out[0]).
template <typename T, typename O>
__device__ __noinline__ void add_part_seen(const AttendParams& a, const Piece& p, int row, int col, int end, O* out) {
  const SeenByAll all = seen_by_all(a, p);
  const int pos = p.span.start + row / a.group;
  const int hi = a.causal ? min(p.span.hi, pos + 1) : p.span.hi, lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
  // the piece's keys from span.lo on
  const int from = (p.span.first + max(p.i0 - p.span.n_sink, 0)) * kKeyTile;
  const int to = min((p.span.first + max(p.i1 - p.span.n_sink, 0)) * kKeyTile, hi);
  auto add = [&](int j0, int j1) {
    for (int j = max(j0, from); j < min(j1, to); ++j) {
      if (j < lo && j >= a.sinks) continue;
      const int page = a.table[(long long)p.b * a.row_pages + (j >> a.page_shift)];
      if (page < 0 || page >= a.pages) continue;
      const T* v = static_cast<const T*>(a.pool[1]) +
                   (((long long)page * a.kv_heads + p.h) * a.page_size + (j & (a.page_size - 1))) * a.dim;
      for (int d = col; d < end; d += 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(v + d);
        if (!non_finite2<T>(w.x) && !non_finite2<T>(w.y)) continue;
        const T* x = reinterpret_cast<const T*>(&w);
        for (int i = 0; i < 4; ++i)
          if (!isfinite(io<T>::to_f(x[i])))
            out[d - col + i] = io<O>::from_f(io<O>::to_f(out[d - col + i]) + io<T>::to_f(x[i]));
      }
    }
  };
  add(max(p.span.lo, a.sinks), min(all.lo, all.hi));
  add(all.hi, p.span.hi);
}

template <int kDim, bool kPair>
struct AttendShape {
  static constexpr int kTiles = kPair ? 2 : 1;      // query tiles
  static constexpr int kRows = 128 * kTiles;
  static constexpr int kHalves = kDim / 64;
  static constexpr int kParts = kPair ? 2 : 1;      // parts of a key tile with scores and weights of their own
  static constexpr int kTileBytes = 128 * kDim * 2;  // a query tile, a K or V tile
  static constexpr int kMergeBytes = kPair ? 0 : 2 * 2 * 128 * kMergeCols * 4;
  static constexpr int kFit = (224 * 1024 - kTiles * kTileBytes - kMergeBytes) / kTileBytes;
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
};

// Behind the tiles in shared memory.
struct AttendShared {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2], o_full[2], q_full, q_empty, wg[2], both;
  uint32_t tmem_base;
  int abort_flag;
  CutShared cut;
  int n_joins;
  JoinItem joins[2];    // a run's first and last item
  // the last piece (counted from 1) with an infinity or a NaN in a key that only some rows see: by stream, with kPair
  // by even and odd pieces
  unsigned odd[2];
  float row_norm[128];
  union {
    float2 row_ml[2][128];
    CutScan scan;  // while the work is cut
  };
};
// All of the 227 KB; the tiles start on a 1024-byte boundary, and there is
// room for the padding that takes (the window starts on one: none).
constexpr int kAttSmem = 227 * 1024;
constexpr int kAttPad = kAttSmem - 224 * 1024 - (int)sizeof(AttendShared);
static_assert(kAttPad >= 0, "tiles and AttendShared must fit 227 KB");

template <typename T, int kDim, bool kPair>
__global__ void __launch_bounds__(kAttThreads, 1)
    attend_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ CUtensorMap map_q, const __grid_constant__ AttendParams a,
                     const __grid_constant__ AttendWork work) {
  using Shape = AttendShape<kDim, kPair>;
  extern __shared__ unsigned char smem_raw[];
  const int pad = (1024 - (smem_u32(smem_raw) & 1023)) & 1023;
  if (pad > kAttPad) {
    if (threadIdx.x == 0) atomicOr(a.status, DD_STATUS_TIMEOUT);
    return;
  }
  unsigned char* sm_q = smem_raw + pad;
  unsigned char* sm_ring = sm_q + Shape::kTiles * Shape::kTileBytes;
  AttendShared& bar = *reinterpret_cast<AttendShared*>(sm_q + 224 * 1024);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.group;
  const int q_tiles = (a.tokens * group + a.item_rows - 1) / a.item_rows;

  if (tid == 0) {
    bar.abort_flag = 0;
    bar.n_joins = 0;
    bar.odd[0] = bar.odd[1] = 0;
    for (int i = 0; i < Shape::kStages; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], 1);
    }
    for (int s = 0; s < 2; ++s) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&bar.s_full[s][k], 1);
        mbar_init(&bar.p_full[s][k], 4);  // one arrival per warp
      }
      mbar_init(&bar.pv_done[s], 1);
      mbar_init(&bar.o_full[s], 1);
      mbar_init(&bar.wg[s], 4);
    }
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_empty, 1);
    mbar_init(&bar.both, 8);
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(&bar.tmem_base, 512);
  if (tid == 32 * 8) {
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  pdl_wait_primary();

  cut_work<kAttThreads>(a, bar.cut, bar.scan, q_tiles, tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem_base;
  volatile int* abort = &bar.abort_flag;
  Piece p = bar.cut.first;
  bool more = p.left > 0;

  if (warp == 8 || warp == 10) {
    // ---------------------------------------------------------------- producers: keys, values
    const bool keys = warp == 8;
    const CUtensorMap* map = keys ? &map_k : &map_v;
    const uint32_t page_bytes = a.page_size * 128u;  // of one 64-value half
    int base = 0;  // loads before this piece, modulo two rounds of the ring
    bool ok = true;
    for (; more && ok; more = piece_next(a, p, q_tiles, a.item_rows)) {
      const int n = p.i1 - p.i0;
      PageWindow window;
      for (int i = 0; i < n; ++i) {
        const int page = window.get(a, p, p.span.tile(p.i0 + i), lane);
        const int c = (base + (keys ? load_index_k<kPair>(i) : load_index_v<kPair>(i, n))) % (2 * Shape::kStages);
        const int st = c >= Shape::kStages ? c - Shape::kStages : c;
        ok = mbar_wait_bounded(&bar.empty[st], (c >= Shape::kStages) ^ 1, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) mbar_arrive_expect_tx(&bar.full[st], __popc(have) * page_bytes * Shape::kHalves);
        __syncwarp();
        if (page >= 0) {
          unsigned char* dst = sm_ring + st * Shape::kTileBytes + lane * page_bytes;
#pragma unroll
          for (int hf = 0; hf < Shape::kHalves; ++hf)
            tma_load_4d(dst + hf * 128 * 128, map, &bar.full[st], hf * 64, 0, p.h, page);
        }
      }
      base = (base + 2 * n) % (2 * Shape::kStages);
    }
    if (!ok) {  // leave no copy in flight behind this CTA: time for all of them to land
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 10 * 1000 * 1000) {
      }
    }
  } else if (warp == 9) {
    // ---------------------------------------------------------------- MMA issuer
    // The whole warp walks the schedule and one elected lane issues: descriptors
    // then stay in uniform registers (issued from inside a lane's own branch, the
    // 16 MMAs of a tile took 1500 cycles, of which the tensor cores need 1024;
    // like this 1130).
    constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr int kPartKeys = kKeyTile / Shape::kParts;
    constexpr uint32_t idesc_s = idesc_f16(kPartKeys, fmt), idesc_o = idesc_f16(kDim, fmt) | kIdescBMnMajor;
    Ring<Shape::kStages> ring;
    uint32_t n_pieces = 0, n_p[2] = {0, 0};  // tiles whose weights stream s has delivered
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t parity) {
      ok = ok && mbar_wait_bounded(b, parity, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
    // the stage of the next load, once it has landed
    auto take = [&]() {
      const int st = ring.stage;
      wait(&bar.full[st], ring.phase);
      ring.next();
      return st;
    };
    const uint32_t ring0 = smem_u32(sm_ring), q0 = smem_u32(sm_q);
    const int copies = kPair ? 1 : a.copies;
    // Scores of stream s from a part of the keys in stage st, and which buffers are free once they are done.
    auto qk = [&](int s, int part, int st, bool free_stage, bool free_q) {
      const uint64_t dq = smem_desc_k_sw128(q0 + (kPair ? s * Shape::kTileBytes : 0));
      const uint64_t dk = smem_desc_k_sw128(ring0 + st * Shape::kTileBytes + part * kPartKeys * 128);
      if (elect_one()) {
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
          const uint64_t off = ((d / 4) * 128 * 128 + (d % 4) * 32) >> 4;
          mma_f16_ss(tmem + s * 128 + part * kPartKeys, dq + off, dk + off, idesc_s, d > 0);
        }
        mma_commit(&bar.s_full[s][part]);
        if (free_stage) mma_commit(&bar.empty[st]);
        if (free_q) mma_commit(&bar.q_empty);
      }
      __syncwarp();
    };
    auto pv = [&](int s, int part, int st, bool accumulate, bool free_stage, bool last) {
      const uint64_t dv = smem_desc_mn_sw128(ring0 + st * Shape::kTileBytes + part * kPartKeys * 128, 128 * 128);
      if (elect_one()) {
#pragma unroll
        for (int d = 0; d < kPartKeys / 16; ++d) {
          const uint32_t to = tmem + 256 + s * kDim, from = tmem + s * 128 + part * kPartKeys + d * 8;
          if (kPair) {
            mma_f16_ts(to, from, dv + ((d * 2048) >> 4), idesc_o, accumulate || d > 0);
          } else {
            // a step of 16 keys is for the copy of the rows that has them: the others' sums stay (a weight of zero
            // would make an infinite value NaN there)
            const int copy = (d * copies) >> 3;
            uint32_t off[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) off[w] = (w * copies) >> 2 == copy ? 0u : ~0u;
            mma_f16_ts_lanes(to, from, dv + ((d * 2048) >> 4), idesc_o, accumulate || ((d * copies) & 7) != 0, off);
          }
        }
        if (Shape::kParts > 1) mma_commit(&bar.pv_done[s]);
        if (free_stage) mma_commit(&bar.empty[st]);
        if (last) mma_commit(&bar.o_full[s]);
      }
      __syncwarp();
    };
    auto wait_p = [&](int s, int part) {
      wait(&bar.p_full[s][part], (part + 1 == Shape::kParts ? n_p[s]++ : n_p[s]) & 1);
      tc_fence_after();
    };
    for (; more && ok; more = piece_next(a, p, q_tiles, a.item_rows)) {
      const int n = p.i1 - p.i0;
      wait(&bar.q_full, n_pieces++ & 1);
      if (!ok) break;
      tc_fence_after();
      if (kPair) {
        constexpr int kSteps = 2 * Shape::kParts;
        int k = take(), v = 0;
        if (!ok) break;
        // parts outside, streams inside: while one stream's exponentials of a
        // part run, the tensor cores have its other part and the other stream
#pragma unroll
        for (int u = 0; u < kSteps; ++u) qk(u & 1, u >> 1, k, u == kSteps - 1, u == kSteps - 1 && n == 1);
        for (int i = 0; i < n && ok; ++i) {
#pragma unroll
          for (int u = 0; u < kSteps; ++u) {
            const int s = u & 1, part = u >> 1;
            wait_p(s, part);
            if (u == 0 && ok) v = take();
            if (!ok) break;
            pv(s, part, v, i > 0 || part > 0, u == kSteps - 1, i + 1 == n && part + 1 == Shape::kParts);
            if (i + 1 < n) {
              if (u == 0) k = take();
              if (!ok) break;
              qk(s, part, k, u == kSteps - 1, u == kSteps - 1 && i + 2 == n);
            }
          }
        }
      } else {
        for (int s = 0; s < min(2, n) && ok; ++s) {
          const int k = take();
          if (ok) qk(s, 0, k, true, s + 1 == n);
        }
        for (int i = 0; i < n && ok; ++i) {
          const int s = i & 1;
          wait_p(s, 0);
          if (!ok) break;
          const int v = take();
          if (!ok) break;
          pv(s, 0, v, i >= 2, true, i + 2 >= n);
          if (i + 2 < n) {
            const int k = take();
            if (ok) qk(s, 0, k, true, i + 3 == n);
          }
        }
      }
    }
  } else if (warp == 11) {
    // ---------------------------------------------------------------- query loader, and the rows of no item
    // A tile holds whole tokens (128 / group of them), so one box of [tokens,
    // heads of the group, 64 values] fills it.  Where q's layout does not allow
    // TMA: 16-byte asynchronous copies, a thread keeping one chunk of the rows,
    // or plain loads.
    constexpr int kChunks = kDim / 8, kRowStep = 32 / kChunks;
    const int ch = lane % kChunks;
    const bool vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_stride[0] % 8 == 0 && a.q_stride[1] % 8 == 0 &&
                     a.q_stride[2] % 8 == 0;
    const int copies = kPair ? 1 : a.copies, copy_rows = 128 / copies, live_rows = kPair ? 128 : copy_rows;
    uint32_t n_pieces = 0;
    bool ok = true;
    for (; more; more = piece_next(a, p, q_tiles, a.item_rows)) {
      ok = mbar_wait_bounded(&bar.q_empty, (n_pieces++ & 1) ^ 1, abort);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int r0 = p.qt * a.item_rows;
      if (a.q_tma) {
        const int box = copy_rows / group;  // tokens
        if (elect_one()) {
          mbar_arrive_expect_tx(&bar.q_full, Shape::kTiles * copies * Shape::kHalves * box * group * 128);
          for (int i = 0; i < Shape::kTiles * copies; ++i)
#pragma unroll
            for (int hf = 0; hf < Shape::kHalves; ++hf)
              tma_load_4d(sm_q + (kPair ? i * Shape::kTileBytes : i * copy_rows * 128) + hf * 128 * 128, &map_q,
                          &bar.q_full, hf * 64, p.h * group, r0 / group + (kPair ? i * box : 0), p.b);
        }
        __syncwarp();
        continue;
      }
      const T* q = static_cast<const T*>(a.q) + p.b * a.q_stride[0] + (long long)p.h * group * a.q_stride[2] + ch * 8;
      const bool in = ch * 8 < a.dim;
      for (int tile = 0; tile < Shape::kTiles; ++tile) {
        const int first_row = r0 + tile * a.tile_rows, rows = min(min(a.tile_rows, live_rows), p.span.rows - first_row);
        int row = lane / kChunks, t = (first_row + row) / group, g = first_row + row - t * group;
        for (; row < rows; row += kRowStep) {
          const T* src = q + t * a.q_stride[1] + g * a.q_stride[2];
          for (int to = row; to < 128; to += live_rows) {
            unsigned char* dst =
                sm_q + tile * Shape::kTileBytes + (ch / 8) * 128 * 128 + to * 128 + ((ch % 8) ^ (to % 8)) * 16;
            if (vec) {
              cp_async16(dst, in ? src : a.q, in ? 16 : 0);
            } else {
              alignas(16) T x[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = in ? src[i] : io<T>::from_f(0.0f);
              *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
            }
          }
          for (g += kRowStep; g >= group; g -= group) ++t;
        }
      }
      cp_async_wait_all();
      fence_proxy_async_shared();
      warp_arrive(&bar.q_full, lane);
    }
    zero_blind_tiles<T>(a, q_tiles, lane, 32);
  } else {
    // ---------------------------------------------------------------- softmax, one thread per query row
    constexpr int kPartKeys = kKeyTile / Shape::kParts;
    constexpr int kCols = kPair ? 2 : 1;  // groups of 32 columns in registers at a time
    constexpr float kTopExponent = std::is_same<T, __half>::value ? 7.0f : 0.0f;
    const int s = warp >> 2, row = tid & 127;
    const uint32_t lanes = ((warp & 3) * 32u) << 16;
    const uint32_t t_s = tmem + s * 128 + lanes, t_o = tmem + 256 + lanes;
    const float sl = a.scale * 1.4426950408889634f;
    uint32_t n_s = 0, n_part = 0, n_o[2] = {0, 0}, n_wg = 0, n_both = 0, n_pieces = 0;
    int base = 0;  // loads before this piece, modulo two rounds of the ring
    bool ok = true, pending = false;
    // Few rows: the tile holds `copies` copies of them, and copy c of a row
    // takes part c of the tile's keys (the products leave its sums alone
    // elsewhere), so that all four warps share the exponentials.  The copies
    // are joined like the streams.
    const int copies = kPair ? 1 : a.copies, copy_rows = 128 / copies;
    const int chunk0 = (row / copy_rows) * (4 / copies), chunk1 = chunk0 + 4 / copies;
    for (; more && ok; more = piece_next(a, p, q_tiles, a.item_rows)) {
      const int n = p.i1 - p.i0;
      ++n_pieces;
      const int tile0 = p.qt * a.item_rows + (kPair ? s * a.tile_rows : 0), in_tile = kPair ? row : row % copy_rows;
      const int rows_here = min(p.span.rows - tile0, a.tile_rows);  // live rows of the tile
      const int r = tile0 + in_tile;
      const bool live = in_tile < rows_here, warp_live = in_tile - lane < rows_here;
      // keys that the row sees: [lo, hi) and, below hi, [0, sinks)
      int hi = 0, lo = 0;
      if (live) {
        const int pos = p.span.start + r / group;
        hi = a.causal ? min(p.span.hi, pos + 1) : p.span.hi;
        lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
      }
      const SeenByAll all = seen_by_all(a, p);
      float m = -INFINITY, l = 0.0f;
      bool have_o = false, far = false;  // far: a row of the warp has m of 2^20 or more
      constexpr int kStep = kPair ? 1 : 2;
      int page = (kPair ? 0 : s) < n ? group_page(a, p.b, p.span.tile(p.i0 + (kPair ? 0 : s)), lane) : 0;
      if (!kPair && pending) {  // the last piece's O, maxima and flags have been read by all
        ok = mbar_wait_bounded(&bar.both, n_both++ & 1, abort);
        if (!ok) break;
        pending = false;
      }
      for (int i = kPair ? 0 : s; i < n && ok; i += kStep) {
        const int tile = p.span.tile(p.i0 + i);
        // 16-key groups without a page (read one tile ahead)
        const unsigned missing = __ballot_sync(0xffffffffu, lane < 8 && (page < 0 || page >= a.pages));
        if (i + kStep < n) page = group_page(a, p.b, p.span.tile(p.i0 + i + kStep), lane);
#pragma unroll
        for (int part = 0; part < Shape::kParts; ++part, ++n_part) {
          const int key0 = tile * kKeyTile, part0 = key0 + part * kPartKeys, part1 = part0 + kPartKeys;
          const bool whole = missing == 0 && part1 <= all.hi && (part0 >= all.lo || part1 <= a.sinks);
          ok = mbar_wait_bounded(&bar.s_full[s][part], n_s & 1, abort);
          if (!ok) break;
          if (part + 1 == Shape::kParts) ++n_s;
          tc_fence_after();
          const int chunk_a = kPair ? part * (kPartKeys / 32) : chunk0, chunk_b = kPair ? chunk_a + kPartKeys / 32 : chunk1;
          if (warp_live) {
            // bit k: the row sees key 32 c + k of the tile
            auto see = [&](int c) {
              const int k0 = key0 + 32 * c;
              const uint32_t gap = (missing >> (2 * c) & 1) * 0xffffu | (missing >> (2 * c + 1) & 1) * 0xffff0000u;
              return low_bits(hi - k0) & (~low_bits(lo - k0) | low_bits(a.sinks - k0)) & ~gap;
            };
            // kCols x 32 scores in registers at a time; where that is not all of
            // the thread's, they are read again for the exponentials.
            uint32_t x[32 * kCols];
            auto fetch = [&](int c) {
#pragma unroll
              for (int d = 0; d < kCols; ++d) tmem_ld32(t_s + 32 * (c + d), x + 32 * d);
              tmem_ld_wait();
              if (!whole)
#pragma unroll
                for (int d = 0; d < kCols; ++d) mask32(x + 32 * d, see(c + d));
            };
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
            for (int c = chunk_a; c < chunk_b; c += kCols) {
              fetch(c);
#pragma unroll
              for (int k = 0; k < 32 * kCols; k += 4) {
                top[0] = max3_nan(top[0], __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                top[1] = max3_nan(top[1], __uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
              }
            }
            const float mt = max3_nan(top[0], top[1], top[1]);
            if (!(mt < INFINITY)) l = __int_as_float(0x7fc00000);  // a NaN or +infinity among the scores: the row is NaN
            const float mt2 = __fmul_rn(mt, sl);
            const bool moves = mt2 - m > 8.0f;
            if (__any_sync(0xffffffffu, moves)) {
              const float m1 = moves ? ceilf(mt2) : m;
              const float keep = moves ? exp2_approx(m - m1) : 1.0f;
              l *= keep;
              m = m1;
              far = __any_sync(0xffffffffu, fabsf(m) >= 1048576.0f && m != -INFINITY);
              if (have_o) {
                // (the scores of part k come after the products of part k - 2; those of k - 1 may still run)
                if (Shape::kParts > 1) ok = mbar_wait_bounded(&bar.pv_done[s], (n_part - 1) & 1, abort);
                if (Shape::kParts > 1) tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < kDim; c += 32) {
                  uint32_t o[32];
                  tmem_ld32(t_o + s * kDim + c, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                  tmem_st32(t_o + s * kDim + c, o);
                }
              }
            }
            have_o = true;
            const float sub = (m == -INFINITY ? 0.0f : m) - kTopExponent;
            uint64_t sum[4] = {0, 0, 0, 0};  // (two fp32 zeros each)
            // With m of 2^20 and more scores are scaled and rounded before m is taken off, as in m, so that none comes
            // out above its maximum (in one step those of 2^29 came out up to 2^5 beside it: infinite weights in fp16).
            const float sl1 = far ? 1.0f : sl;
            const uint64_t sl2 = pack_f32x2(sl1, sl1), sub2 = pack_f32x2(-sub, -sub);
#pragma unroll 1
            for (int c = chunk_a; c < chunk_b; c += kCols) {
              if (chunk_b - chunk_a > kCols) fetch(c);
              if (far)
#pragma unroll
                for (int k = 0; k < 32 * kCols; ++k) x[k] = __float_as_uint(__fmul_rn(__uint_as_float(x[k]), sl));
#pragma unroll
              for (int d = 0; d < kCols; ++d) {
                uint32_t w[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  const float x0 = __uint_as_float(x[32 * d + 2 * k]), x1 = __uint_as_float(x[32 * d + 2 * k + 1]);
                  const uint64_t e = fma_f32x2(pack_f32x2(x0, x1), sl2, sub2);
                  float e0, e1;
                  unpack_f32x2(e, e0, e1);
                  const float p0 = exp2_approx(e0), p1 = exp2_approx(e1);
                  sum[k & 3] = add_f32x2(sum[k & 3], pack_f32x2(p0, p1));
                  w[k] = pack2<T>(p0, p1);
                }
                // over scores that have been read, a part's weights within its own columns
                tmem_st16(t_s + (kPair ? part * kPartKeys + 16 * (c + d - chunk_a) : 16 * (c + d)), w);
              }
            }
            float sum0, sum1;
            unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])), sum0, sum1);
            // the part's largest weight counts as it was rounded: one that takes everything gives its value as it is
            const float top_w = exp2_approx(far ? mt2 - sub : fmaf(mt, sl, -sub));
            l += sum0 + sum1 + (io<T>::to_f(io<T>::from_f(top_w)) - top_w);
            tmem_st_wait();
          }
          if (!whole && (!kPair || s == 0)) {  // (pairs: the other stream's products of a part come after this one's)
            const int c = (base + load_index_v<kPair>(i, n)) % (2 * Shape::kStages);
            const int st = c % Shape::kStages;
            ok = mbar_wait_bounded(&bar.full[st], c / Shape::kStages, abort);
            if (!ok) break;
            // keys that no row of the item sees become zero, and infinities and NaN of those that only some see.
            // Eight lanes a 128-byte row, four rows a step.
            unsigned char* v = sm_ring + st * Shape::kTileBytes + (lane % 8) * 16;
            bool odd = false, wrote = false;
#pragma unroll 1
            for (int k = part * kPartKeys + (warp & 3) * (kPartKeys / 4) + lane / 8, k1 = k + kPartKeys / 4; k < k1; k += 4) {
              const int j = key0 + k;
              const bool seen = j < p.span.hi && (j >= p.span.lo || j < a.sinks) && !(missing >> (k / 16) & 1);
              const bool search = seen && (j >= all.hi || (j < all.lo && j >= a.sinks));
#pragma unroll
              for (int hf = 0; hf < Shape::kHalves; ++hf) {
                uint4* at = reinterpret_cast<uint4*>(v + hf * 128 * 128 + k * 128);
                if (!seen) {
                  *at = make_uint4(0, 0, 0, 0);
                  wrote = true;
                } else if (search) {
                  const uint4 w = *at;
                  if (non_finite2<T>(w.x) || non_finite2<T>(w.y) || non_finite2<T>(w.z) || non_finite2<T>(w.w)) {
                    clean16<T>(at);
                    odd = wrote = true;
                  }
                }
              }
            }
            if (wrote) fence_proxy_async_shared();
            if (odd) bar.odd[kPair ? n_pieces & 1 : s] = n_pieces;
          }
          tc_fence_before();
          warp_arrive(&bar.p_full[s][part], lane);
        }
      }
      if (!ok) break;
      // the piece's result
      const bool split = p.i0 > 0 || p.i1 < p.span.n;
      const size_t slot = 2 * (size_t)blockIdx.x + (p.i0 == 0 ? 1 : 0);
      const int slot_row = (kPair ? s * a.tile_rows : 0) + in_tile;
      const bool in_chunk = in_tile < a.tile_rows && r < a.tokens * group;
      float* part = work.o + slot * Shape::kRows * kDim;
      float2* part_ml = work.ml + slot * Shape::kRows;
      auto out_row = [&](int r) {
        const int t = r / group, g = r - t * group;
        return static_cast<T*>(a.out) + (((long long)p.b * a.tokens + t) * a.heads + p.h * group + g) * a.dim;
      };
      T* const out0 = out_row(kPair ? r : row / 4);  // (the divisions run while the last products do)
      bool odd;
      float f0 = 1.0f, f1 = 0.0f;  // weights of the streams' sums (kPair: only its own)
      if (kPair) {
        ok = mbar_wait_bounded(&bar.o_full[s], n_o[s]++ & 1, abort);
        if (!ok) break;
        // The last products came after all of stream 0's weights, and so after its searches; it reaches the piece after
        // the next, and this word again, only behind the other stream's weights of the next.
        odd = bar.odd[n_pieces & 1] == n_pieces;
      } else {
        bar.row_ml[s][row] = make_float2(m, l);
        ok = mbar_wait_bounded(&bar.o_full[0], n_o[0]++ & 1, abort);
        if (ok && n > 1) ok = mbar_wait_bounded(&bar.o_full[1], n_o[1]++ & 1, abort);
        if (!ok) break;
        warp_arrive(&bar.both, lane);
        ok = mbar_wait_bounded(&bar.both, n_both++ & 1, abort);
        if (!ok) break;
        odd = bar.odd[0] == n_pieces || bar.odd[1] == n_pieces;
        const float m0 = bar.row_ml[0][row].x, m1 = bar.row_ml[1][row].x;
        m = -INFINITY;
        for (int c = row % copy_rows; c < 128; c += copy_rows) m = fmaxf(m, fmaxf(bar.row_ml[0][c].x, bar.row_ml[1][c].x));
        l = 0.0f;
        for (int c = row % copy_rows; c < 128; c += copy_rows)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = bar.row_ml[k][c];
            if (x.y != 0.0f) l += x.y * exp2_approx(x.x - m);
          }
        f0 = m0 == -INFINITY ? 0.0f : exp2_approx(m0 - m);
        f1 = m1 == -INFINITY ? 0.0f : exp2_approx(m1 - m);
      }
      tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (kPair) {
        if (split && in_tile < a.tile_rows) part_ml[slot_row] = make_float2(m, l);
        const float norm = split ? 1.0f : inv;
#pragma unroll 1
        for (int c = 0; c < kDim; c += 32) {
          uint32_t x[32];
          if (warp_live) {
            tmem_ld32(t_o + s * kDim + c, x);
            tmem_ld_wait();
          }
          if (!in_chunk) continue;
          float o[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = live && norm != 0.0f ? __uint_as_float(x[k]) * norm : 0.0f;
          if (split) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(part + (size_t)slot_row * kDim + c + k) =
                  make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              if (c + k < a.dim)
                *reinterpret_cast<uint4*>(out0 + c + k) =
                    make_uint4(pack2<T>(o[k], o[k + 1]), pack2<T>(o[k + 2], o[k + 3]), pack2<T>(o[k + 4], o[k + 5]),
                               pack2<T>(o[k + 6], o[k + 7]));
          }
        }
        if (odd && in_chunk && live) {
          const Piece here = p;
          if (split)
            add_part_seen<T, float>(a, here, r, 0, a.dim, part + (size_t)slot_row * kDim);
          else
            add_part_seen<T, T>(a, here, r, 0, a.dim, out_row(r));
        }
      } else {
        // Each stream's warps take half of the columns, 16 at a time: both
        // streams' sums by row, the copies of a row through shared memory, and
        // out with four lanes a row.
        if (split && s == 0 && row < copy_rows) part_ml[row] = make_float2(m, l);
        bar.row_norm[row] = live ? inv : 0.0f;  // (both streams write the same)
        float4* merge = reinterpret_cast<float4*>(sm_q + 224 * 1024 - Shape::kMergeBytes) + s * 2 * 128 * 4;
        const int rows = min(rows_here, copy_rows), all_rows = min(a.tokens * group, copy_rows);
#pragma unroll 1
        for (int c = s * (kDim / 2), c_end = c + kDim / 2; c < c_end; c += kMergeCols) {
          if (warp_live) {
            uint32_t x[16], y[16];
            tmem_ld16u(t_o + c, x);
            if (n > 1) tmem_ld16u(t_o + kDim + c, y);
            tmem_ld_wait();
            float o[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              o[k] = __uint_as_float(x[k]) * f0;
              if (n > 1) o[k] += __uint_as_float(y[k]) * f1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 16-byte parts of the row, turned by the row against bank conflicts
              merge[row * 4 + (k ^ (row >> 1 & 3))] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          warp_arrive(&bar.wg[s], lane);
          ok = mbar_wait_bounded(&bar.wg[s], n_wg++ & 1, abort);
          if (!ok) break;
          const int part4 = row % 4, col = c + part4 * 4;
          for (int k = row / 4; k < all_rows; k += 32) {
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k < rows)
              for (int from = k; from < 128; from += copy_rows) {
                const float4 x = merge[from * 4 + (part4 ^ (from >> 1 & 3))];
                o.x += x.x;
                o.y += x.y;
                o.z += x.z;
                o.w += x.w;
              }
            if (split) {
              float* to = part + (size_t)k * kDim + col;
              *reinterpret_cast<float4*>(to) = o;
              if (odd && k < rows && col < a.dim) {
                const Piece here = p;
                add_part_seen<T, float>(a, here, k, col, col + 4, to);
              }
            } else if (col < a.dim) {
              const float norm = bar.row_norm[k];
              const uint2 w = make_uint2(pack2<T>(o.x * norm, o.y * norm), pack2<T>(o.z * norm, o.w * norm));
              T* to = (k == row / 4 ? out0 : out_row(k)) + col;
              *reinterpret_cast<uint2*>(to) = norm == 0.0f ? make_uint2(0, 0) : w;
              if (odd && k < rows) {
                const Piece here = p;
                add_part_seen<T, T>(a, here, k, col, col + 4, to);
              }
            }
          }
          // the other buffer next: the wait in between keeps the two apart
          merge = reinterpret_cast<float4*>(sm_q + 224 * 1024 - Shape::kMergeBytes) + s * 2 * 128 * 4 +
                  ((c / kMergeCols) & 1 ? 0 : 128 * 4);
        }
        if (!ok) break;
      }
      if (split) {
        // the piece is in the workspace; whoever brings the item's last adds them up, when its own run is done
        __threadfence();
        warp_arrive(&bar.both, lane);
        ok = mbar_wait_bounded(&bar.both, n_both++ & 1, abort);
        if (!ok) break;
        if (tid == 0) {
          finish_piece(work, bar.cut, p);
          if (bar.cut.join) bar.joins[bar.n_joins++] = JoinItem{p.b, p.qt, p.h, p.span.rows, bar.cut.c0, bar.cut.c1};
        }
      }
      if (!kPair) {  // O, the maxima and the flags have been read; the next piece's first P waits for the other stream's
        tc_fence_before();
        warp_arrive(&bar.both, lane);
        pending = true;
      }
      base = (base + 2 * n) % (2 * Shape::kStages);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) {
    tmem_relinquish();
    tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && bar.abort_flag) atomicOr(a.status, DD_STATUS_TIMEOUT);
  for (int i = 0; i < bar.n_joins; ++i)
    join_pieces<T, kDim, Shape::kRows, kAttThreads / 32, 6, 3>(a, work, bar.joins[i], tid);
}

}  // namespace dd
