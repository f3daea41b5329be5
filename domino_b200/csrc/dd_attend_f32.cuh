// dd_attend_f32.cuh -- paged attention on the FMA units: fp32 caches, whose
// products must not be rounded to 11 or 8 bits, and 16-bit heads of more than
// 128 values.
//
// One CTA of 256 threads holds 16 kR query rows (token t, head g of the group) and
// walks the keys in tiles of kKeys, double-buffered by asynchronous copies.
// Thread (ty, tx) of 16 x 16 computes rows kR ty ..: scores of keys tx, tx + 16,
// .. (a kR x kKeys / 16 register tile, both operands read 16 bytes at a
// time along the head dimension), the running maximum and sum (shuffles among
// the 16 threads of a row), the weights through shared memory, which only the
// row's own half-warp reads, and kR x kDim / 16 sums of weighted values.
// Bound by the FMA units when a tile has many rows, by latency when calls are
// small.  The cut and the join are those of dd_attend_cut.cuh.
//
// A masked weight is stored as -0: its value has no part, even if it is NaN.
#pragma once

#include "dd_attend_cut.cuh"

namespace dd {

constexpr int kF32Threads = 256;
constexpr int kF32Rows = 64;  // at most

// kR rows a thread, 16 kR rows a tile: one for a token or two (more would only
// be empty), four where calls are large, two where that leaves SMs without work.
template <int kDim, int kR>
struct F32Shape {
  static constexpr int kRows = 16 * kR;
  static constexpr int kKeys = kDim > 128 ? 32 : 64;
  static constexpr int kRow = kDim + 4;  // floats of a padded row: 16-byte reads of consecutive rows fall in different banks
  static constexpr int kWeightRow = kKeys + 4;
  static constexpr int kSmem = 4 * (kRows * kRow + 4 * kKeys * kRow + kRows * kWeightRow);
};

template <typename T, int kDim, int kR>
__global__ void __launch_bounds__(kF32Threads) attend_f32_kernel(const __grid_constant__ AttendParams a,
                                                                 const __grid_constant__ AttendWork work) {
  using Shape = F32Shape<kDim, kR>;
  constexpr int kRows = Shape::kRows;
  constexpr int kKeys = Shape::kKeys, kRow = Shape::kRow, kCols = kDim / 64, kScores = kKeys / 16;
  extern __shared__ __align__(16) float sm_f32[];
  __shared__ CutShared cut;
  __shared__ CutScan scan;
  __shared__ int key_seen[2][kKeys];  // whether any row of the item sees the key
  float* sm_q = sm_f32;
  float* sm_k = sm_q + kRows * kRow;   // two buffers
  float* sm_v = sm_k + 2 * kKeys * kRow;  // two buffers
  float* sm_w = sm_v + 2 * kKeys * kRow;
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int group = a.group, q_tiles = (a.tokens * group + a.item_rows - 1) / a.item_rows;
  pdl_wait_primary();
  cut_work<kF32Threads>(a, cut, scan, q_tiles, tid);
  __syncthreads();
  Piece p = cut.first;
  bool more = p.left > 0;
  const int chunks = a.dim / 4;  // 16-byte chunks of an fp32 row
  // (columns behind the head's end and rows behind the last hold anything: they
  // only reach sums that are not stored)
  const bool vec = std::is_same<T, float>::value && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 &&
                   a.q_stride[0] % 4 == 0 && a.q_stride[1] % 4 == 0 && a.q_stride[2] % 4 == 0;

  for (; more; more = piece_next(a, p, q_tiles, a.item_rows)) {
    const int r0 = p.qt * a.item_rows, rows = min(p.span.rows - r0, a.item_rows);
    const T* q = static_cast<const T*>(a.q) + p.b * a.q_stride[0] + (long long)p.h * group * a.q_stride[2];
    for (int i = tid; i < rows * chunks; i += kF32Threads) {
      const int row = i / chunks, d = (i - row * chunks) * 4, t = (r0 + row) / group, g = r0 + row - t * group;
      const T* src = q + t * a.q_stride[1] + g * a.q_stride[2] + d;
      float4 x;
      if (vec)
        x = *reinterpret_cast<const float4*>(src);
      else
        x = make_float4(io<T>::to_f(src[0]), io<T>::to_f(src[1]), io<T>::to_f(src[2]), io<T>::to_f(src[3]));
      *reinterpret_cast<float4*>(sm_q + row * kRow + d) = x;
    }
    constexpr int kSub = kKeyTile / kKeys;
    const int steps = (p.i1 - p.i0) * kSub;
    // tile `step`'s keys and values into buffer step & 1; what no row sees becomes zero
    auto load = [&](int step) {
      const int key0 = p.span.tile(p.i0 + step / kSub) * kKeyTile + step % kSub * kKeys, buf = step & 1;
      // a thread keeps one 16-byte chunk of the rows; all its table entries are read before the first copy
      constexpr int kChunks = kDim / 4, kStep = kF32Threads / kChunks, kLoads = kKeys / kStep;
      const int c = tid % kChunks, k0 = tid / kChunks;
      int page[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int j = key0 + k0 + i * kStep;
        page[i] = -1;
        if (j < p.span.hi && (j >= p.span.lo || j < a.sinks))
          page[i] = a.table[(long long)p.b * a.row_pages + (j >> a.page_shift)];
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int k = k0 + i * kStep, j = key0 + k;
        const bool have = page[i] >= 0 && page[i] < a.pages;
        if (c == 0) key_seen[buf][k] = have;
        if (c >= chunks) continue;
        const long long at =
            (((long long)page[i] * a.kv_heads + p.h) * a.page_size + (j & (a.page_size - 1))) * a.dim + c * 4;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          float* dst = (kv ? sm_v : sm_k) + (buf * kKeys + k) * kRow + c * 4;
          const T* src = static_cast<const T*>(a.pool[kv]) + at;
          if (!have) {
            *reinterpret_cast<float4*>(dst) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          } else if constexpr (std::is_same<T, float>::value) {
            cp_async16(dst, src, 16);
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(src);
            const T* x = reinterpret_cast<const T*>(&w);
            *reinterpret_cast<float4*>(dst) =
                make_float4(io<T>::to_f(x[0]), io<T>::to_f(x[1]), io<T>::to_f(x[2]), io<T>::to_f(x[3]));
          }
        }
      }
      cp_async_commit();
    };
    // the thread's rows: what they see
    int hi[kR], lo[kR];
    float m[kR], l[kR], o[kR][4 * kCols];
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int row = kR * ty + i;
      hi[i] = lo[i] = 0;
      if (row < rows) {
        const int pos = p.span.start + (r0 + row) / group;
        hi[i] = a.causal ? min(p.span.hi, pos + 1) : p.span.hi;
        lo[i] = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
      }
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int c = 0; c < 4 * kCols; ++c) o[i][c] = 0.0f;
    }
    const float sl = a.scale * 1.4426950408889634f;
    const bool busy = kR * (tid / 32 * 2) < rows;  // a warp without rows leaves shared memory to the others
    load(0);
    for (int step = 0; step < steps; ++step) {
      if (step + 1 < steps) load(step + 1);
      if (step + 1 < steps)
        cp_async_wait_1();
      else
        cp_async_wait_all();
      __syncthreads();
      const int key0 = p.span.tile(p.i0 + step / kSub) * kKeyTile + step % kSub * kKeys, buf = step & 1;
      const float* ks = sm_k + buf * kKeys * kRow;
      const float* vs = sm_v + buf * kKeys * kRow;
      if (busy) {
        float s[kR][kScores] = {};
#pragma unroll 2
        for (int d = 0; d < a.dim; d += 4) {
          float4 x[kR], y[kScores];
#pragma unroll
          for (int i = 0; i < kR; ++i) x[i] = *reinterpret_cast<const float4*>(sm_q + (kR * ty + i) * kRow + d);
#pragma unroll
          for (int j = 0; j < kScores; ++j) y[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * kRow + d);
#pragma unroll
          for (int i = 0; i < kR; ++i)
#pragma unroll
            for (int j = 0; j < kScores; ++j) {
              s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
              s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
              s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
              s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
            }
        }
        bool whole = true;
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          float top = -INFINITY;
          bool see[kScores];
#pragma unroll
          for (int j = 0; j < kScores; ++j) {
            const int key = key0 + tx + 16 * j;
            see[j] = key < hi[i] && (key >= lo[i] || key < a.sinks) && key_seen[buf][tx + 16 * j];
            whole = whole && see[j];
            s[i][j] = see[j] ? s[i][j] * sl : -INFINITY;
            top = max3_nan(top, s[i][j], s[i][j]);
          }
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) top = max3_nan(top, __shfl_xor_sync(0xffffffffu, top, d), top);
          if (!(top < INFINITY)) l[i] = __int_as_float(0x7fc00000);  // a NaN or +infinity among the scores: the row is NaN
          const float m1 = fmaxf(m[i], top), sub = m1 == -INFINITY ? 0.0f : m1, keep = exp2f(m[i] - sub);
          m[i] = m1;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < kScores; ++j) {
            const float w = see[j] ? exp2f(s[i][j] - sub) : -0.0f;
            sum += w;
            sm_w[(kR * ty + i) * Shape::kWeightRow + tx + 16 * j] = w;
          }
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          l[i] = l[i] * keep + sum;
#pragma unroll
          for (int c = 0; c < 4 * kCols; ++c) o[i][c] *= keep;
        }
        __syncwarp();
        whole = __all_sync(0xffffffffu, whole);
        auto weigh = [&](auto masked) {
#pragma unroll 2
          for (int k = 0; k < kKeys; k += 4) {
            float4 w4[kR];
#pragma unroll
            for (int i = 0; i < kR; ++i)
              w4[i] = *reinterpret_cast<const float4*>(sm_w + (kR * ty + i) * Shape::kWeightRow + k);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float v[4 * kCols];
#pragma unroll
              for (int c = 0; c < kCols; ++c)
                *reinterpret_cast<float4*>(v + 4 * c) =
                    *reinterpret_cast<const float4*>(vs + (k + u) * kRow + 4 * tx + 64 * c);
#pragma unroll
              for (int i = 0; i < kR; ++i) {
                const float w = u == 0 ? w4[i].x : u == 1 ? w4[i].y : u == 2 ? w4[i].z : w4[i].w;
#pragma unroll
                for (int c = 0; c < 4 * kCols; ++c) {
                  if constexpr (decltype(masked)::value)
                    o[i][c] = __float_as_int(w) < 0 ? o[i][c] : fmaf(w, v[c], o[i][c]);
                  else
                    o[i][c] = fmaf(w, v[c], o[i][c]);
                }
              }
            }
          }
        };
        if (whole)
          weigh(std::false_type());
        else
          weigh(std::true_type());
      }
      __syncthreads();  // the buffer is loaded again in the next step
    }
    // the piece's result
    const bool split = p.i0 > 0 || p.i1 < p.span.n;
    const size_t slot = 2 * (size_t)blockIdx.x + (p.i0 == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int row = kR * ty + i, r = r0 + row;
      if (row >= a.item_rows || r >= a.tokens * group) continue;
      const float inv = l[i] == 0.0f || row >= rows ? 0.0f : 1.0f / l[i];
      if (split) {
        float* part = work.o + (slot * kRows + row) * kDim;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          *reinterpret_cast<float4*>(part + 4 * tx + 64 * c) =
              make_float4(o[i][4 * c], o[i][4 * c + 1], o[i][4 * c + 2], o[i][4 * c + 3]);
        if (tx == 0) work.ml[slot * kRows + row] = make_float2(m[i], l[i]);
      } else {
        const int t = r / group, g = r - t * group;
        T* out = static_cast<T*>(a.out) + (((long long)p.b * a.tokens + t) * a.heads + p.h * group + g) * a.dim;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int d = 4 * tx + 64 * c;
          if (d >= a.dim) continue;
#pragma unroll
          for (int u = 0; u < 4; u += 2) store2(out + d + u, o[i][4 * c + u] * inv, o[i][4 * c + u + 1] * inv);
        }
      }
    }
    if (split) {
      __threadfence();
      __syncthreads();
      if (tid == 0) finish_piece(work, cut, p);
      __syncthreads();
      if (cut.join)
        join_pieces<T, kDim, kRows, kF32Threads / 32, (kDim > 128 ? 2 : 4), 3>(
            a, work, JoinItem{p.b, p.qt, p.h, p.span.rows, cut.c0, cut.c1}, tid);
    }
  }
  zero_blind_tiles<T>(a, q_tiles, tid, kF32Threads);
}

}  // namespace dd
