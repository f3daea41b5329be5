// dd_cache_write.cuh -- a chunk's queries, keys and values on their way into
// the paged cache: RMS norm of each head, rotary position, one rounding, and
// the store of keys and values into their pages.
//
//   y_i  = x_i / sqrt(mean(x^2) + eps) * w_i
//   pair (a, b) at position p:  (f (y_a c - y_b s), f (y_b c + y_a s)),
//   c, s = cos, sin(p * inv_freq)
//
// The angle of a far position needs more than 24 bits: p * inv_freq is exact
// in fp64 (p below 2^29), is reduced to turns there, and only the fraction
// goes to fp32 for the sine and cosine.  One angle serves every head of a
// token, so the fp64 work is rotary / 2 values per token.
//
// Bound by HBM: q, k, v read once, q_out and the pages written once.  A head
// vector lives in the registers of a group of lanes, 8 values a lane.
#pragma once

#include "../../include/domino_draft.h"
#include "dd_ptx.cuh"

namespace dd {

constexpr int kWriteThreads = 256;
constexpr int kMaxHeadDim = 256;

struct WriteParams {
  const void* x[3];          // q (may be null), k, v
  long long stride[3][3];    // batch, token, head
  void* q_out;
  void* pool[2];             // this layer's keys, values
  const int* table;
  const int* refs;
  unsigned* status;
  const long long* start;
  const long long* lens;     // null: all tokens
  const void* norm[2];       // q, k weights or null
  const float* inv_freq;
  float eps, factor;
  int tokens, heads, kv_heads, dim, rotary, pages, page_size, row_pages;
};

// 8 consecutive values to / from fp32 registers.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (kVec) {
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < (int)sizeof(v) / 16; ++i)
      reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = io<T>::to_f(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = io<T>::to_f(p[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  alignas(16) T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = io<T>::from_f(x[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
}

// kPairs: 0 half layout with rotary / 2 a multiple of 8 (the partner values sit
// in the same registers of another lane), 1 half layout otherwise (partners
// through shared memory), 2 interleaved (partners in the same lane).
template <typename T, int kGroup, int kPairs, bool kVec>
__global__ void __launch_bounds__(kWriteThreads) cache_write_kernel(WriteParams a, int tokens_per_cta) {
  extern __shared__ float sm[];
  const int half = a.rotary / 2;
  float* cs = sm;                            // [tokens_per_cta][half] cos, then sin
  float* sn = sm + tokens_per_cta * half;
  float* stage = sm + 2 * tokens_per_cta * half;  // [groups][dim], kPairs == 1 only
  const int b = blockIdx.y, t0 = blockIdx.x * tokens_per_cta;
  const int n_tok = min(tokens_per_cta, a.tokens - t0);
  pdl_wait_primary();
  const long long start = a.start[b];
  const long long n = a.lens ? a.lens[b] : a.tokens;
  for (int i = threadIdx.x; i < n_tok * half; i += kWriteThreads) {
    const int t = i / half, f = i - t * half;
    double turns = (double)(start + t0 + t) * (double)a.inv_freq[f] * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = c * a.factor;
    sn[i] = s * a.factor;
  }
  __syncthreads();
  constexpr int kGroups = kWriteThreads / kGroup;
  const int lane = threadIdx.x % kGroup, group = threadIdx.x / kGroup;
  const int e0 = lane * 8;
  const bool in = e0 < a.dim;
  const int q_heads = a.x[0] ? a.heads : 0;
  const int all = q_heads + 2 * a.kv_heads;
  // the whole CTA runs the same number of rounds, so that shuffles and
  // __syncwarp see full warps
  for (int u0 = 0; u0 < n_tok * all; u0 += kGroups) {
    const int u = u0 + group;
    const bool work = u < n_tok * all;
    const int tt = work ? u / all : 0, hh = work ? u - tt * all : 0;
    const int t = t0 + tt;
    const int kind = hh < q_heads ? 0 : hh < q_heads + a.kv_heads ? 1 : 2;
    const int h = kind == 0 ? hh : kind == 1 ? hh - q_heads : hh - q_heads - a.kv_heads;
    const bool live = work && t < n;
    float x[8] = {};
    if (live && in)
      load8<T, kVec>(static_cast<const T*>(a.x[kind]) + b * a.stride[kind][0] + t * a.stride[kind][1] +
                         h * a.stride[kind][2] + e0, x);
    const void* w = kind < 2 ? a.norm[kind] : nullptr;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int d = kGroup / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    if (w && in) {
      const float r = 1.0f / sqrtf(ss / a.dim + a.eps);
      float wv[8];
      load8<T, kVec>(static_cast<const T*>(w) + e0, wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wv[i];
    }
    // partner of value e: e + half below half, e - half above it
    float y[8];
    if constexpr (kPairs == 0) {
      const int other = e0 < half ? lane + half / 8 : lane - half / 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], other & (kGroup - 1), kGroup);
    } else if constexpr (kPairs == 1) {
      float* row = stage + group * a.dim;
      __syncwarp();
      if (in)
#pragma unroll
        for (int i = 0; i < 8; ++i) row[e0 + i] = x[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        y[i] = e < a.rotary ? row[e < half ? e + half : e - half] : 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
    }
    if (kind < 2 && in && work) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        if (e >= a.rotary) break;
        const int f = kPairs == 2 ? e >> 1 : e < half ? e : e - half;
        const bool low = kPairs == 2 ? (e & 1) == 0 : e < half;
        const float c = cs[tt * half + f], s = sn[tt * half + f];
        x[i] = low ? x[i] * c - y[i] * s : x[i] * c + y[i] * s;
      }
    }
    if (!work || !in) continue;
    if (kind == 0) {  // rows behind the chunk's end are zeros: x was not loaded
      store8(static_cast<T*>(a.q_out) + (((long long)b * a.tokens + t) * a.heads + h) * a.dim + e0, x);
    } else if (live) {
      const long long p = start + t, slot = p / a.page_size;
      int page = -1;
      if (p >= 0 && slot < a.row_pages) page = a.table[(long long)b * a.row_pages + slot];
      unsigned bad = 0;
      if (page < 0 || page >= a.pages)
        bad = DD_STATUS_NO_PAGE;
      else if (a.refs[page] != 1)
        bad = DD_STATUS_SHARED_PAGE;
      if (bad) {
        if (lane == 0) atomicOr(a.status, bad);
      } else {
        store8(static_cast<T*>(a.pool[kind - 1]) +
                   (((long long)page * a.kv_heads + h) * a.page_size + p % a.page_size) * a.dim + e0, x);
      }
    }
  }
}

}  // namespace dd
