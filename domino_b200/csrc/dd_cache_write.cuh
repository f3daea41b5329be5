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
// vector lives in the registers of a group of lanes, 8 values a lane.  The
// arithmetic comes close to being the bound (it was, at 330 us for 805 MB, with
// one loop over all heads, partners by shuffle and an exact square root).
#pragma once

#include <type_traits>

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
  int tokens, heads, kv_heads, dim, rotary, pages, page_size, page_shift, row_pages;  // page_size = 1 << page_shift
};

// Four consecutive values as they lie in memory.
template <typename T>
struct Raw4 {
  using type = uint2;
};
template <>
struct Raw4<float> {
  using type = uint4;
};
template <typename T, bool kVec>
__device__ __forceinline__ typename Raw4<T>::type load4(const T* p) {
  if constexpr (kVec) {
    return __ldcs(reinterpret_cast<const typename Raw4<T>::type*>(p));
  } else {
    alignas(16) T x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = p[k];
    return *reinterpret_cast<const typename Raw4<T>::type*>(x);
  }
}
template <typename T>
__device__ __forceinline__ void widen4(const typename Raw4<T>::type& r, float* x) {
  const T* v = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = io<T>::to_f(v[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* x) {
  alignas(16) T v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = io<T>::from_f(x[i]);
  *reinterpret_cast<typename Raw4<T>::type*>(p) = *reinterpret_cast<const typename Raw4<T>::type*>(v);
}

constexpr int kWriteTokens = 4;  // most tokens of a CTA
constexpr int kWriteAhead = 3;   // head vectors of a thread on their way (one would leave HBM waiting for requests)

// A lane holds 8 values of a head vector, as two runs of four:
//   kPairs 0 (half layout, rotary / 2 a multiple of 4): the lanes of the turned
//            part hold values 4 l .. and rotary / 2 + 4 l .., so both of a pair
//            are at hand; the lanes behind them 8 values in a row
//   kPairs 1 (half layout, any): 8 in a row, partners through shared memory
//   kPairs 2 (interleaved): 8 in a row, partners side by side
template <typename T, int kGroup, int kPairs, bool kVec>
__global__ void __launch_bounds__(kWriteThreads) cache_write_kernel(const __grid_constant__ WriteParams a,
                                                                    int tokens_per_cta) {
  extern __shared__ __align__(16) float sm[];
  __shared__ long long place[kWriteTokens];  // element of the pool where a token's head 0 goes; -1: nowhere
  const int half = a.rotary / 2;
  const int angle_row = (half + 3) / 4 * 4;
  float* cs = sm;                            // [tokens_per_cta][angle_row] cos, then sin
  float* sn = sm + tokens_per_cta * angle_row;
  float* stage = sm + 2 * tokens_per_cta * angle_row;  // [groups][dim], kPairs == 1 only
  const int b = blockIdx.y, t0 = blockIdx.x * tokens_per_cta;
  const int n_tok = min(tokens_per_cta, a.tokens - t0);
  pdl_wait_primary();
  const long long start = a.start[b];
  const long long n = a.lens ? a.lens[b] : a.tokens;
  const int live = (int)min(max(n - t0, 0ll), (long long)n_tok);  // tokens of this CTA that exist
  constexpr int kGroups = kWriteThreads / kGroup;
  const int lane = threadIdx.x % kGroup, group = threadIdx.x / kGroup;
  const bool in = lane * 8 < a.dim;
  const bool split = kPairs == 0 && lane < half / 4;
  const int e0 = split ? 4 * lane : 8 * lane, e1 = split ? half + 4 * lane : 8 * lane + 4;

  for (int i = threadIdx.x; i < live * half; i += kWriteThreads) {
    const int t = i / half, f = i - t * half;
    double turns = (double)(start + t0 + t) * (double)a.inv_freq[f] * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[t * angle_row + f] = c * a.factor;
    sn[t * angle_row + f] = s * a.factor;
  }
  if ((int)threadIdx.x < live) {
    const long long p = start + t0 + threadIdx.x, slot = p >> a.page_shift;
    long long at = -1;
    int page = -1;
    if (p >= 0 && slot < a.row_pages) page = a.table[(long long)b * a.row_pages + slot];
    if (page < 0 || page >= a.pages)
      atomicOr(a.status, DD_STATUS_NO_PAGE);
    else if (a.refs[page] != 1)
      atomicOr(a.status, DD_STATUS_SHARED_PAGE);
    else
      at = ((long long)page * a.kv_heads * a.page_size + (p & (a.page_size - 1))) * a.dim;
    place[threadIdx.x] = at;
  }
  __syncthreads();

  const int head_words = a.page_size * a.dim;
  const float inv_dim = 1.0f / a.dim;
  // one tensor's head vectors: 0 queries, 1 keys, 2 values
  auto pass = [&](auto which, int heads) {
    constexpr int kKind = decltype(which)::value;
    using Raw = typename Raw4<T>::type;
    const T* src = static_cast<const T*>(a.x[kKind]) + b * a.stride[kKind][0] + t0 * a.stride[kKind][1];
    const int s1 = (int)a.stride[kKind][1], s2 = (int)a.stride[kKind][2];
    const int step_t = kGroups / heads, step_h = kGroups - step_t * heads;
    struct Where {
      int t, h;
    };
    auto step = [&](Where& w) {
      w.t += step_t;
      w.h += step_h;
      if (w.h >= heads) {
        w.h -= heads;
        ++w.t;
      }
    };
    auto fetch = [&](const Where& w, Raw& x0, Raw& x1) {
      x0 = x1 = Raw{};
      if (w.t >= live || !in) return;
      const T* at = src + (long long)w.t * s1 + (long long)w.h * s2;
      x0 = load4<T, kVec>(at + e0);
      x1 = load4<T, kVec>(at + e1);
    };
    float wt[8];
    bool norm = false;
    if constexpr (kKind < 2) {
      norm = a.norm[kKind] != nullptr;
      if (norm && in) {
        widen4<T>(load4<T, kVec>(static_cast<const T*>(a.norm[kKind]) + e0), wt);
        widen4<T>(load4<T, kVec>(static_cast<const T*>(a.norm[kKind]) + e1), wt + 4);
      }
    }
    Where now{group / heads, group % heads}, ahead = now;
    Raw next[kWriteAhead][2];
#pragma unroll
    for (int i = 0; i < kWriteAhead; ++i) {
      fetch(ahead, next[i][0], next[i][1]);
      step(ahead);
    }
    // the whole CTA runs the same number of rounds, so that shuffles and
    // __syncwarp see full warps
    for (int u0 = 0; u0 < live * heads; u0 += kGroups) {
      const Where here = now;
      const Raw x0 = next[0][0], x1 = next[0][1];
#pragma unroll
      for (int i = 1; i < kWriteAhead; ++i) {
        next[i - 1][0] = next[i][0];
        next[i - 1][1] = next[i][1];
      }
      step(now);
      fetch(ahead, next[kWriteAhead - 1][0], next[kWriteAhead - 1][1]);
      step(ahead);
      const bool work = here.t < live && in;
      T* dst;
      bool store = work;
      if constexpr (kKind == 0) {
        dst = static_cast<T*>(a.q_out) + (((long long)b * a.tokens + t0 + here.t) * a.heads + here.h) * a.dim;
      } else {
        const long long at = place[min(here.t, live - 1)];
        store = work && at >= 0;
        dst = static_cast<T*>(a.pool[kKind - 1]) + at + (long long)here.h * head_words;
      }
      if constexpr (kKind == 2) {
        if (store) {
          *reinterpret_cast<Raw*>(dst + e0) = x0;
          *reinterpret_cast<Raw*>(dst + e1) = x1;
        }
        continue;
      }
      float x[8];
      widen4<T>(x0, x);
      widen4<T>(x1, x + 4);
      if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int d = kGroup / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float r = rsqrtf(fmaf(ss, inv_dim, a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= r * wt[i];
      }
      const float* c_row = cs + min(here.t, live - 1) * angle_row;
      const float* s_row = sn + min(here.t, live - 1) * angle_row;
      if constexpr (kPairs == 1) {
        float* row = stage + group * a.dim;
        __syncwarp();
        if (in)
#pragma unroll
          for (int i = 0; i < 8; ++i) row[e0 + i] = x[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = e0 + i, f = e < half ? e : e - half;
          if (!in || e >= a.rotary) break;
          x[i] = e < half ? x[i] * c_row[f] - row[e + half] * s_row[f] : x[i] * c_row[f] + row[e - half] * s_row[f];
        }
      } else if (kPairs == 0 ? split : e0 < a.rotary) {
        const int f = 4 * lane;
        const float4 c4 = *reinterpret_cast<const float4*>(c_row + f), s4 = *reinterpret_cast<const float4*>(s_row + f);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int lo = kPairs == 0 ? i : 2 * i, hi = kPairs == 0 ? 4 + i : 2 * i + 1;
          if (kPairs == 2 && e0 + 2 * i >= a.rotary) break;
          const float u = x[lo], v = x[hi];
          x[lo] = u * c[i] - v * s[i];
          x[hi] = v * c[i] + u * s[i];
        }
      }
      if (store) {
        store4(dst + e0, x);
        store4(dst + e1, x + 4);
      }
    }
  };
  if (live > 0) {
    if (a.x[0]) pass(std::integral_constant<int, 0>(), a.heads);
    pass(std::integral_constant<int, 1>(), a.kv_heads);
    pass(std::integral_constant<int, 2>(), a.kv_heads);
  }
  // query rows behind the chunk's end are zeros
  if (a.x[0]) {
    T* out = static_cast<T*>(a.q_out) + ((long long)b * a.tokens + t0) * a.heads * a.dim;
    const float zero[4] = {};
    const long long token = (long long)a.heads * a.dim / 4;
    for (long long i = live * token + threadIdx.x; i < n_tok * token; i += kWriteThreads)
      store4(out + 4 * i, zero);
  }
}

}  // namespace dd
