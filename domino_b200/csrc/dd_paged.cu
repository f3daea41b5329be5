// dd_paged.cu -- host side of the paged key / value cache: argument checks,
// launches, and the C ABI (dd_pages_*, dd_cache_*) of include/domino_draft.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <type_traits>

#include "../../include/domino_draft.h"
#include "dd_attend.cuh"
#include "dd_attend_f32.cuh"
#include "dd_attend_tc.cuh"
#include "dd_cache_write.cuh"
#include "dd_common.h"
#include "dd_pages.cuh"
#include "dd_ptx.cuh"

using namespace dd;

namespace {

int ceil_div(long long x, long long m) { return (int)((x + m - 1) / m); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

#define DD_TRY(call)                                                                                   \
  do {                                                                                                 \
    cudaError_t e_ = (call);                                                                           \
    if (e_ != cudaSuccess) return global_fail(DD_ECUDA, "%s: %s", #call, cudaGetErrorString(e_));      \
  } while (0)

// Makes the cache's device current for one call and puts the caller's back.
struct DeviceScope {
  int prev = -1;
  bool ok = false, moved = false;
  explicit DeviceScope(int device) {
    ok = cudaGetDevice(&prev) == cudaSuccess;
    if (ok && prev != device) ok = moved = cudaSetDevice(device) == cudaSuccess;
  }
  ~DeviceScope() {
    if (moved) cudaSetDevice(prev);
  }
};

struct DeviceInfo {
  int sms = 0, major = 0;
};
// Properties of a device, read once and kept in one word: another thread sees both or neither.
constexpr int kMaxDevices = 64;
int device_info(int device, DeviceInfo* out) {
  static std::atomic<int> known[kMaxDevices];  // SMs, and the major version above them
  if (device < 0 || device >= kMaxDevices) return global_fail(DD_EINVAL, "device %d", device);
  DeviceInfo d;
  int word = known[device].load(std::memory_order_relaxed);
  if (!word) {
    DD_TRY(cudaDeviceGetAttribute(&d.major, cudaDevAttrComputeCapabilityMajor, device));
    DD_TRY(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device));
    word = d.major << 16 | d.sms;
    known[device].store(word, std::memory_order_relaxed);
  }
  d.major = word >> 16;
  d.sms = word & 0xffff;
  if (d.major != 10) return global_fail(DD_EUNSUPPORTED, "device %d is not sm_100; this library is built for sm_100a", device);
  *out = d;
  return DD_OK;
}

int elem_size(int dtype) { return dtype == DD_F32 ? 4 : 2; }

// Shape checks that need no device.
int check_shape(const dd_paged_cache* c) {
  if (!c) return global_fail(DD_EINVAL, "null cache");
  if (c->layers < 1 || c->batch < 1 || c->kv_heads < 1 || c->pages < 1 || c->row_pages < 1)
    return global_fail(DD_EINVAL, "paged cache: layers, batch, kv_heads, pages and row_pages must be positive");
  if (c->batch > kMaxCacheBatch) return global_fail(DD_EINVAL, "paged cache: batch %d above %d", c->batch, kMaxCacheBatch);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return global_fail(DD_EINVAL, "paged cache: page_size %d is not 16, 32, 64 or 128", c->page_size);
  if (c->head_dim < 8 || c->head_dim % 8 || c->head_dim > kMaxHeadDim)
    return global_fail(DD_EINVAL, "paged cache: head_dim %d is not a multiple of 8 up to %d", c->head_dim, kMaxHeadDim);
  if (c->dtype != DD_BF16 && c->dtype != DD_FP16 && c->dtype != DD_F32)
    return global_fail(DD_EINVAL, "paged cache: dtype must be DD_BF16, DD_FP16 or DD_F32");
  if ((long long)c->pages * c->kv_heads > 0x7fffffffll)
    return global_fail(DD_EINVAL, "paged cache: pages x kv_heads must stay below 2^31");
  if ((long long)c->batch * c->row_pages > 0x7fffffffll)
    return global_fail(DD_EINVAL, "paged cache: batch x row_pages must stay below 2^31");
  if ((long long)c->row_pages * c->page_size > (1ll << 30))
    return global_fail(DD_EINVAL, "paged cache: a row holds at most 2^30 tokens");
  return DD_OK;
}

int check_cache(const dd_paged_cache* c) {
  int rc = check_shape(c);
  if (rc) return rc;
  if (!c->data || !c->table || !c->length || !c->refs || !c->scratch || !c->status)
    return global_fail(DD_EINVAL, "paged cache: null pointer");
  if (!aligned16(c->data) || !aligned16(c->scratch))
    return global_fail(DD_EINVAL, "paged cache: data and scratch must be 16-byte aligned");
  return DD_OK;
}

long long plane_bytes(const dd_paged_cache* c) {
  return (long long)c->pages * c->kv_heads * c->page_size * c->head_dim * elem_size(c->dtype);
}
char* plane(const dd_paged_cache* c, int layer, int kv) {
  return static_cast<char*>(c->data) + (2ll * layer + kv) * plane_bytes(c);
}

// The cache's scratch: counters of dd_cache_attend (zero between calls), the
// page calls' lists, and the attention's pieces.
struct Scratch {
  unsigned* count;
  void* pages;
  float* partial;
  size_t bytes;
};
Scratch scratch_of(const dd_paged_cache* c) {
  const size_t lists = (page_scratch_bytes(c->pages, c->batch, c->row_pages) + 255) / 256 * 256;
  const size_t counters = (kMaxAttendCtas * sizeof(unsigned) + 255) / 256 * 256;
  char* p = static_cast<char*>(c->scratch);
  Scratch s;
  s.count = reinterpret_cast<unsigned*>(p);
  s.pages = p + counters;
  s.partial = reinterpret_cast<float*>(p + counters + lists);
  const int dim = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  s.bytes = counters + lists;
  s.bytes += c->dtype != DD_F32 && c->head_dim <= 128 ? attend_work_bytes(kMaxTensorCtas, 256, dim)
                                                      : attend_work_bytes(kMaxAttendCtas, kF32Rows, dim);
  return s;
}

// Launch with programmatic stream serialisation: the kernel may be scheduled
// while its predecessor drains; every kernel here waits for it first thing.
template <typename... K, typename... A>
int launch(const char* what, void (*kernel)(K...), dim3 grid, dim3 block, size_t smem, void* stream, A... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(args)...);
  if (e != cudaSuccess) return global_fail(DD_ECUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return DD_OK;
}

long long* ll(int64_t* p) { return reinterpret_cast<long long*>(p); }
const long long* ll(const int64_t* p) { return reinterpret_cast<const long long*>(p); }

// The planned moves' pages; with `remap` also the table entries that follow them.
int copy_pages(const dd_paged_cache* c, const PageScratch& s, const DeviceInfo& dev, bool remap, void* stream) {
  const long long words = (long long)c->kv_heads * c->page_size * c->head_dim * elem_size(c->dtype) / 16;
  return launch("page copy", pages_copy_kernel, dim3(dev.sms * 8), dim3(kCopyThreads), 0, stream,
                static_cast<uint4*>(c->data), s, 2 * c->layers, c->pages, words, remap ? c->table : nullptr,
                c->batch * c->row_pages);
}

struct PageCall {
  DeviceInfo dev;
  PageScratch s;
};
int page_call(const dd_paged_cache* c, const void* arg, const char* what, const DeviceScope& scope, PageCall* p) {
  if (!arg) return global_fail(DD_EINVAL, "%s: null argument", what);
  if (!scope.ok) return global_fail(DD_ECUDA, "%s: cannot select device %d", what, c->device);
  p->s = page_scratch(scratch_of(c).pages, c->pages, c->batch);
  return device_info(c->device, &p->dev);
}

template <typename T, int kGroup, bool kVec>
int launch_write(const WriteParams& p, int batch, int tokens_per_cta, bool interleaved, void* stream) {
  const int half = p.rotary / 2;
  const int pairs = interleaved ? 2 : half % 4 == 0 ? 0 : 1;
  size_t smem = sizeof(float) * 2 * tokens_per_cta * ((half + 3) / 4 * 4);
  if (pairs == 1) smem += sizeof(float) * (kWriteThreads / kGroup) * p.dim;
  const dim3 grid(ceil_div(p.tokens, tokens_per_cta), batch);
  auto kernel = pairs == 0   ? cache_write_kernel<T, kGroup, 0, kVec>
                : pairs == 1 ? cache_write_kernel<T, kGroup, 1, kVec>
                             : cache_write_kernel<T, kGroup, 2, kVec>;
  return launch("cache write", kernel, grid, dim3(kWriteThreads), smem, stream, p, tokens_per_cta);
}

template <typename T, bool kVec>
int launch_write(const WriteParams& p, int batch, int tokens_per_cta, bool interleaved, void* stream) {
  const int lanes = p.dim / 8;
  if (lanes <= 4) return launch_write<T, 4, kVec>(p, batch, tokens_per_cta, interleaved, stream);
  if (lanes <= 8) return launch_write<T, 8, kVec>(p, batch, tokens_per_cta, interleaved, stream);
  if (lanes <= 16) return launch_write<T, 16, kVec>(p, batch, tokens_per_cta, interleaved, stream);
  return launch_write<T, 32, kVec>(p, batch, tokens_per_cta, interleaved, stream);
}

template <typename T>
int launch_write(const WriteParams& p, int batch, int tokens_per_cta, bool interleaved, bool vec, void* stream) {
  return vec ? launch_write<T, true>(p, batch, tokens_per_cta, interleaved, stream)
             : launch_write<T, false>(p, batch, tokens_per_cta, interleaved, stream);
}

typedef CUresult (*PFN_encodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
PFN_encodeTiled encoder() {
  static PFN_encodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<PFN_encodeTiled>(p) : nullptr;
  }();
  return fn;
}

// One layer's keys or values as [pages, kv_heads, page_size, head_dim], in
// boxes of one head's page x 64 values with 128-byte swizzle.  Values behind
// head_dim read as zero.
int encode_pool(const dd_paged_cache* c, int layer, int kv, CUtensorMap* m) {
  PFN_encodeTiled encode = encoder();
  if (!encode) return global_fail(DD_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t row = (cuuint64_t)c->head_dim * 2;
  cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
  cuuint64_t strides[3] = {row, row * c->page_size, row * c->page_size * c->kv_heads};
  cuuint32_t box[4] = {64, (cuuint32_t)c->page_size, 1, 1}, one[4] = {1, 1, 1, 1};
  CUresult r = encode(m, c->dtype == DD_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                      plane(c, layer, kv), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return global_fail(DD_ECUDA, "cuTensorMapEncodeTiled (page pool) failed (%d)", (int)r);
  return DD_OK;
}

// The queries as [batch, tokens, heads, head_dim] in boxes of `box` tokens x
// one key head's group of heads x 64 values; false where TMA cannot read them.
bool encode_queries(const dd_paged_cache* c, const dd_cache_attend_args* a, int group, int box, CUtensorMap* m) {
  PFN_encodeTiled encode = encoder();
  if (!encode || box < 1 || group > 128 || !aligned16(a->q)) return false;
  // the stride of a dimension of one is free
  long long st[3] = {a->heads == 1 ? c->head_dim : a->q_stride[2], 0, 0};
  st[1] = a->tokens == 1 ? st[0] * a->heads : a->q_stride[1];
  st[2] = c->batch == 1 ? st[1] * a->tokens : a->q_stride[0];
  for (long long x : st)
    if (x <= 0 || x % 8 || x * 2 >= 1ll << 40) return false;
  cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)a->heads, (cuuint64_t)a->tokens, (cuuint64_t)c->batch};
  cuuint64_t strides[3] = {(cuuint64_t)st[0] * 2, (cuuint64_t)st[1] * 2, (cuuint64_t)st[2] * 2};
  cuuint32_t boxes[4] = {64, (cuuint32_t)group, (cuuint32_t)box, 1}, one[4] = {1, 1, 1, 1};
  return encode(m, c->dtype == DD_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                const_cast<void*>(a->q), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Which kernel serves a call: the tensor cores take 16-bit caches with heads
// of up to 128 values; pairs of query tiles from the second tile on.
struct AttendPlan {
  bool tensor, pair;
  int dim;  // head_dim padded to 64 or 128
};
AttendPlan attend_plan(const dd_paged_cache* c, const dd_cache_attend_args* a) {
  AttendPlan p;
  p.tensor = c->dtype != DD_F32 && c->head_dim <= 128;
  p.dim = c->head_dim <= 64 ? 64 : 128;
  p.pair = (long long)a->tokens * (a->heads / c->kv_heads) > 128;
  return p;
}
template <typename T, int kDim, bool kPair>
int launch_attend(const dd_paged_cache* c, const dd_cache_attend_args* args, AttendParams p, const DeviceInfo& dev,
                  void* stream) {
  CUtensorMap mk, mv, mq{};
  int rc = encode_pool(c, args->layer, 0, &mk);
  if (!rc) rc = encode_pool(c, args->layer, 1, &mv);
  if (rc) return rc;
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[c->device]) {
    DD_TRY(cudaFuncSetAttribute(attend_tc_kernel<T, kDim, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttSmem));
    ready[c->device] = true;
  }
  p.tile_rows = p.group <= 128 ? 128 / p.group * p.group : 128;
  p.item_rows = p.tile_rows * (kPair ? 2 : 1);
  p.q_tma = encode_queries(c, args, p.group, (kPair ? 128 : 128 / p.copies) / p.group, &mq);
  const Scratch scratch = scratch_of(c);
  constexpr int kRows = AttendShape<kDim, kPair>::kRows;
  const int grid = std::min(dev.sms, kMaxTensorCtas);
  AttendWork w;
  w.count = scratch.count;
  w.o = scratch.partial;
  w.ml = reinterpret_cast<float2*>(w.o + (size_t)grid * 2 * kRows * kDim);
  return launch("attend", attend_tc_kernel<T, kDim, kPair>, dim3(grid), dim3(kAttThreads), kAttSmem, stream, mk, mv, mq, p, w);
}
template <typename T, int kDim, int kR>
int launch_attend_f32(const dd_paged_cache* c, AttendParams p, const DeviceInfo& dev, void* stream) {
  using Shape = F32Shape<kDim, kR>;
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[c->device]) {
    DD_TRY(cudaFuncSetAttribute(attend_f32_kernel<T, kDim, kR>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem));
    ready[c->device] = true;
  }
  p.item_rows = p.tile_rows = Shape::kRows;
  // a tile takes longer here: with at least 1 / 2 / 3 of them a CTA 1 x 1 token over 528 keys takes 10.2 / 18.0 / 24.3
  // us, 3 x 16 over 1000 22.4 / 23.9 / 39.6 (16 / 4 heads of 64)
  p.min_tiles = 1;
  // two CTAs fit an SM with heads of up to 64 values
  const int grid = std::min(dev.sms * (kDim <= 64 ? 2 : 1), kMaxAttendCtas);
  const Scratch scratch = scratch_of(c);
  AttendWork w;
  w.count = scratch.count;
  w.o = scratch.partial;
  w.ml = reinterpret_cast<float2*>(w.o + (size_t)grid * 2 * Shape::kRows * kDim);
  return launch("attend", attend_f32_kernel<T, kDim, kR>, dim3(grid), dim3(kF32Threads), Shape::kSmem, stream, p, w);
}
// Rows of a tile: with 64 a call of 3 x 16 tokens over 300-1500 keys (12 items of
// 64 rows) took 29 us, of which a tile's products alone are 9 us on one SM.
template <typename T, int kDim>
int launch_attend_f32(const dd_paged_cache* c, const AttendParams& p, const DeviceInfo& dev, void* stream) {
  const long long rows = (long long)p.tokens * p.group, items = (rows + 63) / 64 * p.batch * p.kv_heads;
  if (rows <= 16) return launch_attend_f32<T, kDim, 1>(c, p, dev, stream);
  if (items < dev.sms) return launch_attend_f32<T, kDim, 2>(c, p, dev, stream);
  return launch_attend_f32<T, kDim, 4>(c, p, dev, stream);
}

template <typename T>
int launch_attend(const dd_paged_cache* c, const dd_cache_attend_args* args, const AttendPlan& plan, const AttendParams& p,
                  const DeviceInfo& dev, void* stream) {
  if (plan.dim == 64)
    return plan.pair ? launch_attend<T, 64, true>(c, args, p, dev, stream)
                     : launch_attend<T, 64, false>(c, args, p, dev, stream);
  return plan.pair ? launch_attend<T, 128, true>(c, args, p, dev, stream)
                   : launch_attend<T, 128, false>(c, args, p, dev, stream);
}

int check_attend(const dd_paged_cache* c, const dd_cache_attend_args* a) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!a) return global_fail(DD_EINVAL, "cache attend: null argument");
  if (a->layer < 0 || a->layer >= c->layers) return global_fail(DD_EINVAL, "cache attend: layer %d of %d", a->layer, c->layers);
  if (a->tokens < 1) return global_fail(DD_EINVAL, "cache attend: %d tokens", a->tokens);
  if (a->heads < 1 || a->heads % c->kv_heads)
    return global_fail(DD_EINVAL, "cache attend: %d query heads for %d key heads", a->heads, c->kv_heads);
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return global_fail(DD_EINVAL, "cache attend: scale must be positive");
  if (a->window < 0 || a->sinks < 0 || (a->window == 0 && a->sinks > 0) || (a->window > 0 && !a->causal))
    return global_fail(DD_EINVAL, "cache attend: a window needs causal attention, sinks need a window");
  if ((long long)a->tokens * (a->heads / c->kv_heads) > (1ll << 29) || (long long)a->heads * c->head_dim > 0x7fffffffll)
    return global_fail(DD_EINVAL, "cache attend: chunk too large");
  // the kernels count key tiles of one row and head, and of one SM's share, in 32 bits
  const double tiles = ((double)c->row_pages * c->page_size / 128 + 2) * c->kv_heads;
  const double entries = (double)c->batch * ((double)a->tokens * (a->heads / c->kv_heads) / 128 + 1);
  if (tiles > 1e9 || entries > 1e9 || tiles * entries > 1e11) return global_fail(DD_EINVAL, "cache attend: chunk too large");
  return DD_OK;
}

}  // namespace

extern "C" {

int dd_cache_scratch(const dd_paged_cache* c, uint64_t* bytes) {
  int rc = check_shape(c);
  if (rc) return rc;
  if (!bytes) return global_fail(DD_EINVAL, "null argument");
  *bytes = scratch_of(c).bytes;
  return DD_OK;
}

int dd_pages_reserve(const dd_paged_cache* c, const int64_t* upto, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  DeviceScope scope(c->device);
  PageCall p;
  if ((rc = page_call(c, upto, "dd_pages_reserve", scope, &p))) return rc;
  rc = launch("reserve", pages_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, stream, c->table, ll(c->length), c->refs,
              p.s, c->status, ll(upto), c->batch, c->pages, c->page_size, c->row_pages);
  return rc ? rc : copy_pages(c, p.s, p.dev, false, stream);
}

int dd_pages_crop(const dd_paged_cache* c, const int64_t* to, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  DeviceScope scope(c->device);
  PageCall p;
  if ((rc = page_call(c, to, "dd_pages_crop", scope, &p))) return rc;
  return launch("crop", pages_crop_kernel, dim3(c->batch), dim3(256), 0, stream, c->table, ll(c->length), c->refs,
                ll(to), c->pages, c->page_size, c->row_pages);
}

int dd_pages_fork(const dd_paged_cache* c, const int64_t* src, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  DeviceScope scope(c->device);
  PageCall p;
  if ((rc = page_call(c, src, "dd_pages_fork", scope, &p))) return rc;
  const int blocks = std::min(ceil_div((long long)c->batch * c->row_pages, 1024), p.dev.sms * 2);
  rc = launch("fork snapshot", pages_snapshot_kernel, dim3(blocks), dim3(256), 0, stream, c->table, ll(c->length), p.s,
              c->batch, c->row_pages);
  if (rc) return rc;
  return launch("fork", pages_fork_kernel, dim3(c->batch), dim3(256), 0, stream, c->table, ll(c->length), c->refs, p.s,
                c->status, ll(src), c->batch, c->pages, c->page_size, c->row_pages);
}

int dd_pages_compact(const dd_paged_cache* c, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  DeviceScope scope(c->device);
  PageCall p;
  if ((rc = page_call(c, c, "dd_pages_compact", scope, &p))) return rc;
  rc = launch("compact", pages_compact_kernel, dim3(1), dim3(kPlanThreads), 0, stream, c->refs, p.s, c->pages);
  return rc ? rc : copy_pages(c, p.s, p.dev, true, stream);
}

int dd_cache_write(const dd_paged_cache* c, const dd_cache_write_args* a, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!a || !a->k || !a->v || !a->start) return global_fail(DD_EINVAL, "dd_cache_write: null argument");
  if (a->layer < 0 || a->layer >= c->layers) return global_fail(DD_EINVAL, "dd_cache_write: layer %d of %d", a->layer, c->layers);
  if (a->tokens < 1) return global_fail(DD_EINVAL, "dd_cache_write: %d tokens", a->tokens);
  if (a->q && (!a->q_out || a->heads < 1)) return global_fail(DD_EINVAL, "dd_cache_write: q needs q_out and heads");
  if (a->q && !aligned16(a->q_out)) return global_fail(DD_EINVAL, "dd_cache_write: q_out must be 16-byte aligned");
  if (a->rotary < 0 || a->rotary % 2 || a->rotary > c->head_dim)
    return global_fail(DD_EINVAL, "dd_cache_write: rotary %d is not an even number up to head_dim %d", a->rotary, c->head_dim);
  if (a->rotary && !a->inv_freq) return global_fail(DD_EINVAL, "dd_cache_write: rotary needs inv_freq");
  if ((long long)(a->heads + 2ll * c->kv_heads) * a->tokens > 0x7fffffffll ||
      (a->q && (long long)a->heads * c->head_dim > 0x7fffffffll))
    return global_fail(DD_EINVAL, "dd_cache_write: chunk too large");
  DeviceScope scope(c->device);
  if (!scope.ok) return global_fail(DD_ECUDA, "dd_cache_write: cannot select device %d", c->device);
  DeviceInfo dev;
  if ((rc = device_info(c->device, &dev))) return rc;
  WriteParams p{};
  const void* x[3] = {a->q, a->k, a->v};
  const int64_t* st[3] = {a->q_stride, a->k_stride, a->v_stride};
  const int per16 = 16 / elem_size(c->dtype);
  bool vec = true;
  for (int i = 0; i < 3; ++i) {
    p.x[i] = x[i];
    if (!x[i]) continue;
    vec = vec && aligned16(x[i]);
    for (int k = 0; k < 3; ++k) {
      p.stride[i][k] = st[i][k];
      vec = vec && st[i][k] % per16 == 0;
    }
    if (std::llabs(st[i][1]) > 0x7fffffffll || std::llabs(st[i][2]) > 0x7fffffffll)
      return global_fail(DD_EINVAL, "dd_cache_write: token and head strides must stay below 2^31 elements");
  }
  const void* norm[2] = {a->q_norm, a->k_norm};
  for (int i = 0; i < 2; ++i) {
    p.norm[i] = norm[i];
    vec = vec && (!norm[i] || aligned16(norm[i]));
    p.pool[i] = plane(c, a->layer, i);
  }
  p.q_out = a->q_out;
  p.table = c->table;
  p.refs = c->refs;
  p.status = c->status;
  p.start = ll(a->start);
  p.lens = ll(a->lens);
  p.inv_freq = a->inv_freq;
  p.eps = a->eps;
  p.factor = a->factor;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = c->kv_heads;
  p.dim = c->head_dim;
  p.rotary = a->rotary;
  p.pages = c->pages;
  p.page_size = c->page_size;
  while (1 << p.page_shift < c->page_size) ++p.page_shift;
  p.row_pages = c->row_pages;
  // One token a CTA while all of them are resident at once (four an SM); beyond
  // that four tokens, whose rounds overlap (2331 tokens x 36 heads: 24 us with
  // one, see dd_cache_write.cuh for large calls).
  const int per_cta = (long long)c->batch * a->tokens > 4ll * dev.sms ? kWriteTokens : 1;
  const bool il = a->interleaved != 0;
  if (c->dtype == DD_F32) return launch_write<float>(p, c->batch, per_cta, il, vec, stream);
  if (c->dtype == DD_FP16) return launch_write<__half>(p, c->batch, per_cta, il, vec, stream);
  return launch_write<__nv_bfloat16>(p, c->batch, per_cta, il, vec, stream);
}

int dd_cache_attend(const dd_paged_cache* c, const dd_cache_attend_args* a, void* stream) {
  int rc = check_attend(c, a);
  if (rc) return rc;
  if (!a->q || !a->out || !a->start) return global_fail(DD_EINVAL, "dd_cache_attend: null argument");
  if (!aligned16(a->out)) return global_fail(DD_EINVAL, "dd_cache_attend: out must be 16-byte aligned");
  DeviceScope scope(c->device);
  if (!scope.ok) return global_fail(DD_ECUDA, "dd_cache_attend: cannot select device %d", c->device);
  DeviceInfo dev;
  if ((rc = device_info(c->device, &dev))) return rc;
  AttendParams p{};
  p.q = a->q;
  p.out = a->out;
  for (int i = 0; i < 3; ++i) p.q_stride[i] = a->q_stride[i];
  for (int i = 0; i < 2; ++i) p.pool[i] = plane(c, a->layer, i);
  p.table = c->table;
  p.start = ll(a->start);
  p.lens = ll(a->lens);
  p.scale = a->scale;
  p.batch = c->batch;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = c->kv_heads;
  p.group = a->heads / c->kv_heads;
  p.dim = c->head_dim;
  p.pages = c->pages;
  p.page_size = c->page_size;
  while (1 << p.page_shift < c->page_size) ++p.page_shift;
  p.row_pages = c->row_pages;
  p.causal = a->causal != 0;
  // nothing is further away than 2^30 positions
  p.window = std::min(a->window, 1 << 30);
  p.sinks = std::min(a->sinks, 1 << 30);
  p.status = c->status;
  const AttendPlan plan = attend_plan(c, a);
  const long long rows = (long long)a->tokens * p.group;
  // Copies of the rows in a tile, so that all softmax warps have work, up to the
  // tile's 128 rows (32 / 8 heads of 128, bf16).  4 rows (1 x 1 token over 528 /
  // 4000 keys): 13.4 / 18.3 us with 4 copies, 13.9 / 18.9 with 2, 15.8 / 20.4
  // with 1; 16 rows (2 x 4 tokens over 2560): 18.8, 19.5, 20.8; 64 rows (2 x 16
  // and 8 x 16 tokens over 2560 and 2048): 21.4 and 26.0 us with 2, 22.5 and 28.9 with 1.
  p.copies = rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
  // What a CTA more brings a small call against one piece more to join.  With at
  // least 1 / 2 / 3 / 5 tiles a CTA 1 x 1 token over 528 keys takes 14.1 / 14.6 /
  // 13.4 / 13.4 us, 2 x 16 tokens over 512 keys 17.2 / 18.1 / 16.4 / 16.5, over
  // 2560 keys 21.0 / 21.0 / 21.4 / 22.0.
  p.min_tiles = 3;
  if (plan.tensor) {
    if (c->dtype == DD_FP16) return launch_attend<__half>(c, a, plan, p, dev, stream);
    return launch_attend<__nv_bfloat16>(c, a, plan, p, dev, stream);
  }
  if (c->dtype == DD_F32)
    return c->head_dim <= 64    ? launch_attend_f32<float, 64>(c, p, dev, stream)
           : c->head_dim <= 128 ? launch_attend_f32<float, 128>(c, p, dev, stream)
                                : launch_attend_f32<float, 256>(c, p, dev, stream);
  if (c->dtype == DD_FP16) return launch_attend_f32<__half, 256>(c, p, dev, stream);
  return launch_attend_f32<__nv_bfloat16, 256>(c, p, dev, stream);
}

}  // extern "C"
