// Global gradient norm over many tensors, and clipping to it.
//
//   norm = sqrt(sum_t sum_i g_t[i]^2)   (or max |g_t[i]|),   c = min(1, max_norm / (norm + 1e-6)),
//   out_t[i] = g_t[i] * c
//
// Bound by memory: the norm reads every gradient once, the clip reads it again and writes
// it. Two kernels: one leaves a partial result per workgroup, the other adds all partials in
// every workgroup (16 KB from L2 at most, and always in the same order, so that every
// workgroup and every run has the same factor) and scales. Neither the norm nor the factor
// goes to the host, so the call can be captured into a graph.
//
// The tensor list goes in the kernel arguments (no copy to the device, nothing to keep alive
// until the stream gets there): kTensors of them a launch, found by bisection over the
// tensors' first chunks, which the scalar unit reads. A workgroup takes whole chunks of
// kChunkElems elements, so that tensors of any size share the chip evenly.
//
// 390 fp32 gradients (336 M elements): the norm 225 us (6.0 TB/s), both 785 us: 4.03 GB at 5.1
// TB/s, where a device copy moves 4.94. 198 bf16 ones into fp32 (109 M): 190 us of kernels, 220
// with the host's work on the list, which bounds that call. Three small ones: 4 + 5 us.
//
// Squares are added in 64 bits: an fp32 gradient's square can neither overflow nor vanish,
// and 10^9 terms lose nothing that 32 bits of the result would show. The vector units have
// an order of magnitude more fp64 FMAs than memory brings elements.
#include <math.h>

#include <algorithm>
#include <memory>
#include <new>

#include "tms_common.h"

namespace tms {

constexpr int kTensors = 112;  // 32 bytes each: 3.6 KB of arguments
constexpr int kClipThreads = 256;
constexpr int kVec = 8;                                 // elements a thread moves at once
constexpr int kChunkElems = kClipThreads * kVec * 8;    // 16,384
constexpr int kPartials = 2048;                         // partial results of a call, over all its launches

struct ClipTensor {
  const void* src;
  void* dst;
  int64_t n;
  int32_t first;  // its first chunk among the launch's
  int32_t types;  // source dtype | destination dtype << 8
};
struct ClipTable {
  ClipTensor t[kTensors];
  int32_t count, chunks;
};

template <int DT>
struct Elem;
template <>
struct Elem<TMS_DTYPE_F32> {
  typedef float T;
};
template <>
struct Elem<TMS_DTYPE_F16> {
  typedef _Float16 T;
};
template <>
struct Elem<TMS_DTYPE_BF16> {
  typedef __bf16 T;
};

// Eight elements at an element's alignment: a gradient may be a view that begins anywhere.
// gfx950 takes 16-byte global accesses at any address, so the type only tells the compiler.
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec8 {
  T v[kVec];
};

__device__ __forceinline__ int find_tensor(const ClipTable& tab, int chunk) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].first <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// f(values, element offset in the chunk, how many of the eight are there) over a chunk.
template <int DT, class F>
__device__ __forceinline__ void each8(const void* src, int64_t begin, int64_t n, F&& f) {
  typedef typename Elem<DT>::T T;
  const T* p = (const T*)src + begin;
  if (n >= kChunkElems) {
    Vec8<T> x[8];
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = *(const Vec8<T>*)(p + (k * kClipThreads + threadIdx.x) * kVec);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      float v[kVec];
#pragma unroll
      for (int i = 0; i < kVec; i++) v[i] = (float)x[k].v[i];
      f(v, (k * kClipThreads + (int)threadIdx.x) * kVec, kVec);
    }
    return;
  }
  for (int at = threadIdx.x * kVec; at < n; at += kClipThreads * kVec) {
    const int here = n - at < kVec ? (int)(n - at) : kVec;
    float v[kVec];
    if (here == kVec) {
      const Vec8<T> x = *(const Vec8<T>*)(p + at);
#pragma unroll
      for (int i = 0; i < kVec; i++) v[i] = (float)x.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < kVec; i++) v[i] = i < here ? (float)p[at + i] : 0.f;
    }
    f(v, at, here);
  }
}

template <class F>
__device__ __forceinline__ void each8_typed(int dt, const void* src, int64_t begin, int64_t n, F&& f) {
  if (dt == TMS_DTYPE_F32) each8<TMS_DTYPE_F32>(src, begin, n, f);
  else if (dt == TMS_DTYPE_F16) each8<TMS_DTYPE_F16>(src, begin, n, f);
  else each8<TMS_DTYPE_BF16>(src, begin, n, f);
}

// |x| as an integer: ordered like the values, with NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// The partials: the sum of squares as a double, or the largest |x|'s bits as an integer.
union Partial {
  double sum;
  uint64_t top;
};

template <bool INF>
__device__ __forceinline__ Partial join(Partial a, Partial b) {
  Partial r;
  if constexpr (INF) r.top = a.top > b.top ? a.top : b.top;
  else r.sum = a.sum + b.sum;
  return r;
}

template <bool INF>
__device__ __forceinline__ Partial block_join(Partial x, Partial* lds) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    Partial y;
    y.top = __shfl_xor((unsigned long long)x.top, o);
    x = join<INF>(x, y);
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = lds[0];
#pragma unroll
  for (int w = 1; w < kClipThreads / 64; w++) x = join<INF>(x, lds[w]);
  return x;
}

template <bool INF>
__global__ __launch_bounds__(kClipThreads) void grad_norm_kernel(ClipTable tab, Partial* partials) {
  __shared__ Partial lds[kClipThreads / 64];
  Partial acc;
  acc.top = 0;  // also +0.0
  for (int c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    const ClipTensor& t = tab.t[find_tensor(tab, c)];
    const int64_t begin = (int64_t)(c - t.first) * kChunkElems;
    each8_typed(t.types & 0xff, t.src, begin, t.n - begin, [&](const float(&v)[kVec], int, int) {
      if constexpr (INF) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kVec; i++) m = abs_bits(v[i]) > m ? abs_bits(v[i]) : m;
        acc.top = m > acc.top ? m : acc.top;
      } else {
#pragma unroll
        for (int i = 0; i < kVec; i++) acc.sum += (double)v[i] * (double)v[i];
      }
    });
  }
  acc = block_join<INF>(acc, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// Every thread gets the norm.
template <bool INF>
__device__ __forceinline__ float whole_norm(const Partial* partials, int n, Partial* lds) {
  Partial acc;
  acc.top = 0;
  for (int i = threadIdx.x; i < n; i += kClipThreads) acc = join<INF>(acc, partials[i]);
  acc = block_join<INF>(acc, lds);
  if constexpr (INF) return __builtin_bit_cast(float, (uint32_t)acc.top);
  return (float)sqrt(acc.sum);
}

template <bool INF>
__global__ __launch_bounds__(kClipThreads) void grad_norm_end_kernel(const Partial* partials, int n, float* norm) {
  __shared__ Partial lds[kClipThreads / 64];
  const float x = whole_norm<INF>(partials, n, lds);
  if (threadIdx.x == 0) *norm = x;
}

template <int DT>
__device__ __forceinline__ void put8(void* dst, int64_t at, const float (&v)[kVec], float c, int here) {
  typedef typename Elem<DT>::T T;
  T* p = (T*)dst + at;
  if (here == kVec) {
    Vec8<T> x;
#pragma unroll
    for (int i = 0; i < kVec; i++) x.v[i] = (T)(v[i] * c);
    *(Vec8<T>*)p = x;
  } else {
#pragma unroll
    for (int i = 0; i < kVec; i++)
      if (i < here) p[i] = (T)(v[i] * c);
  }
}

template <bool INF>
__global__ __launch_bounds__(kClipThreads) void grad_clip_kernel(ClipTable tab, const Partial* partials, int n,
                                                                 float max_norm, float* norm) {
  __shared__ Partial lds[kClipThreads / 64];
  const float x = whole_norm<INF>(partials, n, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm != nullptr) *norm = x;
  float c = max_norm / (x + 1e-6f);
  c = c > 1.f ? 1.f : c;  // a NaN norm gives NaN gradients
  for (int k = blockIdx.x; k < tab.chunks; k += gridDim.x) {
    const ClipTensor& t = tab.t[find_tensor(tab, k)];
    const int dt = t.types & 0xff, to = t.types >> 8;
    if (c == 1.f && t.src == t.dst) continue;  // in place, and nothing to scale
    const int64_t begin = (int64_t)(k - t.first) * kChunkElems;
    void* dst = t.dst;
    each8_typed(dt, t.src, begin, t.n - begin, [&](const float(&v)[kVec], int at, int here) {
      if (to == TMS_DTYPE_F32) put8<TMS_DTYPE_F32>(dst, begin + at, v, c, here);
      else if (to == TMS_DTYPE_F16) put8<TMS_DTYPE_F16>(dst, begin + at, v, c, here);
      else put8<TMS_DTYPE_BF16>(dst, begin + at, v, c, here);
    });
  }
}

static int64_t launches_of(int64_t count) { return count <= 0 ? 0 : (count + kTensors - 1) / kTensors; }
// Workgroups a launch may have, so that a call's partials stay within kPartials (or one a launch).
static int64_t most_groups(int64_t count) {
  const int64_t per = kPartials / launches_of(count);
  return per < 1 ? 1 : per;
}

static bool valid_dtype(int dt) { return dt == TMS_DTYPE_F16 || dt == TMS_DTYPE_BF16 || dt == TMS_DTYPE_F32; }

// The tensors from `i` on that fit one launch; empty ones are left out.
static int64_t fill_table(const tms_grad_tensor* tensors, int64_t count, int64_t i, ClipTable& tab) {
  tab.count = 0;
  int64_t chunks = 0;
  const int64_t end = i + kTensors < count ? i + kTensors : count;
  for (; i < end; i++) {
    const tms_grad_tensor& s = tensors[i];
    if (s.n == 0) continue;
    ClipTensor& t = tab.t[tab.count++];
    t = {s.src, s.dst, s.n, (int32_t)chunks, s.src_dtype | s.dst_dtype << 8};
    chunks += (s.n + kChunkElems - 1) / kChunkElems;
  }
  tab.chunks = (int32_t)chunks;
  return end;
}

static int check_tensors(const char* fn, const tms_grad_tensor* tensors, int64_t count, int norm_type, bool dst) {
  if (count < 0) return fail(TMS_ERR_INVALID, "%s: negative tensor count", fn);
  if (norm_type != TMS_NORM_2 && norm_type != TMS_NORM_INF)
    return fail(TMS_ERR_INVALID, "%s: norm_type must be TMS_NORM_2 or TMS_NORM_INF (got %d)", fn, norm_type);
  if (count > 0 && !tensors) return fail(TMS_ERR_INVALID, "%s: NULL tensor list", fn);
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; i++) {
    const tms_grad_tensor& s = tensors[i];
    if (s.n < 0) return fail(TMS_ERR_INVALID, "%s: tensor %lld has a negative size", fn, (long long)i);
    if (!valid_dtype(s.src_dtype) || (dst && !valid_dtype(s.dst_dtype)))
      return fail(TMS_ERR_UNSUPPORTED, "%s: tensor %lld is not fp16, bf16 or fp32", fn, (long long)i);
    if (s.n > 0 && (!s.src || (dst && !s.dst)))
      return fail(TMS_ERR_INVALID, "%s: tensor %lld is NULL", fn, (long long)i);
    if (i % kTensors == 0) chunks = 0;
    chunks += (s.n + kChunkElems - 1) / kChunkElems;
    if (s.n > ((int64_t)1 << 44) || chunks > 0x7fffffff)
      return fail(TMS_ERR_UNSUPPORTED, "%s: tensor %lld is too large", fn, (long long)i);
  }
  return TMS_OK;
}

static int64_t dtype_size(int dt) { return dt == TMS_DTYPE_F32 ? 4 : 2; }

// Refuses what two workgroups would write, or one write and another read: a tensor that is scaled
// and overlaps another one's memory, or its own source other than as a whole. The written ranges
// and the ones only read, each in order of their addresses (a model's mostly are already), are
// gone through together, each against the range that reaches furthest so far.
static int check_overlap(const char* fn, const tms_grad_tensor* tensors, int64_t count) {
  struct Range {
    uintptr_t begin, end;
    int64_t tensor;
    bool operator<(const Range& o) const { return begin < o.begin; }
  };
  Range few[512];
  std::unique_ptr<Range[]> many;
  Range* written = few;
  if (2 * count > 512) {
    many.reset(new (std::nothrow) Range[2 * (size_t)count]);
    written = many.get();
    if (!written) return fail(TMS_ERR_INVALID, "%s: no memory to look %lld tensors over", fn, (long long)count);
  }
  Range* read = written + count;
  int64_t nw = 0, nr = 0;
  for (int64_t i = 0; i < count; i++) {
    const tms_grad_tensor& s = tensors[i];
    if (s.n == 0) continue;
    const uintptr_t src = (uintptr_t)s.src, dst = (uintptr_t)s.dst;
    written[nw++] = {dst, dst + (uintptr_t)(s.n * dtype_size(s.dst_dtype)), i};
    if (src != dst || s.src_dtype != s.dst_dtype) read[nr++] = {src, src + (uintptr_t)(s.n * dtype_size(s.src_dtype)), i};
  }
  if (!std::is_sorted(written, written + nw)) std::sort(written, written + nw);
  if (!std::is_sorted(read, read + nr)) std::sort(read, read + nr);
  Range far = {}, far_written = {};  // of all, and of those written
  for (int64_t w = 0, r = 0; w < nw || r < nr;) {
    const bool writes = r == nr || (w < nw && written[w].begin <= read[r].begin);
    const Range& x = writes ? written[w++] : read[r++];
    const Range& other = writes ? far : far_written;
    if (x.begin < other.end)
      return fail(TMS_ERR_INVALID, "%s: tensors %lld and %lld overlap, and one of them is written", fn, (long long)other.tensor, (long long)x.tensor);
    if (x.end > far.end) far = x;
    if (writes) far_written = x;  // written ranges that passed do not overlap: the last one reaches furthest
  }
  return TMS_OK;
}

static int norm_partials(const tms_grad_tensor* tensors, int64_t count, int norm_type, Partial* ws, hipStream_t st,
                         int& n) {
  ClipTable tab;
  n = 0;
  const int64_t most = most_groups(count);
  for (int64_t i = 0; i < count;) {
    i = fill_table(tensors, count, i, tab);
    if (tab.chunks == 0) continue;
    const unsigned grid = (unsigned)(tab.chunks < most ? tab.chunks : most);
    if (norm_type == TMS_NORM_INF) hipLaunchKernelGGL(grad_norm_kernel<true>, dim3(grid), dim3(kClipThreads), 0, st, tab, ws + n);
    else hipLaunchKernelGGL(grad_norm_kernel<false>, dim3(grid), dim3(kClipThreads), 0, st, tab, ws + n);
    const int rc = check_launch("grad_norm_kernel");
    if (rc) return rc;
    n += (int)grid;
  }
  return TMS_OK;
}

static int norm_only(const Partial* ws, int n, int norm_type, float* norm, hipStream_t st) {
  if (norm_type == TMS_NORM_INF) hipLaunchKernelGGL(grad_norm_end_kernel<true>, dim3(1), dim3(kClipThreads), 0, st, ws, n, norm);
  else hipLaunchKernelGGL(grad_norm_end_kernel<false>, dim3(1), dim3(kClipThreads), 0, st, ws, n, norm);
  return check_launch("grad_norm_end_kernel");
}

}  // namespace tms

using namespace tms;

extern "C" int64_t tms_grad_workspace_size(int64_t count) {
  const int64_t l = launches_of(count);
  return (l > kPartials ? l : (int64_t)kPartials) * (int64_t)sizeof(Partial);
}

extern "C" int tms_grad_norm(const tms_grad_tensor* tensors, int64_t count, int norm_type, void* workspace,
                             int64_t workspace_bytes, float* norm, void* stream) {
  const char* fn = "tms_grad_norm";
  int rc = check_tensors(fn, tensors, count, norm_type, false);
  if (rc) return rc;
  if (!norm || !workspace || workspace_bytes < tms_grad_workspace_size(count))
    return fail(TMS_ERR_INVALID, "%s: NULL norm, or a workspace below tms_grad_workspace_size", fn);
  int n = 0;
  if ((rc = norm_partials(tensors, count, norm_type, (Partial*)workspace, (hipStream_t)stream, n))) return rc;
  return norm_only((const Partial*)workspace, n, norm_type, norm, (hipStream_t)stream);
}

extern "C" int tms_grad_clip(const tms_grad_tensor* tensors, int64_t count, int norm_type, const double* max_norm,
                             void* workspace, int64_t workspace_bytes, float* norm, void* stream) {
  const char* fn = "tms_grad_clip";
  int rc = check_tensors(fn, tensors, count, norm_type, true);
  if (rc || (rc = check_overlap(fn, tensors, count))) return rc;
  if (!max_norm || !(*max_norm >= 0)) return fail(TMS_ERR_INVALID, "%s: max_norm must be a number of at least 0", fn);
  if (!norm || !workspace || workspace_bytes < tms_grad_workspace_size(count))
    return fail(TMS_ERR_INVALID, "%s: NULL norm, or a workspace below tms_grad_workspace_size", fn);
  const hipStream_t st = (hipStream_t)stream;
  Partial* ws = (Partial*)workspace;
  int n = 0;
  if ((rc = norm_partials(tensors, count, norm_type, ws, st, n))) return rc;
  if (n == 0) return norm_only(ws, 0, norm_type, norm, st);
  ClipTable tab;
  float* to = norm;  // the first launch writes it
  for (int64_t i = 0; i < count;) {
    i = fill_table(tensors, count, i, tab);
    if (tab.chunks == 0) continue;
    const unsigned grid = (unsigned)(tab.chunks < kPartials ? tab.chunks : kPartials);
    if (norm_type == TMS_NORM_INF)
      hipLaunchKernelGGL(grad_clip_kernel<true>, dim3(grid), dim3(kClipThreads), 0, st, tab, ws, n, (float)*max_norm, to);
    else
      hipLaunchKernelGGL(grad_clip_kernel<false>, dim3(grid), dim3(kClipThreads), 0, st, tab, ws, n, (float)*max_norm, to);
    if ((rc = check_launch("grad_clip_kernel"))) return rc;
    to = nullptr;
  }
  return TMS_OK;
}
