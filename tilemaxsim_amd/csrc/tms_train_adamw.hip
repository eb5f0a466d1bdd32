// An AdamW step over many tensors.
//
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// c = min(1, max_norm / (norm + 1e-6)), from a norm in device memory, or 1. t is counted on the device, for each
// tensor, so that a captured step goes on counting. Bound by memory: p, m and v are read and
// written and g read once, and what a 16-bit model reads of p is written in the same pass.
//
// The tensor list goes in the kernel arguments, kAdamTensors of them a launch, and a workgroup takes whole
// chunks of them, as gradient clipping does. A first small kernel counts the
// steps and leaves each tensor's factors, which need powers in 64 bits.
//
// States of all tensors stand in flat buffers, each tensor's at a multiple of 128 elements. In
// 8 bits, 128 elements share the exponent of their largest (its fp32 exponent, one byte); a
// code keeps an element's exponent, as far as it is within 31 octaves of that for v (15 for m, and a sign),
// and three bits below the leading one. Code 0 is zero, 255 (127 and its sign) NaN: a state
// that is no number any more. What the code has no room for is cut off after a number below the
// last bit kept has been added, 16 mixed bits of (step, place): the code is above the value as
// often as the value is above the lower code, so that the mean of what is kept is the value.
// With rounding to nearest a v that shrinks by a thousandth a step would never leave its code, an eighth wide.
// A v below its range is kept as the least code, as it divides; an m below it becomes the least code or zero, likewise in the mean.
//
// m and v are formed with each product and sum rounded by itself, so that they (and with them
// the codes) are the same whatever the compiler joins.
#include <math.h>

#include "tms_common.h"
#include "tms_train_ranges.h"

namespace tms {

constexpr int kAdamTensors = 64;
constexpr int kAdamThreads = 256;
constexpr int kAdamBlock = TMS_ADAMW_BLOCK;  // elements that share an exponent
// Elements a thread takes at once: with fp32 states four, so that a wave's accesses are whole lines (336 M parameters:
// 1,815 us, 5.19 TB/s; with eight, in halves of lines, 1,890); with 8-bit ones eight, which share more of a
// block's work (109 M with bf16 gradients and copies: 380 us, 400 with four).
template <bool SMALL>
constexpr int kAdamVec = SMALL ? 8 : 4;
// Elements that a workgroup takes at a time, or 2,048 where those would be fewer than four workgroups a CU
// (98,432 elements, a projection head: 10 us in chunks of 8,192, 5 in smaller ones).
constexpr int kAdamChunk = 8192, kAdamSmallChunk = 2048;
constexpr int64_t kAdamFewChunks = 1024;

struct AdamTensor {
  void* p;
  const void* g;
  void* copy;
  int64_t n;
  int64_t at;      // its first element in the states
  int32_t first;   // its first chunk among the launch's
  int32_t index;   // its counter
  int32_t types;   // p's dtype | g's << 8 | copy's << 16
};
struct AdamTable {
  AdamTensor t[kAdamTensors];
  int32_t count, chunks, chunk;  // chunk: elements of one
};
static_assert(sizeof(AdamTable) <= 3600, "kernel arguments");

struct AdamFactors {
  float step, root, keep;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr decay
  uint32_t key;            // of t, for the mixed bits
};
struct AdamNumbers {
  double lr, b1, b2, decay;
  const float* lr_at;  // device memory, instead of lr; or NULL
};
struct AdamArgs {
  void *m, *v;
  uint8_t *m_exp, *v_exp;
  const AdamFactors* factors;  // by counter
  const float* norm;           // or NULL
  float max_norm, b1, n1, b2, n2, eps;  // n1 = 1 - b1
};

constexpr int kAdamList = 900;  // counters a launch of the first kernel takes
struct AdamList {
  int32_t index[kAdamList];
  int32_t count;
};

// 32 mixed bits of 32: a xor-shift-multiply hash, with the shifts and constants that C. Wellons found for the least bias
// ("Prospecting for Hash Functions", 2018); every input bit reaches every output bit.
__device__ __forceinline__ uint32_t adam_mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x7feb352du;
  x = (x ^ (x >> 15)) * 0x846ca68bu;
  return x ^ (x >> 16);
}

__device__ __forceinline__ double adam_power(double b, int64_t n) {
  double r = 1;
  for (; n > 0; n >>= 1, b *= b)
    if (n & 1) r *= b;
  return r;
}

__global__ __launch_bounds__(256) void adamw_count_kernel(AdamList list, AdamNumbers a, int64_t* steps, AdamFactors* factors) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (i >= list.count) return;
  const int k = list.index[i];
  const int64_t t = steps[k] + 1;
  steps[k] = t;
  const double lr = a.lr_at ? (double)*a.lr_at : a.lr;
  AdamFactors f;
  f.step = (float)(lr / (1 - adam_power(a.b1, t)));
  f.root = (float)(1 / sqrt(1 - adam_power(a.b2, t)));
  f.keep = (float)(1 - lr * a.decay);
  f.key = (uint32_t)t;
  factors[k] = f;
}

template <int DT>
struct AdamElem {
  typedef float T;
};
template <>
struct AdamElem<TMS_DTYPE_F16> {
  typedef _Float16 T;
};
template <>
struct AdamElem<TMS_DTYPE_BF16> {
  typedef __bf16 T;
};
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) AdamVec {  // N elements at an element's alignment
  T v[N];
};

// N elements (or the `here` first of them) from `at` on.
template <int DT, int N>
__device__ __forceinline__ void adam_get(const void* p, int64_t at, int here, float (&x)[N]) {
  typedef typename AdamElem<DT>::T T;
  const T* from = (const T*)p + at;
  if (here == N) {
    const AdamVec<T, N> v = *(const AdamVec<T, N>*)from;
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = (float)v.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = i < here ? (float)from[i] : 0.f;
  }
}
template <int DT, int N>
__device__ __forceinline__ void adam_put(void* p, int64_t at, int here, const float (&x)[N]) {
  typedef typename AdamElem<DT>::T T;
  T* to = (T*)p + at;
  if (here == N) {
    AdamVec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; i++) v.v[i] = (T)x[i];
    *(AdamVec<T, N>*)to = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < here) to[i] = (T)x[i];
  }
}
template <int N>
__device__ __forceinline__ void adam_get_typed(int dt, const void* p, int64_t at, int here, float (&x)[N]) {
  if (dt == TMS_DTYPE_F32) adam_get<TMS_DTYPE_F32>(p, at, here, x);
  else if (dt == TMS_DTYPE_F16) adam_get<TMS_DTYPE_F16>(p, at, here, x);
  else adam_get<TMS_DTYPE_BF16>(p, at, here, x);
}
template <int N>
__device__ __forceinline__ void adam_put_typed(int dt, void* p, int64_t at, int here, const float (&x)[N]) {
  if (dt == TMS_DTYPE_F32) adam_put<TMS_DTYPE_F32>(p, at, here, x);
  else if (dt == TMS_DTYPE_F16) adam_put<TMS_DTYPE_F16>(p, at, here, x);
  else adam_put<TMS_DTYPE_BF16>(p, at, here, x);
}

// ---------------------------------------------------------------- 8 bits

constexpr int kAdamOctavesM = 14, kAdamOctavesV = 30;  // below the shared exponent's

__device__ __forceinline__ float adam_bits(uint32_t x) { return __builtin_bit_cast(float, x); }

// MAG: the codes of magnitudes, 127 with a sign above them or 255.
template <int MAG>
__device__ __forceinline__ float adam_decode(uint32_t code, int exp) {
  const int base = (exp - (MAG == 127 ? kAdamOctavesM : kAdamOctavesV)) * 8;
  const uint32_t c = code & MAG;
  const int r = (int)c + base;
  uint32_t x = r < 0 ? 0u : (uint32_t)r << 20;
  x = c == 0 ? 0u : c == MAG ? 0x7fc00000u : x;
  if constexpr (MAG == 127) x |= (code & 128u) << 24;
  return adam_bits(x);
}

// `dither`: 16 bits. x's block has the largest finite |x| of exponent `exp`.
template <int MAG>
__device__ __forceinline__ uint32_t adam_encode(float x, int exp, uint32_t dither) {
  const int base = (exp - (MAG == 127 ? kAdamOctavesM : kAdamOctavesV)) * 8;
  const uint32_t bits = __builtin_bit_cast(uint32_t, x), a = bits & 0x7fffffffu;
  int c = (int)((a + (dither << 4)) >> 20) - base;
  if (c < 1) {
    if constexpr (MAG == 127) {
      const float least = adam_bits(base + 1 < 0 ? 0u : (uint32_t)(base + 1) << 20);
      c = adam_bits(a) >= (float)dither / 65536.f * least ? 1 : 0;
    } else {
      c = 1;
    }
  }
  c = a == 0 ? 0 : a >= 0x7f800000u ? MAG : c;
  if constexpr (MAG == 127) c |= (int)(bits >> 24 & 128u);
  return (uint32_t)c;
}

// The exponent of the largest finite |x| of a block: of eight in each of 16 lanes, which all get it.
__device__ __forceinline__ int adam_block_exp(const float (&v)[8]) {
  uint32_t x = 0;
  auto up = [&](uint32_t y) { x = y > x ? y : x; };
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t a = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    up(a < 0x7f800000u ? a : 0u);
  }
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));   // lane ^ 1
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));   // lane ^ 2
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));  // the other quad of each half
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));  // the other half
  return (int)(x >> 23);
}

// The root to 2^-23 of it (the correctly rounded one, and a division in the place of the reciprocal below, would
// take as many instructions as the rest of a step); the instruction takes no subnormal numbers.
__device__ __forceinline__ float adam_root(float x) {
  const bool low = x < 0x1p-96f;
  return __builtin_amdgcn_sqrtf(low ? x * 0x1p64f : x) * (low ? 0x1p-32f : 1.f);
}

// ---------------------------------------------------------------- the step

template <bool SMALL>
__global__ __launch_bounds__(kAdamThreads) void adamw_step_kernel(AdamTable tab, AdamArgs a) {
#pragma clang fp contract(off)
  constexpr int N = kAdamVec<SMALL>;
  float c = 1.f;
  if (a.norm) {
    c = a.max_norm / (*a.norm + 1e-6f);
    c = c > 1.f ? 1.f : c;  // a NaN norm gives NaN parameters
  }
  for (int chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    int lo = 0, hi = tab.count;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tab.t[mid].first <= chunk) lo = mid;
      else hi = mid;
    }
    const AdamTensor& t = tab.t[lo];
    const AdamFactors f = a.factors[t.index];
    const int tp = t.types & 0xff, tg = t.types >> 8 & 0xff, tc = t.types >> 16;
    const int64_t begin = (int64_t)(chunk - t.first) * tab.chunk;
    for (int r = (int)threadIdx.x * N; r < tab.chunk; r += kAdamThreads * N) {
      const int64_t at = begin + r, in = t.at + at;
      const int64_t left = t.n - at;
      // whole blocks of states exist behind a tensor's end: lanes there keep to the exchange below
      if (left + kAdamBlock <= 0) break;
      const int here = left >= N ? N : left > 0 ? (int)left : 0;
      float p[N], g[N], m[N], v[N];
      adam_get_typed(tp, t.p, at, here, p);
      adam_get_typed(tg, t.g, at, here, g);
      if constexpr (SMALL) {
        u32x2 cm = {0u, 0u}, cv = {0u, 0u};
        int em = 0, ev = 0;
        if (here > 0) {
          cm = *(const u32x2*)((const uint8_t*)a.m + in);
          cv = *(const u32x2*)((const uint8_t*)a.v + in);
          em = a.m_exp[in / kAdamBlock];
          ev = a.v_exp[in / kAdamBlock];
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
          m[i] = adam_decode<127>(cm[i / 4] >> (8 * (i % 4)) & 0xffu, em);
          v[i] = adam_decode<255>(cv[i / 4] >> (8 * (i % 4)) & 0xffu, ev);
        }
      } else {
        adam_get<TMS_DTYPE_F32>(a.m, in, here, m);
        adam_get<TMS_DTYPE_F32>(a.v, in, here, v);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float x = g[i] * c;
        m[i] = a.b1 * m[i] + a.n1 * x;
        v[i] = a.b2 * v[i] + a.n2 * x * x;
        p[i] = f.keep * p[i] - f.step * m[i] * __builtin_amdgcn_rcpf(adam_root(v[i]) * f.root + a.eps);
        if (i >= here) m[i] = v[i] = 0.f;
      }
      if (here > 0) {
        adam_put_typed(tp, t.p, at, here, p);
        if (t.copy) adam_put_typed(tc, t.copy, at, here, p);
      }
      if constexpr (SMALL) {
        const int em = adam_block_exp(m), ev = adam_block_exp(v);
        const uint32_t key = adam_mix(f.key + (uint32_t)(in >> 32) * 0x9e3779b1u);
        u32x2 cm = {0u, 0u}, cv = {0u, 0u};
#pragma unroll
        for (int i = 0; i < N; i++) {
          const uint32_t mixed = adam_mix((uint32_t)(in + i) ^ key);
          cm[i / 4] |= adam_encode<127>(m[i], em, mixed & 0xffffu) << (8 * (i % 4));
          cv[i / 4] |= adam_encode<255>(v[i], ev, mixed >> 16) << (8 * (i % 4));
        }
        if (here > 0) {
          *(u32x2*)((uint8_t*)a.m + in) = cm;
          *(u32x2*)((uint8_t*)a.v + in) = cv;
          if ((threadIdx.x & 15) == 0) {
            a.m_exp[in / kAdamBlock] = (uint8_t)em;
            a.v_exp[in / kAdamBlock] = (uint8_t)ev;
          }
        }
      } else if (here > 0) {
        adam_put<TMS_DTYPE_F32>(a.m, in, here, m);
        adam_put<TMS_DTYPE_F32>(a.v, in, here, v);
      }
    }
  }
}

// The numbers that 8-bit states stand for: four a thread, whole lines a store (109 M: 1.09 GB in 172 us, 6.3 TB/s).
__global__ __launch_bounds__(256) void adamw_decode_kernel(const uint8_t* m, const uint8_t* m_exp, const uint8_t* v, const uint8_t* v_exp, int64_t n,
                                                           float* mean, float* square) {
  for (int64_t k = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; k < n; k += (int64_t)gridDim.x * 1024) {
    const uint32_t cm = *(const uint32_t*)(m + k), cv = *(const uint32_t*)(v + k);
    const int em = m_exp[k / kAdamBlock], ev = v_exp[k / kAdamBlock];
    f32x4 x, y;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = adam_decode<127>(cm >> (8 * i) & 0xffu, em);
      y[i] = adam_decode<255>(cv >> (8 * i) & 0xffu, ev);
    }
    *(f32x4*)(mean + k) = x;
    *(f32x4*)(square + k) = y;
  }
}

// ---------------------------------------------------------------- host

static bool adam_dtype(int dt) { return dt == TMS_DTYPE_F16 || dt == TMS_DTYPE_BF16 || dt == TMS_DTYPE_F32; }
static int64_t adam_size(int dt) { return dt == TMS_DTYPE_F32 ? 4 : 2; }

static int check_adamw(const char* fn, const tms_adamw_tensor* tensors, int64_t count, const tms_adamw* s) {
  if (!s) return fail(TMS_ERR_INVALID, "%s: NULL state", fn);
  if (count < 0 || s->size < 0 || s->counters < 0) return fail(TMS_ERR_INVALID, "%s: negative size", fn);
  if (s->bits != 8 && s->bits != 32) return fail(TMS_ERR_UNSUPPORTED, "%s: states of 8 or 32 bits (got %lld)", fn, (long long)s->bits);
  if (!(s->lr >= 0) || !(s->lr < 1e30) || !(s->beta1 >= 0 && s->beta1 < 1) || !(s->beta2 >= 0 && s->beta2 < 1) || !(s->eps >= 0) || !(s->eps < 1e30) ||
      !(s->decay >= 0) || !(s->decay < 1e30))
    return fail(TMS_ERR_INVALID, "%s: lr, eps and decay must be at least 0, betas in [0, 1)", fn);
  if (s->norm && !(s->max_norm >= 0)) return fail(TMS_ERR_INVALID, "%s: max_norm must be a number of at least 0", fn);
  if (count == 0) return TMS_OK;
  if (!tensors || !s->m || !s->v || !s->steps || !s->factors || (s->bits == 8 && (!s->m_exp || !s->v_exp))) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if (((uintptr_t)s->m | (uintptr_t)s->v | (uintptr_t)s->factors) % 16 || (uintptr_t)s->steps % 8)
    return fail(TMS_ERR_INVALID, "%s: states must be 16-byte aligned", fn);
  int64_t chunks = 0, last = -1, end = 0;
  for (int64_t i = 0; i < count; i++) {
    const tms_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.at < 0 || t.index < 0) return fail(TMS_ERR_INVALID, "%s: tensor %lld has a negative size or place", fn, (long long)i);
    if (!adam_dtype(t.p_dtype) || !adam_dtype(t.g_dtype) || (t.copy && !adam_dtype(t.copy_dtype)))
      return fail(TMS_ERR_UNSUPPORTED, "%s: tensor %lld is not fp16, bf16 or fp32", fn, (long long)i);
    if (t.n > 0 && (!t.p || !t.g)) return fail(TMS_ERR_INVALID, "%s: tensor %lld is NULL", fn, (long long)i);
    // ascending places and counters: no two tensors share any
    if (t.at % kAdamBlock || t.at < end || t.n > s->size - t.at || t.index <= last || t.index >= s->counters)
      return fail(TMS_ERR_INVALID, "%s: tensor %lld is not at a place of its own in the states", fn, (long long)i);
    last = t.index;
    end = t.at + (t.n + kAdamBlock - 1) / kAdamBlock * kAdamBlock;
    if (i % kAdamTensors == 0) chunks = 0;
    if (t.n > ((int64_t)1 << 43)) return fail(TMS_ERR_UNSUPPORTED, "%s: tensor %lld is too large", fn, (long long)i);
    chunks += (t.n + kAdamSmallChunk - 1) / kAdamSmallChunk;
    if (chunks > 0x7fffffff) return fail(TMS_ERR_UNSUPPORTED, "%s: tensor %lld is too large", fn, (long long)i);
  }
  if (end > s->size) return fail(TMS_ERR_INVALID, "%s: the last tensor's block of states ends behind them", fn);
  return TMS_OK;
}

}  // namespace tms

using namespace tms;

extern "C" int tms_adamw_step(const tms_adamw_tensor* tensors, int64_t count, const tms_adamw* state, void* stream) {
  const char* fn = "tms_adamw_step";
  int rc = check_adamw(fn, tensors, count, state);
  if (rc || count == 0) return rc;
  RangeList ranges;
  if (!ranges.room(3 * count)) return fail(TMS_ERR_INVALID, "%s: no memory to look %lld tensors over", fn, (long long)count);
  for (int64_t i = 0; i < count; i++) {
    const tms_adamw_tensor& t = tensors[i];
    if (t.n == 0) continue;
    ranges.writes(t.p, t.n * adam_size(t.p_dtype), i);
    if (t.copy) ranges.writes(t.copy, t.n * adam_size(t.copy_dtype), i);
    ranges.reads(t.g, t.n * adam_size(t.g_dtype), i);
  }
  int64_t one, other;
  if (ranges.overlap(one, other))
    return fail(TMS_ERR_INVALID, "%s: tensors %lld and %lld overlap, and one of them is written", fn, (long long)one, (long long)other);
  const hipStream_t st = (hipStream_t)stream;
  const AdamNumbers numbers = {state->lr, state->beta1, state->beta2, state->decay, state->lr_at};
  for (int64_t i = 0; i < count;) {
    AdamList list;
    list.count = 0;
    for (; i < count && list.count < kAdamList; i++) list.index[list.count++] = tensors[i].index;
    hipLaunchKernelGGL(adamw_count_kernel, dim3((unsigned)((list.count + 255) / 256)), dim3(256), 0, st, list, numbers, state->steps,
                       (AdamFactors*)state->factors);
    if ((rc = check_launch("adamw_count_kernel"))) return rc;
  }
  AdamArgs a = {};
  a.m = state->m, a.v = state->v;
  a.m_exp = state->m_exp, a.v_exp = state->v_exp;
  a.factors = (const AdamFactors*)state->factors;
  a.norm = state->norm;
  a.max_norm = (float)state->max_norm;
  a.b1 = (float)state->beta1, a.n1 = (float)(1 - state->beta1);
  a.b2 = (float)state->beta2, a.n2 = (float)(1 - state->beta2);
  a.eps = (float)state->eps;
  int64_t all = 0;
  for (int64_t i = 0; i < count; i++) all += (tensors[i].n + kAdamChunk - 1) / kAdamChunk;
  AdamTable tab;
  tab.chunk = all < kAdamFewChunks ? kAdamSmallChunk : kAdamChunk;
  const int64_t chunk = tab.chunk;
  for (int64_t i = 0; i < count;) {
    tab.count = 0;
    int64_t chunks = 0;
    const int64_t end = i + kAdamTensors < count ? i + kAdamTensors : count;
    for (; i < end; i++) {
      const tms_adamw_tensor& t = tensors[i];
      if (t.n == 0) continue;
      tab.t[tab.count++] = {t.p, t.g, t.copy, t.n, t.at, (int32_t)chunks, t.index, t.p_dtype | t.g_dtype << 8 | t.copy_dtype << 16};
      chunks += (t.n + chunk - 1) / chunk;
    }
    tab.chunks = (int32_t)chunks;
    if (chunks == 0) continue;
    const unsigned grid = (unsigned)(chunks < (1 << 20) ? chunks : (1 << 20));
    if (state->bits == 8) hipLaunchKernelGGL(adamw_step_kernel<true>, dim3(grid), dim3(kAdamThreads), 0, st, tab, a);
    else hipLaunchKernelGGL(adamw_step_kernel<false>, dim3(grid), dim3(kAdamThreads), 0, st, tab, a);
    if ((rc = check_launch("adamw_step_kernel"))) return rc;
  }
  return TMS_OK;
}

extern "C" int tms_adamw_moments(const uint8_t* m, const uint8_t* m_exp, const uint8_t* v, const uint8_t* v_exp, int64_t size, float* mean,
                                 float* square, void* stream) {
  const char* fn = "tms_adamw_moments";
  if (size < 0 || size % kAdamBlock) return fail(TMS_ERR_INVALID, "%s: whole blocks of states (got %lld elements)", fn, (long long)size);
  if (size == 0) return TMS_OK;
  if (!m || !m_exp || !v || !v_exp || !mean || !square) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if (((uintptr_t)m | (uintptr_t)v | (uintptr_t)mean | (uintptr_t)square) % 16) return fail(TMS_ERR_INVALID, "%s: tensors must be 16-byte aligned", fn);
  const int64_t groups = (size / 4 + 255) / 256;
  hipLaunchKernelGGL(adamw_decode_kernel, dim3((unsigned)(groups < (1 << 20) ? groups : (1 << 20))), dim3(256), 0, (hipStream_t)stream, m, m_exp, v, v_exp, size,
                     mean, square);
  return check_launch("adamw_decode_kernel");
}
