// What the training operators' matrix products share beside the product itself: operands as rows
// of 16-bit terms, the forms of the tiles, and workspaces.
#pragma once
#include "tms_train_gemm.h"
#include "tms_train_rules.h"

namespace tms {

// Between a wave's stores to its own LDS and its lanes' loads of each other's (and back): LDS takes a
// wave's accesses in order, so this costs nothing, but keeps the compiler from moving one across, or
// from taking lanes of a branch through both first.
__device__ __forceinline__ void wave_meets() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

template <int OUT>
__device__ __forceinline__ uint16_t to16(float x) {
  if constexpr (OUT == TMS_DTYPE_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

template <int IN>
__device__ __forceinline__ float from16(uint16_t x) {
  if constexpr (IN == TMS_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, x);
  return __builtin_bit_cast(float, (uint32_t)x << 16);
}

// Eight elements from column c of a row of d as 16-bit terms (three of a float, 16-bit elements as they
// are), zeros behind d; piece k of the output. `whole`: rows of whole 16-byte pieces. Not `on`: zeros.
template <bool F32>
__device__ __forceinline__ void terms_of_eight(const void* src, uint16_t* dst, int64_t k, int64_t row, int c, int32_t d, int64_t plane, bool whole, bool on) {
  const int64_t at = row * d + c;
  if constexpr (F32) {
    float x[8];
    if (whole) {
      const f32x4 lo = ((const f32x4*)((const float*)src + at))[0], hi = ((const f32x4*)((const float*)src + at))[1];
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = on ? lo[e] : 0.f, x[4 + e] = on ? hi[e] : 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = on && c + e < d ? ((const float*)src)[at + e] : 0.f;
    }
#pragma unroll
    for (int p = 0; p < 3; p++) {
      u32x4 out;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const __bf16 t = (__bf16)x[e];
        const uint32_t bits = __builtin_bit_cast(uint16_t, t);
        out[e / 2] = e % 2 ? out[e / 2] | bits << 16 : bits;
        x[e] -= (float)t;
      }
      *(u32x4*)(dst + p * plane + k * 8) = out;
    }
  } else {
    u32x4 out = {0u, 0u, 0u, 0u};
    if (on && whole) {
      out = *(const u32x4*)((const uint16_t*)src + at);
    } else if (on) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (c + e < d) out[e / 2] |= (uint32_t)((const uint16_t*)src)[at + e] << (16 * (e % 2));
    }
    *(u32x4*)(dst + k * 8) = out;
  }
}

// Rows of d elements as rows of dp (a multiple of 8, zeros behind d) of 16-bit terms, eight a thread.
// With `ref`, rows without a gradient become zeros: what stands in them (NaN included) takes no part.
// 8000 rows of 256 floats: 5 us, bound by the launch.
template <bool F32>
__global__ __launch_bounds__(256) void lce_terms_kernel(const void* src, uint16_t* dst, int64_t rows, int32_t d, int32_t dp, int64_t plane,
                                                        const float* ref) {
  const uint32_t eights = (uint32_t)dp / 8;
  const int64_t n = rows * eights;
  const bool whole = d == dp && (uintptr_t)src % 16 == 0;  // pieces of eight in 16-byte loads (d = 0: dp = 8, nothing to load)
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
    const int64_t row = n >> 32 ? k / eights : (int64_t)((uint32_t)k / eights);
    terms_of_eight<F32>(src, dst, k, row, (int)(k - row * eights) * 8, d, plane, whole, !ref || ref[row] != __builtin_inff());
  }
}

static int planes(int dtype) { return dtype == TMS_DTYPE_F32 ? 3 : 1; }
static bool as_is(const void* p, int64_t d, int dtype) { return dtype != TMS_DTYPE_F32 && d % 8 == 0 && (uintptr_t)p % 16 == 0; }
static unsigned blocks_for(int64_t n) { return (unsigned)(n > 256 * 16384 ? 16384 : n > 0 ? (n + 255) / 256 : 1); }

// The tiles' forms: MI and NI of the kernel (two waves along m, four along n).
template <int S>
struct SizeOf {
  static constexpr int MI = S == kGemm256 ? 8 : S == kGemm128 ? 4 : 2, NI = S == kGemm256 ? 4 : S == kGemm128 ? 2 : 1;
};
template <int PL, class F>
static int with_size(int size, F&& f) {
  if constexpr (PL == 1) {
    if (size == kGemm256) return f(SizeOf<kGemm256>());
  }
  if (size == kGemm128) return f(SizeOf<kGemm128>());
  return f(SizeOf<kGemm64>());
}
// Workspaces, as offsets into one buffer.
struct Carve {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t a = at;
    at += up_to(bytes, 256);
    return a;
  }
};
static int run_terms(const void* src, int dtype, void* dst, int64_t rows, int64_t d, int64_t dp, const float* ref, hipStream_t st) {
  const int64_t n = rows * dp;
  const dim3 grid(blocks_for(n / 8));
  if (dtype == TMS_DTYPE_F32)
    hipLaunchKernelGGL(lce_terms_kernel<true>, grid, dim3(256), 0, st, src, (uint16_t*)dst, rows, (int32_t)d, (int32_t)dp, n, ref);
  else
    hipLaunchKernelGGL(lce_terms_kernel<false>, grid, dim3(256), 0, st, src, (uint16_t*)dst, rows, (int32_t)d, (int32_t)dp, n, ref);
  return check_launch("lce_terms_kernel");
}

}  // namespace tms
