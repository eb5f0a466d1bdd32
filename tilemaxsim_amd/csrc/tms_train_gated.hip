// The gated projection of a feed-forward block, both products and what joins them in one kernel:
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// The forward pass is one matrix product whose tiles take 16 rows of Wg and 16 of Wu in turn, so
// that a wave has g and u of the same places in its registers. The backward pass forms them
// again (4 N F d operations, 260 us at 16384 x 1024 x 4096, where keeping them in 16 bits would take 110 of memory's
// time, 4 N F bytes and one rounding more), with an epilogue that leaves dg and du side by side, (N, 2 F), in 16 bits; two more
// products take them to dx (k over both, and over Wg and Wu one behind the other) and to both
// weights' gradients (their rows one behind the other).
//
// Bound by the matrix cores, the tiles' ends behind them. 16,384 tokens, 1024 x 4096, bf16: forward 267 us (1.03 PFLOP/s), dg
// and du 317 (their ends form two functions and write 268 MB), dx 269, both weights' gradients 273 and 14 for
// the join of two splits. 1229 x 768 x 2043, fp16: 19, 23, 17 + 5 and 17 us, where tiles of 128 fill the chip once
// and a quarter, or less than once (two steps a wait).
//
// Few tokens take a kernel of their own: bound by reading the weights once, which needs every CU to have
// some of them on their way.
//
// Precision. g, u, the activation and all sums are fp32; dg and du are rounded to the inputs' type
// between two products (fp32: three bf16 terms, six products of them), as a product of them
// would take them. The gradients then have two roundings, and an error of 1.4 times that of one: on average, but
// in few tokens, where few elements make up the norm, of up to twice. Up to 64 tokens dg and du are therefore
// two 16-bit terms, which the products take as twice as many tokens (a pass of 2 x 384 x 411 in bf16: 19.4 us, 16.5
// with one; 64 x 4096 x 8192: 163, 145). In fp16 a token's are held times a power of two that
// brings a bound of them, from its largest |dh| and the norms of its x and of the weights, to 2^14 to 2^15: a factor beyond
// fp16's range, as u may be where act(g) is small, does not overflow, and a token whose gradients are far below another's (a loss
// that only some tokens reach leaves many such) keeps its digits. dx takes the power out of its rows; the weights'
// gradients, whose sums go over the tokens, take x over it, in fp16 times one power for all: what that loses of a token is
// 2^-38 of the largest bound there is.
#include <math.h>

#include "tms_train_terms.h"

namespace tms {

enum GatedAct { kSilu = TMS_ACT_SILU, kGelu = TMS_ACT_GELU, kGeluTanh = TMS_ACT_GELU_TANH };

// act(g), and with DERIVATIVE its derivative. FINE: for fp32 results.
//   silu: g s(g), s the logistic function;  gelu: g Phi(g), Phi the normal distribution's function;
//   gelu_tanh: g s(2 sqrt(2 / pi) (g + 0.044715 g^3)), as (1 + tanh z) / 2 = s(2 z)
template <int ACT, bool FINE, bool DERIVATIVE>
__device__ __forceinline__ float gated_act(float g, float& slope) {
  if constexpr (ACT == kGelu) {
    const float phi = 0.5f * erfcf(-0.7071067811865476f * g);
    if constexpr (DERIVATIVE) slope = __builtin_fmaf(g, 0.3989422804014327f * expf(-0.5f * g * g), phi);
    return g * phi;
  }
  constexpr float k0 = 1.5957691216057308f, k1 = 0.044715f * 1.5957691216057308f;
  const float z = ACT == kSilu ? g : g * __builtin_fmaf(k1, g * g, k0);
  float s;
  if constexpr (FINE) s = 1.f / (1.f + expf(-z));
  else s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
  const float y = g * s;
  if constexpr (DERIVATIVE) {
    const float dz = ACT == kSilu ? 1.f : __builtin_fmaf(3.f * k1, g * g, k0);
    // s + g s (1 - s) dz; where s is 0 or 1, the second term is 0, also if the square in dz has overflowed
    if constexpr (ACT == kSilu) slope = __builtin_fmaf(y, 1.f - s, s);
    else slope = __builtin_fmaf(s == 0.f || s == 1.f ? 0.f : y * dz, 1.f - s, s);
  }
  return y;
}

template <int A>
struct ActOf {
  static constexpr int value = A;
};
// f of the activation's type: a branch an epilogue, not one an element, whose code (64 times erfc's) would not stay
// in the instruction cache (16384 x 1024 x 4096 forward: 292 us so).
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act == kSilu) f(ActOf<kSilu>());
  else if (act == kGelu) f(ActOf<kGelu>());
  else f(ActOf<kGeluTanh>());
}

// Eight (four) elements at an element's alignment: rows of an odd F begin anywhere.
template <class T, int N, int ALIGN = sizeof(T)>
struct __attribute__((packed, aligned(ALIGN))) GatedVec {
  T v[N];
};

// h, from the sums of 16 rows of Wg and 16 of Wu in turn: whole lines of a token's row, through the wave's LDS.
template <int OUT, int MIV>
struct GatedEpilogue {
  static constexpr int NP = MIV / 2;
  static constexpr int kRowBytes = OUT == TMS_DTYPE_F32 ? 0 : NP * 32 + 16;
  void* out;
  int32_t rows, F, act;

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int, uint8_t* lds) const {
    with_act(act, [&](auto a) { finish<decltype(a)::value>(acc, m, n, lds); });
  }
  template <int ACT, int MI, int NI>
  __device__ __forceinline__ void finish(f32x4 (&acc)[MI][NI], int m, int n, uint8_t* lds) const {
    static_assert(MI == MIV, "rows of the wave's LDS");
    constexpr bool FINE = OUT == TMS_DTYPE_F32;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, f0 = m / 2;
    float none;
#pragma unroll
    for (int j = 0; j < NI; j++) {
      if constexpr (FINE) {
        const int row = n + 16 * j + c;
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const int f = f0 + 16 * p + 4 * g;
          GatedVec<float, 4> y;
#pragma unroll
          for (int e = 0; e < 4; e++) y.v[e] = gated_act<ACT, FINE, false>(acc[2 * p][j][e], none) * acc[2 * p + 1][j][e];
          float* to = (float*)out + (int64_t)row * F + f;
          if (row >= rows) continue;
          if (f + 4 <= F) *(GatedVec<float, 4>*)to = y;
          else
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (f + e < F) to[e] = y.v[e];
        }
      } else {
#pragma unroll
        for (int p = 0; p < NP; p++) {
          uint16_t y[4];
#pragma unroll
          for (int e = 0; e < 4; e++) y[e] = to16<OUT>(gated_act<ACT, FINE, false>(acc[2 * p][j][e], none) * acc[2 * p + 1][j][e]);
          *(u32x2*)(lds + c * kRowBytes + p * 32 + g * 8) = u32x2{(uint32_t)y[0] | (uint32_t)y[1] << 16, (uint32_t)y[2] | (uint32_t)y[3] << 16};
        }
        wave_meets();
        constexpr int PIECES = NP * 2, ROWS = 64 / PIECES;
#pragma unroll
        for (int k = 0; k < (16 + ROWS - 1) / ROWS; k++) {
          const int rr = k * ROWS + lane / PIECES, f = f0 + lane % PIECES * 8, row = n + 16 * j + rr;
          const u32x4 v = *(const u32x4*)(lds + (rr & 15) * kRowBytes + lane % PIECES * 16);
          uint16_t* to = (uint16_t*)out + (int64_t)row * F + f;
          if (rr < 16 && row < rows) {
            if (f + 8 <= F) *(GatedVec<uint32_t, 4, 2>*)to = GatedVec<uint32_t, 4, 2>{{v[0], v[1], v[2], v[3]}};
            else
#pragma unroll
              for (int e = 0; e < 8; e++)
                if (f + e < F) to[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
          }
        }
        wave_meets();
      }
    }
  }
};

// dg and du, [term][token][2 half]: dg in columns from 0, du from half on; zeros from F up to the next
// multiple of 32 (what follows is not read, or not used).
template <int DT, bool F32, int TERMS, int MIV>
struct GatedGradEpilogue {
  static constexpr int NP = MIV / 2;
  static constexpr int kRowBytes = NP * 32 + 16;
  const void* grad;     // (rows, F), of the inputs' type
  uint16_t* P;
  const float* held;  // fp16: what a token's are held times
  int64_t plane;
  int32_t rows, F, half, act;

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int, uint8_t* lds) const {
    with_act(act, [&](auto a) { finish<decltype(a)::value>(acc, m, n, lds); });
  }
  template <int ACT, int MI, int NI>
  __device__ __forceinline__ void finish(f32x4 (&acc)[MI][NI], int m, int n, uint8_t* lds) const {
    static_assert(MI == MIV, "rows of the wave's LDS");
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, f0 = m / 2;
    typedef typename std::conditional<F32, float, uint16_t>::type T;
    // The dh of the next 16 tokens are on their way while these are used: one by one, their latencies would take
    // as long as a third of the product.
    const bool whole = n + 16 * NI <= rows && f0 + 16 * NP <= F;
    auto load = [&](int j, GatedVec<T, 4>(&to)[NP], float& times) {
      const int row = n + 16 * j + c;
      if constexpr (DT == TMS_DTYPE_F16) times = row < rows ? held[row] : 0.f;
      const T* from = (const T*)grad + (int64_t)row * F + f0 + 4 * g;
#pragma unroll
      for (int p = 0; p < NP; p++) {
        if (whole) {
          to[p] = *(const GatedVec<T, 4>*)(from + 16 * p);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) to[p].v[e] = row < rows && f0 + 16 * p + 4 * g + e < F ? from[16 * p + e] : (T)0;
        }
      }
    };
    GatedVec<T, 4> dhs[2][NP];
    float times[2];
    load(0, dhs[0], times[0]);
#pragma unroll
    for (int j = 0; j < NI; j++) {
      if (j + 1 < NI) load(j + 1, dhs[(j + 1) & 1], times[(j + 1) & 1]);
#pragma unroll
      for (int p = 0; p < NP; p++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float d, slope;
          if constexpr (F32) d = dhs[j & 1][p].v[e];
          else d = from16<DT>(dhs[j & 1][p].v[e]);
          if constexpr (DT == TMS_DTYPE_F16) d *= times[j & 1];
          const float y = gated_act<ACT, F32, true>(acc[2 * p][j][e], slope);
          acc[2 * p][j][e] = d * acc[2 * p + 1][j][e] * slope;
          acc[2 * p + 1][j][e] = d * y;
        }
        if (!whole) {  // columns behind F come from some row of the weights
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (f0 + 16 * p + 4 * g + e >= F) acc[2 * p][j][e] = acc[2 * p + 1][j][e] = 0.f;
        }
      }
#pragma unroll
      for (int which = 0; which < 2; which++)
#pragma unroll
        for (int t = 0; t < TERMS; t++) {
#pragma unroll
          for (int p = 0; p < NP; p++) {
            uint16_t b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float x = acc[2 * p + which][j][e];
              b[e] = to16<DT>(x);
              if constexpr (F32) acc[2 * p + which][j][e] = x - from16<DT>(b[e]);
              else if constexpr (TERMS > 1) acc[2 * p + which][j][e] = fabsf(from16<DT>(b[e])) < __builtin_inff() ? x - from16<DT>(b[e]) : 0.f;  // not inf - inf
            }
            *(u32x2*)(lds + c * kRowBytes + p * 32 + g * 8) = u32x2{(uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16};
          }
          wave_meets();
          constexpr int PIECES = NP * 2, ROWS = 64 / PIECES;
#pragma unroll
          for (int k = 0; k < (16 + ROWS - 1) / ROWS; k++) {
            const int rr = k * ROWS + lane / PIECES, f = f0 + lane % PIECES * 8, r = n + 16 * j + rr;
            const u32x4 v = *(const u32x4*)(lds + (rr & 15) * kRowBytes + lane % PIECES * 16);
            if (rr < 16 && r < rows && f < half) *(u32x4*)(P + t * plane + (int64_t)r * (2 * half) + which * half + f) = v;
          }
          wave_meets();
        }
    }
  }
};

// Rows of a gradient, finished: times *factor, or a factor for each row (NULL: 1), in the inputs' type; row n from `half` on
// is row n - half of the second output.
template <int OUT>
struct GatedRowsEpilogue {
  static constexpr int kRowBytes = 0;
  void *out, *out2;
  const float* factor;
  int32_t rows, half, d, each;  // rows: of each output; each: 1 where rows have factors of their own, or 0

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int, uint8_t*) const {
    typedef typename std::conditional<OUT == TMS_DTYPE_F32, float, uint16_t>::type T;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < NI; j++) {
      int row = n + 16 * j + c;
      T* to = (T*)out;
      if (row >= half) to = (T*)out2, row -= half;
      if (row >= rows || to == nullptr) continue;
      const float k = factor ? factor[row * each] : 1.f;
      to += (int64_t)row * d;
#pragma unroll
      for (int i = 0; i < MI; i++) {
        const int col = m + 16 * i + 4 * g;
        GatedVec<T, 4> v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if constexpr (OUT == TMS_DTYPE_F32) v.v[e] = acc[i][j][e] * k;
          else v.v[e] = to16<OUT>(acc[i][j][e] * k);
        }
        if (col + 4 <= d) *(GatedVec<T, 4>*)(to + col) = v;
        else
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (col + e < d) to[col + e] = v.v[e];
      }
    }
  }
};

// The same rows as sums of a part of k, [split][row][dp].
struct GatedSumEpilogue {
  static constexpr int kRowBytes = 0;
  float* out;
  int64_t split;  // elements of one
  int32_t rows, dp;

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int s, uint8_t*) const {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const int row = n + 16 * j + c;
      if (row >= rows) continue;
#pragma unroll
      for (int i = 0; i < MI; i++) {
        const int col = m + 16 * i + 4 * g;
        if (col < dp) *(f32x4*)(out + s * split + (int64_t)row * dp + col) = acc[i][j];
      }
    }
  }
};

// The splits' sums, in order, as GatedRowsEpilogue finishes rows; four elements a thread. Bound by reading them (two
// splits of 8192 x 1024, 67 MB of fp32, to bf16: 14 us).
template <int OUT>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* sums, int splits, int64_t split, int32_t all, int32_t half, int32_t rows, int32_t d,
                                                         int32_t dp, const float* factor, int32_t each, void* out, void* out2) {
  typedef typename std::conditional<OUT == TMS_DTYPE_F32, float, uint16_t>::type T;
  const int quads = (d + 3) / 4;
  const int64_t n = (int64_t)all * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int col = (int)(i - row * quads) * 4;
    const bool second = row >= half;
    const int64_t r = second ? row - half : row;
    T* to = (T*)(second ? out2 : out);
    if (r >= rows || to == nullptr) continue;
    const float k = factor ? factor[r * each] : 1.f;
    const float* from = sums + row * dp + col;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; s += 4) {
      f32x4 y[4];
#pragma unroll
      for (int v = 0; v < 4; v++) y[v] = s + v < splits ? *(const f32x4*)(from + (s + v) * split) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 4; v++)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += y[v][e];
    }
    GatedVec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if constexpr (OUT == TMS_DTYPE_F32) o.v[e] = x[e] * k;
      else o.v[e] = to16<OUT>(x[e] * k);
    }
    to += r * d + col;
    if (col + 4 <= d) *(GatedVec<T, 4>*)to = o;
    else
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (col + e < d) to[e] = o.v[e];
  }
}

// What fp16's dg and du are bounded by: |dg| <= 1.13 |dh| |u|, |du| <= |dh| |g| (no activation is further from 0 than its
// argument, or steeper than 1.13), and |g|, |u| <= |x| |w| for the norms of the token's row and the weight's. A workgroup has
// tokens (`rows`: their largest |dh| times |x|; `parts`: the largest of those times |x| once more), or four rows of weights at a
// time (squares of their norms: `parts` from kBoundTokens on). Infinite and NaN elements of dh, and rows that have any
// elsewhere, are passed over: they make their own rows what they will. 1229 x 768 x 2043: 6.3 us; 16,384 x
// 1024 x 4096: 38, bound by reading them (5.0 TB/s).
constexpr int kBoundTokens = 2048, kBoundWeights = 1024;
constexpr float kBoundSlope = 1.2f;

__device__ __forceinline__ float gated_finite(float x) { return x < __builtin_inff() ? x : 0.f; }  // 0 for NaN, too

// Thread `t` of `all`'s share of a row of n elements: f(bits) for each.
template <class F>
__device__ __forceinline__ void gated_row(const uint16_t* row, int n, int t, int all, F&& f) {
  for (int k = t * 8; k < n; k += all * 8) {
    if (k + 8 <= n) {
      const GatedVec<uint16_t, 8> v = *(const GatedVec<uint16_t, 8>*)(row + k);
#pragma unroll
      for (int e = 0; e < 8; e++) f(v.v[e]);
    } else {
      for (int e = k; e < n; e++) f(row[e]);
    }
  }
}
__device__ __forceinline__ float gated_square_of(const uint16_t* row, int n, int t, int all) {
  float s = 0.f;
  gated_row(row, n, t, all, [&](uint16_t x) {
    const float y = from16<TMS_DTYPE_F16>(x);
    s = __builtin_fmaf(y, y, s);
  });
  return s;
}
__global__ __launch_bounds__(256) void gated_bounds_kernel(const uint16_t* dh, const uint16_t* x, const uint16_t* wg, const uint16_t* wu, int32_t N, int32_t d,
                                                           int32_t F, int32_t tokens, float* parts, float* rows) {
  __shared__ float lds[2][4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  float most = 0.f;
  if ((int)blockIdx.x < tokens) {
    for (int64_t n = blockIdx.x; n < N; n += tokens) {
      uint32_t top = 0;
      gated_row(dh + n * F, F, t, 256, [&](uint16_t y) {
        const uint32_t a = y & 0x7fffu;
        top = a < 0x7c00u && a > top ? a : top;
      });
      float h = from16<TMS_DTYPE_F16>((uint16_t)top), s = gated_square_of(x + n * d, d, t, 256);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        h = fmaxf(h, __shfl_xor(h, o));
        s += __shfl_xor(s, o);
      }
      __syncthreads();  // the last token's have been read
      if (lane == 0) lds[0][wave] = h, lds[1][wave] = s;
      __syncthreads();
      h = fmaxf(fmaxf(lds[0][0], lds[0][1]), fmaxf(lds[0][2], lds[0][3]));
      s = (lds[1][0] + lds[1][1]) + (lds[1][2] + lds[1][3]);
      const float norm = sqrtf(s);
      if (t == 0) rows[n] = h * norm;
      most = fmaxf(most, gated_finite(h * norm * norm));
    }
    if (t == 0) parts[blockIdx.x] = most;
    return;
  }
  for (int64_t r = (int64_t)(blockIdx.x - tokens) * 4 + wave; r < 2 * (int64_t)F; r += (int64_t)(gridDim.x - tokens) * 4) {
    float s = gated_square_of(r < F ? wg + r * d : wu + (r - F) * d, d, lane, 64);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    most = fmaxf(most, gated_finite(s));
  }
  if (lane == 0) lds[0][wave] = most;
  __syncthreads();
  if (t == 0) parts[kBoundTokens + (int)blockIdx.x - tokens] = fmaxf(fmaxf(lds[0][0], lds[0][1]), fmaxf(lds[0][2], lds[0][3]));
}
// The largest of both kinds of parts in all of the workgroup's threads.
__device__ __forceinline__ void gated_largest(const float* parts, int tokens, int weights, float& h, float& w) {
  __shared__ float lds[2][4];
  h = w = 0.f;
#pragma unroll
  for (int k = 0; k < kBoundTokens / 256; k++) {
    const int i = k * 256 + (int)threadIdx.x;
    h = fmaxf(h, i < tokens ? parts[i] : 0.f);
  }
#pragma unroll
  for (int k = 0; k < kBoundWeights / 256; k++) {
    const int i = k * 256 + (int)threadIdx.x;
    w = fmaxf(w, i < weights ? parts[kBoundTokens + i] : 0.f);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    h = fmaxf(h, __shfl_xor(h, o));
    w = fmaxf(w, __shfl_xor(w, o));
  }
  if ((threadIdx.x & 63) == 0) lds[0][threadIdx.x >> 6] = h, lds[1][threadIdx.x >> 6] = w;
  __syncthreads();
  h = fmaxf(fmaxf(lds[0][0], lds[0][1]), fmaxf(lds[0][2], lds[0][3]));
  w = fmaxf(fmaxf(lds[1][0], lds[1][1]), fmaxf(lds[1][2], lds[1][3]));
}
// The exponent of the power of two that brings x > 0 to 2^14 to 2^15: half of fp16's range, so that rounding stays within it.
__device__ __forceinline__ int gated_up(float x) { return 14 + 127 - (int)(__builtin_bit_cast(uint32_t, x) >> 23); }
__device__ __forceinline__ float gated_power(int e) { return e < -126 ? 0.f : __builtin_bit_cast(float, (uint32_t)(127 + (e > 127 ? 127 : e)) << 23); }

// What each token's dg and du are held times, its reciprocal, and x times that reciprocal and a power of two that brings the
// largest bound of that to 2^14 to 2^15 (`xs`, `terms` times one behind the other; *back: what takes the power out again).
// 1229 x 768: 5.1 us, most of them the way of the parts; 16,384 x 1024: 17.
__global__ __launch_bounds__(256) void gated_scale_kernel(const float* parts, int tokens, int weights, const float* rows, const uint16_t* x, int32_t N, int32_t d,
                                                          int32_t dp, int32_t terms, uint16_t* xs, float* held, float* held_back, float* back) {
  float h, w;
  gated_largest(parts, tokens, weights, h, w);
  w = kBoundSlope * sqrtf(w);
  const float all = h * w * 0x1p-14f;  // a token's power takes its bound's exponent from 14
  const int up = all > 0.f ? gated_up(all) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *back = gated_power(-up);
  const int eights = dp / 8;
  const int64_t n = (int64_t)N * eights;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
    const int64_t row = k / eights;
    const int c = (int)(k - row * eights) * 8;
    const float bound = rows[row] * w;
    const bool some = bound > 0.f && bound < __builtin_inff();  // dg and du of others are zeros, or not finite
    const int e = some ? gated_up(bound) : 0;
    const float f = some ? gated_power(up - e) : 1.f;
    if (c == 0) held[row] = gated_power(e), held_back[row] = gated_power(-e);
    const uint16_t* from = x + row * d + c;
    GatedVec<uint16_t, 8> v;
    if (c + 8 <= d) {
      v = *(const GatedVec<uint16_t, 8>*)from;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v.v[i] = c + i < d ? from[i] : (uint16_t)0;
    }
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; i++)
      out[i] = (uint32_t)to16<TMS_DTYPE_F16>(from16<TMS_DTYPE_F16>(v.v[2 * i]) * f) | (uint32_t)to16<TMS_DTYPE_F16>(from16<TMS_DTYPE_F16>(v.v[2 * i + 1]) * f) << 16;
    for (int t = 0; t < terms; t++) *(u32x4*)(xs + ((int64_t)t * N + row) * dp + c) = out;
  }
}

// ---------------------------------------------------------------- few tokens

constexpr int kFewWaves = 8;
constexpr int kFewTokens = 64;  // of a workgroup

// Bound by reading the weights: 16 tokens, 2048 x 5504 in bf16, 13.4 us (3.4 TB/s); 768 x 2048, 4 us, the launch and two
// trips to memory. Eight rows of Wg and eight of Wu are one operand's 16 rows; the waves share k, 32 in turn, and add
// up through LDS. fp32 goes through the fp32 matrix instructions as it is; tokens behind 64 are another row of workgroups.
template <int DT, int NI>
__global__ __launch_bounds__(kFewWaves * 64) void gated_few_kernel(const void* x, int32_t N, int32_t d, const void* wg, const void* wu, int32_t F,
                                                                   int32_t act, int32_t whole, void* out) {
  typedef typename std::conditional<DT == TMS_DTYPE_F32, float, uint16_t>::type T;
  __shared__ f32x4 parts[kFewWaves][NI][64];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int f0 = (int)blockIdx.x * 8, n0 = (int)blockIdx.y * kFewTokens;
  const int fr = f0 + (c & 7) < F ? f0 + (c & 7) : F - 1;
  const T* w = (const T*)(c < 8 ? wg : wu) + (int64_t)fr * d;
  const T* xs[NI];
#pragma unroll
  for (int j = 0; j < NI; j++) xs[j] = (const T*)x + (int64_t)(n0 + 16 * j + c < N ? n0 + 16 * j + c : N - 1) * d;
  f32x4 acc[NI];
#pragma unroll
  for (int j = 0; j < NI; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto eight = [&](const T* p, int k) {  // elements k .. k + 8 of a row, zeros behind its end
    GatedVec<T, 8> v;
    if (whole ? k < d : k + 8 <= d) {
      v = *(const GatedVec<T, 8>*)(p + k);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v.v[e] = k + e < d ? p[k + e] : (T)0;
    }
    return v;
  };
#pragma unroll 4
  for (int k0 = wave * 32; k0 < d; k0 += kFewWaves * 32) {
    const GatedVec<T, 8> a = eight(w, k0 + 8 * g);
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const GatedVec<T, 8> b = eight(xs[j], k0 + 8 * g);
      if constexpr (DT == TMS_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc[j], 0, 0, 0);
      } else {
        acc[j] = mfma16x16x32<DT>(__builtin_bit_cast(u32x4, a), __builtin_bit_cast(u32x4, b), acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NI; j++) parts[wave][j][lane] = acc[j];
  __syncthreads();
  // thread (c, g, j) with g < 2: token 16 j + c, columns f0 + 4 g ..; g from lanes 32 on has u's
  for (int i = threadIdx.x; i < 32 * NI; i += kFewWaves * 64) {
    const int j = i / 32, l = i % 32, row = n0 + 16 * j + (l & 15), f = f0 + 4 * (l >> 4);
    f32x4 gate = {0.f, 0.f, 0.f, 0.f}, up = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kFewWaves; v++) {
      const f32x4 a = parts[v][j][l], b = parts[v][j][l + 32];
#pragma unroll
      for (int e = 0; e < 4; e++) gate[e] += a[e], up[e] += b[e];
    }
    if (row >= N) continue;
    with_act(act, [&](auto a) {
      float none;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float y = gated_act<decltype(a)::value, (DT == TMS_DTYPE_F32), false>(gate[e], none) * up[e];
        if (f + e < F) {
          if constexpr (DT == TMS_DTYPE_F32) ((float*)out)[(int64_t)row * F + f + e] = y;
          else ((uint16_t*)out)[(int64_t)row * F + f + e] = to16<DT>(y);
        }
      }
    });
  }
}

// ---------------------------------------------------------------- host

struct GatedSpace {
  int64_t x, wg, wu, p, sums, bytes;
  int64_t parts, rows, xs, held, held_back, back;  // fp16
  GemmSplit dx, dw;  // how the gradients' products go
  int terms;         // of dg and du, as that many times the tokens
};

// How often x is laid out one behind the other for the weights' product: fp16 has another x for that.
static int gated_laid(const GatedSpace& s, int dtype) { return dtype == TMS_DTYPE_F16 ? 1 : s.terms; }

static GatedSpace gated_space(int64_t N, int64_t d, int64_t F, int dtype, bool backward) {
  GatedSpace s = {};
  Carve c;
  if (!backward && gated_few(N, d, F, dtype == TMS_DTYPE_F32)) return s;
  const int64_t dp = up_to(d, 8);
  s.terms = backward && dtype != TMS_DTYPE_F32 && N <= kFewTokens ? 2 : 1;
  const int laid = gated_laid(s, dtype);
  if (dtype == TMS_DTYPE_F32 || d % 8 || laid > 1) s.x = c.take(N * dp * 2 * planes(dtype) * laid);
  if (dtype == TMS_DTYPE_F32 || d % 8) {
    s.wg = c.take(F * dp * 2 * planes(dtype));
    s.wu = c.take(F * dp * 2 * planes(dtype));
  }
  if (backward) {
    s.p = c.take(N * 2 * up_to(F, 64) * 2 * planes(dtype) * s.terms);
    if (dtype == TMS_DTYPE_F16) {
      s.parts = c.take((kBoundTokens + kBoundWeights) * 4);
      s.rows = c.take(N * 4);
      s.xs = c.take(N * dp * 2 * s.terms);
      s.held = c.take(N * 4);
      s.held_back = c.take(N * 4);
      s.back = c.take(4);
    }
    const int64_t half = up_to(F, 64);
    s.dx = gemm_split(dp, N * s.terms, 2 * half, planes(dtype));
    s.dw = gemm_split(dp, 2 * half, N * s.terms, planes(dtype));
    const int64_t one = s.dx.splits * s.terms > 1 ? s.dx.splits * s.terms * N : 0, other = s.dw.splits > 1 ? s.dw.splits * 2 * half : 0;
    s.sums = c.take((one > other ? one : other) * dp * 4);  // one product after the other
  }
  s.bytes = c.at;
  return s;
}

static int check_gated(const char* fn, const void* x, int64_t N, int64_t d, const void* wg, const void* wu, int64_t F, int dtype, int act, bool backward,
                       const void* ws, int64_t bytes, GatedSpace& s) {
  if (N < 0 || d < 0 || F < 0) return fail(TMS_ERR_INVALID, "%s: negative size", fn);
  if (dtype != TMS_DTYPE_F16 && dtype != TMS_DTYPE_BF16 && dtype != TMS_DTYPE_F32)
    return fail(TMS_ERR_UNSUPPORTED, "%s: dtype must be fp16, bf16 or fp32", fn);
  if (act != TMS_ACT_SILU && act != TMS_ACT_GELU && act != TMS_ACT_GELU_TANH) return fail(TMS_ERR_INVALID, "%s: unknown activation %d", fn, act);
  if (d == 0) return fail(TMS_ERR_INVALID, "%s: rows of no elements", fn);
  // 256 rows of dg and du side by side are less than 2^31 bytes: the product's offsets in a tile have 32 bits
  if (d > 65536 || N > (1 << 24) || F > (1 << 20)) return fail(TMS_ERR_UNSUPPORTED, "%s: sizes up to d = 65536, N = 2^24, F = 2^20", fn);
  if (N == 0 || F == 0) return TMS_OK;
  if (!x || !wg || !wu) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  const uintptr_t all = (uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu;
  if (all % 16) return fail(TMS_ERR_INVALID, "%s: x and the weights must be 16-byte aligned", fn);
  s = gated_space(N, d, F, dtype, backward);
  if (s.bytes > 0 && (!ws || (uintptr_t)ws % 256 || bytes < s.bytes))
    return fail(TMS_ERR_INVALID, "%s: a workspace of %lld bytes is needed, 256-byte aligned", fn, (long long)s.bytes);
  return TMS_OK;
}

// The operands as the products take them.
struct GatedOperands {
  const uint16_t *x, *wg, *wu;
};
// x (twice in a row, where dg and du are two terms) and both weights as rows of terms, in one launch.
struct GatedTerms {
  const void* src[4];
  uint16_t* dst[4];
  int64_t rows[4];
};
template <bool F32>
__global__ __launch_bounds__(256) void gated_terms_kernel(GatedTerms t, int32_t d, int32_t dp) {
  const int which = blockIdx.y;
  const bool whole = d == dp && (uintptr_t)t.src[which] % 16 == 0;
  const int eights = dp / 8;
  const int64_t n = t.rows[which] * eights;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
    const int64_t row = k / eights;
    terms_of_eight<F32>(t.src[which], t.dst[which], k, row, (int)(k - row * eights) * 8, d, t.rows[which] * dp, whole, true);
  }
}
static int gated_operands(const void* x, int64_t N, int64_t d, const void* wg, const void* wu, int64_t F, int dtype, uint8_t* ws, const GatedSpace& s,
                          GatedOperands& o, hipStream_t st) {
  o = {(const uint16_t*)x, (const uint16_t*)wg, (const uint16_t*)wu};
  const bool all = dtype == TMS_DTYPE_F32 || d % 8;
  const int laid = gated_laid(s, dtype);
  if (!all && laid <= 1) return TMS_OK;
  const int64_t dp = up_to(d, 8);
  uint16_t *px = (uint16_t*)(ws + s.x), *pg = (uint16_t*)(ws + s.wg), *pu = (uint16_t*)(ws + s.wu);
  GatedTerms t = {};
  unsigned n = 0;
  auto lay = [&](const void* src, uint16_t* dst, int64_t rows) {
    t.src[n] = src, t.dst[n] = dst, t.rows[n] = rows;
    n++;
  };
  lay(x, px, N);
  if (laid > 1) lay(x, px + N * dp, N);
  o.x = px;
  if (all) {
    lay(wg, pg, F);
    lay(wu, pu, F);
    o.wg = pg, o.wu = pu;
  }
  const dim3 grid(blocks_for((all && F > N ? F : N) * dp / 8), n);
  if (dtype == TMS_DTYPE_F32) hipLaunchKernelGGL(gated_terms_kernel<true>, grid, dim3(256), 0, st, t, (int32_t)d, (int32_t)dp);
  else hipLaunchKernelGGL(gated_terms_kernel<false>, grid, dim3(256), 0, st, t, (int32_t)d, (int32_t)dp);
  return check_launch("gated_terms_kernel");
}

// g and u: m over rows of Wg and Wu in turn, n over tokens.
static GemmArgs gated_args(const GatedOperands& o, int64_t N, int64_t F, int64_t dp) {
  GemmArgs a = {};
  a.A = o.wg;
  a.A2 = o.wu;
  a.B = o.x;
  a.aplane = F * dp;
  a.bplane = N * dp;
  a.lda = a.ldb = (int32_t)dp;
  a.M = (int32_t)(2 * F);
  a.N = (int32_t)N;
  a.K = (int32_t)dp;
  a.splits = 1;
  return a;
}

template <int DT>
static int gated_few_rows(const void* x, int64_t N, int64_t d, const void* wg, const void* wu, int64_t F, int act, void* h, hipStream_t st) {
  const dim3 grid((unsigned)((F + 7) / 8), (unsigned)((N + kFewTokens - 1) / kFewTokens)), threads(kFewWaves * 64);
  const int whole = d % 8 == 0;
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, threads, 0, st, x, (int32_t)N, (int32_t)d, wg, wu, (int32_t)F, (int32_t)act, whole, h); };
  if (N <= 16) go(gated_few_kernel<DT, 1>);
  else if (N <= 32) go(gated_few_kernel<DT, 2>);
  else go(gated_few_kernel<DT, 4>);
  return check_launch("gated_few_kernel");
}

// A product with the tiles of `size`; epi(SizeOf) is its epilogue.
template <int DT, int PL, bool AO, bool BO, int PAIR, class F>
static int gated_product(const GemmArgs& a, int size, F&& epi, const char* what, hipStream_t st) {
  return with_size<PL>(size, [&](auto z) {
    using Z = decltype(z);
    if constexpr (PL == 1 && Z::MI < 8) {
      if (product_deep(size, a.M, a.N, a.splits)) return run_gemm<DT, PL, Z::MI, Z::NI, AO, BO, PAIR, true>(a, epi(z), st, what);
    }
    return run_gemm<DT, PL, Z::MI, Z::NI, AO, BO, PAIR>(a, epi(z), st, what);
  });
}

template <int DT, int PL, int OUT>
static int gated_forward(const void* x, int64_t N, int64_t d, const void* wg, const void* wu, int64_t F, int dtype, int act, uint8_t* ws, const GatedSpace& s,
                         void* h, hipStream_t st) {
  if (gated_few(N, d, F, dtype == TMS_DTYPE_F32)) return gated_few_rows<OUT>(x, N, d, wg, wu, F, act, h, st);
  GatedOperands o;
  int rc = gated_operands(x, N, d, wg, wu, F, dtype, ws, s, o, st);
  if (rc) return rc;
  const int64_t dp = up_to(d, 8);
  const GemmArgs a = gated_args(o, N, F, dp);
  auto epi = [&](auto z) { return GatedEpilogue<OUT, decltype(z)::MI>{h, (int32_t)N, (int32_t)F, (int32_t)act}; };
  return gated_product<DT, PL, false, false, kPairRows>(a, product_size(2 * F, N, dp, PL), epi, "train_gemm_kernel (gated)", st);
}

// A product to rows of d elements, at once or in splits; with terms > 1, of so many times `all` rows, summed.
template <int DT, int PL, int OUT, bool BO, int PAIR>
static int gated_rows(GemmArgs b, GemmSplit plan, int terms, int64_t all, int64_t half, int64_t rows, int64_t d, int64_t dp, const float* factor, int each, float* sums,
                      void* out, void* out2, const char* what, hipStream_t st) {
  b.splits = plan.splits;
  if (plan.splits * terms == 1) {
    const GatedRowsEpilogue<OUT> e = {out, out2, factor, (int32_t)rows, (int32_t)half, (int32_t)d, (int32_t)each};
    return gated_product<DT, PL, true, BO, PAIR>(b, plan.size, [&](auto) { return e; }, what, st);
  }
  const GatedSumEpilogue e = {sums, terms * all * dp, (int32_t)(terms * all), (int32_t)dp};
  const int rc = gated_product<DT, PL, true, BO, PAIR>(b, plan.size, [&](auto) { return e; }, what, st);
  if (rc) return rc;
  hipLaunchKernelGGL(gated_join_kernel<OUT>, dim3(blocks_for(all * ((d + 3) / 4))), dim3(256), 0, st, sums, plan.splits * terms, all * dp, (int32_t)all,
                     (int32_t)half, (int32_t)rows, (int32_t)d, (int32_t)dp, factor, (int32_t)each, out, out2);
  return check_launch("gated_join_kernel");
}

template <int DT, int PL, int OUT>
static int gated_backward(const void* x, int64_t N, int64_t d, const void* wg, const void* wu, int64_t F, int dtype, int act, const void* grad, uint8_t* ws,
                          const GatedSpace& s, void* dx, void* dwg, void* dwu, hipStream_t st) {
  GatedOperands o;
  int rc = gated_operands(x, N, d, wg, wu, F, dtype, ws, s, o, st);
  if (rc) return rc;
  const int64_t dp = up_to(d, 8), half = up_to(F, 64), plane = N * 2 * half;
  uint16_t* P = (uint16_t*)(ws + s.p);
  const float *held = nullptr, *held_back = nullptr, *back = nullptr;
  const uint16_t* xs = o.x;
  if (DT == TMS_DTYPE_F16) {
    const int tokens = (int)(N < kBoundTokens ? N : kBoundTokens), rows = (int)((2 * F + 3) / 4), weights = rows < kBoundWeights ? rows : kBoundWeights;
    float* parts = (float*)(ws + s.parts);
    hipLaunchKernelGGL(gated_bounds_kernel, dim3((unsigned)(tokens + weights)), dim3(256), 0, st, (const uint16_t*)grad, (const uint16_t*)x, (const uint16_t*)wg,
                       (const uint16_t*)wu, (int32_t)N, (int32_t)d, (int32_t)F, tokens, parts, (float*)(ws + s.rows));
    if ((rc = check_launch("gated_bounds_kernel"))) return rc;
    const int64_t groups = (N * dp / 8 + 255) / 256;
    hipLaunchKernelGGL(gated_scale_kernel, dim3((unsigned)(groups < 2048 ? groups : 2048)), dim3(256), 0, st, (const float*)parts, tokens, weights,
                       (const float*)(ws + s.rows), (const uint16_t*)x, (int32_t)N, (int32_t)d, (int32_t)dp, (int32_t)s.terms, (uint16_t*)(ws + s.xs),
                       (float*)(ws + s.held), (float*)(ws + s.held_back), (float*)(ws + s.back));
    if ((rc = check_launch("gated_scale_kernel"))) return rc;
    held = (const float*)(ws + s.held), held_back = (const float*)(ws + s.held_back), back = (const float*)(ws + s.back);
    xs = (const uint16_t*)(ws + s.xs);
  }
  const GemmArgs a = gated_args(o, N, F, dp);
  auto form = [&](auto terms) {
    auto epi = [&](auto z) {
      return GatedGradEpilogue<DT, (PL > 1), decltype(terms)::value, decltype(z)::MI>{grad, P, held, plane, (int32_t)N, (int32_t)F, (int32_t)half, (int32_t)act};
    };
    return gated_product<DT, PL, false, false, kPairRows>(a, product_size(2 * F, N, dp, PL), epi, "train_gemm_kernel (dg, du)", st);
  };
  if (PL == 1 && s.terms > 1) rc = form(std::integral_constant<int, PL == 1 ? 2 : PL>());
  else rc = form(std::integral_constant<int, PL>());
  if (rc) return rc;
  if (dx) {  // m over d, n over tokens, k over F columns of dg and du and the rows of Wg and Wu
    GemmArgs b = {};
    b.A = o.wg;
    b.A2 = o.wu;
    b.B = P;
    b.aplane = F * dp;
    b.bplane = plane;
    b.lda = (int32_t)dp;
    b.ldb = b.K = (int32_t)(2 * half);
    b.M = (int32_t)dp;
    b.N = (int32_t)(N * s.terms);
    b.half = (int32_t)half;
    b.real = (int32_t)F;
    rc = gated_rows<DT, PL, OUT, false, kPairDepth>(b, s.dx, s.terms, N, 0x7fffffff, N, d, dp, held_back, 1, (float*)(ws + s.sums), dx, nullptr,
                                               "train_gemm_kernel (dx)", st);
    if (rc) return rc;
  }
  if (dwg || dwu) {  // m over d, n over F columns of dg and du, k over tokens
    GemmArgs b = {};
    b.A = xs;
    b.B = P;
    b.aplane = N * dp;
    b.bplane = plane;
    b.lda = (int32_t)dp;
    b.ldb = b.N = (int32_t)(2 * half);
    b.M = (int32_t)dp;
    b.K = (int32_t)(N * s.terms);
    rc = gated_rows<DT, PL, OUT, true, kSingle>(b, s.dw, 1, 2 * half, half, F, d, dp, back, 0, (float*)(ws + s.sums), dwg, dwu,
                                            "train_gemm_kernel (dWg, dWu)", st);
  }
  return rc;
}

}  // namespace tms

using namespace tms;

extern "C" int64_t tms_gated_workspace_size(int64_t N, int64_t d, int64_t F, int dtype, int backward) {
  if (N <= 0 || d <= 0 || F <= 0) return 0;
  return gated_space(N, d, F, dtype, backward != 0).bytes;
}

extern "C" int tms_gated_linear(const void* x, int64_t N, int64_t d, const void* w_gate, const void* w_up, int64_t F, int dtype, int activation,
                                void* workspace, int64_t workspace_bytes, void* h, void* stream) {
  const char* fn = "tms_gated_linear";
  GatedSpace s = {};
  const int rc = check_gated(fn, x, N, d, w_gate, w_up, F, dtype, activation, false, workspace, workspace_bytes, s);
  if (rc || N == 0 || F == 0) return rc;
  if (!h) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if ((uintptr_t)h % 16) return fail(TMS_ERR_INVALID, "%s: h must be 16-byte aligned", fn);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  if (dtype == TMS_DTYPE_F16) return gated_forward<TMS_DTYPE_F16, 1, TMS_DTYPE_F16>(x, N, d, w_gate, w_up, F, dtype, activation, ws, s, h, st);
  if (dtype == TMS_DTYPE_BF16) return gated_forward<TMS_DTYPE_BF16, 1, TMS_DTYPE_BF16>(x, N, d, w_gate, w_up, F, dtype, activation, ws, s, h, st);
  return gated_forward<TMS_DTYPE_BF16, 3, TMS_DTYPE_F32>(x, N, d, w_gate, w_up, F, dtype, activation, ws, s, h, st);
}

extern "C" int tms_gated_linear_grad(const void* x, int64_t N, int64_t d, const void* w_gate, const void* w_up, int64_t F, int dtype, int activation,
                                     const void* grad, void* workspace, int64_t workspace_bytes, void* dx, void* dw_gate, void* dw_up, void* stream) {
  const char* fn = "tms_gated_linear_grad";
  GatedSpace s = {};
  const int rc = check_gated(fn, x, N, d, w_gate, w_up, F, dtype, activation, true, workspace, workspace_bytes, s);
  if (rc || N == 0 || F == 0 || (!dx && !dw_gate && !dw_up)) return rc;  // no rows or columns: the caller's zeros
  if (!grad) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if (((uintptr_t)grad | (uintptr_t)dx | (uintptr_t)dw_gate | (uintptr_t)dw_up) % 16) return fail(TMS_ERR_INVALID, "%s: tensors must be 16-byte aligned", fn);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  if (dtype == TMS_DTYPE_F16)
    return gated_backward<TMS_DTYPE_F16, 1, TMS_DTYPE_F16>(x, N, d, w_gate, w_up, F, dtype, activation, grad, ws, s, dx, dw_gate, dw_up, st);
  if (dtype == TMS_DTYPE_BF16)
    return gated_backward<TMS_DTYPE_BF16, 1, TMS_DTYPE_BF16>(x, N, d, w_gate, w_up, F, dtype, activation, grad, ws, s, dx, dw_gate, dw_up, st);
  return gated_backward<TMS_DTYPE_BF16, 3, TMS_DTYPE_F32>(x, N, d, w_gate, w_up, F, dtype, activation, grad, ws, s, dx, dw_gate, dw_up, st);
}
