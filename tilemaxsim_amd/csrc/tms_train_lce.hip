// Softmax cross entropy of the logits scale * H W^T, from the hidden states and the
// vocabulary's weights, without the logits.
//
//   x[n, v] = scale <H[n], W[v]>,  loss[n] = log sum_v exp x[n, v] - x[n, t[n]]
//   P[n, v] = exp x[n, v] / sum_u exp x[n, u] - [v = t[n]]
//   dH[n] = g[n] scale sum_v P[n, v] W[v],   dW[v] = scale sum_n g[n] P[n, v] H[n]
//
// Forward: one product whose epilogue reduces each tile's logits to a maximum and a sum of
// exponentials per row and block of the vocabulary, and a kernel that joins the blocks
// (8 bytes per row and block instead of 4 per logit).
// Backward: piece by piece of the vocabulary the logits are formed again (2 N V d operations,
// where writing and reading them in fp32 would take 8 N V bytes: at d = 768 as long, at less
// shorter), become P in 16 bits in a workspace, and two more products take P to dH and dW.
//
// Everything is in powers of two: x log2(e) goes into exp2. A row keeps its largest logit, the
// sum of exp2 relative to it, and the others' share of that sum (all but the target's): with
// rest = sum over v != t of exp(x[v] - x[t]), the loss is log(1 + rest) and P at the target
// -rest / (1 + rest). Neither is a difference of two numbers of the logits' size, or of a
// softmax near 1 and 1, so a row that is nearly right keeps its digits. (From one log-sum-exp a
// row, a loss of 2e-11 came out as 1.3e-6, others below zero, and P at the target as far off.)
//
// Precision. Logits, maxima, sums, and the sums of both gradients are fp32. P is rounded to
// the inputs' type, as the matrix cores take it (bf16: 2^-9 of each term; fp16: 2^-12, and P is
// held times 2^15, so that 2^-29 is still a normal number). In dH its element at the target, as
// large as the others of the row together, is made whole again, so dH is as near to 64 bits as
// with a P of 32 bits (512 x 8000 x 256 in fp16, rows of W with ten times their spread in
// common: 2.3e-4, 1.2e-3 without). dW has both roundings, P's and its own: where a word is the
// target of one row, 1.4 times the error of the second alone (1024 x 16384 x 128, unit vectors:
// 2.9e-4 against 2.2e-4 in fp16). fp32 inputs are three bf16 terms, and so is their P. P is times
// g[n] / u before it is rounded, for both gradients, and their sums are times u: u is what a
// reduction gives every row alike (the ratio is 1), or a power of two above the largest |g| of
// rows with their own.
#include <math.h>

#include "tms_train_terms.h"

namespace tms {

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kP16 = 15;  // fp16: P times 2^15

struct RowStat {
  float top, sum;  // of a block: the largest x log2(e), and the sum of exp2 relative to it but the target's
};

// The forward pass's statistics, from the sums in registers: a lane has four rows of the
// vocabulary for each of its hidden rows, and a wave one RowStat a hidden row and tile. 8192 x
// 131072 x 768 in bf16: 1.38 to 1.46 ms, 1.19 to 1.13 PFLOP/s; the matrix cores are busy for 54 % of
// it, at 1.9 GHz, and with twelve steps a tile its first loads and its exponentials take 6 us in 25.
struct LseEpilogue {
  static constexpr int kRowBytes = 0;
  RowStat* parts;  // [block of the vocabulary][rows]
  const int64_t* target;  // per row; outside the vocabulary: in no block
  float* hit_sum;         // per row: the product's sum at its target
  int32_t rows, V;
  float s2;  // scale log2(e)

  // The sum of a lane's elements of one row, and its target's element, which takes no part.
  template <bool HIT, int MI, int NI>
  __device__ __forceinline__ float sum_of(const f32x4 (&acc)[MI][NI], int j, float ref, int hit, float& at_hit) const {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], s2, -ref));
        if constexpr (HIT) {
          const bool at = hit == 16 * i + e;
          at_hit = at ? acc[i][j][e] : at_hit;
          sum += at ? 0.f : p;
        } else {
          sum += p;
        }
      }
    return sum;
  }

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int, uint8_t*) const {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const float NEG = -__builtin_inff();
    int64_t t[NI];  // on their way while the maxima are formed
#pragma unroll
    for (int j = 0; j < NI; j++) t[j] = n + 16 * j + c < rows ? target[n + 16 * j + c] : -1;
    if (m + 16 * MI > V) {  // past the vocabulary
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (m + 16 * i + 4 * g + e >= V)
#pragma unroll
            for (int j = 0; j < NI; j++) acc[i][j][e] = NEG;
    }
    float tops[NI];
#pragma unroll
    for (int j = 0; j < NI; j++) {
      float top = NEG;
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, acc[i][j][e]);
      tops[j] = cross_row_max(top) * s2;  // scale > 0
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const float top = tops[j], ref = top == NEG ? 0.f : top;
      const int row = n + 16 * j + c;
      const int hit = t[j] >= 0 && t[j] < V ? (int)t[j] - (m + 4 * g) : -1;  // the target's place among this lane's 16 i + e
      float sum, at_hit = 0.f;
      if (__ballot(hit >= 0 && hit < 16 * MI) != 0ull) {
        sum = sum_of<true>(acc, j, ref, hit, at_hit);
        if (hit >= 0 && hit < 16 * MI && (hit & 15) < 4) hit_sum[row] = at_hit;
      } else {
        sum = sum_of<false>(acc, j, ref, hit, at_hit);
      }
      sum = cross_row_sum(sum);
      if (g == 0 && row < rows && m < V) parts[(int64_t)(m / (16 * MI)) * rows + row] = {top, sum};
    }
  }
};

// P of one piece: [plane][row][ldp]; rows and columns that do not exist are zero. A lane holds
// four neighbouring columns of a row, so a wave's rows pass through its LDS and leave as whole
// lines (eight-byte stores left half-written lines: a quarter more time). 8192 x 65,536 of them
// at d = 768 in bf16: 0.79 to 0.82 ms, 1.05 to 1.0 PFLOP/s, bound like the statistics' product (matrix
// cores busy for 47 %); 1 GB leaves with it.
template <int DT, int PL, int MIV>
struct ProbEpilogue {
  static constexpr int kRowBytes = MIV * 32 + 16;  // 16 more: the rows of four lanes fall on other banks
  uint16_t* P;
  const float* top;       // per row: its largest logit; +inf for a row without a gradient
  const float* g_row;     // per row: g / u over the sum of exp2
  const float* hit_row;   // per row: what P is at its target
  const int32_t* target;  // per row; -1 for none
  int64_t plane;
  int32_t ldp, rows, V, v0;  // V: columns of the piece that exist; v0: its first
  float s2;

  // p = exp2(x - top) w of a lane's elements of one row, at its target at_hit, and its terms
  template <bool HIT, int MI>
  __device__ __forceinline__ void row(const f32x4 (&x)[MI], float ref, float w, int hit, float at_hit, u32x2 (&out)[PL][MI]) const {
#pragma unroll
    for (int i = 0; i < MI; i++) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][e], s2, -ref)) * w;
        if constexpr (HIT) p[e] = hit == 16 * i + e ? at_hit : p[e];
      }
#pragma unroll
      for (int t = 0; t < PL; t++) {
        uint16_t b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if constexpr (DT == TMS_DTYPE_F16) {
            b[e] = __builtin_bit_cast(uint16_t, (_Float16)p[e]);
          } else {
            const __bf16 h = (__bf16)p[e];
            b[e] = __builtin_bit_cast(uint16_t, h);
            if constexpr (PL > 1) p[e] -= (float)h;
          }
        }
        out[t][i] = u32x2{(uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16};
      }
    }
  }

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int, uint8_t* lds) const {
    static_assert(MI == MIV, "rows of the wave's LDS");
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    if (m + 16 * MI > V) {  // past the vocabulary: exp2 gives 0
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (m + 16 * i + 4 * g + e >= V)
#pragma unroll
            for (int j = 0; j < NI; j++) acc[i][j][e] = -__builtin_inff();
    }
    constexpr int PIECES = MI * 2, ROWS = 64 / PIECES;  // 16-byte pieces of a row; rows a wave stores at once
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const int r = n + 16 * j + c;
      const bool in = r < rows;
      const float ref = in ? top[r] : __builtin_inff(), w = in ? g_row[r] : 0.f;
      const int hit = in ? target[r] - v0 - (m + 4 * g) : -1;  // its place among this lane's 16 i + e
      f32x4 x[MI];
#pragma unroll
      for (int i = 0; i < MI; i++) x[i] = acc[i][j];
      u32x2 out[PL][MI];
      if (__ballot(hit >= 0 && hit < 16 * MI) != 0ull) row<true>(x, ref, w, hit, in ? hit_row[r] : 0.f, out);
      else row<false>(x, ref, w, hit, 0.f, out);
#pragma unroll
      for (int t = 0; t < PL; t++) {
#pragma unroll
        for (int i = 0; i < MI; i++) *(u32x2*)(lds + c * kRowBytes + i * 32 + g * 8) = out[t][i];
#pragma unroll
        for (int k = 0; k < 16 / ROWS; k++) {
          const int rr = k * ROWS + lane / PIECES, piece = lane % PIECES;
          const u32x4 v = *(const u32x4*)(lds + rr * kRowBytes + piece * 16);
          *(u32x4*)(P + t * plane + (int64_t)(n + 16 * j + rr) * ldp + m + piece * 8) = v;
        }
      }
    }
  }
};

// Sums of dH: [split][row][d], added to from the second piece on. A piece of 65,536 at 8192 rows
// of 768 in bf16, five splits: 0.89 to 0.92 ms, 0.92 to 0.9 PFLOP/s: 480 workgroups are two rounds, the second
// not full (matrix cores busy for 40 %), and 250 MB of sums are read and written.
struct SumEpilogue {
  static constexpr int kRowBytes = 0;
  float* out;
  int64_t split;  // elements of one
  int32_t rows, d;
  int32_t first;

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
        if (col >= d) continue;
        f32x4* to = (f32x4*)(out + s * split + (int64_t)row * d + col);
        f32x4 v = acc[i][j];
        if (!first) {
          const f32x4 old = *to;
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] += old[e];
        }
        *to = v;
      }
    }
  }
};

// dW of one piece, finished: times *factor, in the inputs' type. 65,536 rows of 768 over 8192 in
// bf16: 0.69 to 0.72 ms, 1.2 PFLOP/s (three whole rounds of workgroups; pieces half as large take one and a half).
template <int OUT>
struct WeightEpilogue {
  static constexpr int kRowBytes = 0;
  void* out;  // the piece's first row
  const float* factor;
  int32_t rows, d;

  template <int MI, int NI>
  __device__ __forceinline__ void operator()(f32x4 (&acc)[MI][NI], int m, int n, int, uint8_t*) const {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const float f = *factor;
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const int row = n + 16 * j + c;
      if (row >= rows) continue;
#pragma unroll
      for (int i = 0; i < MI; i++) {
        const int col = m + 16 * i + 4 * g;
        if (col >= d) continue;
        const int64_t at = (int64_t)row * d + col;
        if constexpr (OUT == TMS_DTYPE_F32) {
          float* to = (float*)out + at;
          if ((d & 3) == 0) *(f32x4*)to = f32x4{acc[i][j][0] * f, acc[i][j][1] * f, acc[i][j][2] * f, acc[i][j][3] * f};
          else
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (col + e < d) to[e] = acc[i][j][e] * f;
        } else {
          uint16_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = to16<OUT>(acc[i][j][e] * f);
          uint16_t* to = (uint16_t*)out + at;
          if ((d & 3) == 0) *(u32x2*)to = u32x2{(uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16};
          else
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (col + e < d) to[e] = w[e];
        }
      }
    }
  }
};

// ---------------------------------------------------------------- rows

// (top, sum) of two parts of a row
__device__ __forceinline__ RowStat join_stats(RowStat a, RowStat b) {
  const float t = fmaxf(a.top, b.top), ref = t == -__builtin_inff() ? 0.f : t;
  return {t, a.sum * __builtin_amdgcn_exp2f(a.top - ref) + b.sum * __builtin_amdgcn_exp2f(b.top - ref)};
}

// Joins a row's blocks and its target's exponential; LANES lanes a row. Writes what the backward
// pass takes, [row] each: the largest logit, 1 over the sum of exp2 relative to it, and in the
// place of hit_sum the others' share. A target outside the vocabulary (and not ignored) makes the
// row NaN. With `loss` and one workgroup, that goes over all rows and then reduces them as the
// kernel below does: a call of a few rows is bound by its launches. Bound by the latency of a
// row's statistics: 1024 rows of 128 blocks 5 us, 8192 of 1024 20 us (67 MB read).
template <int LANES>
__global__ __launch_bounds__(256) void lce_join_kernel(const RowStat* parts, int32_t blocks, int32_t rows, int32_t V, const int64_t* target,
                                                       int64_t ignore, float s2, float* top, float* inv_sum, float* hit_sum,
                                                       float* rows_loss, float* loss, float* count, int mean) {
  constexpr int ROWS = 256 / LANES;
  __shared__ RowStat stats[4];
  const int lane = threadIdx.x % LANES;
  double all = 0;
  int kept_rows = 0;
  for (int row0 = blockIdx.x * ROWS; row0 < rows; row0 += gridDim.x * ROWS) {
    const int row = row0 + threadIdx.x / LANES;
    const bool in = row < rows;
    const int64_t t = in ? target[row] : ignore;
    const bool kept = t != ignore, fine = t >= 0 && t < V;
    const float hit = lane == 0 && kept && fine ? hit_sum[row] : 0.f;
    RowStat r = {-__builtin_inff(), 0.f};
    for (int b = lane; in && b < blocks; b += 8 * LANES) {  // eight loads at a time
      RowStat x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int at = b + i * LANES;
        x[i] = at < blocks ? parts[(int64_t)at * rows + row] : RowStat{-__builtin_inff(), 0.f};
      }
#pragma unroll
      for (int i = 0; i < 8; i++) r = join_stats(r, x[i]);
    }
#pragma unroll
    for (int o = (LANES < 64 ? LANES : 64) / 2; o >= 1; o >>= 1) r = join_stats(r, RowStat{__shfl_xor(r.top, o), __shfl_xor(r.sum, o)});
    if constexpr (LANES > 64) {
      __syncthreads();  // the last row's are read
      if ((threadIdx.x & 63) == 0) stats[threadIdx.x >> 6] = r;
      __syncthreads();
      r = stats[0];
#pragma unroll
      for (int w = 1; w < 4; w++) r = join_stats(r, stats[w]);
    }
    const float y = __builtin_fmaf(hit, s2, -r.top);  // of the target, as every other exponent is formed
    float sum = r.sum + __builtin_amdgcn_exp2f(y), x = 0.f;
    if (kept && !fine) r.top = sum = __builtin_nanf("");
    // Near the top the loss is log(1 + rest); away from it, at least ln 2, a sum of two positive numbers.
    if (kept) x = !fine ? sum : y > -1.f ? log1pf(r.sum * __builtin_amdgcn_exp2f(-y)) : (log2f(sum) - y) * kLn2;
    if (in && lane == 0) {
      top[row] = r.top;
      inv_sum[row] = 1.f / sum;
      hit_sum[row] = r.sum / sum;
      if (rows_loss) rows_loss[row] = x;
    }
    all += (double)x;
    kept_rows += kept;
  }
  if (LANES == 256 && loss && threadIdx.x == 0) {
    *count = (float)kept_rows;
    *loss = mean ? (float)(all / (double)kept_rows) : (float)all;
  }
}

// The sum or mean of the rows' losses, and how many rows count: in 64 bits and one workgroup,
// bound by its loads' latency, 5 us for 8192 rows.
__global__ __launch_bounds__(1024) void lce_reduce_kernel(const float* rows_loss, const int64_t* target, int64_t ignore, int32_t rows,
                                                          int mean, float* loss, float* count) {
  __shared__ double sums[16];
  __shared__ int counts[16];
  double s = 0;
  int c = 0;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    s += (double)rows_loss[i];
    c += target[i] != ignore;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    s += __shfl_xor(s, o);
    c += __shfl_xor(c, o);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = s;
    counts[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; w++) {
      s += sums[w];
      c += counts[w];
    }
    *count = (float)c;
    *loss = mean ? (float)(s / (double)c) : (float)s;
  }
}

// What the backward kernels take for each row: g / u over its sum of exp2, its reference for
// exp2, its target and what P is there; and u with the factor of both gradients' sums. P is held
// times 2^up. One workgroup, 12 us for 8192 rows.
__global__ __launch_bounds__(1024) void lce_rows_kernel(const float* top, const float* inv_sum, const float* others, const int64_t* target,
                                                        int64_t ignore, int32_t V, int32_t rows, const float* grad, int per_row,
                                                        const float* count, int up, float scale, float* g, float* ref, int32_t* hit,
                                                        float* at_hit, float* factor) {
  __shared__ float tops[16];
  float unit = 1.f;
  if (per_row) {
    float most = 0.f;
    for (int i = threadIdx.x; i < rows; i += 1024)
      if (target[i] != ignore) most = fmaxf(most, fabsf(grad[i]));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = most;
    __syncthreads();
    for (int w = 0; w < 16; w++) most = fmaxf(most, tops[w]);
    int e = (int)((__builtin_bit_cast(uint32_t, most) >> 23) & 0xffu) + 1;  // 2^(e - 127) > most
    e = most == 0.f || e > 252 ? 127 : e < 2 ? 2 : e;  // an infinite factor stays as it is
    unit = __builtin_bit_cast(float, (uint32_t)e << 23);
  } else {
    const float all = *grad / (count ? *count : 1.f);
    if (all != 0.f && fabsf(all) < 1e38f) unit = all;
  }
  const float held = (float)(1 << up);
  if (threadIdx.x == 0) *factor = unit * scale / held;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const int64_t t = target[i];
    const bool kept = t != ignore;
    const float w = !kept ? 0.f : (per_row ? grad[i] : *grad / (count ? *count : 1.f)) / unit * held;
    g[i] = kept ? w * inv_sum[i] : 0.f;
    at_hit[i] = kept ? -w * others[i] : 0.f;
    ref[i] = kept ? top[i] : __builtin_inff();
    hit[i] = kept && t >= 0 && t < V ? (int32_t)t : -1;
  }
}

// dH: the splits' sums, in order, times the factor, in the inputs' type. To them comes what P's
// rounding to 16 bits took off its element at the target, times the target's row: that element is
// as large as all others of its row together, and what the vocabulary's rows have in common
// cancels between the two. Four elements of a row a thread (rows of sums and of w are whole
// multiples of four), eight splits' loads at a time. 8192 x 768, five splits: 31 us, 4.9 TB/s.
template <int OUT>
__global__ __launch_bounds__(256) void lce_hidden_kernel(const float* sums, int splits, int64_t split, int32_t rows, int32_t d, int32_t dp,
                                                         const float* factor, const uint16_t* w, const int32_t* hit, const float* at_hit,
                                                         void* dH) {
  const int quads = (d + 3) / 4;
  const int64_t n = (int64_t)rows * quads;
  const float f = *factor;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
    const int64_t row = k / quads;
    const int col = (int)(k - row * quads) * 4;
    const float* from = sums + row * dp + col;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; s += 8) {
      f32x4 y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = s + i < splits ? *(const f32x4*)(from + (s + i) * split) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += y[i][e];
    }
    if constexpr (OUT != TMS_DTYPE_F32) {  // three terms leave nothing
      const int t = hit[row];
      if (t >= 0) {
        const float left = at_hit[row] - from16<OUT>(to16<OUT>(at_hit[row]));
        const u32x2 at = *(const u32x2*)(w + (int64_t)t * dp + col);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(left, from16<OUT>((uint16_t)(at[e / 2] >> (16 * (e & 1)))), x[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (col + e >= d) break;
      const float v = x[e] * f;
      if constexpr (OUT == TMS_DTYPE_F32) ((float*)dH)[row * d + col + e] = v;
      else ((uint16_t*)dH)[row * d + col + e] = to16<OUT>(v);
    }
  }
}

// ---------------------------------------------------------------- host

static int logits_size(int64_t N, int64_t V, int64_t dp, int dtype) {
  return terms_size(V, N, dp, planes(dtype), gemm_largest(planes(dtype)));
}
// Vocabulary rows that one RowStat of the forward pass covers: a wave's share of a tile.
static int64_t stat_rows(int size) { return gemm_side(size) / 2; }
// Rows up to which one workgroup joins them all: below that its launch would take longer.
constexpr int64_t kJoinAlone = 4;

struct LceSpace {
  int64_t h, w, parts, loss, g, ref, hit, at_hit, factor, p, sums, bytes;
};
static LceSpace lce_space(int64_t N, int64_t V, int64_t d, int dtype, bool backward, bool terms) {
  LceSpace s = {};
  Carve c;
  const int64_t dp = up_to(d > 0 ? d : 8, 8);
  if (terms || backward) s.h = c.take(N * dp * 2 * planes(dtype));
  if (terms) s.w = c.take(V * dp * 2 * planes(dtype));
  if (!backward) {
    const int64_t per = stat_rows(logits_size(N, V, dp, dtype));
    s.parts = c.take((V + per - 1) / per * N * (int64_t)sizeof(RowStat));
    s.loss = c.take(N * 4);
  } else {
    const LcePlan p = lce_plan(N, V, d, planes(dtype));
    s.g = c.take(N * 4);
    s.ref = c.take(N * 4);
    s.hit = c.take(N * 4);
    s.at_hit = c.take(N * 4);
    s.factor = c.take(4);
    s.p = c.take(p.rows_p * p.piece * 2 * planes(dtype));
    s.sums = c.take(p.splits * N * dp * 4);
  }
  s.bytes = c.at;
  return s;
}

static int check_lce(const char* fn, int64_t N, int64_t d, int64_t V, int dtype, const double* scale, int reduction) {
  if (N < 0 || d < 0 || V < 0) return fail(TMS_ERR_INVALID, "%s: negative size", fn);
  if (dtype != TMS_DTYPE_F16 && dtype != TMS_DTYPE_BF16 && dtype != TMS_DTYPE_F32)
    return fail(TMS_ERR_UNSUPPORTED, "%s: dtype must be fp16, bf16 or fp32", fn);
  if (reduction != TMS_REDUCE_NONE && reduction != TMS_REDUCE_SUM && reduction != TMS_REDUCE_MEAN)
    return fail(TMS_ERR_INVALID, "%s: unknown reduction %d", fn, reduction);
  if (!scale || !(*scale > 0) || !(*scale < 1e30)) return fail(TMS_ERR_INVALID, "%s: scale must be positive and finite", fn);
  if (V == 0 && N > 0) return fail(TMS_ERR_INVALID, "%s: an empty vocabulary", fn);
  if (d > 65536 || N > (1 << 24) || V > (1 << 28)) return fail(TMS_ERR_UNSUPPORTED, "%s: sizes up to d = 65536, N = 2^24, V = 2^28", fn);
  return TMS_OK;
}

// The logits' product: m over vocabulary rows, n over hidden rows.
static GemmArgs logits_args(const void* H, const void* W, int64_t N, int64_t V, int64_t Vall, int64_t dp, int dtype) {
  GemmArgs a = {};
  a.A = (const uint16_t*)W;
  a.B = (const uint16_t*)H;
  a.aplane = Vall * dp;
  a.bplane = N * dp;
  a.lda = a.ldb = (int32_t)dp;
  a.M = (int32_t)V;
  a.N = (int32_t)N;
  a.K = (int32_t)dp;
  a.splits = 1;
  return a;
}

template <int DT, int PL>  // the terms' type and number: fp32 inputs have three bf16 ones
static int lce_forward(const void* H, int64_t N, int64_t d, const void* W, int64_t V, int dtype, const int64_t* target, int64_t ignore,
                       float s2, int reduction, uint8_t* ws, const LceSpace& s, bool terms, float* loss, float* stats, hipStream_t st) {
  const int64_t dp = up_to(d > 0 ? d : 8, 8);
  const void *h = H, *w = W;
  int rc;
  if (terms) {
    h = ws + s.h;
    w = ws + s.w;
    if ((rc = run_terms(H, dtype, ws + s.h, N, d, dp, nullptr, st))) return rc;
    if ((rc = run_terms(W, dtype, ws + s.w, V, d, dp, nullptr, st))) return rc;
  }
  const GemmArgs a = logits_args(h, w, N, V, V, dp, dtype);
  float *top = stats, *inv_sum = stats + N, *hit_sum = stats + 2 * N, *count = stats + 3 * N;
  LseEpilogue e = {(RowStat*)(ws + s.parts), target, hit_sum, (int32_t)N, (int32_t)V, s2};
  const int size = logits_size(N, V, dp, dtype);
  rc = with_size<PL>(size, [&](auto z) { return run_gemm<DT, PL, decltype(z)::MI, decltype(z)::NI, false, false>(a, e, st, "train_gemm_kernel (lse)"); });
  if (rc) return rc;
  const bool rows = reduction == TMS_REDUCE_NONE, alone = !rows && N <= kJoinAlone;
  float* rows_loss = rows ? loss : (float*)(ws + s.loss);
  const int32_t blocks = (int32_t)((V + stat_rows(size) - 1) / stat_rows(size));
  const RowStat* parts = (const RowStat*)(ws + s.parts);
  // Few rows of many blocks take a workgroup each, many rows sixteen lanes each, which read
  // sixteen rows' neighbouring statistics together.
  if (N <= 1024)
    hipLaunchKernelGGL(lce_join_kernel<256>, dim3(alone ? 1u : (unsigned)N), dim3(256), 0, st, parts, blocks, (int32_t)N, (int32_t)V, target,
                       ignore, s2, top, inv_sum, hit_sum, rows_loss, alone ? loss : nullptr, count, reduction == TMS_REDUCE_MEAN ? 1 : 0);
  else
    hipLaunchKernelGGL(lce_join_kernel<16>, dim3((unsigned)((N + 15) / 16)), dim3(256), 0, st, parts, blocks, (int32_t)N, (int32_t)V, target,
                       ignore, s2, top, inv_sum, hit_sum, rows_loss, nullptr, nullptr, 0);
  if ((rc = check_launch("lce_join_kernel")) || rows || alone) return rc;
  hipLaunchKernelGGL(lce_reduce_kernel, dim3(1), dim3(1024), 0, st, rows_loss, target, ignore, (int32_t)N, reduction == TMS_REDUCE_MEAN ? 1 : 0,
                     loss, count);
  return check_launch("lce_reduce_kernel");
}

template <int DT, int PL, int OUT>
static int lce_backward(const void* H, int64_t N, int64_t d, const void* W, int64_t V, int dtype, const int64_t* target, int64_t ignore,
                        float scale, float s2, int reduction, const float* stats, const float* grad, uint8_t* ws, const LceSpace& s, bool terms,
                        void* dH, void* dW, hipStream_t st) {
  const LcePlan p = lce_plan(N, V, d, planes(dtype));
  const int up = DT == TMS_DTYPE_F16 ? kP16 : 0;
  float *g = (float*)(ws + s.g), *ref = (float*)(ws + s.ref), *factor = (float*)(ws + s.factor), *sums = (float*)(ws + s.sums);
  float* at_hit = (float*)(ws + s.at_hit);
  int32_t* hit = (int32_t*)(ws + s.hit);
  uint16_t *h = (uint16_t*)(ws + s.h), *P = (uint16_t*)(ws + s.p);
  const void* w = terms ? ws + s.w : W;
  int rc;
  hipLaunchKernelGGL(lce_rows_kernel, dim3(1), dim3(1024), 0, st, stats, stats + N, stats + 2 * N, target, ignore, (int32_t)V, (int32_t)N, grad,
                     reduction == TMS_REDUCE_NONE ? 1 : 0, reduction == TMS_REDUCE_MEAN ? stats + 3 * N : nullptr, up, scale, g, ref, hit, at_hit,
                     factor);
  if ((rc = check_launch("lce_rows_kernel"))) return rc;
  if ((rc = run_terms(H, dtype, h, N, d, p.dp, ref, st))) return rc;
  if (terms && (rc = run_terms(W, dtype, ws + s.w, V, d, p.dp, nullptr, st))) return rc;
  const int64_t pplane = p.rows_p * p.piece;
  for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
    const int64_t nv = V - v0 < p.piece ? V - v0 : p.piece;
    GemmArgs a = logits_args(h, (const uint16_t*)w + v0 * p.dp, N, nv, V, p.dp, dtype);
    rc = with_size<PL>(p.size_p, [&](auto z) {
      using Z = decltype(z);
      const ProbEpilogue<DT, PL, Z::MI> e = {P, ref, g, at_hit, hit, pplane, (int32_t)p.piece, (int32_t)N, (int32_t)nv, (int32_t)v0, s2};
      return run_gemm<DT, PL, Z::MI, Z::NI, false, false>(a, e, st, "train_gemm_kernel (P)");
    });
    if (rc) return rc;
    if (dH && d > 0) {  // m over d, n over rows, k over the piece
      GemmArgs b = {};
      b.A = (const uint16_t*)w + v0 * p.dp;
      b.B = P;
      b.aplane = V * p.dp;
      b.bplane = pplane;
      b.lda = (int32_t)p.dp;
      b.ldb = (int32_t)p.piece;
      b.M = (int32_t)p.dp;
      b.N = (int32_t)N;
      b.K = (int32_t)nv;
      b.splits = p.splits;
      SumEpilogue se = {sums, N * p.dp, (int32_t)N, (int32_t)p.dp, v0 == 0};
      rc = with_size<PL>(p.size_h, [&](auto z) {
        return run_gemm<DT, PL, decltype(z)::MI, decltype(z)::NI, true, false>(b, se, st, "train_gemm_kernel (dH)");
      });
      if (rc) return rc;
    }
    if (dW && d > 0) {  // m over d, n over the piece, k over rows
      GemmArgs b = {};
      b.A = h;
      b.B = P;
      b.aplane = N * p.dp;
      b.bplane = pplane;
      b.lda = (int32_t)p.dp;
      b.ldb = (int32_t)p.piece;
      b.M = (int32_t)p.dp;
      b.N = (int32_t)up_to(nv, 8);
      b.K = (int32_t)N;
      b.splits = 1;
      WeightEpilogue<OUT> we = {(uint8_t*)dW + v0 * d * (OUT == TMS_DTYPE_F32 ? 4 : 2), factor, (int32_t)nv, (int32_t)d};
      rc = with_size<PL>(p.size_w, [&](auto z) {
        return run_gemm<DT, PL, decltype(z)::MI, decltype(z)::NI, true, true>(b, we, st, "train_gemm_kernel (dW)");
      });
      if (rc) return rc;
    }
  }
  if (dH && d > 0) {
    hipLaunchKernelGGL(lce_hidden_kernel<OUT>, dim3(blocks_for(N * ((d + 3) / 4))), dim3(256), 0, st, sums, p.splits, N * p.dp, (int32_t)N, (int32_t)d,
                       (int32_t)p.dp, factor, (const uint16_t*)w, hit, at_hit, dH);
    return check_launch("lce_hidden_kernel");
  }
  return TMS_OK;
}

}  // namespace tms

using namespace tms;

extern "C" int64_t tms_lce_stats(int64_t N) { return N < 0 ? 0 : 3 * N + 1; }

extern "C" int64_t tms_lce_workspace_size(int64_t N, int64_t d, int64_t V, int dtype, int backward) {
  if (N <= 0 || d < 0 || V <= 0) return 0;
  return lce_space(N, V, d, dtype, backward != 0, dtype == TMS_DTYPE_F32 || d % 8 != 0 || d == 0).bytes;
}

static int lce_workspace(const char* fn, const void* H, const void* W, int64_t N, int64_t d, int64_t V, int dtype, bool backward,
                         const void* ws, int64_t bytes, bool& terms, LceSpace& s) {
  terms = dtype == TMS_DTYPE_F32 || d % 8 != 0 || d == 0;
  if (!terms && !(as_is(H, d, dtype) && as_is(W, d, dtype))) return fail(TMS_ERR_INVALID, "%s: hidden and weight must be 16-byte aligned", fn);
  s = lce_space(N, V, d, dtype, backward, terms);
  if (!ws || (uintptr_t)ws % 256 || bytes < s.bytes)
    return fail(TMS_ERR_INVALID, "%s: a workspace of %lld bytes is needed, 256-byte aligned", fn, (long long)s.bytes);
  return TMS_OK;
}

extern "C" int tms_linear_cross_entropy(const void* hidden, int64_t N, int64_t d, const void* weight, int64_t V, int dtype,
                                        const int64_t* target, int64_t ignore_index, const double* scale, int reduction, void* workspace,
                                        int64_t workspace_bytes, float* loss, float* stats, void* stream) {
  const char* fn = "tms_linear_cross_entropy";
  int rc = check_lce(fn, N, d, V, dtype, scale, reduction);
  if (rc) return rc;
  if ((!loss && (N > 0 || reduction != TMS_REDUCE_NONE)) || !stats || (N > 0 && (!target || (d > 0 && (!hidden || !weight)))))
    return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  LceSpace s = {};
  bool terms = false;
  if (N > 0) {
    if ((rc = lce_workspace(fn, hidden, weight, N, d, V, dtype, false, ws, workspace_bytes, terms, s))) return rc;
    const float s2 = (float)(*scale * kLog2e);
    if (dtype == TMS_DTYPE_F16) rc = lce_forward<TMS_DTYPE_F16, 1>(hidden, N, d, weight, V, dtype, target, ignore_index, s2, reduction, ws, s, terms, loss, stats, st);
    else if (dtype == TMS_DTYPE_BF16) rc = lce_forward<TMS_DTYPE_BF16, 1>(hidden, N, d, weight, V, dtype, target, ignore_index, s2, reduction, ws, s, terms, loss, stats, st);
    else rc = lce_forward<TMS_DTYPE_BF16, 3>(hidden, N, d, weight, V, dtype, target, ignore_index, s2, reduction, ws, s, terms, loss, stats, st);
    if (rc) return rc;
  }
  if (N > 0 || reduction == TMS_REDUCE_NONE) return TMS_OK;
  hipLaunchKernelGGL(lce_reduce_kernel, dim3(1), dim3(1024), 0, st, nullptr, target, ignore_index, 0, reduction == TMS_REDUCE_MEAN ? 1 : 0, loss, stats);
  return check_launch("lce_reduce_kernel");
}

extern "C" int tms_linear_cross_entropy_grad(const void* hidden, int64_t N, int64_t d, const void* weight, int64_t V, int dtype,
                                             const int64_t* target, int64_t ignore_index, const double* scale, int reduction,
                                             const float* stats, const float* grad, void* workspace, int64_t workspace_bytes, void* dH,
                                             void* dW, void* stream) {
  const char* fn = "tms_linear_cross_entropy_grad";
  int rc = check_lce(fn, N, d, V, dtype, scale, reduction);
  if (rc) return rc;
  if (N == 0 || (!dH && !dW)) return TMS_OK;  // no rows: the caller's zeros
  if (!target || !stats || !grad || (d > 0 && (!hidden || !weight))) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  LceSpace s = {};
  bool terms = false;
  if ((rc = lce_workspace(fn, hidden, weight, N, d, V, dtype, true, workspace, workspace_bytes, terms, s))) return rc;
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  const float sc = (float)*scale, s2 = (float)(*scale * kLog2e);  // s2: the forward pass's
  if (dtype == TMS_DTYPE_F16)
    return lce_backward<TMS_DTYPE_F16, 1, TMS_DTYPE_F16>(hidden, N, d, weight, V, dtype, target, ignore_index, sc, s2, reduction, stats, grad, ws, s, terms, dH, dW, st);
  if (dtype == TMS_DTYPE_BF16)
    return lce_backward<TMS_DTYPE_BF16, 1, TMS_DTYPE_BF16>(hidden, N, d, weight, V, dtype, target, ignore_index, sc, s2, reduction, stats, grad, ws, s, terms, dH, dW, st);
  return lce_backward<TMS_DTYPE_BF16, 3, TMS_DTYPE_F32>(hidden, N, d, weight, V, dtype, target, ignore_index, sc, s2, reduction, stats, grad, ws, s, terms, dH, dW, st);
}
