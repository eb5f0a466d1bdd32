// Rules on sizes of the training operators: plain C++, so that tests can ask them.
#pragma once
#include <stdint.h>

namespace tms {

inline int64_t up_to(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// The matrix product's tiles (tms_train_gemm.h): m x n of 256 x 256, 128 x 128 and 64 x 64.
enum GemmSize { kGemm256 = 0, kGemm128 = 1, kGemm64 = 2 };
constexpr int kGemmSizes = 3;
inline int64_t gemm_side(int size) { return size == kGemm256 ? 256 : size == kGemm128 ? 128 : 64; }

// Microseconds of a product of m x n tiles over `steps` 64-steps of k, `splits` times: the
// rounds of workgroups that the 256 CUs take, each as long as its steps and what surrounds
// them. Measured in bf16 (4096 deep, a step of one, two and four workgroups a CU): 256 x 256
// 1.58; 128 x 128 0.87, 1.05; 64 x 64 0.64, 0.68, 0.95. The large tile's steps alone make 1.36
// PFLOP/s once they fill the chip; below that, the smaller ones do the same work on more CUs.
inline double gemm_us(int size, int64_t m, int64_t n, int64_t steps, int64_t splits) {
  const int64_t side = gemm_side(size);
  const int64_t groups = up_to(m, side) / side * (up_to(n, side) / side) * splits, each = (steps + splits - 1) / splits;
  if (size == kGemm256) return (double)((groups + 255) / 256) * ((double)each * 1.58 + 6.0);
  if (size == kGemm128) return groups <= 256 ? (double)each * 0.87 + 4.0 : (double)((groups + 511) / 512) * ((double)each * 1.05 + 4.0);
  if (groups <= 256) return (double)each * 0.64 + 3.0;
  if (groups <= 512) return (double)each * 0.68 + 3.0;
  return (double)((groups + 1023) / 1024) * ((double)each * 0.95 + 3.0);
}

// Products of rows of three bf16 terms take six products a 64-step with seven tiles' loads:
// as long as four steps. Their largest tile is 128 x 128: 256 x 256 has no registers for the
// fragments that the next product shares (4096 x 32000 x 1024, k inside: 1.23 PFLOP/s against 1.32).
inline int64_t gemm_steps(int64_t k, int planes) { return up_to(k, 64) / 64 * (planes == 3 ? 4 : 1); }
inline int gemm_largest(int planes) { return planes == 3 ? kGemm128 : kGemm256; }

inline int gemm_size(int64_t m, int64_t n, int64_t steps, int largest = kGemm256) {  // largest: the largest tile to take
  int best = largest;
  for (int s = best + 1; s < kGemmSizes; s++)
    if (gemm_us(s, m, n, steps, 1) < gemm_us(best, m, n, steps, 1)) best = s;
  return best;
}

inline int64_t gemm_groups(int size, int64_t m, int64_t n, int64_t splits) {
  const int64_t side = gemm_side(size);
  return up_to(m, side) / side * (up_to(n, side) / side) * splits;
}

// Microseconds of a product of m x n over k. Of three planes, tiles of 64 x 64 wait once a 64-step, with one workgroup a CU:
// rounds of up to 256 of them, 0.97 a step. (fp32 logits of 500 x 8000 x 64, 1000 tiles of one step: 11.7, in tiles of 128
// 7.5; 1024 x 4000 x 128: 15.4 / 11.6; 600 x 4000 x 64: 8.7 / 7.1, x 1024: 50 / 54; 400 x 4000 x 64: 6.2 / 6.9, x 256: 12.1 /
// 16.0. 176 tiles over 2048: 33.0.)
inline double terms_us(int size, int64_t m, int64_t n, int64_t k, int planes, int64_t splits) {
  if (planes != 3 || size != kGemm64) return gemm_us(size, m, n, gemm_steps(k, planes), splits);
  const double each = (double)((up_to(k, 64) / 64 + splits - 1) / splits);
  return (double)((gemm_groups(size, m, n, splits) + 255) / 256) * (each * 0.97 + 1.6) + 1.5;
}
inline int terms_size(int64_t m, int64_t n, int64_t k, int planes, int largest) {  // largest: the largest tile to take
  int best = largest;
  for (int s = best + 1; s < kGemmSizes; s++)
    if (terms_us(s, m, n, k, planes, 1) < terms_us(best, m, n, k, planes, 1)) best = s;
  return best;
}

// How linear cross entropy's backward pass goes over the vocabulary.
struct LcePlan {
  int64_t dp;      // width of a row of terms
  int64_t rows_p;  // rows of P: N up to a multiple of 256 (64 for up to 64 rows), whole tiles of size_p
  int64_t piece;   // columns of P, a multiple of 256
  int splits;      // of the vocabulary in dH's product
  int size_p, size_h, size_w;  // tiles of the three products
};

constexpr int64_t kFewRows = 64;

// The splits and tiles of dH's product (d x N, over a piece of the vocabulary): its tiles are
// few, so the piece is split until they fill the chip, as long as a split's sums (written,
// and read but for the first piece, at about 4 TB/s) cost less than idle CUs.
inline double lce_split(LcePlan& p, int64_t N, int64_t piece, int planes) {
  static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64};
  double least = 1e30;
  for (int s : kSplits) {
    if (s > 1 && s * 2 > piece / 64) break;
    for (int size = gemm_largest(planes); size < kGemmSizes; size++) {
      const double us = terms_us(size, p.dp, N, piece, planes, s) + (double)s * (double)N * (double)p.dp * 8 / 4e6;
      if (us < least) least = us, p.splits = s, p.size_h = size;
    }
  }
  return least;
}

// A piece of P takes up to 2^29 terms (1 GB, of 288): pieces of one size, as few as fit or up
// to three more, whichever the three products take least over. (8192 x 131072 x 768 in bf16,
// forward and backward: 6.9 ms in pieces of 512 MB, 6.3 of 1 GB, 6.25 of 2 GB: the products' last
// round of workgroups is a smaller part of a larger piece.)
inline LcePlan lce_plan(int64_t N, int64_t V, int64_t d, int planes) {
  LcePlan best = {};
  const int64_t dp = up_to(d > 0 ? d : 8, 8);
  const int largest = gemm_largest(planes);
  const int64_t rows_p = N <= kFewRows ? kFewRows : up_to(N, 256);
  const int64_t tiles = up_to(V, 256) / 256;
  int64_t most = ((int64_t)1 << 29) / planes / rows_p / 256;
  most = most < 1 ? 1 : most > tiles ? tiles : most;
  const int64_t fewest = (tiles + most - 1) / most;
  double least = 1e30;
  for (int64_t n = fewest; n <= fewest + (fewest > 1 ? 3 : 0) && n <= tiles; n++) {
    LcePlan p = {};
    p.dp = dp;
    p.rows_p = rows_p;
    p.piece = (tiles + n - 1) / n * 256;
    // P's product stores whole tiles: none taller than P, whatever the times say.
    p.size_p = terms_size(p.piece, N, dp, planes, rows_p % gemm_side(largest) == 0 ? largest : kGemm64);
    p.size_w = terms_size(dp, p.piece, N, planes, largest);
    const double us = terms_us(p.size_p, p.piece, N, dp, planes, 1) + terms_us(p.size_w, dp, p.piece, N, planes, 1) + lce_split(p, N, p.piece, planes);
    const double all = us * (double)((tiles * 256 + p.piece - 1) / p.piece);
    if (all < least) least = all, best = p;
  }
  return best;
}

// Whether a product of one plane takes two 64-steps with one wait: where there are no more workgroups than LDS then has room
// for. Rows of weights in turn, bf16, one step a wait / two: 256 tiles of 128 over 2048, 29.5 / 23.6 us; 112 of 64 over 1024, 11.6 /
// 8.2; 512 of 64 over 4096, 41.8 / 31.0. With k outside, 256 of 128 over 1024: 20.8 / 17.6.
inline bool product_deep(int size, int64_t m, int64_t n, int64_t splits) {
  if (size == kGemm256) return false;
  return gemm_groups(size, m, n, splits) <= (size == kGemm128 ? 256 : 512);
}

// Microseconds of a product of m x n over k that may take two steps a wait.
inline double product_us(int size, int64_t m, int64_t n, int64_t k, int planes, int64_t splits) {
  if (planes != 1 || !product_deep(size, m, n, splits)) return terms_us(size, m, n, k, planes, splits);
  const double each = (double)((up_to(k, 64) / 64 + splits - 1) / splits);
  return size == kGemm128 ? each * 0.7 + 5.0 : each * (gemm_groups(size, m, n, splits) <= 256 ? 0.42 : 0.57) + 3.5;
}
inline int product_size(int64_t m, int64_t n, int64_t k, int planes) {
  int best = gemm_largest(planes);
  for (int s = best + 1; s < kGemmSizes; s++)
    if (product_us(s, m, n, k, planes, 1) < product_us(best, m, n, k, planes, 1)) best = s;
  return best;
}

// Tiles and splits of k of a product of m x n whose sums go to 16 bits at once, or through fp32 and another kernel where that
// is shorter: splits fill the chip where tiles are few. A split's sums are written and read at about 4 TB/s, and the
// second kernel takes 4 us. (500 x 256 over 1408 in three terms, a wait a product: 53 us whole, 17 in eight splits.)
struct GemmSplit {
  int size, splits;
};
inline GemmSplit gemm_split(int64_t m, int64_t n, int64_t k, int planes) {
  static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32};
  GemmSplit best = {};
  double least = 1e30;
  for (int s : kSplits) {
    if (s > 1 && s * 2 > up_to(k, 64) / 64) break;
    for (int size = gemm_largest(planes); size < kGemmSizes; size++) {
      const double us = product_us(size, m, n, k, planes, s) + (s > 1 ? (double)s * (double)m * (double)n * 8 / 4e6 + 4.0 : 0.0);
      if (us < least) least = us, best = {size, s};
    }
  }
  return best;
}

// Whether the gated projection's forward pass takes the kernel of few tokens, whose workgroups read all of x each and
// eight columns of the weights, or the matrix product's tiles, which need rows of whole 16 bytes. Few / tiles, us, in
// bf16: 768 x 2048, 16 tokens 4.1 / 5.5, 32 tokens 4.7 / 5.5, 64 tokens 6.1 / 5.6; 1024 x 2816, 16 tokens 6.0 / 6.5, 32 tokens
// 7.9 / 6.5; 2048 x 5504, 16 tokens 13.4 / 14.6; 4096 x 11008, 1 token 34 / 28, 16 tokens 46 / 28. Rows that have to be laid out
// anew first: 1020 x 4096, 64 tokens 8.7 / 23. fp32, whose tiles take terms: 768 x 2048, 64 tokens 9.7 / 24, 128 tokens
// 16.5 / 24; 4096 x 11008, 64 tokens 221 / 450.
inline bool gated_few(int64_t N, int64_t d, int64_t F, bool f32) {
  if (f32) return N <= 128;
  if (d % 8) return N <= 64;
  const int64_t weights = 2 * d * F;
  return (N <= 16 && weights <= (int64_t)1 << 25) || (N <= 32 && weights <= (int64_t)1 << 22);
}

// Attention over packed texts (tms_train_attn_kernel.h). Numbers that tiles of `rows` rows may have: those of
// B texts, and of what stands before and behind them.
inline int64_t attn_slots(int64_t T, int64_t B, int64_t rows) { return T / rows + B + 2; }

// Whether a wave takes 32 queries (or keys) and not 16: each row that passes through LDS then serves twice
// as many, but tiles of 128 rows fill short texts badly, and few of them the chip. 16,384 tokens, 8 heads of
// 64 in bf16, forward and both backward kernels, 16 / 32: texts of 128 tokens 27, 29, 32 / 35, 38, 44 us; of 512
// 43, 48, 71 / 44, 48, 55; of 8192 414, 477, 657 / 363, 412, 526; heads of 128, texts of 512: 79, 88 / 62, 73.
// One text of 2048 tokens: 28, 29, 40 / 36, 42, 50.
inline bool attn_wide(int64_t T, int64_t B, int64_t heads) { return T >= 512 * B && T / 128 * heads >= 512; }

// Whether most texts are a tile of keys or less.
inline bool attn_short(int64_t T, int64_t B) { return T <= 64 * B; }

// Workgroups that share the heads of a tile of keys (a divisor of how many those are), where there are
// fewer than two a CU without. Their sums, in fp32, are joined by another kernel.
inline int64_t attn_parts(int64_t T, int64_t B, int64_t kv_heads, int64_t many) {
  const int64_t groups = attn_slots(T, B, 64) * kv_heads;
  int64_t parts = (512 + groups - 1) / groups;
  parts = parts < 1 ? 1 : parts > many ? many : parts;
  while (many % parts) parts++;
  return parts;
}

// Whether keys beyond a bias's reach are looked for: in texts so long that there are some. The norms' kernel and the
// other order of the tiles cost texts of 2048 tokens 6 % under a bias that reaches all of them (16,384 tokens, 8
// heads of 64: 510 us, 470 without) and save as much under slopes of 2^-1 to 2^-8 (445, 464 without); two texts of
// 8192 under 2^-0.7 to 2^-8 take 1,530 us, 2,020 without.
inline bool attn_reaches(int64_t T, int64_t B) { return T >= 2048 * B; }

}  // namespace tms
