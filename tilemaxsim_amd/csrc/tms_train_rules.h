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
  const int64_t steps = gemm_steps(piece, planes);
  double least = 1e30;
  for (int s : kSplits) {
    if (s > 1 && s * 2 > piece / 64) break;
    for (int size = gemm_largest(planes); size < kGemmSizes; size++) {
      const double us = gemm_us(size, p.dp, N, steps, s) + (double)s * (double)N * (double)p.dp * 8 / 4e6;
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
  const int64_t dp = up_to(d > 0 ? d : 8, 8), steps_d = gemm_steps(dp, planes), steps_n = gemm_steps(N, planes);
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
    p.size_p = gemm_size(p.piece, N, steps_d, rows_p % gemm_side(largest) == 0 ? largest : kGemm64);
    p.size_w = gemm_size(dp, p.piece, steps_n, largest);
    const double us = gemm_us(p.size_p, p.piece, N, steps_d, 1) + gemm_us(p.size_w, dp, p.piece, steps_n, 1) + lce_split(p, N, p.piece, planes);
    const double all = us * (double)((tiles * 256 + p.piece - 1) / p.piece);
    if (all < least) least = all, best = p;
  }
  return best;
}

}  // namespace tms
