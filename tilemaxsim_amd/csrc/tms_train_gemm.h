// The matrix product of the training operators: C[m, n] = sum_k A[m, k] B[n, k] over 16-bit
// operands with fp32 sums, either of which may lie in memory with k inside (rows of k) or
// outside (rows of m or n), and an epilogue that takes the sums from registers.
//
// Eight waves, 2 along m and 4 along n, share tiles of BM x BN with k in steps of 64; a wave
// keeps MI x NI sums of 16 x 16 (256 x 256: 128 VGPRs). A step's operands go from memory
// through registers into one of two LDS buffers, in MFMA fragment order, one barrier a step:
// the loads have a whole step's products to arrive in. Operands with k outside are read back
// with ds_read_b64_tr_b16 (in each 16 lanes, lane l receives element l % 4 of lanes
// l / 4, 4 + l / 4, 8 + l / 4, 12 + l / 4), so no transposed copy of anything is made.
//
// A 16 x 16 block of sums has lane (c, g) hold column n = c and rows m = 4 g + i: what is
// reduced over m stays in a lane, and four neighbouring m are one store.
#pragma once
#include "tms_common.h"

namespace tms {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// fp32 operands are three bf16 terms ("planes"); of the nine products of two such operands
// the six above 2^-24 of the whole are formed, small ones first.
constexpr int kTermPairs = 6;
__device__ constexpr int kTermA[kTermPairs] = {2, 0, 1, 1, 0, 0};
__device__ constexpr int kTermB[kTermPairs] = {0, 2, 1, 0, 1, 0};

struct GemmArgs {
  const uint16_t* A;
  const uint16_t* B;
  int64_t aplane, bplane;  // elements between planes
  int32_t lda, ldb;        // elements between rows (multiples of 8)
  int32_t M, N, K;         // k inside: K is a multiple of 8, or zeros follow it up to one; outside: M (N) is
  int32_t pairs;           // 1, or kTermPairs
  int32_t splits, per;     // splits of k, 64-steps each
  int32_t tm, tn;          // tiles
};

constexpr int kGemmThreads = 512;
constexpr int kOuterBlock = 2080;  // bytes of 16 columns x 64 k: 32 more than they need, so that blocks fall on other banks

constexpr int gemm_lds(int rows, bool outer) { return outer ? rows / 16 * kOuterBlock : rows * 128; }

// One operand's share of a step: R rows (or columns) x 64 k.
template <int R, bool OUTER>
struct GemmTile {
  static constexpr int L = R / 64;  // 16-byte loads a thread
  u32x4 reg[L];
  int32_t off[L];  // elements from the tile's first, at k = 0 of the step
  int16_t kk[L];   // k within the step
  int32_t place[L];

  __device__ __forceinline__ void init(int ld, int limit) {  // limit: rows (columns) of the tile that exist
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < L; i++) {
      if constexpr (OUTER) {
        const int idx = i * kGemmThreads + (int)threadIdx.x, k = idx / (R / 8), c = idx % (R / 8);
        kk[i] = (int16_t)k;
        off[i] = k * ld + (c * 8 < limit ? c * 8 : 0);
        place[i] = (c >> 1) * kOuterBlock + (k >> 5) * 1024 + ((k >> 2) & 1) * 512 + (((k >> 3) & 3) * 16 + (k & 3) * 4 + 2 * (c & 1)) * 8;
      } else {
        const int f = i * 8 + wave, row = (f >> 1) * 16 + (lane & 15);
        kk[i] = (int16_t)((f & 1) * 32 + (lane >> 4) * 8);
        off[i] = (row < limit ? row : limit - 1) * ld + kk[i];
        place[i] = f * 1024 + lane * 16;
      }
    }
  }
  // base: the tile's first element at this step's first k; left: how many k there are from it on
  __device__ __forceinline__ void load(const uint16_t* base, int ld, int left) {
    if (left >= 64) {
#pragma unroll
      for (int i = 0; i < L; i++) reg[i] = *(const u32x4*)(base + off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < L; i++) {
        const bool in = kk[i] < left;
        const u32x4 v = *(const u32x4*)(base + (in ? off[i] : off[i] - (OUTER ? kk[i] * ld : kk[i])));
        reg[i] = in ? v : u32x4{0u, 0u, 0u, 0u};
      }
    }
  }
  __device__ __forceinline__ void put(uint8_t* lds) const {
#pragma unroll
    for (int i = 0; i < L; i++) *(u32x4*)(lds + place[i]) = reg[i];
  }
  // the fragment of 16 rows and 32 k
  __device__ static __forceinline__ u32x4 frag(const uint8_t* lds, int block, int ks, int lane) {
    if constexpr (OUTER) {
      typedef __attribute__((address_space(3))) s16x4* LP;
      const uint8_t* p = lds + block * kOuterBlock + ks * 1024 + lane * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(p + 512));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      return u32x4{a[0], a[1], b[0], b[1]};
    } else {
      return *(const u32x4*)(lds + (block * 2 + ks) * 1024 + lane * 16);
    }
  }
};

// Tile numbers in the order of the launch: each XCD takes a run of its own (workgroups go to
// the XCDs in turn), and a run goes over four m tiles for each n tile, so that the workgroups
// that an XCD holds at a time share rows of both operands in its L2.
__device__ __forceinline__ bool gemm_tile_of(const GemmArgs& a, int& m, int& n) {
  const int total = a.tm * a.tn, each = (total + 7) / 8;
  const int id = ((int)blockIdx.x % 8) * each + (int)blockIdx.x / 8;
  if ((int)blockIdx.x / 8 >= each || id >= total) return false;
  const int wide = 4 * a.tn, first = id / wide * 4, in = id % wide;
  const int rows = a.tm - first < 4 ? a.tm - first : 4;
  m = first + in % rows;
  n = in / rows;
  return true;
}
static inline unsigned gemm_grid(int tm, int tn) { return (unsigned)(((int64_t)tm * tn + 7) / 8 * 8); }

template <int DT, int MI, int NI, bool AO, bool BO, class Epi>
__global__ __launch_bounds__(kGemmThreads, 2) void train_gemm_kernel(GemmArgs a, Epi epi) {
  constexpr int BM = 32 * MI, BN = 64 * NI;
  constexpr int ASZ = gemm_lds(BM, AO), BSZ = gemm_lds(BN, BO);
  extern __shared__ uint8_t gemm_mem[];
  int tm, tn;
  if (!gemm_tile_of(a, tm, tn)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = tm * BM, n0 = tn * BN;

  GemmTile<BM, AO> ta;
  GemmTile<BN, BO> tb;
  ta.init(a.lda, a.M - m0);
  tb.init(a.ldb, a.N - n0);
  const int k0 = (int)blockIdx.y * a.per;
  const int steps_all = (a.K + 63) / 64;
  const int nk = k0 + a.per < steps_all ? a.per : steps_all - k0;
  const int steps = nk > 0 ? nk * a.pairs : 0;
  const uint16_t* A = a.A + (AO ? (int64_t)m0 : (int64_t)m0 * a.lda);
  const uint16_t* B = a.B + (BO ? (int64_t)n0 : (int64_t)n0 * a.ldb);
  int pair = kTermPairs - a.pairs, kt = 0;  // the step that is loaded next
  auto load = [&]() {
    const int64_t k = (int64_t)(k0 + kt) * 64;
    const int left = a.K - (int)k;
    ta.load(A + kTermA[pair] * a.aplane + (AO ? k * a.lda : k), a.lda, left);
    tb.load(B + kTermB[pair] * a.bplane + (BO ? k * a.ldb : k), a.ldb, left);
    if (++kt == nk) {
      kt = 0;
      pair++;
    }
  };

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NI; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (steps > 0) {
    load();
    ta.put(gemm_mem);
    tb.put(gemm_mem + ASZ);
    if (steps > 1) load();
  }
  __syncthreads();
  int buf = 0;
  for (int t = 0; t < steps; t++) {
    const uint8_t* la = gemm_mem + buf * (ASZ + BSZ);
    const uint8_t* lb = la + ASZ;
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      u32x4 fa[MI], fb[NI];
#pragma unroll
      for (int j = 0; j < NI; j++) fb[j] = GemmTile<BN, BO>::frag(lb, wn * NI + j, ks, lane);
#pragma unroll
      for (int i = 0; i < MI; i++) fa[i] = GemmTile<BM, AO>::frag(la, wm * MI + i, ks, lane);
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) acc[i][j] = mfma16x16x32<DT>(fa[i], fb[j], acc[i][j]);
    }
    if (t + 1 < steps) {
      uint8_t* to = gemm_mem + (buf ^ 1) * (ASZ + BSZ);
      ta.put(to);
      tb.put(to + ASZ);
    }
    if (t + 2 < steps) load();
    __syncthreads();
    buf ^= 1;
  }
  epi(acc, m0 + wm * MI * 16, n0 + wn * NI * 16, (int)blockIdx.y);
}

template <int DT, int MI, int NI, bool AO, bool BO, class Epi>
static int run_gemm(GemmArgs a, const Epi& epi, hipStream_t st, const char* what) {
  a.tm = (a.M + 32 * MI - 1) / (32 * MI);
  a.tn = (a.N + 64 * NI - 1) / (64 * NI);
  const int steps = (a.K + 63) / 64;
  a.per = (steps + a.splits - 1) / a.splits;
  const size_t lds = 2 * (size_t)(gemm_lds(32 * MI, AO) + gemm_lds(64 * NI, BO));
  hipLaunchKernelGGL((train_gemm_kernel<DT, MI, NI, AO, BO, Epi>), dim3(gemm_grid(a.tm, a.tn), (unsigned)a.splits), dim3(kGemmThreads),
                     lds, st, a, epi);
  return check_launch(what);
}

}  // namespace tms
