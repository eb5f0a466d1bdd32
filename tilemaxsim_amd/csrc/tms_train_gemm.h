// The matrix product of the training operators: C[m, n] = sum_k A[m, k] B[n, k] over 16-bit
// operands with fp32 sums, either of which may lie in memory with k inside (rows of k) or
// outside (rows of m or n), and an epilogue that takes the sums from registers.
//
// Eight waves, 2 along m and 4 along n, share tiles of BM x BN with k in steps of 64; a wave
// keeps MI x NI sums of 16 x 16 (256 x 256: 128 VGPRs). The next step's operands go from
// memory straight to one of two LDS buffers while this step's are multiplied: a wave first
// reads all its fragments of the step, then issues the loads (an LDS read behind them would
// wait for them), then multiplies, waits for its loads and meets the others: one barrier a
// step. Both kinds of operand come in units of 1 KB, eight rows of 128 bytes (whole lines),
// whose 16-byte pieces are stored permuted so that the fragment reads fall evenly on the
// LDS banks:
//  * k inside: rows are m (n); piece p of row r is stored at p ^ (r % 8). A fragment is one
//    ds_read_b128 a lane.
//  * k outside: rows are k, 64 of m (n); piece p of row r of the unit of k / 8 = u is stored
//    at p ^ (4 (r / 2 % 2) + 2 (u % 2) + u / 2 % 2), which spreads each half of a wave over all
//    banks (4 (r / 2 % 2) + u % 4 spreads the wave but not its halves: twice the LDS cycles, and
//    7 % of the product's time). A fragment is two ds_read_b64_tr_b16: in each 16 lanes,
//    lane l receives element l % 4 of lanes l / 4, 4 + l / 4, 8 + l / 4 and 12 + l / 4, so no
//    transposed copy of anything is made.
//
// Tiles of 256 x 256 with their epilogues, 8192^3 in bf16, random data: 1.30 PFLOP/s with k inside,
// 1.22 outside in one operand, 1.20 in both (the library's products: 1.61, 1.41, 1.21); 4096^3, one
// round of workgroups: 1.16, 1.01, 0.91. At 8192 x 131072 x 768 the matrix cores are busy for 40 to 54 %
// of the cycles, at 1.9 to 2.2 GHz (power), and waves wait for operands for a third to a half of
// theirs. Smaller tiles are bound by the operands' way: 10 TB/s into LDS over the chip.
//
// A 16 x 16 block of sums has lane (c, g) hold column n = c and rows m = 4 g + i: what is
// reduced over m stays in a lane, and four neighbouring m are one store.
#pragma once
#include "tms_common.h"

namespace tms {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// fp32 operands are three bf16 terms ("planes"); of the nine products of two such operands
// the six above 2^-24 of the whole are formed. A 64-step of k takes them in the order (2, 0),
// (1, 0), (1, 1), (0, 1), (0, 2), (0, 0): each differs from the one before in one operand, whose tile
// alone is loaded and read from LDS, so that the six cost seven tiles and not twelve.
struct GemmArgs {
  const uint16_t* A;
  const uint16_t* B;
  int64_t aplane, bplane;  // elements between planes
  int32_t lda, ldb;        // elements between rows (multiples of 8)
  int32_t M, N, K;         // k inside: K is a multiple of 8, or zeros follow it up to one; outside: M (N) is
  int32_t splits, per;     // splits of k, 64-steps each
  int32_t tm, tn;          // tiles
};

constexpr int kGemmThreads = 512;

// Epilogues are called with the wave's sums, its first m and n, its split, and LDS of its
// own: kRowBytes for each of its columns n (0: none).

// What stands for the elements past the end of k.
__device__ const u32x4 kGemmZeros = {0u, 0u, 0u, 0u};

// One operand's share of a step: R rows (or columns) x 64 k, R / 8 units.
template <int R, bool OUTER>
struct GemmTile {
  static constexpr int L = R / 64;  // units a wave loads (R is a multiple of 64)
  uint32_t off[L];                  // bytes from the tile's first element, at k = 0 of the step
  int32_t kk;                       // k within the step, of unit 0 (k outside: + 8 a unit, see load)

  // Units go to the waves in turn: wave w loads units w, w + 8, ...: k inside, rows 8 unit ..;
  // outside, k 8 (unit % 8) .. of columns 64 (unit / 8) ..
  __device__ __forceinline__ void init(int ld, int limit, int lane, int wave) {  // limit: rows (columns) that exist
    const int r = lane >> 3, slot = lane & 7;
    if constexpr (OUTER) {
      const int p = slot ^ (4 * ((r >> 1) & 1) + 2 * (wave & 1) + ((wave >> 1) & 1));  // unit % 8 is the wave
      kk = 8 * wave + r;
#pragma unroll
      for (int i = 0; i < L; i++) {
        const int col = 64 * i + 8 * p;
        off[i] = 2u * (uint32_t)(kk * ld + (col < limit ? col : 0));
      }
    } else {
      kk = 8 * (slot ^ r);
#pragma unroll
      for (int i = 0; i < L; i++) {
        const int row = (i * 8 + wave) * 8 + r;
        off[i] = 2u * (uint32_t)((row < limit ? row : limit - 1) * ld + kk);
      }
    }
  }
  // base: the tile's first element at this step's first k; left: how many k there are from it on
  __device__ __forceinline__ void load(const uint16_t* base, int left, uint8_t* lds, int wave) const {
    typedef __attribute__((address_space(1))) const void* GP;
    typedef __attribute__((address_space(3))) void* LP;
    const uint8_t* from = (const uint8_t*)base;
    if (left >= 64) {
#pragma unroll
      for (int i = 0; i < L; i++) __builtin_amdgcn_global_load_lds((GP)(from + off[i]), (LP)(lds + (i * 8 + wave) * 1024), 16, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < L; i++) {
        const uint8_t* p = kk < left ? from + off[i] : (const uint8_t*)&kGemmZeros;
        __builtin_amdgcn_global_load_lds((GP)p, (LP)(lds + (i * 8 + wave) * 1024), 16, 0, 0);
      }
    }
  }
  // The fragment of 16 rows and 32 k. at: this lane's part of the address (frag_at), which
  // the unrolled block and ks only add constants to.
  __device__ static __forceinline__ u32x4 frag(const uint8_t* lds, int block, int ks, int lane) {
    if constexpr (OUTER) {
      typedef __attribute__((address_space(3))) s16x4* LP;
      const int g = lane >> 4, j = (lane >> 2) & 3, q = lane & 3;
      // rows 4 h + j of unit (block / 4, 4 ks + g)
      const int x = 4 * ((j >> 1) & 1) + 2 * (g & 1) + (g >> 1), piece = ((block & 3) * 2 + (q >> 1)) ^ x;
      const uint8_t* p = lds + ((block >> 2) * 8 + ks * 4 + g) * 1024 + j * 128 + piece * 16 + (q & 1) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(p + 512));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      return u32x4{a[0], a[1], b[0], b[1]};
    } else {
      const int r = lane & 15, g = lane >> 4;
      return *(const u32x4*)(lds + (block * 2 + (r >> 3)) * 1024 + (r & 7) * 128 + (((ks * 4 + g) ^ (r & 7)) * 16));
    }
  }
};

// Tile numbers in the order of the launch: each XCD takes a run of its own (workgroups go to
// the XCDs in turn), and a run goes over four m tiles for each n tile, so that the workgroups
// that an XCD holds at a time share rows of both operands in its L2. One axis of a launch takes
// 2^32 threads: workgroups beyond kAxisTiles (a multiple of 8) stand in further rows of it.
constexpr int kAxisTiles = 1 << 22;
__device__ __forceinline__ bool gemm_tile_of(const GemmArgs& a, int& m, int& n) {
  const int total = a.tm * a.tn, each = (total + 7) / 8;
  const int at = (int)blockIdx.z * kAxisTiles + (int)blockIdx.x;
  const int id = (at % 8) * each + at / 8;
  if (at / 8 >= each || id >= total) return false;
  const int wide = 4 * a.tn, first = id / wide * 4, in = id % wide;
  const int rows = a.tm - first < 4 ? a.tm - first : 4;
  m = first + in % rows;
  n = in / rows;
  return true;
}
static inline dim3 gemm_grid(int tm, int tn, int splits) {
  const int64_t n = ((int64_t)tm * tn + 7) / 8 * 8;
  return dim3((unsigned)(n < kAxisTiles ? n : kAxisTiles), (unsigned)splits, (unsigned)((n + kAxisTiles - 1) / kAxisTiles));
}

template <bool V>
struct More {
  static constexpr bool value = V;
};

// PL: planes of both operands, 1 or 3.
template <int DT, int PL, int MI, int NI, bool AO, bool BO, class Epi>
__global__ __launch_bounds__(kGemmThreads, MI == 8 ? 2 : 4) void train_gemm_kernel(GemmArgs a, Epi epi) {
  constexpr int BM = 32 * MI, BN = 64 * NI;
  constexpr int ASZ = BM * 128, BSZ = BN * 128;
  extern __shared__ __attribute__((aligned(1024))) uint8_t gemm_mem[];
  int tm, tn;
  if (!gemm_tile_of(a, tm, tn)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = tm * BM, n0 = tn * BN;

  GemmTile<BM, AO> ta;
  GemmTile<BN, BO> tb;
  ta.init(a.lda, a.M - m0, lane, wave);
  tb.init(a.ldb, a.N - n0, lane, wave);
  const int k0 = (int)blockIdx.y * a.per;
  const int steps_all = (a.K + 63) / 64;
  const int nk = k0 + a.per < steps_all ? a.per : steps_all - k0;
  const uint16_t* A = a.A + (AO ? (int64_t)m0 : (int64_t)m0 * a.lda);
  const uint16_t* B = a.B + (BO ? (int64_t)n0 : (int64_t)n0 * a.ldb);
  uint8_t* const lds_a = gemm_mem;
  uint8_t* const lds_b = gemm_mem + 2 * ASZ;
  auto load_a = [&](int buf, int step, int plane) {
    const int64_t k = (int64_t)(k0 + step) * 64;
    ta.load(A + plane * a.aplane + (AO ? k * a.lda : k), a.K - (int)k, lds_a + buf * ASZ, wave);
  };
  auto load_b = [&](int buf, int step, int plane) {
    const int64_t k = (int64_t)(k0 + step) * 64;
    tb.load(B + plane * a.bplane + (BO ? k * a.ldb : k), a.K - (int)k, lds_b + buf * BSZ, wave);
  };
  auto meet = [&]() {  // this wave's loads are in LDS, then everyone's
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
  };

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NI; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 fa[2][MI], fb[2][NI];
  auto read_a = [&](int buf) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int i = 0; i < MI; i++) fa[ks][i] = GemmTile<BM, AO>::frag(lds_a + buf * ASZ, wm * MI + i, ks, lane);
  };
  auto read_b = [&](int buf) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int j = 0; j < NI; j++) fb[ks][j] = GemmTile<BN, BO>::frag(lds_b + buf * BSZ, wn * NI + j, ks, lane);
  };
  // The products of the fragments; `next`: the next step's loads, which go out once some of the
  // products are issued (behind the loads, a product would wait for all of the wave's LDS
  // reads together): a quarter of them, or an eighth with k outside in both operands (8192^3 in
  // bf16, an eighth / a quarter: 1.25 / 1.28 PFLOP/s with k inside, 1.21 / 1.19 outside in both; outside
  // in one, 1.24 / 1.22 on one card and 1.23 / 1.29 on another). The scheduler would otherwise move
  // products behind the wait for the loads.
  constexpr int kBefore = AO && BO ? MI / 4 : MI / 2;
  auto multiply = [&](auto&& next) {
    auto products = [&](int ks, int i0, int i1) {
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++)
          if (i >= i0 && i < i1) acc[i][j] = mfma16x16x32<DT>(fa[ks][i], fb[ks][j], acc[i][j]);
    };
    products(0, 0, kBefore);
    __builtin_amdgcn_sched_barrier(0);
    next();
    __builtin_amdgcn_sched_barrier(0);
    products(0, kBefore, MI);
    products(1, 0, MI);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (nk > 0) {
    load_a(0, 0, PL - 1);
    load_b(0, 0, 0);
    meet();
  }
  int buf = 0;
  auto step = [&](int t, auto more) {
    read_b(PL == 3 ? 0 : buf);
    read_a(buf);
    if constexpr (PL == 3) {  // the fragments of the tile that stays, stay
      multiply([&]() { load_a(buf ^ 1, t, 1); });
      meet();
      read_a(buf ^ 1);
      multiply([&]() { load_b(1, t, 1); });
      meet();
      read_b(1);
      multiply([&]() { load_a(buf, t, 0); });
      meet();
      read_a(buf);
      multiply([&]() { load_b(0, t, 2); });
      meet();
      read_b(0);
      multiply([&]() { load_b(1, t, 0); });
      meet();
      read_b(1);
    }
    multiply([&]() {
      if constexpr (decltype(more)::value) {
        load_a(buf ^ 1, t + 1, PL - 1);
        load_b(PL == 3 ? 0 : buf ^ 1, t + 1, 0);
      }
    });
    if constexpr (decltype(more)::value) meet();
    buf ^= 1;
  };
  for (int t = 0; t + 1 < nk; t++) step(t, More<true>());
  if (nk > 0) step(nk - 1, More<false>());
  if constexpr (Epi::kRowBytes > 0) __syncthreads();  // the operands' LDS is the epilogue's
  epi(acc, m0 + wm * MI * 16, n0 + wn * NI * 16, (int)blockIdx.y, gemm_mem + wave * (NI * 16 * Epi::kRowBytes));
}

template <int DT, int PL, int MI, int NI, bool AO, bool BO, class Epi>
static int run_gemm(GemmArgs a, const Epi& epi, hipStream_t st, const char* what) {
  a.tm = (a.M + 32 * MI - 1) / (32 * MI);
  a.tn = (a.N + 64 * NI - 1) / (64 * NI);
  if ((int64_t)a.tm * a.tn > 1 << 30) return fail(TMS_ERR_UNSUPPORTED, "%s: %d x %d tiles are too many", what, a.tm, a.tn);
  const int steps = (a.K + 63) / 64;
  a.per = (steps + a.splits - 1) / a.splits;
  size_t lds = 2 * (size_t)(32 * MI + 64 * NI) * 128;
  if (lds < (size_t)8 * NI * 16 * Epi::kRowBytes) lds = (size_t)8 * NI * 16 * Epi::kRowBytes;
  hipLaunchKernelGGL((train_gemm_kernel<DT, PL, MI, NI, AO, BO, Epi>), gemm_grid(a.tm, a.tn, a.splits), dim3(kGemmThreads),
                     lds, st, a, epi);
  return check_launch(what);
}

}  // namespace tms
