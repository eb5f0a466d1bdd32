// MaxSim of query and document batches for training: scores with the position of every
// maximum, and the gradients of both sides.
//
//   score[q, b] = sum_i s_i,  s_i = max_j <Q[q, i], D[b, j]>  (real tokens i, j),   a[q, b, i] = the first j with s_i
//   dQ[q, i]    = sum_b G[q, b] D[b, a[q, b, i]]
//   dD[b, j]    = sum_{q, i: a[q, b, i] = j} G[q, b] Q[q, i]
//
// Pairs are every query with every document, or (nway > 0) each query with its own nway
// documents. Positions are uint16, [document][query][token], kNone where a token or the
// whole document is masked: 2 bytes a maximum instead of the similarities' 2 * Nd or more.
#include "tms_common.h"

namespace tms {

constexpr int kNone = 0xffff;       // no position: nothing flows back
constexpr int kMaxTokens = 0xffff;  // a document's tokens: positions 0 .. 65,534
constexpr int kStage = 64;          // document tokens per LDS stage
constexpr int kMaskWords = 1024;    // 64-token mask words of a workgroup's documents

struct PairsArgs {
  const uint8_t* Q;      // [plane][nQ * nq][d] 16-bit terms, d a multiple of 32, 16-byte aligned
  const uint8_t* D;      // [plane][B * nd][d]
  const uint8_t* qmask;  // (nQ, nq) bytes, or null
  const uint8_t* dmask;  // (B, nd) bytes, or null
  float* scores;         // (nQ, B), or (nQ, nway)
  uint16_t* arg;         // [pair][nqp], or null
  int64_t B, qplane, dplane;  // planes' strides in bytes
  int32_t nQ, nq, nqp, nd, d, nway;
  int32_t nbq, qpw, docs_per_wg;  // shared form: 32-token blocks a query, queries a wave, documents a workgroup
};

__device__ __forceinline__ int64_t score_at(const PairsArgs& a, int q, int64_t b) {
  return a.nway ? b : (int64_t)q * a.B + b;
}
__device__ __forceinline__ int64_t arg_at(const PairsArgs& a, int q, int64_t b) {
  return (a.nway ? b : b * a.nQ + q) * a.nqp;
}

// Running maximum and its token over one 16-token tile: lane (c, g) sees query token c
// against tokens base + 4 g + i. A strict comparison keeps the first of equal ones, as
// tokens rise. Three VALU instructions a value; at d = 128 the four MFMAs behind a value's
// 16 x 16 block take longer than that, and the two waves of a SIMD overlap them.
struct Best {
  float v;
  int at;
};
__device__ __forceinline__ void take(Best& r, const f32x4& s, int first) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const bool up = s[i] > r.v;
    r.v = up ? s[i] : r.v;
    r.at = up ? first + i : r.at;
  }
}
__device__ __forceinline__ Best better(Best x, Best y) {
  const bool up = y.v > x.v || (y.v == x.v && y.at < x.at);
  return {up ? y.v : x.v, up ? y.at : x.at};
}
// Over the four 16-lane rows; every lane receives the result.
__device__ __forceinline__ Best across_rows(Best r) {
  const unsigned v = __builtin_bit_cast(unsigned, r.v), i = (unsigned)r.at;
  const auto v0 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const auto i0 = __builtin_amdgcn_permlane32_swap(i, i, false, false);
  r = better({__builtin_bit_cast(float, (unsigned)v0[0]), (int)i0[0]}, {__builtin_bit_cast(float, (unsigned)v0[1]), (int)i0[1]});
  const unsigned w = __builtin_bit_cast(unsigned, r.v), j = (unsigned)r.at;
  const auto v1 = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  const auto i1 = __builtin_amdgcn_permlane16_swap(j, j, false, false);
  return better({__builtin_bit_cast(float, (unsigned)v1[0]), (int)i1[0]}, {__builtin_bit_cast(float, (unsigned)v1[1]), (int)i1[1]});
}

// Values of masked tokens never win: bit t of `live` is token base + t of the tile.
__device__ __forceinline__ void mask_tile(f32x4& s, uint32_t live, int g) {
#pragma unroll
  for (int i = 0; i < 4; i++) s[i] = (live >> (4 * g + i)) & 1u ? s[i] : -__builtin_inff();
}

// fp32 products from three bf16 terms a side: the six pairs whose product is above 2^-24
// of the whole, small ones first.
__device__ constexpr int kPairQ[6] = {2, 0, 1, 1, 0, 0};
__device__ constexpr int kPairD[6] = {0, 2, 1, 0, 1, 0};

// ---------------------------------------------------------------- one pair a workgroup

// Four waves take a document's 16-token tiles in turn, and join through LDS: the form of
// small calls and of documents that one query alone sees, whose tokens are read once and
// straight into MFMA fragments. KS > 0: d = 32 KS, the query block's fragments in registers.
// KS = 0: any d and any number of planes, fragments read as they are used.
template <int DT, int KS, int PL>
__global__ __launch_bounds__(256) void pairs_direct_kernel(PairsArgs a) {
  __shared__ Best joined[4][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t b = blockIdx.x;
  const int q = a.nway ? (int)(b / a.nway) : (int)blockIdx.y;
  const int64_t drow = b * a.nd, qrow = (int64_t)q * a.nq;
  const int64_t width = (int64_t)a.d * 2;
  const int tiles = (a.nd + 15) >> 4;
  float total = 0.f;
  bool some = false;  // a real document token, in any lane of the workgroup
  for (int blk = 0; blk < a.nbq; blk++) {
    bool real[2];
    u32x4 qf[KS ? KS : 1][2];
    const uint8_t* qp[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int tok = blk * 32 + 16 * h + r;
      real[h] = tok < a.nq && (!a.qmask || a.qmask[qrow + tok] != 0);
      qp[h] = a.Q + (qrow + (tok < a.nq ? tok : 0)) * width + 16 * g;
      if constexpr (KS > 0) {
#pragma unroll
        for (int s = 0; s < KS; s++) {
          const u32x4 v = *(const u32x4*)(qp[h] + 64 * s);
          qf[s][h] = real[h] ? v : u32x4{0u, 0u, 0u, 0u};
        }
      }
    }
    Best best[2] = {{-__builtin_inff(), kNone}, {-__builtin_inff(), kNone}};
    for (int t = wave; t < tiles; t += 4) {
      int tok = t * 16 + r;
      const bool in = tok < a.nd;
      tok = in ? tok : a.nd - 1;
      const bool live = in && (!a.dmask || a.dmask[drow + tok] != 0);
      const uint32_t bits = (uint32_t)__ballot(live) & 0xffffu;
      if (bits == 0) continue;
      some = true;
      const uint8_t* dp = a.D + (drow + tok) * width + 16 * g;
      f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if constexpr (KS > 0) {
        u32x4 df[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) df[s] = *(const u32x4*)(dp + 64 * s);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int h = 0; h < 2; h++) acc[h] = mfma16x16x32<DT>(df[s], qf[s][h], acc[h]);
      } else {
        for (int p = PL == 1 ? 5 : 0; p < 6; p++)
          for (int s = 0; s * 64 < width; s++) {
            const u32x4 df = *(const u32x4*)(dp + kPairD[p] * a.dplane + 64 * s);
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const u32x4 v = *(const u32x4*)(qp[h] + kPairQ[p] * a.qplane + 64 * s);
              acc[h] = mfma16x16x32<DT>(df, v, acc[h]);
            }
          }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (bits != 0xffffu) mask_tile(acc[h], bits, g);
        take(best[h], acc[h], t * 16 + 4 * g);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      best[h] = across_rows(best[h]);
      if (!real[h]) best[h] = {0.f, kNone};
      if (g == 0) joined[wave][16 * h + r] = best[h];
    }
    __syncthreads();
    if (wave == 0) {
      Best x = {0.f, kNone};
      if (lane < 32) {
        x = joined[0][lane];
#pragma unroll
        for (int w = 1; w < 4; w++) x = better(x, joined[w][lane]);
        const int tok = blk * 32 + lane;
        if (a.arg && tok < a.nqp) a.arg[arg_at(a, q, b) + tok] = (uint16_t)x.at;
      }
      float s = x.v;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor(s, o);
      total += s;
    }
    __syncthreads();
  }
  some = __syncthreads_or(some);
  if (threadIdx.x == 0) a.scores[score_at(a, q, b)] = some ? total : -__builtin_inff();
}

// ---------------------------------------------------------------- shared document tiles

// Eight waves hold up to 8 NB blocks of 32 query tokens in registers and walk the same
// documents: each 64-token stage comes from memory once, through registers into one of two
// LDS buffers in MFMA fragment order (the reads are whole and conflict-free), so a token
// costs 1 / (8 NB) of a load per block. Bound by the matrix cores and the maxima's VALU work.
// One barrier a stage: a stage is written to the buffer that every wave left before the
// last one. Masks become 64-bit words in LDS first; stages of padding are never loaded.
// Whole queries belong to a wave, so a score is summed in one place and in one order.
template <int DT, int KS, int NB, int PL>
__global__ __launch_bounds__(512, 2) void pairs_shared_kernel(PairsArgs a) {
  constexpr int FS = 4 * PL * KS;  // fragments of a stage
  constexpr int LD = (FS + 7) / 8;  // fragments a wave loads
  __shared__ u32x4 ring[2][FS][64];
  __shared__ uint64_t words[kMaskWords];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = lane & 15, g = lane >> 4;
  const int64_t b0 = (int64_t)blockIdx.x * a.docs_per_wg;
  const int ndocs = (int)(b0 + a.docs_per_wg < a.B ? a.docs_per_wg : a.B - b0);
  const int stages = (a.nd + kStage - 1) / kStage;
  const int64_t width = (int64_t)a.d * 2;
  const int q0 = ((int)blockIdx.y * 8 + wave) * a.qpw;  // this wave's first query

  for (int w = wave; w < ndocs * stages; w += 8) {
    const int doc = w / stages, tok = (w - doc * stages) * kStage + lane;
    const bool live = tok < a.nd && (!a.dmask || a.dmask[(b0 + doc) * a.nd + tok] != 0);
    const uint64_t bits = __ballot(live);
    if (lane == 0) words[w] = bits;
  }

  u32x4 qf[NB][PL][KS][2];
  uint32_t real = 0;  // bit 2 j + h: this lane's token of half h of block j
#pragma unroll
  for (int j = 0; j < NB; j++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int q = q0 + j / a.nbq, tok = (j % a.nbq) * 32 + 16 * h + r;
      const bool in = j < a.qpw * a.nbq && q < a.nQ && tok < a.nq;
      const int64_t row = in ? (int64_t)q * a.nq + tok : 0;
      const bool on = in && (!a.qmask || a.qmask[row] != 0);
      real |= (on ? 1u : 0u) << (2 * j + h);
#pragma unroll
      for (int p = 0; p < PL; p++)
#pragma unroll
        for (int s = 0; s < KS; s++) {
          const u32x4 v = *(const u32x4*)(a.Q + p * a.qplane + row * width + 64 * s + 16 * g);
          qf[j][p][s][h] = on ? v : u32x4{0u, 0u, 0u, 0u};
        }
    }
  __syncthreads();

  const int total = ndocs * stages;
  // the first stage from w on with a real token; `total` past the end
  auto seek = [&](int w) -> int {
    while (w < total && words[w] == 0) w++;
    return __builtin_amdgcn_readfirstlane(w);
  };
  u32x4 stg[LD];
  auto load = [&](int w) {
    if (w >= total) return;
    const int doc = w / stages, t0 = (w - doc * stages) * kStage;
#pragma unroll
    for (int k = 0; k < LD; k++) {
      const int f = wave + 8 * k;  // fragment: tile, plane, k-step
      if (FS % 8 == 0 || f < FS) {
        const int tile = f / (PL * KS), p = (f / KS) % PL, s = f % KS;
        int tok = t0 + tile * 16 + r;
        tok = tok < a.nd ? tok : a.nd - 1;
        stg[k] = *(const u32x4*)(a.D + p * a.dplane + ((b0 + doc) * a.nd + tok) * width + 64 * s + 16 * g);
      }
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int k = 0; k < LD; k++) {
      const int f = wave + 8 * k;
      if (FS % 8 == 0 || f < FS) ring[buf][f][lane] = stg[k];
    }
  };

  Best best[NB][2];
#pragma unroll
  for (int j = 0; j < NB; j++) best[j][0] = best[j][1] = {-__builtin_inff(), kNone};

  int cur = seek(0), nxt = cur < total ? seek(cur + 1) : total;
  load(cur);
  if (cur < total) put(0);
  load(nxt);
  __syncthreads();
  int buf = 0;
  while (cur < total) {
    const int doc = cur / stages, t0 = (cur - doc * stages) * kStage;
    const uint64_t bits64 = words[cur];
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)bits64);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(bits64 >> 32));
#pragma unroll
    for (int tile = 0; tile < 4; tile++) {
      const uint32_t bits = ((tile & 2 ? hi : lo) >> (16 * (tile & 1))) & 0xffffu;
      if (bits == 0) continue;
      u32x4 df[PL][KS];
#pragma unroll
      for (int p = 0; p < PL; p++)
#pragma unroll
        for (int s = 0; s < KS; s++) df[p][s] = ring[buf][(tile * PL + p) * KS + s][lane];
#pragma unroll
      for (int j = 0; j < NB; j++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = PL == 1 ? 5 : 0; p < 6; p++)
#pragma unroll
            for (int s = 0; s < KS; s++) acc = mfma16x16x32<DT>(df[kPairD[p]][s], qf[j][kPairQ[p]][s][h], acc);
          if (bits != 0xffffu) mask_tile(acc, bits, g);
          take(best[j][h], acc, t0 + tile * 16 + 4 * g);
        }
    }
    const int after = nxt < total ? seek(nxt + 1) : total;
    if (nxt >= total || nxt / stages != doc) {  // the document's end
      const int64_t b = b0 + doc;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NB; j++) {
        const int q = q0 + j / a.nbq, blk = j % a.nbq;
        const Best x0 = across_rows(best[j][0]), x1 = across_rows(best[j][1]);
        best[j][0] = best[j][1] = {-__builtin_inff(), kNone};
        if (j < a.qpw * a.nbq && q < a.nQ) {
          const bool on0 = (real >> (2 * j)) & 1u, on1 = (real >> (2 * j + 1)) & 1u;
          if (a.arg && g < 2) {
            const int tok = blk * 32 + lane;
            const int at = g == 0 ? (on0 ? x0.at : kNone) : (on1 ? x1.at : kNone);
            if (tok < a.nqp) a.arg[arg_at(a, q, b) + tok] = (uint16_t)at;
          }
          const float s = row_sum16((on0 ? x0.v : 0.f) + (on1 ? x1.v : 0.f));
          sum = blk == 0 ? s : sum + s;
          if (blk == a.nbq - 1 && lane == 0) a.scores[score_at(a, q, b)] = sum;
        }
      }
    }
    if (nxt < total) put(buf ^ 1);
    load(after);
    __syncthreads();
    buf ^= 1;
    cur = nxt;
    nxt = after;
  }

  // documents without a real token
  for (int doc = 0; doc < ndocs; doc++) {
    bool any = false;
    for (int s = 0; s < stages && !any; s++) any = words[doc * stages + s] != 0;
    if (any) continue;
    for (int j = 0; j < a.qpw && q0 + j < a.nQ; j++) {
      const int q = q0 + j;
      if (lane == 0) a.scores[score_at(a, q, b0 + doc)] = -__builtin_inff();
      if (a.arg)
        for (int i = lane; i < a.nqp; i += 64) a.arg[arg_at(a, q, b0 + doc) + i] = (uint16_t)kNone;
    }
  }
}

// ---------------------------------------------------------------- 16-bit terms

// Rows of d elements as rows of dp (a multiple of 32; the rest zero) in the type the matrix
// cores take: a copy of 16-bit rows whose width or address they do not take as they are, or
// fp32 rows as three bf16 terms, x = t0 + t1 + t2 with 24 bits between them.
template <int DT>
__global__ __launch_bounds__(256) void pairs_terms_kernel(const void* src, uint16_t* dst, int64_t rows, int32_t d, int32_t dp,
                                                          int64_t plane) {
  const int64_t n = rows * dp;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
    const int64_t row = k / dp;
    const int c = (int)(k - row * dp);
    if constexpr (DT == TMS_DTYPE_F32) {
      float x = c < d ? ((const float*)src)[row * d + c] : 0.f;
#pragma unroll
      for (int p = 0; p < 3; p++) {
        const __bf16 t = (__bf16)x;
        dst[p * plane + k] = __builtin_bit_cast(uint16_t, t);
        x -= (float)t;
      }
    } else {
      dst[k] = c < d ? ((const uint16_t*)src)[row * d + c] : (uint16_t)0;
    }
  }
}

// ---------------------------------------------------------------- gradients

template <int DT>
struct El;
template <>
struct El<TMS_DTYPE_F16> {
  typedef _Float16 T;
};
template <>
struct El<TMS_DTYPE_BF16> {
  typedef __bf16 T;
};
template <>
struct El<TMS_DTYPE_F32> {
  typedef float T;
};

struct PairsGradArgs {
  const void* Q;
  const void* D;
  const uint16_t* arg;
  const float* G;  // (nQ, B) or (nQ, nway)
  void* dQ;
  void* dD;
  float* parts;  // [split][nQ * nq][d]
  int64_t B;
  int32_t nQ, nq, nqp, nd, d, nway;
  int32_t rows;            // dD: document tokens whose sums a workgroup keeps
  int32_t splits, chunk;   // dQ: splits of the documents, documents each
};

// dD: one wave keeps 64 columns of a document's gradient in LDS, a column a lane, and adds
// every maximum's query token to the row that won it. Only the column's own lane touches a
// sum, in the order of the queries, so that the result does not depend on timing. Positions
// and G come through the scalar unit, eight maxima at a time; the query rows are read ahead.
template <int DT>
__global__ __launch_bounds__(64) void pairs_grad_d_kernel(PairsGradArgs a) {
  extern __shared__ float sums[];  // [rows + 1][64]: the last row takes what is not ours
  typedef typename El<DT>::T T;
  const int lane = threadIdx.x;
  const int64_t b = blockIdx.x;
  const int col = (int)blockIdx.y * 64 + lane, t0 = (int)blockIdx.z * a.rows;
  const int rows = t0 + a.rows < a.nd ? a.rows : a.nd - t0;
  for (int i = 0; i <= rows; i++) sums[i * 64 + lane] = 0.f;
  const bool in = col < a.d;
  const int qa = a.nway ? (int)(b / a.nway) : 0, qn = a.nqp == 0 ? 0 : a.nway ? 1 : a.nQ;
  const uint16_t* arg = a.arg + (a.nway ? b : b * a.nQ) * a.nqp;
  const T* Q = (const T*)a.Q + (int64_t)qa * a.nq * a.d + (in ? col : 0);
  for (int q = 0; q < qn; q++) {
    const float w = a.G[a.nway ? b : (int64_t)(qa + q) * a.B + b];
    for (int i = 0; i < a.nqp; i += 8) {
      const u32x4 at = *(const u32x4*)(arg + (int64_t)q * a.nqp + i);  // nqp is a multiple of 8
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int tok = i + k < a.nq ? i + k : a.nq - 1;
        x[k] = (float)Q[((int64_t)q * a.nq + tok) * a.d];
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        uint32_t j = (at[k / 2] >> (16 * (k & 1))) & 0xffffu;
        j = __builtin_amdgcn_readfirstlane(j) - (uint32_t)t0;
        j = j < (uint32_t)rows ? j : (uint32_t)rows;  // kNone is beyond every document
        __hip_atomic_fetch_add(&sums[j * 64 + lane], w * x[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
      }
    }
  }
  if (in) {
    T* out = (T*)a.dD + ((int64_t)b * a.nd + t0) * a.d + col;
    for (int i = 0; i < rows; i++) out[(int64_t)i * a.d] = (T)sums[i * 64 + lane];
  }
}

// dQ: a wave takes eight query tokens and 128 columns (two a lane) over a run of documents,
// and adds the token that each document answered with. Runs are a power of two to the XCDs,
// so that the waves of an XCD walk the same documents and find their rows in its L2.
template <int DT>
__global__ __launch_bounds__(64) void pairs_grad_q_kernel(PairsGradArgs a) {
  typedef typename El<DT>::T T;
  const int lane = threadIdx.x;
  const int split = (int)(blockIdx.x % a.splits);
  const int unit = (int)(blockIdx.x / a.splits);
  const int groups = a.nqp / 8;
  const int q = unit / groups, i0 = (unit - q * groups) * 8;
  const int col = (int)blockIdx.y * 128 + 2 * lane;
  const bool in0 = col < a.d, in1 = col + 1 < a.d;
  const int64_t first = a.nway ? (int64_t)q * a.nway : 0, n = a.nway ? a.nway : a.B;
  const int64_t e0 = (int64_t)split * a.chunk, e1 = e0 + a.chunk < n ? e0 + a.chunk : n;
  float acc[8][2] = {};
  const T* D = (const T*)a.D;
  for (int64_t k = e0; k < e1; k++) {
    const int64_t b = first + k;
    const float w = a.G[a.nway ? b : (int64_t)q * a.B + b];
    const u32x4 at = *(const u32x4*)(a.arg + (a.nway ? b : b * a.nQ + q) * a.nqp + i0);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t j = __builtin_amdgcn_readfirstlane((at[i / 2] >> (16 * (i & 1))) & 0xffffu);
      if (j >= (uint32_t)a.nd) continue;  // kNone
      const T* row = D + ((int64_t)b * a.nd + j) * a.d;
      const float x0 = in0 ? (float)row[col] : 0.f, x1 = in1 ? (float)row[col + 1] : 0.f;
      acc[i][0] += w * x0;
      acc[i][1] += w * x1;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (i0 + i >= a.nq) break;
    const int64_t row = (int64_t)q * a.nq + i0 + i;
    if (a.splits == 1) {
      T* out = (T*)a.dQ + row * a.d + col;
      if (in0) out[0] = (T)acc[i][0];
      if (in1) out[1] = (T)acc[i][1];
    } else {
      float* out = a.parts + ((int64_t)split * a.nQ * a.nq + row) * a.d + col;
      if (in0) out[0] = acc[i][0];
      if (in1) out[1] = acc[i][1];
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void pairs_grad_q_join_kernel(const float* parts, void* dQ, int64_t n, int splits) {
  typedef typename El<DT>::T T;
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (k >= n) return;
  float x = 0.f;
  for (int s = 0; s < splits; s++) x += parts[s * n + k];
  ((T*)dQ)[k] = (T)x;
}

// ---------------------------------------------------------------- host

constexpr int64_t kLdsBytes = 160 * 1024;

static int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Whether the forward kernels take these rows as they are.
static bool as_is(const void* p, int64_t d, int dtype) {
  return dtype != TMS_DTYPE_F32 && d % 32 == 0 && (uintptr_t)p % 16 == 0;
}
static int planes(int dtype) { return dtype == TMS_DTYPE_F32 ? 3 : 1; }

// The splits of dQ's documents: enough waves for four on each SIMD's worth of the chip
// (1,024 SIMDs), at least 16 documents each, a multiple of 8 where there are several.
static int grad_q_splits(int64_t nQ, int64_t nqp, int64_t cols, int64_t n) {
  const int64_t units = nQ * (nqp / 8) * cols;
  int64_t s = units > 0 ? 4096 / units : 1;
  if (s > n / 16) s = n / 16;
  if (s >= 8) s = s / 8 * 8;
  return (int)(s < 1 ? 1 : s > 512 ? 512 : s);
}

static int check_pairs(const char* fn, int64_t nQ, int64_t nq, int64_t d, int64_t B, int64_t nd, int64_t nway, int dtype) {
  if (nQ < 0 || nq < 0 || d < 0 || B < 0 || nd < 0 || nway < 0) return fail(TMS_ERR_INVALID, "%s: negative size", fn);
  if (dtype != TMS_DTYPE_F16 && dtype != TMS_DTYPE_BF16 && dtype != TMS_DTYPE_F32)
    return fail(TMS_ERR_UNSUPPORTED, "%s: dtype must be fp16, bf16 or fp32", fn);
  if (nway > 0 && B != nQ * nway)
    return fail(TMS_ERR_INVALID, "%s: B=%lld is not nQ * nway = %lld", fn, (long long)B, (long long)(nQ * nway));
  if (nd > kMaxTokens) return fail(TMS_ERR_UNSUPPORTED, "%s: documents of more than %d tokens", fn, kMaxTokens);
  if (d > 65536 || nq > 65536) return fail(TMS_ERR_UNSUPPORTED, "%s: d and nq go up to 65536", fn);
  if (nQ > 65535 || B > 0x7fffffff || (d > 0 && B * nd > ((int64_t)1 << 48) / d))
    return fail(TMS_ERR_UNSUPPORTED, "%s: more than 65535 queries or 2^31 - 1 documents", fn);
  return TMS_OK;
}

template <int DT, int KS, int PL>
static int run_direct(const PairsArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.B, a.nway ? 1u : (unsigned)a.nQ);
  hipLaunchKernelGGL((pairs_direct_kernel<DT, KS, PL>), grid, dim3(256), 0, st, a);
  return check_launch("pairs_direct_kernel");
}

template <int DT, int KS, int NB, int PL>
static int run_shared(PairsArgs a, hipStream_t st) {
  a.qpw = NB / a.nbq;
  const int64_t groups = (a.nQ + 8 * a.qpw - 1) / (8 * a.qpw);
  const int64_t stages = (a.nd + kStage - 1) / kStage;
  // Documents a workgroup: its mask words, and at least four workgroups a CU over the launch
  // (1,024) where there are that many documents, so that the last round is a small part.
  int64_t docs = kMaskWords / (stages > 0 ? stages : 1);
  const int64_t even = (a.B * groups + 1023) / 1024;
  if (docs > even) docs = even;
  if (docs < 1) docs = 1;
  a.docs_per_wg = (int32_t)docs;
  hipLaunchKernelGGL((pairs_shared_kernel<DT, KS, NB, PL>), dim3((unsigned)((a.B + docs - 1) / docs), (unsigned)groups), dim3(512), 0,
                     st, a);
  return check_launch("pairs_shared_kernel");
}

template <int DT, int KS, int PL>
static int run_width(const PairsArgs& a, int64_t blocks, hipStream_t st) {
  if constexpr (PL == 3) return run_shared<DT, KS, 1, 3>(a, st);
  else {
    if (a.nbq <= 1 && blocks <= 8) return run_shared<DT, KS, 1, 1>(a, st);
    if (a.nbq <= 2 && blocks <= 16) return run_shared<DT, KS, 2, 1>(a, st);
    return run_shared<DT, KS, 4, 1>(a, st);
  }
}

template <int DT, int PL>
static int run_pairs(PairsArgs& a, hipStream_t st) {
  const int64_t blocks = (int64_t)a.nQ * a.nbq;
  const int ks = a.d / 32;
  // Sharing pays once the waves are mostly filled; a call of few pairs needs a workgroup for
  // each instead. A document takes at most kMaskWords stages (65,535 tokens).
  const bool shared = !a.nway && ks <= 4 && a.nbq <= (PL == 3 ? 1 : 4) && blocks >= 4 && a.B * a.nQ > 2048;
  if (shared) {
    switch (ks) {
      case 1: return run_width<DT, 1, PL>(a, blocks, st);
      case 2: return run_width<DT, 2, PL>(a, blocks, st);
      case 3: return run_width<DT, 3, PL>(a, blocks, st);
      default: return run_width<DT, 4, PL>(a, blocks, st);
    }
  }
  if (PL == 1) switch (ks) {
      case 1: return run_direct<DT, 1, 1>(a, st);
      case 2: return run_direct<DT, 2, 1>(a, st);
      case 3: return run_direct<DT, 3, 1>(a, st);
      case 4: return run_direct<DT, 4, 1>(a, st);
    }
  return run_direct<DT, 0, PL>(a, st);
}

static int run_terms(const void* src, void* dst, int64_t rows, int64_t d, int64_t dp, int dtype, hipStream_t st) {
  const int64_t n = rows * dp;
  if (n == 0) return TMS_OK;
  const unsigned grid = (unsigned)(n > 256 * 8192 ? 8192 : (n + 255) / 256);
  if (dtype == TMS_DTYPE_F32)
    hipLaunchKernelGGL(pairs_terms_kernel<TMS_DTYPE_F32>, dim3(grid), dim3(256), 0, st, src, (uint16_t*)dst, rows, (int32_t)d, (int32_t)dp, n);
  else
    hipLaunchKernelGGL(pairs_terms_kernel<TMS_DTYPE_F16>, dim3(grid), dim3(256), 0, st, src, (uint16_t*)dst, rows, (int32_t)d, (int32_t)dp, n);
  return check_launch("pairs_terms_kernel");
}

// Scores of no tokens: 0 for a query without any, -inf for a document without any.
__global__ void pairs_fill_kernel(float* scores, int64_t n, float v, uint16_t* arg, int64_t m) {
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < (n > m ? n : m); k += (int64_t)gridDim.x * 256) {
    if (k < n) scores[k] = v;
    if (k < m) arg[k] = (uint16_t)kNone;
  }
}

template <int DT>
static int run_grads(PairsGradArgs a, hipStream_t st) {
  int rc;
  if (a.dD && a.B > 0 && a.nd > 0 && a.d > 0) {
    const unsigned cols = (unsigned)((a.d + 63) / 64);
    const int tiles = (a.nd + 510) / 511;  // at most 512 rows of 256 bytes: 128 KB of LDS
    a.rows = (a.nd + tiles - 1) / tiles;
    const size_t lds = (size_t)(a.rows + 1) * 256;
    hipLaunchKernelGGL(pairs_grad_d_kernel<DT>, dim3((unsigned)a.B, cols, (unsigned)tiles), dim3(64), lds, st, a);
    if ((rc = check_launch("pairs_grad_d_kernel"))) return rc;
  }
  if (a.dQ && a.nQ > 0 && a.nq > 0 && a.d > 0) {
    const unsigned cols = (unsigned)((a.d + 127) / 128);
    const int64_t n = a.nway ? a.nway : a.B;
    a.chunk = (int32_t)((n + a.splits - 1) / a.splits);
    hipLaunchKernelGGL(pairs_grad_q_kernel<DT>, dim3((unsigned)((int64_t)a.nQ * (a.nqp / 8) * a.splits), cols), dim3(64), 0, st, a);
    if ((rc = check_launch("pairs_grad_q_kernel"))) return rc;
    if (a.splits > 1) {
      const int64_t m = (int64_t)a.nQ * a.nq * a.d;
      hipLaunchKernelGGL(pairs_grad_q_join_kernel<DT>, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, st, a.parts, a.dQ, m, a.splits);
      if ((rc = check_launch("pairs_grad_q_join_kernel"))) return rc;
    }
  }
  return TMS_OK;
}

}  // namespace tms

using namespace tms;

extern "C" int64_t tms_pairs_workspace_size(int64_t nQ, int64_t nq, int64_t d, int64_t B, int64_t nd, int dtype) {
  if (nQ < 0 || nq < 0 || d < 0 || B < 0 || nd < 0) return 0;
  const int64_t dp = d > 0 ? round_up(d, 32) : 32;
  if (dtype != TMS_DTYPE_F32 && d == dp) return 0;
  return (round_up(nQ * nq * dp * 2, 256) + B * nd * dp * 2) * planes(dtype);
}

extern "C" int64_t tms_pairs_positions(int64_t nQ, int64_t nq, int64_t B, int64_t nway) {
  if (nQ < 0 || nq < 0 || B < 0) return 0;
  return (nway > 0 ? B : nQ * B) * round_up(nq, 8);
}

extern "C" int tms_maxsim_pairs(const void* Qs, int64_t nQ, int64_t nq, int64_t d, const void* D, int64_t B, int64_t nd,
                                int64_t nway, const uint8_t* qmask, const uint8_t* dmask, int dtype, void* workspace,
                                int64_t workspace_bytes, float* scores, uint16_t* positions, void* stream) {
  const char* fn = "tms_maxsim_pairs";
  int rc = check_pairs(fn, nQ, nq, d, B, nd, nway, dtype);
  if (rc) return rc;
  if (nQ == 0 || B == 0) return TMS_OK;
  if (!scores || (nq * d > 0 && !Qs) || (nd * d > 0 && !D)) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  PairsArgs a = {};
  a.qmask = qmask;
  a.dmask = dmask;
  a.scores = scores;
  a.arg = positions;
  a.B = B;
  a.nQ = (int32_t)nQ;
  a.nq = (int32_t)nq;
  a.nqp = (int32_t)round_up(nq, 8);
  a.nd = (int32_t)nd;
  a.nway = (int32_t)nway;
  a.nbq = (int32_t)((nq + 31) / 32);
  const int64_t npairs = nway ? B : nQ * B;
  if (nd == 0 || nq == 0) {
    const int64_t m = positions ? npairs * a.nqp : 0, most = npairs > m ? npairs : m;
    hipLaunchKernelGGL(pairs_fill_kernel, dim3((unsigned)(most > 256 * 4096 ? 4096 : (most + 255) / 256)), dim3(256), 0, st, scores,
                       npairs, nd == 0 ? -__builtin_inff() : 0.f, positions, m);
    return check_launch("pairs_fill_kernel");
  }
  const int64_t dp = d > 0 ? round_up(d, 32) : 32;
  a.d = (int32_t)dp;
  const bool keep = d > 0 && as_is(Qs, d, dtype) && as_is(D, d, dtype);
  a.Q = (const uint8_t*)Qs;
  a.D = (const uint8_t*)D;
  if (!keep) {
    const int64_t qbytes = round_up(nQ * nq * dp * 2, 256) * planes(dtype), dbytes = B * nd * dp * 2 * planes(dtype);
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < qbytes + dbytes)
      return fail(TMS_ERR_INVALID, "%s: these rows need a workspace of %lld bytes, 16-byte aligned", fn, (long long)(qbytes + dbytes));
    uint8_t* wq = (uint8_t*)workspace;
    uint8_t* wd = wq + qbytes;
    if ((rc = run_terms(Qs, wq, nQ * nq, d, dp, dtype, st))) return rc;
    if ((rc = run_terms(D, wd, B * nd, d, dp, dtype, st))) return rc;
    a.Q = wq;
    a.D = wd;
    a.qplane = nQ * nq * dp * 2;
    a.dplane = B * nd * dp * 2;
  }
  if (dtype == TMS_DTYPE_F16) return run_pairs<TMS_DTYPE_F16, 1>(a, st);
  if (dtype == TMS_DTYPE_BF16) return run_pairs<TMS_DTYPE_BF16, 1>(a, st);
  return run_pairs<TMS_DTYPE_BF16, 3>(a, st);
}

extern "C" int64_t tms_pairs_grad_workspace_size(int64_t nQ, int64_t nq, int64_t d, int64_t B, int64_t nway) {
  if (nQ <= 0 || nq <= 0 || d <= 0 || B <= 0) return 0;
  const int s = grad_q_splits(nQ, round_up(nq, 8), (d + 127) / 128, nway > 0 ? nway : B);
  return s > 1 ? s * nQ * nq * d * 4 : 0;
}

extern "C" int tms_maxsim_pairs_grad(const void* Qs, int64_t nQ, int64_t nq, int64_t d, const void* D, int64_t B, int64_t nd,
                                     int64_t nway, const uint16_t* positions, const float* grad, int dtype, void* workspace,
                                     int64_t workspace_bytes, void* dQ, void* dD, void* stream) {
  const char* fn = "tms_maxsim_pairs_grad";
  const int rc = check_pairs(fn, nQ, nq, d, B, nd, nway, dtype);
  if (rc) return rc;
  const int64_t nqp = round_up(nq, 8);
  if ((dQ && nQ * nq * d > 0 && B > 0 && nd > 0 && !D) || (dD && B * nd * d > 0 && nQ * nq > 0 && !Qs) ||
      (nQ * nq > 0 && B > 0 && (!positions || !grad)))
    return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if ((uintptr_t)positions % 16) return fail(TMS_ERR_INVALID, "%s: positions must be 16-byte aligned", fn);
  const int64_t need = dQ ? tms_pairs_grad_workspace_size(nQ, nq, d, B, nway) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(TMS_ERR_INVALID, "%s: a workspace of %lld bytes is needed", fn, (long long)need);
  PairsGradArgs a = {};
  a.Q = Qs;
  a.D = D;
  a.arg = positions;
  a.G = grad;
  a.dQ = dQ;
  a.dD = dD;
  a.parts = (float*)workspace;
  a.B = B;
  a.nQ = (int32_t)nQ;
  a.nq = (int32_t)nq;
  a.nqp = (int32_t)nqp;
  a.nd = (int32_t)nd;
  a.d = (int32_t)d;
  a.nway = (int32_t)nway;
  a.splits = B > 0 ? grad_q_splits(nQ, nqp, (d + 127) / 128, nway > 0 ? nway : B) : 1;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TMS_DTYPE_F16) return run_grads<TMS_DTYPE_F16>(a, st);
  if (dtype == TMS_DTYPE_BF16) return run_grads<TMS_DTYPE_BF16>(a, st);
  return run_grads<TMS_DTYPE_F32>(a, st);
}
