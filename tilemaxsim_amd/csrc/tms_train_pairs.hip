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

// Workgroups beyond what one axis of a launch takes (2^32 threads) stand in further rows of it.
constexpr int64_t kAxisGroups = 1 << 21;
__device__ __forceinline__ int64_t workgroup() { return (int64_t)blockIdx.z * gridDim.x + blockIdx.x; }
static dim3 grid_of(int64_t groups, unsigned y) {
  const int64_t rows = (groups + kAxisGroups - 1) / kAxisGroups;
  return dim3((unsigned)((groups + rows - 1) / rows), y, (unsigned)rows);
}

// Running maximum and its token over one 16-token tile: lane (c, g) sees query token c
// against tokens base + 4 g + i. A strict comparison keeps the first of equal ones, as
// tokens rise; the maximum keeps a NaN, which has to reach the loss. Three VALU instructions
// a value, half of one without positions.
struct Best {
  float v;
  int at;
};
__device__ __forceinline__ float top(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <bool POS>
__device__ __forceinline__ void take(Best& r, const f32x4& s, int first) {
  if constexpr (POS) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      r.at = s[i] > r.v ? first + i : r.at;
      r.v = top(r.v, s[i]);
    }
  } else {
    r.v = top(top(r.v, s[0]), s[1]);
    r.v = top(top(r.v, s[2]), s[3]);
  }
}
__device__ __forceinline__ Best better(Best x, Best y) {
  const bool up = y.v > x.v || (y.v == x.v && y.at < x.at);
  return {top(x.v, y.v), up ? y.at : x.at};
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

// Two registers' rows in one, compared: with 32, lanes 0-31 get x over both halves of the wave
// and lanes 32-63 y; with 16, even rows get x over their pair of rows and odd rows y.
template <int N>
__device__ __forceinline__ Best swap_rows(Best x, Best y) {
  const unsigned xv = __builtin_bit_cast(unsigned, x.v), yv = __builtin_bit_cast(unsigned, y.v);
  if constexpr (N == 32) {
    const auto v = __builtin_amdgcn_permlane32_swap(xv, yv, false, false);
    const auto i = __builtin_amdgcn_permlane32_swap((unsigned)x.at, (unsigned)y.at, false, false);
    return better({__builtin_bit_cast(float, (unsigned)v[0]), (int)i[0]}, {__builtin_bit_cast(float, (unsigned)v[1]), (int)i[1]});
  } else {
    const auto v = __builtin_amdgcn_permlane16_swap(xv, yv, false, false);
    const auto i = __builtin_amdgcn_permlane16_swap((unsigned)x.at, (unsigned)y.at, false, false);
    return better({__builtin_bit_cast(float, (unsigned)v[0]), (int)i[0]}, {__builtin_bit_cast(float, (unsigned)v[1]), (int)i[1]});
  }
}

template <bool V>
struct Flag {
  static constexpr bool value = V;
};

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
// KS = 0: any d, fragments read as they are used. Bound by the latency of a tile's loads: 32 queries
// x 8 documents of their own of 171 tokens, d = 128, fp16: 7 us.
template <int DT, int KS, int PL>
__global__ __launch_bounds__(256) void pairs_direct_kernel(PairsArgs a) {
  __shared__ Best joined[4][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t b = workgroup();
  if (b >= a.B) return;
  const int q = a.nway ? (int)(b / a.nway) : (int)blockIdx.y;
  const int64_t drow = b * a.nd, qrow = (int64_t)q * a.nq;
  const int64_t width = (int64_t)a.d * 2;
  const int tiles = (a.nd + 15) >> 4;
  float total = 0.f;
  bool some = false;  // a real document token, in any lane of the workgroup
  for (int blk = 0; blk < a.nbq; blk++) {
    bool real[2];
    u32x4 qf[PL][KS ? KS : 1][2];
    const uint8_t* qp[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int tok = blk * 32 + 16 * h + r;
      real[h] = tok < a.nq && (!a.qmask || a.qmask[qrow + tok] != 0);
      qp[h] = a.Q + (qrow + (tok < a.nq ? tok : 0)) * width + 16 * g;
      if constexpr (KS > 0) {
#pragma unroll
        for (int p = 0; p < PL; p++)
#pragma unroll
          for (int s = 0; s < KS; s++) {
            const u32x4 v = *(const u32x4*)(qp[h] + p * a.qplane + 64 * s);
            qf[p][s][h] = real[h] ? v : u32x4{0u, 0u, 0u, 0u};
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
        u32x4 df[PL][KS];
#pragma unroll
        for (int p = 0; p < PL; p++)
#pragma unroll
          for (int s = 0; s < KS; s++) df[p][s] = *(const u32x4*)(dp + p * a.dplane + 64 * s);
#pragma unroll
        for (int p = PL == 1 ? 5 : 0; p < 6; p++)
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) acc[h] = mfma16x16x32<DT>(df[kPairD[p]][s], qf[kPairQ[p]][s][h], acc[h]);
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
        mask_tile(acc[h], bits, g);  // not behind a branch, for one would follow an MFMA
        take<true>(best[h], acc[h], t * 16 + 4 * g);
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
// costs 1 / (8 NB) of a load per block. One barrier a stage: a stage is written to the buffer
// that every wave left before the last one. Masks become 64-bit words in LDS first, and the
// words with a real token a list, so that stages of padding are neither loaded nor looked at.
// Whole queries belong to a wave, so a score is summed in one place and in one order.
//
// A block's 16 x 16 similarities are a chain of MFMAs (4 of 16 cycles at d = 128), and
// their maxima twelve VALU instructions of 4 cycles (POS: with positions), or two without; a
// wave issues in order, so the maxima of one block are put between the MFMAs of the next.
// 64 queries x 4096 documents of 60 to 180 tokens, d = 128, 16 bits: 315 us with positions (with
// one block after the other 80 more), 250 without, bound by the SIMDs' issue of the two, which
// do not overlap there: products 38 % of the cycles, other VALU work 44 %. (32 x 32 products, which overlap half of it, take 365 and
// 274: documents then end on 32 tokens, and the registers do not hold the next fragments.)
template <int DT, int KS, int NB, int PL, bool POS>
__global__ __launch_bounds__(512, 2) void pairs_shared_kernel(PairsArgs a) {
  constexpr int FS = 4 * PL * KS;  // fragments of a stage
  constexpr int LD = (FS + 7) / 8;  // fragments a wave loads
  constexpr int NP = (NB + 1) / 2;  // pairs of blocks, at a document's end
  __shared__ u32x4 ring[2][FS][64];
  __shared__ uint64_t words[kMaskWords];
  __shared__ uint32_t list[kMaskWords + 2];  // document << 16 | stage of the words that are not 0
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = lane & 15, g = lane >> 4;
  const int64_t b0 = (int64_t)blockIdx.x * a.docs_per_wg;
  const int ndocs = (int)(b0 + a.docs_per_wg < a.B ? a.docs_per_wg : a.B - b0);
  const int stages = (a.nd + kStage - 1) / kStage;
  const int64_t width = (int64_t)a.d * 2;
  const int q0 = ((int)blockIdx.y * 8 + wave) * a.qpw;  // this wave's first query

  // Everything below reads memory once or twice and then waits: loads first, in batches.
  const int nwords = ndocs * stages;
  auto mask_words = [&](int w0) {
    bool live[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int w = w0 + 8 * k, doc = w / stages, tok = (w - doc * stages) * kStage + lane;
      live[k] = w < nwords && tok < a.nd;
      if (live[k] && a.dmask) live[k] = a.dmask[(b0 + doc) * a.nd + tok] != 0;
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const uint64_t bits = __ballot(live[k]);
      if (lane == 0 && w0 + 8 * k < nwords) words[w0 + 8 * k] = bits;
    }
  };
  u32x4 qf[NB][PL][KS][2];
  uint32_t real = 0;  // bit 2 j + h: this lane's token of half h of block j
#pragma unroll
  for (int j = 0; j < NB; j++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int q = q0 + j / a.nbq, tok = (j % a.nbq) * 32 + 16 * h + r;
      const bool in = j < a.qpw * a.nbq && q < a.nQ && tok < a.nq;
      const int64_t row = in ? (int64_t)q * a.nq + tok : 0;
      uint8_t on = in ? 1 : 0;
      if (a.qmask) on = in ? a.qmask[row] : 0;
      real |= (on ? 1u : 0u) << (2 * j + h);
#pragma unroll
      for (int p = 0; p < PL; p++)
#pragma unroll
        for (int s = 0; s < KS; s++) qf[j][p][s][h] = *(const u32x4*)(a.Q + p * a.qplane + row * width + 64 * s + 16 * g);
    }
  for (int w = wave; w < nwords; w += 64) mask_words(w);
#pragma unroll
  for (int j = 0; j < NB; j++)
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int p = 0; p < PL; p++)
#pragma unroll
        for (int s = 0; s < KS; s++) qf[j][p][s][h] = (real >> (2 * j + h)) & 1u ? qf[j][p][s][h] : u32x4{0u, 0u, 0u, 0u};
  __syncthreads();
  if (wave == 0) {
    int n = 0;
    for (int w = lane; w - lane < nwords; w += 64) {
      const bool some = w < nwords && words[w] != 0;
      const uint64_t all = __ballot(some);
      const int doc = w / stages;
      if (some) list[n + __popcll(all & ((1ull << lane) - 1))] = (uint32_t)doc << 16 | (uint32_t)(w - doc * stages);
      n += __popcll(all);
    }
    if (lane == 0) list[kMaskWords + 1] = (uint32_t)n;
  }
  __syncthreads();
  const int total = __builtin_amdgcn_readfirstlane((int)list[kMaskWords + 1]);

  u32x4 stg[LD];
  // the n-th stage of the list, and which of its tokens are real: looked up two stages ahead
  auto entry = [&](int n) -> uint32_t { return __builtin_amdgcn_readfirstlane(list[n < total ? n : 0]); };
  auto bits_of = [&](uint32_t e) -> uint64_t {
    const uint64_t w = words[(int)(e >> 16) * stages + (int)(e & 0xffffu)];
    return (uint64_t)wave_uniform((int64_t)w);
  };
  auto load = [&](uint32_t e) {
    const int t0 = (int)(e & 0xffffu) * kStage;
    const int64_t row0 = (b0 + (e >> 16)) * a.nd;
#pragma unroll
    for (int k = 0; k < LD; k++) {
      const int f = wave + 8 * k;  // fragment: tile, plane, k-step
      if (FS % 8 == 0 || f < FS) {
        const int tile = f / (PL * KS), p = (f / KS) % PL, s = f % KS;
        int tok = t0 + tile * 16 + r;
        tok = tok < a.nd ? tok : a.nd - 1;
        stg[k] = *(const u32x4*)(a.D + p * a.dplane + (row0 + tok) * width + 64 * s + 16 * g);
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

  uint32_t cur = 0, nxt = 0;
  uint64_t cur_bits = 0, nxt_bits = 0;
  if (total > 0) {
    cur = entry(0);
    load(cur);
    nxt = entry(1);
    cur_bits = bits_of(cur);
    nxt_bits = bits_of(nxt);
    put(0);
    if (total > 1) load(nxt);
  }
  __syncthreads();
  for (int n = 0; n < total; n++) {
    const int buf = n & 1;
    const int doc = (int)(cur >> 16), t0 = (int)(cur & 0xffffu) * kStage;
    const uint32_t after_at = list[n + 2 < total ? n + 2 : 0];  // read ahead of the products
    // a tile's fragments are read while the tile before is scored (three planes have no room)
    constexpr int AHEAD = PL == 1 ? 2 : 1;
    u32x4 frags[AHEAD][PL][KS];
    auto read = [&](int tile) {
#pragma unroll
      for (int p = 0; p < PL; p++)
#pragma unroll
        for (int s = 0; s < KS; s++) frags[tile % AHEAD][p][s] = ring[buf][(tile * PL + p) * KS + s][lane];
    };
    if constexpr (AHEAD == 2) read(0);
#pragma unroll
    for (int tile = 0; tile < 4; tile++) {
      if constexpr (AHEAD == 1) read(tile);
      else if (tile < 3) read(tile + 1);
      const uint32_t bits = (uint32_t)(cur_bits >> (16 * tile)) & 0xffffu;
      if (bits == 0) continue;
      const auto& df = frags[tile % AHEAD];
      const int first = t0 + tile * 16 + 4 * g;
      // one body for whole tiles and one for masked ones: no branch behind an MFMA
      auto score = [&](auto masked) {
        f32x4 acc[2][2];  // a block's two halves, and the block's before
#pragma unroll
        for (int j = 0; j <= NB; j++) {
          if (j < NB) {
            f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int p = PL == 1 ? 5 : 0; p < 6; p++)
#pragma unroll
              for (int s = 0; s < KS; s++)
#pragma unroll
                for (int h = 0; h < 2; h++) v[h] = mfma16x16x32<DT>(df[kPairD[p]][s], qf[j < NB ? j : 0][kPairQ[p]][s][h], v[h]);
            acc[j & 1][0] = v[0];
            acc[j & 1][1] = v[1];
          }
          if (j > 0) {
            f32x4(&v)[2] = acc[(j - 1) & 1];
            if constexpr (decltype(masked)::value) mask_tile(v[0], bits, g), mask_tile(v[1], bits, g);
            take<POS>(best[j - 1][0], v[0], first);
            take<POS>(best[j - 1][1], v[1], first);
          }
          constexpr int MF = (PL == 1 ? KS : 6 * KS) * 2, VA = ((POS ? 24 : 4) + MF - 1) / MF;
          if (j == 0) __builtin_amdgcn_sched_group_barrier(0x008, MF, 0);
          if (j > 0 && j < NB) {
#pragma unroll
            for (int s = 0; s < MF; s++) {  // an MFMA, then a share of the maxima
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x002, VA, 0);
            }
          }
        }
      };
      if (bits == 0xffffu) score(Flag<false>());
      else score(Flag<true>());
    }
    const uint32_t after = __builtin_amdgcn_readfirstlane(after_at);
    const uint64_t after_bits = bits_of(after);
    if (n + 1 >= total || (nxt >> 16) != (uint32_t)doc) {  // the document's end
      const int64_t b = b0 + doc;
      float sums[NB];
#pragma unroll
      for (int P = 0; P < NP; P++) {
        // Row g of the wave ends with half g / 2 of block 2 P + g % 2: each swap brings two
        // registers' rows together in one, so two blocks take three comparisons.
        constexpr int last = NB - 1;
        const int j1 = 2 * P + 1 < NB ? 2 * P + 1 : last;
        const Best x = swap_rows<32>(best[2 * P][0], best[2 * P][1]);
        const Best y = 2 * P + 1 < NB ? swap_rows<32>(best[j1][0], best[j1][1]) : x;
        const Best z = swap_rows<16>(x, y);
        const int j = 2 * P + (2 * P + 1 < NB ? (g & 1) : 0), h = g >> 1;
        const bool on = (real >> (2 * j + h)) & 1u;
        const int q = q0 + j / a.nbq, tok = (j % a.nbq) * 32 + 16 * h + r;
        if (POS && j < a.qpw * a.nbq && q < a.nQ && tok < a.nqp && (2 * P + 1 < NB || (g & 1) == 0))
          a.arg[arg_at(a, q, b) + tok] = (uint16_t)(on ? z.at : kNone);
        float s = row_sum16(on ? z.v : 0.f);
        const auto hs = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, s), __builtin_bit_cast(unsigned, s), false, false);
        s = __builtin_bit_cast(float, (unsigned)hs[0]) + __builtin_bit_cast(float, (unsigned)hs[1]);  // the halves of a block
        sums[2 * P] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), 0));
        if (2 * P + 1 < NB) sums[j1] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), 16));
      }
      float score = 0.f;  // lane k: query q0 + k
#pragma unroll
      for (int j = 0; j < NB; j++) {
        score += lane == j / a.nbq ? sums[j] : 0.f;
        best[j][0] = best[j][1] = {-__builtin_inff(), kNone};
      }
      if (lane < a.qpw && q0 + lane < a.nQ) a.scores[score_at(a, q0 + lane, b)] = score;
    }
    if (n + 1 < total) put(buf ^ 1);
    if (n + 2 < total) load(after);
    __syncthreads();
    cur = nxt;
    nxt = after;
    cur_bits = nxt_bits;
    nxt_bits = after_bits;
  }

  // documents without a real token
  for (int d0 = 0; d0 < ndocs; d0 += 64) {
    bool none = d0 + lane < ndocs;
    for (int s = 0; s < stages && none; s++) none = words[(d0 + lane) * stages + s] == 0;
    for (uint64_t left = __ballot(none); left != 0; left &= left - 1) {
      const int64_t b = b0 + d0 + __builtin_ctzll(left);
      for (int j = 0; j < a.qpw && q0 + j < a.nQ; j++) {
        if (lane == 0) a.scores[score_at(a, q0 + j, b)] = -__builtin_inff();
        if (POS)
          for (int i = lane; i < a.nqp; i += 64) a.arg[arg_at(a, q0 + j, b) + i] = (uint16_t)kNone;
      }
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
  float* sums;   // (B * nd, d): dD's sums between two runs of queries
  int64_t B;
  int32_t nQ, nq, nqp, nd, d, nway;
  int32_t nbq, blocks;            // blocks of 32 tokens a query, blocks in all
  int32_t run;                    // dD: blocks sorted at a time
  int32_t splits, chunk, tokens;  // dQ: splits of the documents, documents each; document tokens per LDS stage
};

__device__ __forceinline__ float grad_of(const PairsGradArgs& a, int q, int64_t b) {
  return a.G[a.nway ? b : (int64_t)q * a.B + b];
}

// Two neighbouring columns of a row, as floats.
template <int DT>
__device__ __forceinline__ f32x2 two(const uint8_t* p) {
  if constexpr (DT == TMS_DTYPE_F32) {
    return *(const f32x2*)p;
  } else {
    const uint32_t x = *(const uint32_t*)p;
    if constexpr (DT == TMS_DTYPE_BF16) {
      return f32x2{__builtin_bit_cast(float, x << 16), __builtin_bit_cast(float, x & 0xffff0000u)};
    } else {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      const f16x2 h = __builtin_bit_cast(f16x2, x);
      return f32x2{(float)h[0], (float)h[1]};
    }
  }
}

// dD: a document's maxima are sorted by the token that won them, and each token adds the query
// tokens that it won, read one 256-byte row a wave's access, in the order of the queries: no
// sum depends on timing, and only rows that won or were won are touched. A workgroup has a
// document and 128 columns (two a lane). The sort is a counting sort in LDS, four bits of the
// token at a time: a thread counts and places its own run of maxima, so equal tokens keep their
// order. Then each wave takes a quarter of the sorted maxima, cut between tokens, with the
// rows of the next eight in flight while eight are added. 64 queries of 32 tokens x 4096
// documents of 60 to 180 tokens, d = 128, 16 bits: 158 us; 7.2 vector and 3.7 scalar instructions a
// maximum with the sort's, the vector units busy for 63 % of it. The rest is waits of the sort
// (LDS, half of its cycles conflicts, and barriers) and for rows. (Products with a matrix of ones made from the positions cost a multiply-add for each
// column, token and query block as well: 560 us.)
// More than kRun blocks are sorted in runs; the sums stand in memory between them, in fp32.
constexpr int kRun = 128;  // blocks of 32 maxima: 32 KB of LDS

// Two columns of a row of Q, of any width.
template <int DT>
__device__ __forceinline__ f32x2 columns(const typename El<DT>::T* row, int col, int d) {
  return f32x2{(float)row[col], col + 1 < d ? (float)row[col + 1] : 0.f};
}

// PAIR: an even width, and Q below 4 GB: two columns are one load, at a 32-bit offset.
template <int DT, bool PAIR>
__global__ __launch_bounds__(256) void pairs_grad_d_kernel(PairsGradArgs a) {
  typedef typename El<DT>::T T;
  constexpr int AHEAD = 8;
  extern __shared__ __attribute__((aligned(16))) uint8_t sort_mem[];
  const int most = a.run * 32;
  uint16_t* tok = (uint16_t*)sort_mem;                // the maxima's tokens; nd for none
  uint16_t* order[2] = {tok + most, tok + 2 * most};  // maxima in sorted order
  uint16_t* count = tok + 3 * most;                   // [digit][thread]
  float* weight = (float*)(count + 16 * 256);         // G of the run's blocks
  __shared__ int totals[4], cuts[5];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t b = workgroup();
  if (b >= a.B) return;
  const int col = (int)blockIdx.y * 128 + 2 * lane;
  const bool in = col < a.d;
  const uint32_t at_col = (uint32_t)((in ? col : 0) * (int)sizeof(T));
  const int first = a.nway ? (int)(b / a.nway) * a.nbq : 0, blocks = a.nway ? a.nbq : a.blocks;
  const uint16_t* arg = a.arg + (a.nway ? b : b * a.nQ) * a.nqp;
  const T* Q = (const T*)a.Q;
  int bits = 0;
  while ((a.nd >> bits) != 0) bits++;

  for (int k0 = 0; k0 < blocks || k0 == 0; k0 += a.run) {
    const int nb = blocks - k0 < a.run ? blocks - k0 : a.run, n = nb * 32;
    const int per = (n + 255) / 256;  // maxima a thread, in a row
    const bool begun = k0 > 0, last = k0 + a.run >= blocks;
    __syncthreads();  // the run before has read what is written here, and its sums are in memory
    for (int i = t * 8; i < n; i += 256 * 8) {
      const u32x4 v = *(const u32x4*)(arg + (int64_t)k0 * 32 + i);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t j = (v[e / 2] >> (16 * (e & 1))) & 0xffffu;
        tok[i + e] = (uint16_t)(j < (uint32_t)a.nd ? j : (uint32_t)a.nd);
      }
    }
    for (int k = t; k < nb; k += 256) weight[k] = grad_of(a, (first + k0 + k) / a.nbq, b);
    int from = 0;
    for (int shift = 0; shift < bits || shift == 0; shift += 4) {
#pragma unroll
      for (int g = 0; g < 16; g++) count[g * 256 + t] = 0;
      __syncthreads();
      const int i0 = t * per, i1 = i0 + per < n ? i0 + per : n;
      for (int i = i0; i < i1; i++) {
        const int e = shift == 0 ? i : order[from][i];
        count[((tok[e] >> shift) & 15) * 256 + t]++;
      }
      __syncthreads();
      // exclusive sums over (digit, thread): sixteen in a row a thread, then over the threads
      u32x4* mine = (u32x4*)(count + 16 * t);
      u32x4 c[2] = {mine[0], mine[1]};
      int sum = 0;
#pragma unroll
      for (int g = 0; g < 16; g++) {
        const int x = (int)((c[g / 8][(g / 2) & 3] >> (16 * (g & 1))) & 0xffffu);
        sum += x;
      }
      int before = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(before, o);
        before += lane >= o ? x : 0;
      }
      if (lane == 63) totals[wave] = before;
      __syncthreads();
      before -= sum;
      for (int w = 0; w < wave; w++) before += totals[w];
#pragma unroll
      for (int h = 0; h < 8; h++) {
        const uint32_t x = c[h / 4][h & 3], lo = x & 0xffffu, hi = x >> 16;
        c[h / 4][h & 3] = (uint32_t)before | (uint32_t)(before + (int)lo) << 16;
        before += (int)(lo + hi);
      }
      mine[0] = c[0];
      mine[1] = c[1];
      __syncthreads();
      const int to = shift == 0 ? 0 : from ^ 1;
      for (int i = i0; i < i1; i++) {
        const int e = shift == 0 ? i : order[from][i];
        order[to][count[((tok[e] >> shift) & 15) * 256 + t]++] = (uint16_t)e;
      }
      from = to;
      __syncthreads();
    }
    // The waves' shares, cut at the first maximum of a token; those of no token come last.
    const uint16_t* sorted = order[from];
    if (t < 5) {
      int lo = 0, hi = n;
      while (lo < hi) {  // how many have a token
        const int mid = (lo + hi) / 2;
        if (tok[sorted[mid]] < a.nd) lo = mid + 1;
        else hi = mid;
      }
      const int real = lo;
      int k = (int)((int64_t)real * t / 4);
      if (k > 0 && k < real) {  // the first one of the next token, if this one's is cut
        const int j = tok[sorted[k - 1]];
        hi = real;
        while (k < hi) {
          const int mid = (k + hi) / 2;
          if (tok[sorted[mid]] <= j) k = mid + 1;
          else hi = mid;
        }
      }
      cuts[t] = k;
    }
    __syncthreads();
    const int m0 = __builtin_amdgcn_readfirstlane(cuts[wave]), m1 = __builtin_amdgcn_readfirstlane(cuts[wave + 1]);
    // this wave's tokens: from the first of its share up to the next wave's first
    const int real = __builtin_amdgcn_readfirstlane(cuts[4]);
    const int j0 = wave == 0 ? 0 : m0 < real ? tok[sorted[m0]] : a.nd;
    const int j1 = wave == 3 || m1 >= real ? a.nd : tok[sorted[m1]];
    int cur = __builtin_amdgcn_readfirstlane(j0);
    const int end = __builtin_amdgcn_readfirstlane(j1);
    float x0 = 0.f, x1 = 0.f;
    int64_t at = ((int64_t)b * a.nd + cur) * a.d + col;
    auto flush = [&]() {  // token `cur` is done
      if (in) {
        if (begun) {
          x0 += a.sums[at];
          if (PAIR || col + 1 < a.d) x1 += a.sums[at + 1];
        }
        if (!last) {
          a.sums[at] = x0;
          if (PAIR || col + 1 < a.d) a.sums[at + 1] = x1;
        } else {
          T* out = (T*)a.dD + at;
          if constexpr (PAIR) {
            struct alignas(2 * sizeof(T)) Two {
              T v[2];
            };
            *(Two*)out = Two{{(T)x0, (T)x1}};
          } else {
            out[0] = (T)x0;
            if (col + 1 < a.d) out[1] = (T)x1;
          }
        }
      }
      x0 = x1 = 0.f;
      cur++;
      at += a.d;
    };
    // Sixty-four maxima at a time: each lane finds one's row, factor and whether it is the first
    // of its token, and the wave takes them from the lanes one after another. Past the end the
    // last one stands in with a factor of 0.
    for (int m = m0; m < m1; m += 64) {
      const int here = m1 - m < 64 ? m1 - m : 64;
      const int e = sorted[m + (lane < here ? lane : here - 1)];
      const int k = first + k0 + (e >> 5), q = a.nbq == 1 ? k : k / a.nbq;
      const uint32_t row = (uint32_t)(q * a.nq + (k - q * a.nbq) * 32 + (e & 31));
      const uint32_t from = PAIR ? row * (uint32_t)(a.d * (int)sizeof(T)) : row;  // bytes, below 2^32
      const int j = tok[e];
      const int before = __shfl_up(j, 1);
      const uint64_t firsts = __ballot(lane == 0 ? j != cur : j != before);
      const float w = lane < here ? weight[e >> 5] : 0.f;
      f32x2 x[2][AHEAD];
      auto load = [&](int buf, int s) {
        if (s >= here || s >= 64) return;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
          const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)from, s + i);
          if constexpr (PAIR) x[buf][i] = two<DT>((const uint8_t*)a.Q + (r + at_col));
          else x[buf][i] = in ? columns<DT>(Q + (int64_t)r * a.d, col, a.d) : f32x2{0.f, 0.f};
        }
      };
      auto add = [&](int buf, int s) {
        if (s >= here) return;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
          if ((firsts >> (s + i)) & 1) {
            const int js = __builtin_amdgcn_readlane(j, s + i);
            while (cur < js) flush();
          }
          const float ws = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s + i));
          x0 = __builtin_fmaf(ws, x[buf][i][0], x0);
          x1 = __builtin_fmaf(ws, x[buf][i][1], x1);
        }
      };
      load(0, 0);
#pragma unroll
      for (int s = 0; s < 64; s += 2 * AHEAD) {  // lanes and bits are constants: half of the scalar work
        load(1, s + AHEAD);
        add(0, s);
        load(0, s + 2 * AHEAD);
        add(1, s + AHEAD);
      }
    }
    while (cur < end) flush();
  }
}

// Where dQ's sums go: the gradient itself, or a split's part.
template <int DT>
__device__ __forceinline__ void put_q(const PairsGradArgs& a, int split, int64_t row, int col, float x0, float x1) {
  typedef typename El<DT>::T T;
  if (col >= a.d) return;
  const int64_t at = row * a.d + col;
  if (a.splits == 1) {
    T* out = (T*)a.dQ + at;
    out[0] = (T)x0;
    if (col + 1 < a.d) out[1] = (T)x1;
  } else {
    float* out = a.parts + (int64_t)split * a.nQ * a.nq * a.d + at;
    out[0] = x0;
    if (col + 1 < a.d) out[1] = x1;
  }
}

// dQ, many queries: sixteen waves, each with a block of 32 query tokens and 128 columns (two
// a lane) in registers, walk the same run of documents. A document's tokens come to LDS
// once for the 512 query tokens, while the one before is added up: each query token reads the
// row that answered it, 256 bytes in one wave's access. A lane finds its token's row, and the
// wave takes the rows from the lanes one after another: 6.1 vector and 4.7 scalar instructions a
// maximum in all. Where there is none, a row of zeros stands in. The runs' sums are joined by
// the kernel below, in order. 64 queries of 32 tokens x 4096 documents, d = 128, 16 bits: 155 us
// (with the positions through the scalar unit 278): the vector units busy for 53 % of it, the waves, four
// a SIMD, waiting for 48 % of theirs, at a barrier a document; padding is loaded too, a third of
// the bytes. The join takes 11 us.
// WHOLE: rows in pieces of 16 bytes, on their way in registers meanwhile; others element by element.
template <int DT, bool WHOLE>
__global__ __launch_bounds__(1024) void pairs_grad_q_kernel(PairsGradArgs a) {
  using T = typename El<DT>::T;
  constexpr int ES = DT == TMS_DTYPE_F32 ? 4 : 2, ROW = 128 * ES;
  constexpr int LD = 4;  // 16-byte loads a thread and stage: 64 KB
  extern __shared__ __attribute__((aligned(16))) uint8_t docs[];  // [2][tokens + 1][ROW]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t id = workgroup();
  const int split = (int)(id % a.splits), group = (int)(id / a.splits);
  if (group * 16 >= a.blocks) return;
  const int kb = group * 16 + wave;
  const bool mine = kb < a.blocks;
  const int q = mine ? kb / a.nbq : 0;
  const int col0 = (int)blockIdx.y * 128, cols = a.d - col0 < 128 ? a.d - col0 : 128;
  const int64_t e0 = (int64_t)split * a.chunk, e1 = e0 + a.chunk < a.B ? e0 + a.chunk : a.B;
  const int size = (a.tokens + 1) * ROW;

  for (int k = threadIdx.x; k < 2 * ROW / 4; k += 1024)  // the rows of zeros
    *(uint32_t*)(docs + (k / (ROW / 4)) * size + a.tokens * ROW + (k % (ROW / 4)) * 4) = 0u;

  struct Stage {  // a document and its tokens from t0 on
    int64_t b;
    int t0;
  };
  auto next = [&](Stage& s) {
    s.t0 += a.tokens;
    if (s.t0 >= a.nd) {
      s.t0 = 0;
      s.b++;
    }
  };
  auto tokens = [&](const Stage& s) { return a.nd - s.t0 < a.tokens ? a.nd - s.t0 : a.tokens; };
  auto from = [&](const Stage& s) { return (const uint8_t*)a.D + ((s.b * a.nd + s.t0) * a.d + col0) * ES; };
  u32x4 reg[WHOLE ? LD : 1];
  auto load = [&](const Stage& s) {
    if constexpr (WHOLE) {
      if (s.b >= e1) return;
      const uint8_t* base = from(s);
      const int n = tokens(s);
#pragma unroll
      for (int i = 0; i < LD; i++) {
        const int k = i * 1024 + (int)threadIdx.x, row = k / (ROW / 16), at = k % (ROW / 16);
        if (row < n && at * (16 / ES) < cols) reg[i] = *(const u32x4*)(base + (row * a.d * ES + at * 16));
      }
    }
  };
  auto put = [&](const Stage& s, int buf) {
    if (s.b >= e1) return;
    const int n = tokens(s);
    if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < LD; i++) {
        const int k = i * 1024 + (int)threadIdx.x;
        if (k / (ROW / 16) < n) *(u32x4*)(docs + buf * size + k * 16) = reg[i];
      }
    } else {
      const T* base = (const T*)from(s);
      for (int k = threadIdx.x; k < n * (ROW / ES); k += 1024) {
        const int row = k / (ROW / ES), col = k % (ROW / ES);
        if (col < cols) ((T*)(docs + buf * size))[k] = base[(int64_t)row * a.d + col];
      }
    }
  };

  // Lane i's position of the block's token i, and G, read a stage ahead.
  uint32_t at_next = kNone;
  float w_next = 0.f;
  auto look = [&](const Stage& s) {
    if (!mine || s.b >= e1) return;
    if (lane < 32) at_next = a.arg[s.b * a.nQ * a.nqp + (int64_t)kb * 32 + lane];
    w_next = grad_of(a, q, s.b);
  };

  float acc[32][2] = {};
  Stage now = {e0, 0}, soon = now;  // the one added up, and the last one asked for
  load(now);
  look(now);
  put(now, 0);
  next(soon);
  load(soon);
  __syncthreads();
  for (int buf = 0; now.b < e1; buf ^= 1) {
    const uint32_t j = at_next - (uint32_t)now.t0;
    const bool here = j < (uint32_t)tokens(now);  // of the tokens that there are: kNone is none of them
    const uint32_t row = (here ? j : (uint32_t)a.tokens) * ROW + buf * size;
    const float w = w_next;
    look(soon);
    if (mine) {
      const uint8_t* base = docs + lane * 2 * ES;
      // A row of zeros takes any factor but infinities and NaN away: the factor is 0 there too.
      const uint32_t answered = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)__ballot(here));
      const float ws = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, w)));
#pragma unroll
      for (int i = 0; i < 32; i++) {
        const f32x2 x = two<DT>(base + (uint32_t)__builtin_amdgcn_readlane((int)row, i));
        const float f = (answered >> i) & 1 ? ws : 0.f;
        acc[i][0] = __builtin_fmaf(f, x[0], acc[i][0]);
        acc[i][1] = __builtin_fmaf(f, x[1], acc[i][1]);
      }
    }
    put(soon, buf ^ 1);
    now = soon;
    next(soon);
    load(soon);
    __syncthreads();
  }
  if (!mine) return;
  const int i0 = (kb - q * a.nbq) * 32;
#pragma unroll
  for (int i = 0; i < 32; i++)
    if (i0 + i < a.nq) put_q<DT>(a, split, (int64_t)q * a.nq + i0 + i, col0 + 2 * lane, acc[i][0], acc[i][1]);
}

// dQ, few queries or documents of their own: eight waves share eight query tokens and 128
// columns, take the documents in turn straight from memory, and join through LDS in order.
// Bound by the latency of a position and then its row, eight of each in flight: 32 queries x 8
// documents of their own, d = 128: 5 us.
template <int DT>
__global__ __launch_bounds__(512) void pairs_grad_q_few_kernel(PairsGradArgs a) {
  constexpr int ES = DT == TMS_DTYPE_F32 ? 4 : 2;
  typedef typename El<DT>::T T;
  __shared__ float sums[8][8][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t id = workgroup();
  const int split = (int)(id % a.splits), unit = (int)(id / a.splits);
  const int groups = (a.nq + 7) / 8;
  const int q = unit / groups, i0 = (unit - q * groups) * 8;
  if (q >= a.nQ) return;
  const int col = (int)blockIdx.y * 128 + 2 * lane;
  const int64_t first = a.nway ? (int64_t)q * a.nway : 0, n = a.nway ? a.nway : a.B;
  const int64_t e0 = (int64_t)split * a.chunk, e1 = e0 + a.chunk < n ? e0 + a.chunk : n;
  const bool pair = a.d % 2 == 0 && (uintptr_t)a.D % (2 * ES) == 0;
  float acc[8][2] = {};
  for (int64_t k = e0 + wave; k < e1; k += 8) {
    const int64_t b = first + k;
    const float w = grad_of(a, q, b);
    const uint32_t* at = (const uint32_t*)(a.arg + (a.nway ? b : b * a.nQ + q) * a.nqp + i0);
    f32x2 x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t j = (at[i / 2] >> (16 * (i & 1))) & 0xffffu;
      x[i] = f32x2{0.f, 0.f};
      if (j < (uint32_t)a.nd && col < a.d) {  // kNone is beyond every document
        const T* row = (const T*)a.D + ((int64_t)b * a.nd + j) * a.d + col;
        if (pair) {
          x[i] = two<DT>((const uint8_t*)row);
        } else {
          x[i][0] = (float)row[0];
          x[i][1] = col + 1 < a.d ? (float)row[1] : 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t j = (at[i / 2] >> (16 * (i & 1))) & 0xffffu;
      const float f = j < (uint32_t)a.nd ? w : 0.f;
      acc[i][0] = __builtin_fmaf(f, x[i][0], acc[i][0]);
      acc[i][1] = __builtin_fmaf(f, x[i][1], acc[i][1]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; i++) *(f32x2*)&sums[wave][i][2 * lane] = f32x2{acc[i][0], acc[i][1]};
  __syncthreads();
  if (i0 + wave >= a.nq) return;
  f32x2 x = {0.f, 0.f};
#pragma unroll
  for (int v = 0; v < 8; v++) {
    x[0] += sums[v][wave][2 * lane];
    x[1] += sums[v][wave][2 * lane + 1];
  }
  put_q<DT>(a, split, (int64_t)q * a.nq + i0 + wave, col, x[0], x[1]);
}

// The splits' sums: four waves take a quarter of the splits each for 64 elements, eight loads at
// a time, and join in order. Bound by latency where there are few elements, else by the read.
template <int DT>
__global__ __launch_bounds__(256) void pairs_grad_q_join_kernel(const float* parts, void* dQ, int64_t n, int splits) {
  typedef typename El<DT>::T T;
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t k = (int64_t)blockIdx.x * 64 + lane;
  const int each = (splits + 3) / 4, s0 = wave * each, s1 = s0 + each < splits ? s0 + each : splits;
  float x = 0.f;
  if (k < n) {
    for (int s = s0; s < s1; s += 8) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = s + i < s1 ? parts[(s + i) * n + k] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) x += y[i];
    }
  }
  sums[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && k < n) ((T*)dQ)[k] = (T)(sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]);
}

// ---------------------------------------------------------------- host

static int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Whether the forward kernels take these rows as they are.
static bool as_is(const void* p, int64_t d, int dtype) {
  return dtype != TMS_DTYPE_F32 && d % 32 == 0 && (uintptr_t)p % 16 == 0;
}
static int planes(int dtype) { return dtype == TMS_DTYPE_F32 ? 3 : 1; }

// dQ's form and its splits of the documents. The form that shares documents takes one workgroup
// a CU, and pays from about 8,192 blocks of 32 maxima on (32-token queries x documents of 180
// tokens, d = 128, 16 bits, few / shared: 64 x 100 19 / 28 us, 16 x 1000 53 / 38, 4 x 4000 55 / 40, 64 x 4096 761 / 158).
// The other fills the chip twice over, with at least eight documents (one a wave) a split. The
// sums of a split are written and read once, so no more splits than fill the chip. A multiple
// of 8 where there are several: workgroups go to the XCDs in turn, so an XCD then keeps to its
// own documents.
struct GradQ {
  bool shared;
  int splits;
};
static GradQ grad_q_form(int64_t nQ, int64_t nq, int64_t d, int64_t B, int64_t nway) {
  const int64_t cols = (d + 127) / 128, blocks = nQ * ((nq + 31) / 32);
  GradQ f;
  f.shared = nway == 0 && blocks >= 4 && blocks * B > 8192;
  const int64_t units = (f.shared ? (blocks + 15) / 16 : nQ * ((nq + 7) / 8)) * cols;
  const int64_t most = f.shared ? B / 4 : (nway ? nway : B) / 8;
  int64_t s = (f.shared ? 256 : 512) / (units > 0 ? units : 1);
  if (s > most) s = most;
  if (s >= 8) s = s / 8 * 8;
  f.splits = (int)(s < 1 ? 1 : s);
  return f;
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
  const dim3 grid = grid_of(a.B, a.nway ? 1u : (unsigned)a.nQ);
  hipLaunchKernelGGL((pairs_direct_kernel<DT, KS, PL>), grid, dim3(256), 0, st, a);
  return check_launch("pairs_direct_kernel");
}

template <int DT, int KS, int NB, int PL>
static int run_shared(PairsArgs a, hipStream_t st) {
  a.qpw = NB / a.nbq;
  const int64_t groups = (a.nQ + 8 * a.qpw - 1) / (8 * a.qpw);
  const int64_t stages = (a.nd + kStage - 1) / kStage;
  // Documents a workgroup: its mask words, and as many workgroups as run at once, for each reads
  // its queries first: one a CU of the forms with the most registers (64 queries x 4096
  // documents, d = 128: 315 us in 256 workgroups, 324 in 512, 342 in 768), else two.
  constexpr int kWhole = NB * KS * PL >= 6 ? 256 : 512;
  int64_t docs = kMaskWords / (stages > 0 ? stages : 1);
  const int64_t even = (a.B * groups + kWhole - 1) / kWhole;
  if (docs > even) docs = even;
  if (docs < 1) docs = 1;
  a.docs_per_wg = (int32_t)docs;
  const dim3 grid((unsigned)((a.B + docs - 1) / docs), (unsigned)groups);
  if (a.arg) hipLaunchKernelGGL((pairs_shared_kernel<DT, KS, NB, PL, true>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((pairs_shared_kernel<DT, KS, NB, PL, false>), grid, dim3(512), 0, st, a);
  return check_launch("pairs_shared_kernel");
}

template <int DT, int KS, int PL>
static int run_width(const PairsArgs& a, hipStream_t st) {
  if constexpr (PL == 3) return run_shared<DT, KS, 1, 3>(a, st);
  else {
    // Blocks a wave: more share a document's fragments, fewer leave less of the last group of
    // waves empty. A block takes 1.2, 1.13 and 1 times as long with one, two and four a wave
    // (64 queries x 4096 documents, d = 128, with positions: 480, 476 and 421 us; 37 x 501 documents
    // of 300 tokens, d = 96, without: 44, 48 and 53; 48 x 2000, d = 64: 95, 69 and 88).
    auto time = [&](int nb, int each) {
      const int64_t queries = 8 * (nb / a.nbq);
      return (a.nQ + queries - 1) / queries * nb * each;
    };
    const int64_t four = time(4, 100), two = a.nbq <= 2 ? time(2, 113) : four + 1, one = a.nbq <= 1 ? time(1, 120) : four + 1;
    if (one < two && one < four) return run_shared<DT, KS, 1, 1>(a, st);
    if (two < four) return run_shared<DT, KS, 2, 1>(a, st);
    return run_shared<DT, KS, 4, 1>(a, st);
  }
}

template <int DT, int PL>
static int run_pairs(PairsArgs& a, hipStream_t st) {
  const int64_t blocks = (int64_t)a.nQ * a.nbq;
  const int ks = a.d / 32;
  // Sharing pays once there are workgroups enough; a call of few pairs needs one for each
  // instead. (16 bits, d = 128, 180 tokens, direct / shared: 32 x 32 pairs 11 / 17 us, 8 x 128 11 / 11, 8 x 256
  // 20 / 11, 2 x 2000 41 / 27, 1 x 4000 42 / 46; fp32: 8 x 32 19 / 26, 4 x 125 32 / 31, 32 x 32 42 / 27, 2 x 2000
  // 234 / 201.) A document takes at most kMaskWords stages (65,535 tokens).
  const bool shared = !a.nway && ks <= 4 && a.nbq <= (PL == 3 ? 1 : 4) && blocks >= 2 && a.B * a.nQ > (PL == 3 ? 512 : 1024);
  if (shared) {
    switch (ks) {
      case 1: return run_width<DT, 1, PL>(a, st);
      case 2: return run_width<DT, 2, PL>(a, st);
      case 3: return run_width<DT, 3, PL>(a, st);
      default: return run_width<DT, 4, PL>(a, st);
    }
  }
  switch (ks) {
    case 1: return run_direct<DT, 1, PL>(a, st);
    case 2: return run_direct<DT, 2, PL>(a, st);
    case 3: return run_direct<DT, 3, PL>(a, st);
    case 4: return run_direct<DT, 4, PL>(a, st);
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
static int run_grads(PairsGradArgs a, const GradQ& form, hipStream_t st) {
  int rc;
  if (a.dD && a.B > 0 && a.nd > 0 && a.d > 0) {
    const int n = a.nway ? a.nbq : a.blocks;
    a.run = n < 1 ? 1 : n < kRun ? n : kRun;
    const size_t lds = (size_t)a.run * 32 * 6 + 16 * 256 * 2 + (size_t)a.run * 4;
    const dim3 grid = grid_of(a.B, (unsigned)((a.d + 127) / 128));
    const bool pair = a.d % 2 == 0 && (int64_t)a.nQ * a.nq * a.d * (int64_t)sizeof(typename El<DT>::T) < ((int64_t)1 << 32) && (uintptr_t)a.Q % 8 == 0 && (uintptr_t)a.dD % 8 == 0;
    if (pair) hipLaunchKernelGGL((pairs_grad_d_kernel<DT, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((pairs_grad_d_kernel<DT, false>), grid, dim3(256), lds, st, a);
    if ((rc = check_launch("pairs_grad_d_kernel"))) return rc;
  }
  if (a.dQ && a.nQ > 0 && a.nq > 0 && a.d > 0) {
    const unsigned cols = (unsigned)((a.d + 127) / 128);
    const int64_t n = a.nway ? a.nway : a.B;
    a.splits = form.splits;
    a.chunk = (int32_t)((n + a.splits - 1) / a.splits);
    if (form.shared && a.nd > 0) {
      constexpr int es = DT == TMS_DTYPE_F32 ? 4 : 2;
      const int most = 65536 / (128 * es);  // a stage is at most 64 KB
      const int stages = (a.nd + most - 1) / most;
      a.tokens = stages > 0 ? (a.nd + stages - 1) / stages : 0;
      const size_t lds = 2 * (size_t)(a.tokens + 1) * 128 * es;
      const bool whole = a.d * es % 16 == 0 && (uintptr_t)a.D % 16 == 0;
      const dim3 grid = grid_of((int64_t)(a.blocks + 15) / 16 * a.splits, cols);
      if (whole) hipLaunchKernelGGL((pairs_grad_q_kernel<DT, true>), grid, dim3(1024), lds, st, a);
      else hipLaunchKernelGGL((pairs_grad_q_kernel<DT, false>), grid, dim3(1024), lds, st, a);
      if ((rc = check_launch("pairs_grad_q_kernel"))) return rc;
    } else {
      hipLaunchKernelGGL(pairs_grad_q_few_kernel<DT>, grid_of((int64_t)a.nQ * ((a.nq + 7) / 8) * a.splits, cols), dim3(512), 0, st, a);
      if ((rc = check_launch("pairs_grad_q_few_kernel"))) return rc;
    }
    if (a.splits > 1) {
      const int64_t m = (int64_t)a.nQ * a.nq * a.d;
      hipLaunchKernelGGL(pairs_grad_q_join_kernel<DT>, dim3((unsigned)((m + 63) / 64)), dim3(256), 0, st, a.parts, a.dQ, m, a.splits);
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
  return (nway > 0 ? B : nQ * B) * round_up(nq, 32);
}

extern "C" int tms_maxsim_pairs(const void* Qs, int64_t nQ, int64_t nq, int64_t d, const void* D, int64_t B, int64_t nd,
                                int64_t nway, const uint8_t* qmask, const uint8_t* dmask, int dtype, void* workspace,
                                int64_t workspace_bytes, float* scores, uint16_t* positions, void* stream) {
  const char* fn = "tms_maxsim_pairs";
  int rc = check_pairs(fn, nQ, nq, d, B, nd, nway, dtype);
  if (rc) return rc;
  if (nQ == 0 || B == 0) return TMS_OK;
  if (!scores || (nq * d > 0 && !Qs) || (nd * d > 0 && !D)) return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if ((uintptr_t)positions % 16) return fail(TMS_ERR_INVALID, "%s: positions must be 16-byte aligned", fn);
  const hipStream_t st = (hipStream_t)stream;
  PairsArgs a = {};
  a.qmask = qmask;
  a.dmask = dmask;
  a.scores = scores;
  a.arg = positions;
  a.B = B;
  a.nQ = (int32_t)nQ;
  a.nq = (int32_t)nq;
  a.nqp = (int32_t)round_up(nq, 32);
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

static int64_t parts_bytes(int64_t nQ, int64_t nq, int64_t d, const GradQ& f) { return f.splits > 1 ? round_up(f.splits * nQ * nq * d * 4, 256) : 0; }

extern "C" int64_t tms_pairs_grad_workspace_size(int64_t nQ, int64_t nq, int64_t d, int64_t B, int64_t nd, int64_t nway) {
  if (nQ <= 0 || nq <= 0 || d <= 0 || B <= 0 || nd < 0) return 0;
  const int64_t runs = nway > 0 ? (nq + 31) / 32 : nQ * ((nq + 31) / 32);
  return parts_bytes(nQ, nq, d, grad_q_form(nQ, nq, d, B, nway)) + (runs > kRun ? B * nd * d * 4 : 0);
}

extern "C" int tms_maxsim_pairs_grad(const void* Qs, int64_t nQ, int64_t nq, int64_t d, const void* D, int64_t B, int64_t nd,
                                     int64_t nway, const uint16_t* positions, const float* grad, int dtype, void* workspace,
                                     int64_t workspace_bytes, void* dQ, void* dD, void* stream) {
  const char* fn = "tms_maxsim_pairs_grad";
  const int rc = check_pairs(fn, nQ, nq, d, B, nd, nway, dtype);
  if (rc) return rc;
  if ((dQ && nQ * nq * d > 0 && B > 0 && nd > 0 && !D) || (dD && B * nd * d > 0 && nQ * nq > 0 && !Qs) ||
      (nQ * nq > 0 && B > 0 && (!positions || !grad)))
    return fail(TMS_ERR_INVALID, "%s: NULL pointer", fn);
  if ((uintptr_t)positions % 16) return fail(TMS_ERR_INVALID, "%s: positions must be 16-byte aligned", fn);
  const int64_t need = tms_pairs_grad_workspace_size(nQ, nq, d, B, nd, nway);
  if (need > 0 && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
    return fail(TMS_ERR_INVALID, "%s: a workspace of %lld bytes is needed, 16-byte aligned", fn, (long long)need);
  PairsGradArgs a = {};
  a.Q = Qs;
  a.D = D;
  a.arg = positions;
  a.G = grad;
  a.dQ = dQ;
  a.dD = dD;
  const GradQ form = grad_q_form(nQ, nq, d, B, nway);
  a.parts = (float*)workspace;
  a.sums = (float*)((uint8_t*)workspace + parts_bytes(nQ, nq, d, form));
  a.B = B;
  a.nQ = (int32_t)nQ;
  a.nq = (int32_t)nq;
  a.nqp = (int32_t)round_up(nq, 32);
  a.nd = (int32_t)nd;
  a.d = (int32_t)d;
  a.nway = (int32_t)nway;
  a.nbq = (int32_t)((nq + 31) / 32);
  a.blocks = a.nQ * a.nbq;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TMS_DTYPE_F16) return run_grads<TMS_DTYPE_F16>(a, form, st);
  if (dtype == TMS_DTYPE_BF16) return run_grads<TMS_DTYPE_BF16>(a, form, st);
  return run_grads<TMS_DTYPE_F32>(a, form, st);
}
