// Attention over packed texts, forward and backward.
//
//   x[i, j] = scale <q[i], k[j]>,  with a cap x = cap tanh(x / cap),  with a bias x -= slope |i - j|
//   P[i, j] = exp(x[i, j] - L[i]) over the j that i sees,  L[i] = log sum_j exp x[i, j]
//   o[i] = sum_j P[i, j] v[j]
//   dv[j] = sum_i P[i, j] do[i],  dP[i, j] = <do[i], v[j]>,  delta[i] = <do[i], o[i]>
//   dS[i, j] = P[i, j] (dP[i, j] - delta[i])  (times 1 - tanh^2 under a cap)
//   dq[i] = scale sum_j dS[i, j] k[j],  dk[j] = scale sum_i dS[i, j] q[i]
//
// Texts stand one behind another. A token sees its own text alone: all of it, or (with
// prefixes) the text's first prefix tokens and those up to itself. A workgroup takes a tile of
// one text's rows, so nothing of another text, NaN included, comes near its sums; tiles of
// short texts are partly empty, but a wave without rows only loads.
//
// All three kernels have one shape. What a wave owns (16 NB queries, or keys in the kernel for
// dk and dv) stands in registers as columns of the matrix instructions; what it goes over comes
// through LDS, 64 rows at a time, as their rows:
//   S^T = K Q^T: a lane has four neighbouring keys of one query: the softmax runs in a lane, and
//   two exchanges between the wave's four rows of lanes finish a maximum;
//   o^T += V^T P^T: a lane's P are in the place where the next product takes them, when the
//   keys of a step are numbered as the first product left them. V^T's fragments come
//   out of LDS by transposing reads, from the rows as they lie in memory.
// With queries and keys in each other's place that is the kernel for dk and dv, where P and dS
// are formed once more: seven products for a backward pass and not five, and no atomics: every
// sum has one order. Each row's text is found from its tile's number alone (AttnTile), without
// a list of tiles and without the host knowing the lengths.
//
// In LDS a row of 32 elements takes 64 bytes (fp32: 128), two rows a line of 128, whose 16-byte
// pieces stand at p ^ (line % 8): the row fragments (a lane's eight neighbouring elements) and the
// transposing reads both fall evenly on the banks.
//
// Precision. Scores, statistics, sums and gradients are fp32. P and dS are rounded to the
// inputs' type between two products (2^-9 of each term in bf16, 2^-12 in fp16), as the matrix
// cores take them. fp16 has no range to spare for gradients: P is held times 2^15, and dS times
// a power of two for each row (column of sums) that follows the largest |dS| so far. delta is
// taken from o in two 16-bit terms (2^-17 of it): from o as it is returned, dS would have o's rounding
// even where P is 1 and dS 0. fp32 goes through the fp32 matrix instructions.
#pragma once
#include <math.h>

#include "tms_common.h"

namespace tms {

typedef short attn_s16x4 __attribute__((ext_vector_type(4)));

constexpr int kAttnThreads = 256;
constexpr float kAttnLog2e = 1.4426950408889634f;
constexpr int kAttnP16 = 15;  // fp16: P times 2^15 in the backward pass

struct AttnArgs {
  const void *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;  // elements between tokens and heads
  const int64_t* offsets;          // B + 1
  const int64_t* prefix;           // B, or NULL: a text sees all of itself
  const float* slopes;             // H, or NULL
  int64_t T;
  int32_t B, H, KV, slots;
  float scale, cap;  // cap 0: none
  void* out;         // (T, H, D)
  void* low;         // what out's rounding left, of out's type, or NULL
  float* lse;        // (H, T): log2 of the sums of exponentials; or NULL
  // backward
  const void* grad;  // (T, H, D)
  float* delta;      // (H, T)
  void *dq, *dk, *dv;
};

template <int DT>
struct AttnType {
  typedef uint16_t E;
  typedef u32x4 Frag;  // eight elements
  static constexpr int kRows = 64;  // rows of a tile that passes through LDS
};
template <>
struct AttnType<TMS_DTYPE_F32> {
  typedef float E;
  typedef u32x8 Frag;
  static constexpr int kRows = 32;
};

// One product of 16 x 16 over 32: lane (c, g) gives eight elements of row (column) c each; which k
// they are is the caller's, the same for both operands.
template <int DT>
__device__ __forceinline__ f32x4 attn_mfma(typename AttnType<DT>::Frag a, typename AttnType<DT>::Frag b, f32x4 c) {
  if constexpr (DT == TMS_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t x = a[e], y = b[e];
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y), c, 0, 0, 0);
    }
    return c;
  } else {
    return mfma16x16x32<DT>(a, b, c);
  }
}

// A fragment of eight fp32 values in the inputs' type, rounded to nearest.
template <int DT>
__device__ __forceinline__ typename AttnType<DT>::Frag attn_pack(f32x4 lo, f32x4 hi) {
  typename AttnType<DT>::Frag r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (DT == TMS_DTYPE_F32) {
      const float a = lo[i], b = hi[i];
      r[i] = __builtin_bit_cast(uint32_t, a);
      r[4 + i] = __builtin_bit_cast(uint32_t, b);
    } else {
      const float a = i < 2 ? lo[2 * i] : hi[2 * i - 4], b = i < 2 ? lo[2 * i + 1] : hi[2 * i - 3];
      if constexpr (DT == TMS_DTYPE_BF16) {
        const f32x2 v = {a, b};
        r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
      } else {
        r[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
      }
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ float attn_float(typename AttnType<DT>::E x) {
  if constexpr (DT == TMS_DTYPE_F32) return x;
  else if constexpr (DT == TMS_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, x);
  else return __builtin_bit_cast(float, (uint32_t)x << 16);
}
template <int DT>
__device__ __forceinline__ typename AttnType<DT>::E attn_round(float x) {
  if constexpr (DT == TMS_DTYPE_F32) return x;
  else if constexpr (DT == TMS_DTYPE_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
  else return __builtin_bit_cast(uint16_t, (__bf16)x);
}
// Element e of a fragment.
template <int DT>
__device__ __forceinline__ float attn_elem(const typename AttnType<DT>::Frag& f, int e) {
  if constexpr (DT == TMS_DTYPE_F32) {
    const uint32_t x = f[e];
    return __builtin_bit_cast(float, x);
  } else {
    return attn_float<DT>((uint16_t)(f[e / 2] >> (16 * (e & 1))));
  }
}

// The tile of `rows` rows with number w. Text t (0: what stands before the first text, B + 1: behind
// the last) has the numbers from floor(begin / rows) + t on: texts that follow each other never share
// one, whatever their lengths, and floor(T / rows) + B + 2 numbers hold all. A few of them
// have no rows. Offsets are taken within [0, T]; where they descend, some rows have no tile, or two.
struct AttnTile {
  int32_t text;  // -1: no rows
  bool real;     // rows of a text
  int32_t first, begin, end;  // the tile's first row; the text's rows
  int32_t prefix_end;         // rows before it are seen by the whole text; end without prefixes

  __device__ __forceinline__ static int32_t offset(const AttnArgs& a, int i) {
    if (i == 0) return 0;
    if (i > a.B + 1) return (int32_t)a.T;
    const int64_t x = a.offsets[i - 1];
    return (int32_t)(x < 0 ? 0 : x > a.T ? a.T : x);
  }
  __device__ __forceinline__ void find(const AttnArgs& a, int w, int rows) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.B + 2;
    while (n > 1) {  // 64 candidates at a time
      const int step = (n + 63) / 64, i = lane * step;
      const bool in = i < n;
      const uint64_t hit = __ballot(in && (lane == 0 || offset(a, lo + i) / rows + lo + i <= w));
      const int at = (63 - __builtin_clzll(hit)) * step;  // the last one at or before w
      lo += at;
      n = n - at < step ? n - at : step;
    }
    text = __builtin_amdgcn_readfirstlane(lo);
    begin = __builtin_amdgcn_readfirstlane(offset(a, text));
    end = __builtin_amdgcn_readfirstlane(offset(a, text + 1));
    const int64_t at = (int64_t)begin + (int64_t)(w - (begin / rows + text)) * rows;
    if (at < begin || at >= end) {
      text = -1;
      return;
    }
    first = (int32_t)at;
    real = text > 0 && text <= a.B;
    prefix_end = end;
    if (real && a.prefix) {
      const int64_t p = a.prefix[text - 1], len = end - begin;
      prefix_end = begin + (int32_t)(p < 0 ? 0 : p > len ? len : p);
      prefix_end = __builtin_amdgcn_readfirstlane(prefix_end);
    }
  }
};

// Which tile and head a workgroup takes: each XCD (workgroups go to the eight in turn) takes a run of its
// own, head by head, so that the tiles of a long text that read the same keys share an L2.
__device__ __forceinline__ bool attn_place(const AttnArgs& a, int heads, int& slot, int& head) {
  const int64_t total = (int64_t)a.slots * heads, each = (total + 7) / 8;
  const int64_t at = blockIdx.x % 8 * each + blockIdx.x / 8;
  if (blockIdx.x / 8 >= each || at >= total) return false;
  head = (int)(at / a.slots);
  slot = (int)(at - (int64_t)head * a.slots);
  return true;
}

// Rows of D elements in LDS, and the way there: from memory to registers, and (after the wait that
// the store makes) to LDS. Rows from `limit` on are zeros.
template <int DT, int D>
struct AttnRows {
  typedef AttnType<DT> Ty;
  typedef typename Ty::Frag Frag;
  static constexpr int R = Ty::kRows, ES = sizeof(typename Ty::E);
  static constexpr int kBytes = R * D * ES;
  static constexpr int kPanel = R * 32 * ES;                 // bytes of 32 columns
  static constexpr int kLoads = kBytes / 16 / kAttnThreads;  // 16-byte pieces a thread
  static_assert(kBytes % (16 * kAttnThreads) == 0, "whole pieces");
  u32x4 held[kLoads];

  // Piece n of the tile, in the order of LDS: its row and first element.
  __device__ __forceinline__ static void piece(int n, int& row, int& col) {
    const int panel = n / (kPanel / 16), in = n % (kPanel / 16), line = in / 8, p = (in % 8) ^ (line % 8);
    if constexpr (ES == 4) row = line, col = panel * 32 + p * 4;
    else row = 2 * line + (p >> 2), col = panel * 32 + (p & 3) * 8;
  }
  __device__ __forceinline__ void load(const typename Ty::E* base, int64_t stride, int first, int limit) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      int row, col;
      piece(i * kAttnThreads + (int)threadIdx.x, row, col);
      held[i] = u32x4{0u, 0u, 0u, 0u};
      if (first + row < limit) held[i] = *(const u32x4*)(base + (int64_t)(first + row) * stride + col);
    }
  }
  __device__ __forceinline__ void store(uint8_t* lds) const {
#pragma unroll
    for (int i = 0; i < kLoads; i++) *(u32x4*)(lds + (i * kAttnThreads + (int)threadIdx.x) * 16) = held[i];
  }
  // Row 16 block + c, elements 32 ks + 8 g ..
  __device__ __forceinline__ static Frag row_frag(const uint8_t* lds, int block, int ks, int c, int g) {
    if constexpr (ES == 4) {
      const int row = block * 16 + c;
      const uint8_t* p = lds + ks * kPanel + row * 128;
      const u32x4 lo = *(const u32x4*)(p + ((2 * g) ^ (row & 7)) * 16), hi = *(const u32x4*)(p + ((2 * g + 1) ^ (row & 7)) * 16);
      return u32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      const int line = block * 8 + (c >> 1);
      return *(const u32x4*)(lds + ks * kPanel + line * 128 + ((((c & 1) << 2) + g) ^ (line & 7)) * 16);
    }
  }
  // Column 16 db + c, rows 32 step + 4 g + (0 .. 3) and 16 further.
  __device__ __forceinline__ static Frag col_frag(const uint8_t* lds, int step, int db, int c, int g) {
    if constexpr (ES == 4) {
      u32x8 r;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int row = step * 32 + (e >> 2) * 16 + 4 * g + (e & 3);
        r[e] = *(const uint32_t*)(lds + (db >> 1) * kPanel + row * 128 + ((((db & 1) << 2) + (c >> 2)) ^ (row & 7)) * 16 + (c & 3) * 4);
      }
      return r;
    } else {
      typedef __attribute__((address_space(3))) attn_s16x4* LP;
      // 16 lanes read rows 4 g + (0 .. 3) of 16 columns: lane c four elements from 4 (c % 4) of row c / 4
      const int row = step * 32 + 4 * g + (c >> 2), line = row >> 1, p = ((row & 1) << 2) + ((db & 1) << 1) + ((c >> 1) & 1);
      const uint8_t* at = lds + (db >> 1) * kPanel + line * 128 + (p ^ (line & 7)) * 16 + (c & 1) * 8;
      const attn_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)at);
      const attn_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(at + 8 * 128));  // 16 rows on: the same line % 8
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      return u32x4{x[0], x[1], y[0], y[1]};
    }
  }
};

// A wave's own rows, as columns of the products: lane (c, g) has elements 32 ks + 8 g .. of row c.
template <int DT, int D>
__device__ __forceinline__ void attn_own(const typename AttnType<DT>::E* base, int64_t row_elems, int g,
                                         typename AttnType<DT>::Frag (&f)[D / 32]) {
  typedef typename AttnType<DT>::Frag Frag;
#pragma unroll
  for (int ks = 0; ks < D / 32; ks++) f[ks] = *(const Frag*)(base + row_elems + ks * 32 + 8 * g);
}

// A score in powers of two from the sum of products, and (under a cap) its derivative's factor.
struct AttnScore {
  float c1, cap2, inv_cap, slope2;  // scale log2(e), cap log2(e), scale / cap, slope log2(e)
  __device__ __forceinline__ void init(const AttnArgs& a, int head) {
    c1 = a.scale * kAttnLog2e;
    cap2 = a.cap * kAttnLog2e;
    inv_cap = a.cap > 0.f ? a.scale / a.cap : 0.f;
    slope2 = a.slopes ? a.slopes[head] * kAttnLog2e : 0.f;
  }
  template <int DT>
  __device__ __forceinline__ static float tanh_of(float z) {
    if constexpr (DT == TMS_DTYPE_F32) return tanhf(z);
    // 1 - 2 / (1 + e^2z): to 2^-22 or so of the cap, where the operands have 2^-9 or 2^-12
    return __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * (2.f * kAttnLog2e))), 1.f);
  }
  template <int DT>
  __device__ __forceinline__ float operator()(float s, int far, float* factor) const {
    float x;
    if (cap2 > 0.f) {  // uniform
      const float t = tanh_of<DT>(s * inv_cap);
      x = t * cap2;
      if (factor) *factor = __builtin_fmaf(-t, t, 1.f);
    } else {
      x = s * c1;
      if (factor) *factor = 1.f;
    }
    return __builtin_fmaf(-slope2, (float)(far < 0 ? -far : far), x);
  }
};

// ---------------------------------------------------------------- forward

// GENERAL: with a cap or a bias. NB: blocks of 16 queries a wave.
template <int DT, int D, int NB, bool GENERAL>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_forward_kernel(AttnArgs a) {
  typedef AttnRows<DT, D> Rows;
  typedef typename AttnType<DT>::E E;
  typedef typename AttnType<DT>::Frag Frag;
  constexpr int R = Rows::R, KB = R / 16, DB = D / 16, KS = D / 32, BQ = 64 * NB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t attn_mem[];
  int slot, head;
  if (!attn_place(a, a.H, slot, head)) return;
  AttnTile t;
  t.find(a, slot, BQ);
  if (t.text < 0) return;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int row0 = t.first + wave * 16 * NB;
  const float NEG = -__builtin_inff();

  f32x4 acc[DB][NB];
#pragma unroll
  for (int d = 0; d < DB; d++)
#pragma unroll
    for (int j = 0; j < NB; j++) acc[d][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top[NB], sum[NB];
#pragma unroll
  for (int j = 0; j < NB; j++) top[j] = NEG, sum[j] = 0.f;

  if (t.real) {
    const int kvh = head / (a.H / a.KV);
    const E* K = (const E*)a.k + kvh * a.kh;
    const E* V = (const E*)a.v + kvh * a.vh;
    AttnScore score;
    score.init(a, head);
    Frag q[NB][KS];
    int sees[NB];  // a row's last visible key, plus one
    int least = t.end;
#pragma unroll
    for (int j = 0; j < NB; j++) {
      const int row = row0 + 16 * j + c, in = row < t.end ? row : t.end - 1;
      attn_own<DT, D>((const E*)a.q + head * a.qh, (int64_t)in * a.qt, g, q[j]);
      sees[j] = in + 1 > t.prefix_end ? in + 1 : t.prefix_end;
    }
    if (row0 + 1 > t.prefix_end) least = row0 + 1;
    else least = t.prefix_end;
    // keys that any of the workgroup's rows sees, and any of this wave's
    const int last = t.first + BQ < t.end ? t.first + BQ : t.end;
    const int keys = last > t.prefix_end ? last : t.prefix_end;
    int mine = row0 + 16 * NB < t.end ? row0 + 16 * NB : t.end;
    mine = row0 >= t.end ? t.begin : mine > t.prefix_end ? mine : t.prefix_end;

    Rows rk, rv;
    rk.load(K, a.kt, t.begin, keys);
    rv.load(V, a.vt, t.begin, keys);
    int buf = 0;
    for (int k0 = t.begin; k0 < keys; k0 += R) {
      uint8_t* lk = attn_mem + buf * 2 * Rows::kBytes;
      uint8_t* lv = lk + Rows::kBytes;
      rk.store(lk);
      rv.store(lv);
      __syncthreads();
      if (k0 + R < keys) {
        rk.load(K, a.kt, k0 + R, keys);
        rv.load(V, a.vt, k0 + R, keys);
      }
      __builtin_amdgcn_sched_barrier(0);
      buf ^= 1;
      if (k0 >= mine) continue;  // uniform in the wave

      f32x4 s[KB][NB];
#pragma unroll
      for (int b = 0; b < KB; b++) {
#pragma unroll
        for (int j = 0; j < NB; j++) s[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const Frag f = Rows::row_frag(lk, b, ks, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) s[b][j] = attn_mfma<DT>(f, q[j][ks], s[b][j]);
        }
      }
      if constexpr (GENERAL) {
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              s[b][j][e] = score.template operator()<DT>(s[b][j][e], row0 + 16 * j + c - (k0 + 16 * b + 4 * g + e), nullptr);
      }
      if (k0 + R > least) {  // some row does not see all of the tile
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[b][j][e] = k0 + 16 * b + 4 * g + e < sees[j] ? s[b][j][e] : NEG;
      }
      Frag p[NB][R / 32];
#pragma unroll
      for (int j = 0; j < NB; j++) {
        float m = NEG;
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int e = 0; e < 4; e++) m = fmaxf(m, s[b][j][e]);
        m = cross_row_max(m);
        if constexpr (!GENERAL) m *= score.c1;
        if (__ballot(m > top[j]) != 0ull) {
          const float up = fmaxf(m, top[j]);
          const float k = up == NEG ? 1.f : __builtin_amdgcn_exp2f(top[j] - up);
          top[j] = up;
          sum[j] *= k;
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[d][j][e] *= k;
        }
        const float ref = top[j] == NEG ? 0.f : top[j];
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float x;
            if constexpr (GENERAL) x = s[b][j][e] - ref;
            else x = __builtin_fmaf(s[b][j][e], score.c1, -ref);
            s[b][j][e] = __builtin_amdgcn_exp2f(x);
            sum[j] += s[b][j][e];
          }
#pragma unroll
        for (int h = 0; h < R / 32; h++) p[j][h] = attn_pack<DT>(s[2 * h][j], s[2 * h + 1][j]);
      }
#pragma unroll
      for (int h = 0; h < R / 32; h++)
#pragma unroll
        for (int d = 0; d < DB; d++) {
          const Frag f = Rows::col_frag(lv, h, d, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) acc[d][j] = attn_mfma<DT>(f, p[j][h], acc[d][j]);
        }
    }
  }

#pragma unroll
  for (int j = 0; j < NB; j++) {
    const int row = row0 + 16 * j + c;
    if (row >= t.end) continue;
    const float all = t.real ? sum[j] : 0.f;
    float z = all;
    z += __shfl_xor(z, 16);
    z += __shfl_xor(z, 32);
    const float inv = t.real ? 1.f / z : 0.f;
    if (a.lse && g == 0) a.lse[(int64_t)head * a.T + row] = t.real ? top[j] + log2f(z) : __builtin_inff();
    const int64_t at = ((int64_t)row * a.H + head) * D;
#pragma unroll
    for (int d = 0; d < DB; d++) {
      E o[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float x = acc[d][j][e] * inv;
        o[e] = attn_round<DT>(x);
        l[e] = attn_round<DT>(x - attn_float<DT>(o[e]));
      }
      struct __attribute__((packed, aligned(4 * sizeof(E)))) Four { E x[4]; };
      *(Four*)((E*)a.out + at + 16 * d + 4 * g) = Four{{o[0], o[1], o[2], o[3]}};
      if (DT != TMS_DTYPE_F32 && a.low) *(Four*)((E*)a.low + at + 16 * d + 4 * g) = Four{{l[0], l[1], l[2], l[3]}};
    }
  }
}

// ---------------------------------------------------------------- backward

// Sums of products of dS in fp16: dS is held times a power of two a column, which goes down
// when a larger one comes. `most`: the largest |dS| of this round in the column.
struct AttnRange {
  float held = 0x1p100f;
  template <int DB, int NB>
  __device__ __forceinline__ void follow(float most, f32x4 (&acc)[DB][NB], int j) {
    most = cross_row_max(most);
    if (__ballot(most * held > 32768.f) == 0ull) return;
    const int e = (int)((__builtin_bit_cast(uint32_t, most) >> 23) & 0xffu);  // most < 2^(e - 126)
    int s = 14 + 126 - e;
    s = s < -100 ? -100 : s > 100 ? 100 : s;
    const float to = most * held > 32768.f ? __builtin_bit_cast(float, (uint32_t)(s + 127) << 23) : held;
    const float k = to / held;
    held = to;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[d][j][i] *= k;
  }
};

// A lane's gradients: four neighbouring elements of row `row` (16 d + 4 g ..), times f.
template <int DT, int DB, int NB>
__device__ __forceinline__ void attn_store(void* out, int64_t at, const f32x4 (&acc)[DB][NB], int j, float f, int g) {
  typedef typename AttnType<DT>::E E;
  struct __attribute__((packed, aligned(4 * sizeof(E)))) Four { E x[4]; };
#pragma unroll
  for (int d = 0; d < DB; d++) {
    Four o;
#pragma unroll
    for (int e = 0; e < 4; e++) o.x[e] = attn_round<DT>(acc[d][j][e] * f);
    *(Four*)((E*)out + at + 16 * d + 4 * g) = o;
  }
}

// delta and dq: a workgroup has a tile of queries and goes over their keys.
template <int DT, int D, int NB, bool GENERAL>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_dq_kernel(AttnArgs a) {
  typedef AttnRows<DT, D> Rows;
  typedef typename AttnType<DT>::E E;
  typedef typename AttnType<DT>::Frag Frag;
  constexpr int R = Rows::R, KB = R / 16, DB = D / 16, KS = D / 32, BQ = 64 * NB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t attn_mem[];
  int slot, head;
  if (!attn_place(a, a.H, slot, head)) return;
  AttnTile t;
  t.find(a, slot, BQ);
  if (t.text < 0) return;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int row0 = t.first + wave * 16 * NB;

  f32x4 acc[DB][NB];
#pragma unroll
  for (int d = 0; d < DB; d++)
#pragma unroll
    for (int j = 0; j < NB; j++) acc[d][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  AttnRange range[NB];

  if (t.real) {
    const int kvh = head / (a.H / a.KV);
    const E* K = (const E*)a.k + kvh * a.kh;
    const E* V = (const E*)a.v + kvh * a.vh;
    AttnScore score;
    score.init(a, head);
    Frag q[NB][KS], go[NB][KS];
    int sees[NB];
    float lse[NB], delta[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) {
      const int row = row0 + 16 * j + c, in = row < t.end ? row : t.end - 1;
      const int64_t at = ((int64_t)in * a.H + head) * D;
      attn_own<DT, D>((const E*)a.q + head * a.qh, (int64_t)in * a.qt, g, q[j]);
      attn_own<DT, D>((const E*)a.grad, at, g, go[j]);
      lse[j] = a.lse[(int64_t)head * a.T + in];
      sees[j] = in + 1 > t.prefix_end ? in + 1 : t.prefix_end;
      Frag o[KS], low[KS];
      attn_own<DT, D>((const E*)a.out, at, g, o);
      if constexpr (DT != TMS_DTYPE_F32) attn_own<DT, D>((const E*)a.low, at, g, low);
      float x = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          float y = attn_elem<DT>(o[ks], e);
          if constexpr (DT != TMS_DTYPE_F32) y += attn_elem<DT>(low[ks], e);
          x = __builtin_fmaf(attn_elem<DT>(go[j][ks], e), y, x);
        }
      delta[j] = cross_row_sum(x);
      if (g == 0 && row < t.end) a.delta[(int64_t)head * a.T + row] = delta[j];
    }
    const int least = row0 + 1 > t.prefix_end ? row0 + 1 : t.prefix_end;
    const int last = t.first + BQ < t.end ? t.first + BQ : t.end;
    const int keys = last > t.prefix_end ? last : t.prefix_end;
    int mine = row0 + 16 * NB < t.end ? row0 + 16 * NB : t.end;
    mine = row0 >= t.end ? t.begin : mine > t.prefix_end ? mine : t.prefix_end;

    Rows rk, rv;
    rk.load(K, a.kt, t.begin, keys);
    rv.load(V, a.vt, t.begin, keys);
    int buf = 0;
    for (int k0 = t.begin; k0 < keys; k0 += R) {
      uint8_t* lk = attn_mem + buf * 2 * Rows::kBytes;
      uint8_t* lv = lk + Rows::kBytes;
      rk.store(lk);
      rv.store(lv);
      __syncthreads();
      if (k0 + R < keys) {
        rk.load(K, a.kt, k0 + R, keys);
        rv.load(V, a.vt, k0 + R, keys);
      }
      __builtin_amdgcn_sched_barrier(0);
      buf ^= 1;
      if (k0 >= mine) continue;
      const bool part = k0 + R > least;

      f32x4 s[KB][NB];
      float most[NB];
#pragma unroll
      for (int j = 0; j < NB; j++) most[j] = 0.f;
#pragma unroll
      for (int b = 0; b < KB; b++) {
        f32x4 dp[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) s[b][j] = dp[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const Frag fk = Rows::row_frag(lk, b, ks, c, g), fv = Rows::row_frag(lv, b, ks, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            s[b][j] = attn_mfma<DT>(fk, q[j][ks], s[b][j]);
            dp[j] = attn_mfma<DT>(fv, go[j][ks], dp[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float x, f = 1.f;
            if constexpr (GENERAL) x = score.template operator()<DT>(s[b][j][e], row0 + 16 * j + c - (k0 + 16 * b + 4 * g + e), &f) - lse[j];
            else x = __builtin_fmaf(s[b][j][e], score.c1, -lse[j]);
            float y = __builtin_amdgcn_exp2f(x) * (dp[j][e] - delta[j]);
            if constexpr (GENERAL) y *= f;
            if (part) y = k0 + 16 * b + 4 * g + e < sees[j] ? y : 0.f;
            s[b][j][e] = y;
            if constexpr (DT == TMS_DTYPE_F16) most[j] = fmaxf(most[j], fabsf(y));
          }
      }
      Frag ds[NB][R / 32];
#pragma unroll
      for (int j = 0; j < NB; j++) {
        if constexpr (DT == TMS_DTYPE_F16) {
          range[j].follow(most[j], acc, j);
#pragma unroll
          for (int b = 0; b < KB; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[b][j][e] *= range[j].held;
        }
#pragma unroll
        for (int h = 0; h < R / 32; h++) ds[j][h] = attn_pack<DT>(s[2 * h][j], s[2 * h + 1][j]);
      }
#pragma unroll
      for (int h = 0; h < R / 32; h++)
#pragma unroll
        for (int d = 0; d < DB; d++) {
          const Frag f = Rows::col_frag(lk, h, d, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) acc[d][j] = attn_mfma<DT>(f, ds[j][h], acc[d][j]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < NB; j++) {
    const int row = row0 + 16 * j + c;
    if (row >= t.end) continue;
    const float f = !t.real ? 0.f : DT == TMS_DTYPE_F16 ? a.scale / range[j].held : a.scale;
    if (a.dq) attn_store<DT>(a.dq, ((int64_t)row * a.H + head) * D, acc, j, f, g);
  }
}

// dk and dv: a workgroup has a tile of keys and goes over the queries that see them, head by head of
// those that share the keys.
template <int DT, int D, int NB, bool GENERAL>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_dkv_kernel(AttnArgs a) {
  typedef AttnRows<DT, D> Rows;
  typedef typename AttnType<DT>::E E;
  typedef typename AttnType<DT>::Frag Frag;
  constexpr int R = Rows::R, QB = R / 16, DB = D / 16, KS = D / 32, BK = 64 * NB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t attn_mem[];
  float* const stats = (float*)(attn_mem + 4 * Rows::kBytes);  // [buffer][lse, delta][R]
  int slot, kvh;
  if (!attn_place(a, a.KV, slot, kvh)) return;
  AttnTile t;
  t.find(a, slot, BK);
  if (t.text < 0) return;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int key0 = t.first + wave * 16 * NB;

  f32x4 dk[DB][NB], dv[DB][NB];
#pragma unroll
  for (int d = 0; d < DB; d++)
#pragma unroll
    for (int j = 0; j < NB; j++) dk[d][j] = dv[d][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  AttnRange range[NB];

  if (t.real) {
    Frag k[NB][KS], v[NB][KS];
    int from[NB];  // the first row that sees the key
#pragma unroll
    for (int j = 0; j < NB; j++) {
      const int key = key0 + 16 * j + c, in = key < t.end ? key : t.end - 1;
      attn_own<DT, D>((const E*)a.k + kvh * a.kh, (int64_t)in * a.kt, g, k[j]);
      attn_own<DT, D>((const E*)a.v + kvh * a.vh, (int64_t)in * a.vt, g, v[j]);
      from[j] = key < t.prefix_end ? t.begin : key;
    }
    // the first row that sees any key of the workgroup, and any of this wave's; the first one that sees all of the wave's
    const int rows = t.first < t.prefix_end ? t.begin : t.first;
    const int mine = key0 >= t.end ? 0x7fffffff : key0 < t.prefix_end ? t.begin : key0;
    const int all = key0 + 16 * NB <= t.prefix_end || t.prefix_end == t.end ? t.begin : key0 + 16 * NB - 1;
    const int many = a.H / a.KV, tiles = (t.end - rows + R - 1) / R, total = tiles * many;

    Rows rq, rg;
    float st = 0.f;  // a thread's share of the tile's statistics: lse (the first R), delta (the next)
    auto load = [&](int n) {
      const int head = kvh * many + n / tiles, r0 = rows + n % tiles * R;
      rq.load((const E*)a.q + head * a.qh, a.qt, r0, t.end);
      rg.load((const E*)a.grad + (int64_t)head * D, (int64_t)a.H * D, r0, t.end);
      if ((int)threadIdx.x < 2 * R) {
        const int r = r0 + (int)threadIdx.x % R;
        const float* from_ = (int)threadIdx.x < R ? a.lse : a.delta;
        st = r < t.end ? from_[(int64_t)head * a.T + r] : (int)threadIdx.x < R ? __builtin_inff() : 0.f;
      }
    };
    AttnScore score;
    load(0);
    int buf = 0;
    for (int n = 0; n < total; n++) {
      uint8_t* lq = attn_mem + buf * 2 * Rows::kBytes;
      uint8_t* lg = lq + Rows::kBytes;
      float* ls = stats + buf * 2 * R;
      rq.store(lq);
      rg.store(lg);
      if ((int)threadIdx.x < 2 * R) ls[threadIdx.x] = st;
      __syncthreads();
      if (n + 1 < total) load(n + 1);
      __builtin_amdgcn_sched_barrier(0);
      buf ^= 1;
      const int r0 = rows + n % tiles * R;
      if (n % tiles == 0) score.init(a, kvh * many + n / tiles);
      if (r0 + R <= mine) continue;  // uniform in the wave
      const bool part = r0 < all;

      f32x4 p[QB][NB], s[QB][NB];
      float most[NB];
#pragma unroll
      for (int j = 0; j < NB; j++) most[j] = 0.f;
#pragma unroll
      for (int b = 0; b < QB; b++) {
        f32x4 dp[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) s[b][j] = dp[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const Frag fq = Rows::row_frag(lq, b, ks, c, g), fg = Rows::row_frag(lg, b, ks, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            s[b][j] = attn_mfma<DT>(fq, k[j][ks], s[b][j]);
            dp[j] = attn_mfma<DT>(fg, v[j][ks], dp[j]);
          }
        }
        const f32x4 lse = *(const f32x4*)(ls + 16 * b + 4 * g), delta = *(const f32x4*)(ls + R + 16 * b + 4 * g);
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int row = r0 + 16 * b + 4 * g + e;
            float x, f = 1.f;
            if constexpr (GENERAL) x = score.template operator()<DT>(s[b][j][e], row - (key0 + 16 * j + c), &f) - lse[e];
            else x = __builtin_fmaf(s[b][j][e], score.c1, -lse[e]);
            float y = __builtin_amdgcn_exp2f(x);
            if (part) y = row >= from[j] ? y : 0.f;
            float z = y * (dp[j][e] - delta[e]);
            if constexpr (GENERAL) z *= f;
            if (part) z = row >= from[j] ? z : 0.f;
            p[b][j][e] = DT == TMS_DTYPE_F16 ? y * (float)(1 << kAttnP16) : y;
            s[b][j][e] = z;
            if constexpr (DT == TMS_DTYPE_F16) most[j] = fmaxf(most[j], fabsf(z));
          }
      }
      Frag pf[NB][R / 32], sf[NB][R / 32];
#pragma unroll
      for (int j = 0; j < NB; j++) {
        if constexpr (DT == TMS_DTYPE_F16) {
          range[j].follow(most[j], dk, j);
#pragma unroll
          for (int b = 0; b < QB; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[b][j][e] *= range[j].held;
        }
#pragma unroll
        for (int h = 0; h < R / 32; h++) {
          pf[j][h] = attn_pack<DT>(p[2 * h][j], p[2 * h + 1][j]);
          sf[j][h] = attn_pack<DT>(s[2 * h][j], s[2 * h + 1][j]);
        }
      }
#pragma unroll
      for (int h = 0; h < R / 32; h++)
#pragma unroll
        for (int d = 0; d < DB; d++) {
          const Frag fg = Rows::col_frag(lg, h, d, c, g), fq = Rows::col_frag(lq, h, d, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            dv[d][j] = attn_mfma<DT>(fg, pf[j][h], dv[d][j]);
            dk[d][j] = attn_mfma<DT>(fq, sf[j][h], dk[d][j]);
          }
        }
    }
  }
#pragma unroll
  for (int j = 0; j < NB; j++) {
    const int key = key0 + 16 * j + c;
    if (key >= t.end) continue;
    const int64_t at = ((int64_t)key * a.KV + kvh) * D;
    const float fk = !t.real ? 0.f : DT == TMS_DTYPE_F16 ? a.scale / range[j].held : a.scale;
    const float fv = !t.real ? 0.f : DT == TMS_DTYPE_F16 ? 1.f / (float)(1 << kAttnP16) : 1.f;
    if (a.dk) attn_store<DT>(a.dk, at, dk, j, fk, g);
    if (a.dv) attn_store<DT>(a.dv, at, dv, j, fv, g);
  }
}

// ---------------------------------------------------------------- launches

enum AttnPass { kAttnForward = 0, kAttnDq = 1, kAttnDkv = 2 };

static inline int64_t attn_slots(int64_t T, int64_t B, int64_t rows) { return T / rows + B + 2; }

template <int DT, int D, int NB, bool GENERAL>
static int attn_launch(AttnArgs a, AttnPass pass, hipStream_t st) {
  typedef AttnRows<DT, D> Rows;
  a.slots = (int32_t)attn_slots(a.T, a.B, 64 * NB);
  const int64_t total = (int64_t)a.slots * (pass == kAttnDkv ? a.KV : a.H), grid = (total + 7) / 8 * 8;
  size_t lds = 4 * (size_t)Rows::kBytes;
  if (pass == kAttnForward) {
    hipLaunchKernelGGL((attn_forward_kernel<DT, D, NB, GENERAL>), dim3((unsigned)grid), dim3(kAttnThreads), lds, st, a);
    return check_launch("attn_forward_kernel");
  }
  if (pass == kAttnDq) {
    hipLaunchKernelGGL((attn_dq_kernel<DT, D, NB, GENERAL>), dim3((unsigned)grid), dim3(kAttnThreads), lds, st, a);
    return check_launch("attn_dq_kernel");
  }
  lds += 4 * Rows::R * sizeof(float);
  hipLaunchKernelGGL((attn_dkv_kernel<DT, D, NB, GENERAL>), dim3((unsigned)grid), dim3(kAttnThreads), lds, st, a);
  return check_launch("attn_dkv_kernel");
}

// One of these for each dtype, in a file of its own.
int attn_run_f16(const AttnArgs& a, int D, AttnPass pass, hipStream_t st);
int attn_run_bf16(const AttnArgs& a, int D, AttnPass pass, hipStream_t st);
int attn_run_f32(const AttnArgs& a, int D, AttnPass pass, hipStream_t st);

template <int DT, int D>
static int attn_run_d(const AttnArgs& a, AttnPass pass, hipStream_t st) {
  constexpr int NB = 1;
  if (a.cap > 0.f || a.slopes) return attn_launch<DT, D, NB, true>(a, pass, st);
  return attn_launch<DT, D, NB, false>(a, pass, st);
}
template <int DT>
static int attn_run(const AttnArgs& a, int D, AttnPass pass, hipStream_t st) {
  switch (D) {
    case 32: return attn_run_d<DT, 32>(a, pass, st);
    case 64: return attn_run_d<DT, 64>(a, pass, st);
    case 96: return attn_run_d<DT, 96>(a, pass, st);
    default: return attn_run_d<DT, 128>(a, pass, st);
  }
}

}  // namespace tms
