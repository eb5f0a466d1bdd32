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
// through LDS, 32 or 64 rows at a time, as their rows:
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
// What bounds them. Long texts: issue. A score takes about seven vector instructions, one of them an exponential,
// beside its products, and the two take turns rather than overlap. Two texts of 8192 tokens under biases, 12 heads of 64, in
// bf16: forward 434 us, dq 513, dk and dv 701; vector instructions issue for 56, 41 and 39 % of the time, matrix
// cores are busy for 25, 32 and 31 %, without a bank conflict. Without a bias, 8 heads over texts of 8192 (16,384 tokens):
// 367, 395 and 521 us in heads of 64 (0.75, 1.05 and 1.06 PFLOP/s, the products formed again counted),
// 565, 690 and 1,165 in heads of 128 (0.97, 1.2, 0.94). Short texts: the way to a tile's first products. 128 texts
// of 32 to 300 tokens, 12 heads of 64: 67, 71 and 96 us, where their bytes take 81 for all three at a copy's rate.
//
// In LDS a row of 32 elements takes 64 bytes (fp32: 128), two rows a line of 128, whose 16-byte
// pieces stand at p ^ (line % 8): the row fragments (a lane's eight neighbouring elements) and the
// transposing reads both fall evenly on the banks.
//
// Precision. Scores, statistics, sums and gradients are fp32. P and dS are rounded to the
// inputs' type between two products (2^-9 of each term in bf16, 2^-12 in fp16), as the matrix
// cores take them; where most texts are short, to two terms in the backward pass. fp16 has no range to spare: P is held times 2^15 in all three
// kernels (a key e^-17 below a row's best is nothing in fp16 as it is, and 16,000 of them half a step of o), and dS times
// a power of two for each row (column of sums) that follows the largest |dS| so far. delta is
// taken from o in two 16-bit terms (2^-17 of it): from o as it is returned, dS would have o's rounding
// even where P is 1 and dS 0. fp32 goes through the fp32 matrix instructions.
#pragma once
#include <math.h>

#include "tms_common.h"
#include "tms_train_rules.h"

namespace tms {

typedef short attn_s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 attn_f16x2 __attribute__((ext_vector_type(2)));

constexpr int kAttnThreads = 256;
constexpr float kAttnLog2e = 1.4426950408889634f;
constexpr float kAttnNothing = 160.f;  // so many powers of two below, exp2 is 0
// P is held times 2^this between two products.
template <int DT>
constexpr int attn_up() {
  return DT == TMS_DTYPE_F16 ? 15 : 0;
}

constexpr int kAttnNorms = 64;  // numbers a head

struct AttnArgs {
  const void *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;  // elements between tokens and heads
  const int64_t* offsets;          // B + 1
  const int64_t* prefix;           // B, or NULL: a text sees all of itself
  const float* slopes;             // H, or NULL
  int64_t T;
  int32_t B, H, KV, many, slots;  // many: heads that share keys
  int32_t parts;                  // workgroups that share a tile's heads in the kernel for dk and dv
  float scale, cap;  // cap 0: none
  void* out;         // (T, H, D)
  void* low;         // what out's rounding left, of out's type, or NULL
  float* lse;        // (H, T): log2 of the sums of exponentials; or NULL
  // backward
  const void* grad;  // (T, H, D)
  float* delta;      // (H, T)
  float* sums;       // [part][dk, dv][T, KV, D], where parts > 1
  void *dq, *dk, *dv;
  float* norms;  // [H + KV][kAttnNorms]: largest squares of rows of q and k; or NULL
};

template <int DT>
struct AttnType {
  typedef uint16_t E;
  typedef u32x4 Frag;  // eight elements
};
template <>
struct AttnType<TMS_DTYPE_F32> {
  typedef float E;
  typedef u32x8 Frag;
};

enum AttnPass { kAttnForward = 0, kAttnDq = 1, kAttnDkv = 2 };

// Rows of a tile that passes through LDS: 64, but for rows so wide that two workgroups fill a CU's LDS with them,
// where 32 leave room for another one (37 texts of 1 to 701 tokens, 8 heads of 128, forward and dq: 62 and 74
// us with 64, 52 and 65 with 32; a wave of 32 queries needs fewer of them at a time: texts of 8192, 565 and 668).
template <int DT, int D, int NB>
constexpr int attn_rows(AttnPass pass) {
  if (DT == TMS_DTYPE_F32) return 32;
  if (D < 128 || pass == kAttnDkv || (pass == kAttnForward && NB == 2)) return 64;
  return 32;
}

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
        const f32x2 v = {a, b};
        r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, attn_f16x2));
      }
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ typename AttnType<DT>::E attn_round(float x);
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
// What attn_pack's rounding leaves of the values, in the inputs' type.
template <int DT>
__device__ __forceinline__ typename AttnType<DT>::Frag attn_rest(f32x4 lo, f32x4 hi) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    lo[e] -= attn_float<DT>(attn_round<DT>(lo[e]));
    hi[e] -= attn_float<DT>(attn_round<DT>(hi[e]));
  }
  return attn_pack<DT>(lo, hi);
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
  template <int ROWS>
  __device__ __forceinline__ void find(const AttnArgs& a, int w) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.B + 2;
    while (n > 255) {  // 64 candidates at a time
      const int step = (n + 63) / 64, i = lane * step;
      const uint64_t hit = __ballot(i < n && (lane == 0 || offset(a, lo + i) / ROWS + lo + i <= w));
      const int at = (63 - __builtin_clzll(hit)) * step;  // the last one at or before w
      lo += at;
      n = n - at < step ? n - at : step;
    }
    // four a lane, and the one behind the last: one round trip, and both ends of the text's rows are at hand
    int v[4], hits = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = lo + lane * 4 + k <= a.B + 2 ? offset(a, lo + lane * 4 + k) : 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = lane * 4 + k;
      hits += __builtin_popcountll(__ballot(i < n && (i == 0 || v[k] / ROWS + lo + i <= w)));
    }
    auto value = [&](int i) {  // uniform i
      int x = 0;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int y = __builtin_amdgcn_readlane(v[k], i / 4);
        x = i % 4 == k ? y : x;
      }
      return x;
    };
    hits = hits < 1 ? 1 : hits > n ? n : hits;
    text = lo + hits - 1;
    begin = value(hits - 1);
    end = value(hits);
    constexpr int rows = ROWS;
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

// Which tile and head a workgroup takes. Workgroups go to the eight XCDs in turn. Each XCD takes a run of its
// own, head by head: the tiles of a long text read the same keys through one L2 (2048 tokens, 8 heads
// of 64, forward and backward: 98 us, 124 without). Where heads differ in how far they reach, each XCD takes
// every eighth group of four neighbouring tiles instead, and so its share of each head (two texts of
// 8192 under biases of 2^-0.7 to 2^-8: 1,533 us, 2,019 in runs, as long as the XCD with the flattest ones).
constexpr int kAttnGroup = 4;
static inline int64_t attn_grid(int64_t slots, int64_t heads) {
  return ((slots + kAttnGroup - 1) / kAttnGroup * heads + 7) / 8 * 8 * kAttnGroup;
}
__device__ __forceinline__ bool attn_place(const AttnArgs& a, int heads, int& slot, int& head) {
  const uint32_t slots = (uint32_t)a.slots, xcd = blockIdx.x % 8, i = blockIdx.x / 8;
  if (a.norms != nullptr) {
    const uint32_t groups = (slots + kAttnGroup - 1) / kAttnGroup, unit = i / kAttnGroup * 8 + xcd;
    if (unit >= groups * (uint32_t)heads) return false;
    head = (int)(unit / groups);
    slot = (int)((unit - (uint32_t)head * groups) * kAttnGroup + i % kAttnGroup);
    return slot < a.slots;
  }
  const uint32_t total = slots * (uint32_t)heads, each = (total + 7) / 8, at = xcd * each + i;
  if (i >= each || at >= total) return false;
  head = (int)(at / slots);
  slot = (int)(at - (uint32_t)head * slots);
  return true;
}

// Rows of D elements in LDS, and the way there: from memory to registers, and (after the wait that
// the store makes) to LDS. Rows from `limit` on are zeros.
template <int DT, int D, int R_>
struct AttnRows {
  typedef AttnType<DT> Ty;
  typedef typename Ty::Frag Frag;
  static constexpr int R = R_, ES = sizeof(typename Ty::E);
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
  uint32_t off[kLoads];  // bytes from the tile's first row: 64 rows are less than 2^32 apart
  __device__ __forceinline__ void init(int64_t stride) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      int row, col;
      piece(i * kAttnThreads + (int)threadIdx.x, row, col);
      off[i] = (uint32_t)(row * (int)stride + col) * (uint32_t)ES;
    }
  }
  // Rows from `first` (uniform) on.
  __device__ __forceinline__ void load(const typename Ty::E* base, int64_t stride, int first, int limit) {
    const uint8_t* at = (const uint8_t*)(base + first * stride);
    if (first + R <= limit) {
#pragma unroll
      for (int i = 0; i < kLoads; i++) held[i] = *(const u32x4*)(at + off[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      int row, col;
      piece(i * kAttnThreads + (int)threadIdx.x, row, col);
      held[i] = u32x4{0u, 0u, 0u, 0u};
      if (first + row < limit) held[i] = *(const u32x4*)(at + off[i]);
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

constexpr float kAttnCoarse = 64.f;  // 2^-22 of it: 1.5e-5 of a score
template <bool V>
struct AttnYes {
  static constexpr bool value = V;
};

// What a score takes besides the products: nothing, a bias, or a cap (and perhaps a bias).
enum AttnKind { kAttnPlain = 0, kAttnBias = 1, kAttnCap = 2 };

// Scores x from sums of products s, as y with x log2(e) = unit y + shift: y = s - lean |i - j|, or under
// a cap y = cap log2(e) tanh(s scale / cap) - lean |i - j| with a unit of 1. The unit goes into the exponent's
// one FMA. Without a cap, a bias costs next to nothing in tiles that lie on one side of a wave's own rows:
// there it is a part of the tile's row, which the products' sums begin with, and a part of
// the wave's own row, which is in the shift.
template <int DT, int KIND, int R>
struct AttnScore {
  float unit, cap2, inv_cap, lean;
  int side = 2;  // of the tile: its rows before the wave's (-1), behind them (1), or both (0)
  f32x4 begin[KIND == kAttnBias ? R / 16 : 1];  // -lean of rows 16 b + 4 g + e by side

  __device__ __forceinline__ void init(const AttnArgs& a, int head) {
    unit = KIND == kAttnCap ? 1.f : a.scale * kAttnLog2e;
    cap2 = a.cap * kAttnLog2e;
    inv_cap = KIND == kAttnCap ? a.scale / a.cap * (DT == TMS_DTYPE_F32 ? 1.f : 2.f * kAttnLog2e) : 0.f;
    lean = a.slopes ? a.slopes[head] * (KIND == kAttnCap ? kAttnLog2e : 1.f / a.scale) : 0.f;
    side = 2;
  }
  // The tile of rows from `first` on, against the wave's own from `own` up to `own_end`.
  __device__ __forceinline__ void tile(int first, int own, int own_end, int g) {
    if constexpr (KIND == kAttnBias) {
      const int now = first + R <= own ? -1 : first >= own_end ? 1 : 0;
      if (now == side) return;
      side = now;
#pragma unroll
      for (int b = 0; b < R / 16; b++)
#pragma unroll
        for (int e = 0; e < 4; e++) begin[b][e] = lean * (float)(-now * (16 * b + 4 * g + e));
    }
  }
  __device__ __forceinline__ f32x4 start(int b) const {
    if constexpr (KIND == kAttnBias) return begin[b];
    return f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // What the scores of the wave's own row `own` have in common with the tile from `first` on.
  __device__ __forceinline__ float shift(int own, int first) const {
    if constexpr (KIND == kAttnBias) return unit * lean * (float)(side * (own - first));
    return 0.f;
  }
  // Whether the bias has to be taken off element by element.
  __device__ __forceinline__ bool single() const { return (KIND == kAttnCap && lean != 0.f) || (KIND == kAttnBias && side == 0); }
  // Under a cap, y from s, and kSlope times the derivative's factor, 1 - tanh^2. In 16 bits tanh z is taken as
  // 1 - 2 r with r = 1 / (1 + e^2z), to 2^-22 or so of the cap, where the operands have 2^-9 or 2^-12. A cap above
  // kAttnCoarse takes the series z (1 - z^2 / 3 + 2 z^4 / 15) up to |z| = 2^-4 (the next term, 17 z^6 / 315, is
  // below 2^-28 there), as scores far below their cap would have its error: FINE.
  static constexpr float kSlope = KIND == kAttnCap && DT != TMS_DTYPE_F32 ? 0.25f : 1.f;
  template <bool FINE>
  __device__ __forceinline__ float capped(float s, float& slope) const {
    if constexpr (DT == TMS_DTYPE_F32) {
      const float t = tanhf(s * inv_cap);
      slope = __builtin_fmaf(-t, t, 1.f);
      return t * cap2;
    }
    const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * inv_cap));  // inv_cap has 2 log2(e) in it
    slope = __builtin_fmaf(-r, r, r);  // (1 - t^2) / 4
    float y = __builtin_fmaf(-2.f * cap2, r, cap2);
    if constexpr (FINE) {
      const float z = s * inv_cap * (0.5f / kAttnLog2e), zz = z * z;
      y = zz < 0x1p-8f ? z * cap2 * __builtin_fmaf(zz, __builtin_fmaf(zz, 2.f / 15.f, -1.f / 3.f), 1.f) : y;
    }
    return y;
  }
  // y of all of a wave's s, and (with dp) their factors: f(place, slope) for each.
  template <int N, class F>
  __device__ __forceinline__ void cap_all(f32x4 (&s)[N], F&& f) const {
    auto all = [&](auto fine) {
#pragma unroll
      for (int j = 0; j < N; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float slope;
          s[j][e] = capped<decltype(fine)::value>(s[j][e], slope);
          f(j, e, slope);
        }
    };
    if (cap2 > kAttnCoarse * kAttnLog2e) all(AttnYes<true>());  // uniform
    else all(AttnYes<false>());
  }
  // far: i - j, or its negative.
  __device__ __forceinline__ float biased(float y, float far) const { return __builtin_fmaf(-lean, fabsf(far), y); }
};

// How far from a token its keys can matter under a bias alone (T without one). With |q|, |k| the largest
// norms, scores but for the bias lie within scale |q| |k| of 0, and a row's largest is at least its own
// token's: P of a token n away is at most exp(2 scale |q| |k| - slope n), and 0 in fp32 where that is
// below 2^-160. Where a norm is not finite, nothing is left out.
__device__ __forceinline__ int attn_reach(const AttnArgs& a, int head) {
  if (a.norms == nullptr) return (int)a.T;
  const int lane = threadIdx.x & 63;
  float q = a.norms[head * kAttnNorms + lane], k = a.norms[(a.H + head / a.many) * kAttnNorms + lane];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    q = __builtin_elementwise_maximum(q, __shfl_xor(q, o));
    k = __builtin_elementwise_maximum(k, __shfl_xor(k, o));
  }
  const float far = (kAttnNothing + 2.f * kAttnLog2e * a.scale * sqrtf(q) * sqrtf(k) * 1.001f) / (a.slopes[head] * kAttnLog2e);
  const int reach = far >= 0.f && far < (float)a.T ? (int)far + 1 : (int)a.T;  // no slope, a negative one, NaN: all
  return __builtin_amdgcn_readfirstlane(reach);
}

// The larger of the two; NaN if either is.
__device__ __forceinline__ float attn_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The largest over the four lanes that have a column's rows, in all of them.
__device__ __forceinline__ float attn_cross_max(float m) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, m), __builtin_bit_cast(unsigned, m), false, false);
  m = attn_max(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, m), __builtin_bit_cast(unsigned, m), false, false);
  return attn_max(__builtin_bit_cast(float, (unsigned)q[0]), __builtin_bit_cast(float, (unsigned)q[1]));
}

// ---------------------------------------------------------------- norms

// The largest squared norms of q's and k's rows: 16 lanes a row, a part of the tokens a workgroup. Bound by reading
// them (16,384 tokens, 24 heads of 64 in bf16: 50 MB in 10 us).
template <int DT, int D>
__global__ __launch_bounds__(kAttnThreads) void attn_norms_kernel(AttnArgs a) {
  typedef typename AttnType<DT>::E E;
  constexpr int EACH = D / 16;
  __shared__ float lds[kAttnThreads / 64];
  const int head = blockIdx.x / kAttnNorms, part = blockIdx.x % kAttnNorms;
  const bool of_q = head < a.H;
  const E* base = of_q ? (const E*)a.q + head * a.qh : (const E*)a.k + (head - a.H) * a.kh;
  const int64_t stride = of_q ? a.qt : a.kt;
  float most = 0.f;
  for (int64_t row = part * 16 + (int)threadIdx.x / 16; row < a.T; row += 16 * kAttnNorms) {
    const E* x = base + row * stride + (threadIdx.x & 15) * EACH;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EACH; e++) s = __builtin_fmaf(attn_float<DT>(x[e]), attn_float<DT>(x[e]), s);
    most = attn_max(most, row_sum16(s));
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) most = attn_max(most, __shfl_xor(most, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0) a.norms[blockIdx.x] = attn_max(attn_max(lds[0], lds[1]), attn_max(lds[2], lds[3]));
}

// ---------------------------------------------------------------- rows by themselves

// Under a prefix mask a row shares tiles with tokens that it does not see, and if one of those is NaN or infinite, the 0 that
// stands for it in the matrix instructions makes the row NaN. Rows of sums that are not finite are therefore formed
// once more by one wave, from what they see alone, in fp32: 64 of the others at a time, one a lane for the scores, then one
// after the other with the row's elements on the lanes. A row that is not finite by what it does see stays so. That takes
// 50 times as long as with the matrix instructions, so rows that need not are not formed again: those whose own
// statistic is not finite; all of a wave where every token in reach that some row does not see is finite; and those that are finite but in
// columns where their own token, or one that all of the wave's rows see, is not. What is left are rows close to the first bad token
// of a column. (Two causal texts of 8192, 12 heads of 64, both directions: 1.4 ms; with NaN or infinities in one
// token, one column, every 64th token or all of them 1.2 to 2.7.)
// What it needs is formed anew or read again, so that next to nothing stays in registers for it while the tiles are gone over; calls without
// prefixes take kernels without it (MASK: 100 causal texts of 200, 12 heads of 64, forward 38.9 us and backward 122.9, without the check 38.4 and 117.8).
__device__ __forceinline__ int attn_lane() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }
__device__ __forceinline__ bool attn_finite(float x) { return fabsf(x) < __builtin_inff(); }

// Whether a lane's sums of column j are all finite: their sum is, then (and where they are near fp32's limit perhaps not,
// which only costs time).
template <int DB, int NB>
__device__ __forceinline__ bool attn_all_finite(const f32x4 (&acc)[DB][NB], int j) {
  f32x4 x = acc[0][j];
#pragma unroll
  for (int d = 1; d < DB; d++)
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] += acc[d][j][e];
  return attn_finite((x[0] + x[1]) + (x[2] + x[3]));
}
// The 16 rows (columns of the products) that any of a wave's lanes reports.
__device__ __forceinline__ uint32_t attn_odd(bool here) {
  const uint64_t b = __ballot(here);
  return (uint32_t)(b | b >> 16 | b >> 32 | b >> 48) & 0xffffu;
}

// Whether all elements of rows from `from` up to `to` are finite: one row a lane.
template <int DT, int D>
__device__ bool attn_rows_finite(const typename AttnType<DT>::E* x, int64_t stride, int from, int to) {
  typedef typename AttnType<DT>::Frag Frag;
  bool bad = false;
  for (int r = from + attn_lane(); r < to; r += 64)
    for (int k = 0; k < D; k += 8) {
      const Frag f = *(const Frag*)(x + r * stride + k);
#pragma unroll
      for (int e = 0; e < 8; e++) bad |= !attn_finite(attn_elem<DT>(f, e));
    }
  return __ballot(bad) == 0ull;
}

// The columns in which any of those rows is not finite, as bits (of all lanes).
template <int D>
struct AttnColumns {
  uint32_t bits[D / 32] = {};
  template <int DT>
  __device__ void add(const typename AttnType<DT>::E* x, int64_t stride, int from, int to) {
    typedef typename AttnType<DT>::Frag Frag;
    for (int r = from + attn_lane(); r < to; r += 64)
#pragma unroll
      for (int k = 0; k < D; k += 8) {
        const Frag f = *(const Frag*)(x + r * stride + k);
#pragma unroll
        for (int e = 0; e < 8; e++) bits[k / 32] |= attn_finite(attn_elem<DT>(f, e)) ? 0u : 1u << ((k + e) % 32);
      }
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) bits[i] |= __shfl_xor(bits[i], o);
  }
};
// Whether a lane's sums of column j (elements 16 d + 4 g + e) are not finite where neither those columns nor its own token explain it.
template <int DT, int D, int DB, int NB>
__device__ __forceinline__ bool attn_unexplained(const f32x4 (&acc)[DB][NB], int j, const AttnColumns<D>& bad, const typename AttnType<DT>::E* own, int g) {
  bool some = false;
#pragma unroll
  for (int d = 0; d < DB; d++) {
    const uint32_t four = bad.bits[d / 2] >> (16 * (d & 1) + 4 * g) & 15u;
#pragma unroll
    for (int e = 0; e < 4; e++) some |= !attn_finite(acc[d][j][e]) && !(four >> e & 1) && attn_finite(attn_float<DT>(own[16 * d + 4 * g + e]));
  }
  return some;
}

template <int DT, int D>
__device__ __forceinline__ float attn_dot(const typename AttnType<DT>::E* x, const typename AttnType<DT>::E* y) {
  typedef typename AttnType<DT>::Frag Frag;
  float s = 0.f;
#pragma unroll 2
  for (int k = 0; k < D; k += 8) {
    const Frag f = *(const Frag*)(x + k), h = *(const Frag*)(y + k);
#pragma unroll
    for (int e = 0; e < 8; e++) s = __builtin_fmaf(attn_elem<DT>(f, e), attn_elem<DT>(h, e), s);
  }
  return s;
}

// One row against those from `from` up to `to`, which it sees (or which see it). `own` is the row, and `x` its partners, of the
// scores; `own2` and `y` of dP. Added to sum, element 64 u + lane: forward, P y; dq, dS x; dk and dv, dS x and (sum2) P y.
template <int DT, int D, int KIND, AttnPass PASS>
__device__ void attn_alone(const AttnArgs& a, int head, int row, int from, int to, const typename AttnType<DT>::E* own, const typename AttnType<DT>::E* own2,
                           const typename AttnType<DT>::E* x, int64_t xs, const typename AttnType<DT>::E* y, int64_t ys, float lse, float delta,
                           float (&sum)[(D + 63) / 64], float (&sum2)[(D + 63) / 64]) {
  const int lane = attn_lane();
  AttnScore<DT, KIND, 64> score;
  score.init(a, head);
  for (int r0 = from; r0 < to; r0 += 64) {
    const int r = r0 + lane, n = to - r0 < 64 ? to - r0 : 64;
    float p = 0.f, ds = 0.f;
    if (r < to) {
      float s = attn_dot<DT, D>(own, x + r * xs), slope = 1.f;
      if constexpr (KIND == kAttnCap) {
        s = score.cap2 > kAttnCoarse * kAttnLog2e ? score.template capped<true>(s, slope) : score.template capped<false>(s, slope);
        slope *= 1.f / score.kSlope;
      }
      if (score.lean != 0.f) s = score.biased(s, (float)(row - r));
      if constexpr (PASS == kAttnDkv) lse = a.lse[(int64_t)head * a.T + r], delta = a.delta[(int64_t)head * a.T + r];
      p = __builtin_amdgcn_exp2f(__builtin_fmaf(s, score.unit, -lse));
      if constexpr (PASS != kAttnForward) ds = p * (attn_dot<DT, D>(own2, y + r * ys) - delta) * slope;
    }
    for (int i = 0; i < n; i++) {
      const float pi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), i));
      const float di = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ds), i));
#pragma unroll
      for (int u = 0; u < (D + 63) / 64; u++) {
        const int d = 64 * u + lane;
        if (d >= D) continue;
        if constexpr (PASS != kAttnForward) sum[u] = __builtin_fmaf(di, attn_float<DT>(x[(r0 + i) * xs + d]), sum[u]);
        if constexpr (PASS == kAttnForward) sum[u] = __builtin_fmaf(pi, attn_float<DT>(y[(r0 + i) * ys + d]), sum[u]);
        if constexpr (PASS == kAttnDkv) sum2[u] = __builtin_fmaf(pi, attn_float<DT>(y[(r0 + i) * ys + d]), sum2[u]);
      }
    }
  }
}

// ---------------------------------------------------------------- forward

// A workgroup has a tile of queries and goes over their keys; the running maximum, sum and o are in registers, and
// the next tile's keys and values on their way while one is used. NB: blocks of 16 queries a wave. Times: above.
template <int DT, int D, int NB, int KIND, bool MASK>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_forward_kernel(AttnArgs a) {
  typedef AttnRows<DT, D, attn_rows<DT, D, NB>(kAttnForward)> Rows;
  typedef typename AttnType<DT>::E E;
  typedef typename AttnType<DT>::Frag Frag;
  constexpr int R = Rows::R, KB = R / 16, DB = D / 16, KS = D / 32, BQ = 64 * NB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t attn_mem[];
  int slot, head;
  if (!attn_place(a, a.H, slot, head)) return;
  AttnTile t;
  t.find<BQ>(a, slot);
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
    const int kvh = head / a.many;
    const E* K = (const E*)a.k + kvh * a.kh;
    const E* V = (const E*)a.v + kvh * a.vh;
    AttnScore<DT, KIND, R> score;
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
    int keys = last > t.prefix_end ? last : t.prefix_end, key0 = t.begin;
    if constexpr (KIND == kAttnBias) {
      const int reach = attn_reach(a, head);
      if (t.first - reach > key0) key0 += (t.first - reach - key0) / R * R;
      if (last + reach < keys) keys = last + reach;
    }
    int mine = row0 + 16 * NB < t.end ? row0 + 16 * NB : t.end;
    mine = row0 >= t.end ? t.begin : mine > t.prefix_end ? mine : t.prefix_end;

    Rows rk, rv;
    rk.init(a.kt);
    rv.init(a.vt);
    rk.load(K, a.kt, key0, keys);
    rv.load(V, a.vt, key0, keys);
    int buf = 0;
    for (int k0 = key0; k0 < keys; k0 += R) {
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
      score.tile(k0, row0, row0 + 16 * NB, g);
#pragma unroll
      for (int b = 0; b < KB; b++) {
#pragma unroll
        for (int j = 0; j < NB; j++) s[b][j] = score.start(b);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const Frag f = Rows::row_frag(lk, b, ks, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) s[b][j] = attn_mfma<DT>(f, q[j][ks], s[b][j]);
        }
      }
      if constexpr (KIND == kAttnCap) {
#pragma unroll
        for (int b = 0; b < KB; b++) score.cap_all(s[b], [](int, int, float) {});
      }
      if (score.single()) {
        const float near = (float)(row0 + c - k0 - 4 * g);
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[b][j][e] = score.biased(s[b][j][e], near + (float)(16 * j - 16 * b - e));
      }
      if (k0 + R > least) {  // some row does not see all of the tile
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[b][j][e] = k0 + 16 * b + 4 * g + e < sees[j] ? s[b][j][e] : NEG;
      }
      // A row's reference is its maximum so far, so that its largest P is 1 and not rounded: rows that look at few keys
      // have their error from the others.
      float m[NB], shift[NB];
      bool over = false, some = false;
#pragma unroll
      for (int j = 0; j < NB; j++) {
        m[j] = NEG;
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
          for (int e = 0; e < 4; e += 2) m[j] = attn_max(attn_max(s[b][j][e], s[b][j][e + 1]), m[j]);
        shift[j] = score.shift(row0 + 16 * j + c, k0);
        m[j] = __builtin_fmaf(attn_cross_max(m[j]), score.unit, shift[j]);
        over |= m[j] > top[j];
        some |= !(m[j] < top[j] - kAttnNothing);
      }
      if (__ballot(some) == 0ull) continue;  // every P of the tile is 0, as far behind as it is by its bias
      if (__ballot(over) != 0ull) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
          const float up = fmaxf(m[j], top[j]);
          const float k = up == NEG ? 1.f : __builtin_amdgcn_exp2f(top[j] - up);
          top[j] = up;
          sum[j] *= k;
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[d][j][e] *= k;
        }
      }
      float ref[NB];
#pragma unroll
      for (int j = 0; j < NB; j++) ref[j] = (top[j] == NEG ? 0.f : top[j]) - shift[j] - (float)attn_up<DT>();
#pragma unroll
      for (int h = 0; h < R / 32; h++) {  // 32 keys at a time
        Frag p[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
          for (int b = 2 * h; b < 2 * h + 2; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              s[b][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j][e], score.unit, -ref[j]));
              sum[j] += s[b][j][e];
            }
          p[j] = attn_pack<DT>(s[2 * h][j], s[2 * h + 1][j]);
        }
#pragma unroll
        for (int d = 0; d < DB; d++) {
          const Frag f = Rows::col_frag(lv, h, d, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) acc[d][j] = attn_mfma<DT>(f, p[j], acc[d][j]);
        }
      }
    }
  }

  uint32_t odd[NB];
#pragma unroll
  for (int j = 0; j < NB; j++) {
    const int row = row0 + 16 * j + c;
    const float all = t.real ? sum[j] : 0.f;
    float z = all;
    z += __shfl_xor(z, 16);
    z += __shfl_xor(z, 32);
    const float inv = t.real ? 1.f / z : 0.f;
    top[j] = t.real ? top[j] + (log2f(z) - (float)attn_up<DT>()) : __builtin_inff();
    odd[j] = 0;
    if constexpr (MASK) {
      odd[j] = attn_odd(!attn_all_finite(acc, j) && row < t.end && attn_finite(top[j]));
      if (odd[j] != 0) {
        const E* v = (const E*)a.v + head / a.many * a.vh;
        const int unseen = row0 + 1 > t.prefix_end ? row0 + 1 : t.prefix_end, past = row0 + 16 * NB, end = (past > t.prefix_end ? past : t.prefix_end) + R;
        if (attn_rows_finite<DT, D>(v, a.vt, unseen, end < t.end ? end : t.end)) {
          odd[j] = 0;
        } else {
          AttnColumns<D> bad;
          bad.template add<DT>(v, a.vt, t.begin, unseen);
          odd[j] &= attn_odd(row < t.end && attn_unexplained<DT, D>(acc, j, bad, v + row * a.vt, g));
        }
      }
    }
    if (row >= t.end) continue;
    if (a.lse && g == 0) a.lse[(int64_t)head * a.T + row] = top[j];
    if (odd[j] >> c & 1) continue;
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
#pragma unroll
  for (int j = 0; j < NB; j++) {
    for (uint32_t m = MASK ? odd[j] : 0; m != 0; m &= m - 1) {
      const int i = __builtin_ctz(m), row = row0 + 16 * j + i, kvh = head / a.many;
      const int ln = attn_lane();
      const float lse = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, top[j]), i));
      float x[(D + 63) / 64] = {};
      attn_alone<DT, D, KIND, kAttnForward>(a, head, row, t.begin, row + 1 > t.prefix_end ? row + 1 : t.prefix_end, (const E*)a.q + head * a.qh + row * a.qt, nullptr,
                                            (const E*)a.k + kvh * a.kh, a.kt, (const E*)a.v + kvh * a.vh, a.vt, lse, 0.f, x, x);
#pragma unroll
      for (int u = 0; u < (D + 63) / 64; u++) {
        const int64_t at = ((int64_t)row * a.H + head) * D + 64 * u + ln;
        if (64 * u + ln >= D) continue;
        const E o = attn_round<DT>(x[u]);
        ((E*)a.out)[at] = o;
        if (DT != TMS_DTYPE_F32 && a.low) ((E*)a.low)[at] = attn_round<DT>(x[u] - attn_float<DT>(o));
      }
    }
  }
}

// ---------------------------------------------------------------- backward

// Sums of products of dS in fp16: dS is held times a power of two a column, which goes down
// when a larger one comes.
struct AttnRange {
  float held = 0x1p100f;
  // Two blocks of dS on their way to fp16; j: their column of sums.
  template <int DB, int NB>
  __device__ __forceinline__ void follow(f32x4& x, f32x4& y, f32x4 (&acc)[DB][NB], int j) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) most = attn_max(attn_max(fabsf(x[e]), fabsf(y[e])), most);
    most = attn_cross_max(most);
    if (__ballot(most * held > 32768.f) != 0ull) {
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
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] *= held, y[i] *= held;
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

// delta and dq: a workgroup has a tile of queries and goes over their keys. SHORT: texts of one tile of keys
// have their delta from P and dP, before dS is formed: where few keys share a row, o's own error (P is
// rounded there) would be as large as that of dS's rounding. (For all: 128 documents of 32 to 300 tokens take 70 us
// and not 62.) And dS goes into its products as two 16-bit terms, as do P and dS in the kernel for dk and dv: where
// few elements make up a gradient's norm, one rounding more than its own can be twice the error (256 texts of 64, 12 heads of
// 64: 48 and 61 us, 46 and 58 with one term; 1024 of 16: 74 and 93, 72 and 88).
template <int DT, int D, int NB, int KIND, bool SHORT, bool MASK>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_dq_kernel(AttnArgs a) {
  typedef AttnRows<DT, D, attn_rows<DT, D, NB>(kAttnDq)> Rows;
  typedef typename AttnType<DT>::E E;
  typedef typename AttnType<DT>::Frag Frag;
  constexpr int R = Rows::R, DB = D / 16, KS = D / 32, BQ = 64 * NB;
  constexpr bool TWO = SHORT && DT != TMS_DTYPE_F32;
  extern __shared__ __attribute__((aligned(1024))) uint8_t attn_mem[];
  int slot, head;
  if (!attn_place(a, a.H, slot, head)) return;
  AttnTile t;
  t.find<BQ>(a, slot);
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
    const int kvh = head / a.many;
    const E* K = (const E*)a.k + kvh * a.kh;
    const E* V = (const E*)a.v + kvh * a.vh;
    AttnScore<DT, KIND, R> score;
    score.init(a, head);
    Frag q[NB][KS], go[NB][KS];
    int sees[NB];
    float lse[NB], delta[NB];
    const bool alone = SHORT && t.end - t.begin <= R;  // all keys in one tile
#pragma unroll
    for (int j = 0; j < NB; j++) {
      const int row = row0 + 16 * j + c, in = row < t.end ? row : t.end - 1;
      const int64_t at = ((int64_t)in * a.H + head) * D;
      attn_own<DT, D>((const E*)a.q + head * a.qh, (int64_t)in * a.qt, g, q[j]);
      attn_own<DT, D>((const E*)a.grad, at, g, go[j]);
      lse[j] = a.lse[(int64_t)head * a.T + in];
      sees[j] = in + 1 > t.prefix_end ? in + 1 : t.prefix_end;
      delta[j] = 0.f;
      if (alone) continue;
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
    int keys = last > t.prefix_end ? last : t.prefix_end, key0 = t.begin;
    if constexpr (KIND == kAttnBias) {
      const int reach = attn_reach(a, head);
      if (t.first - reach > key0) key0 += (t.first - reach - key0) / R * R;
      if (last + reach < keys) keys = last + reach;
    }
    int mine = row0 + 16 * NB < t.end ? row0 + 16 * NB : t.end;
    mine = row0 >= t.end ? t.begin : mine > t.prefix_end ? mine : t.prefix_end;

    Rows rk, rv;
    rk.init(a.kt);
    rv.init(a.vt);
    rk.load(K, a.kt, key0, keys);
    rv.load(V, a.vt, key0, keys);
    int buf = 0;
    for (int k0 = key0; k0 < keys; k0 += R) {
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
      float ref[NB];
      score.tile(k0, row0, row0 + 16 * NB, g);
#pragma unroll
      for (int j = 0; j < NB; j++) ref[j] = score.shift(row0 + 16 * j + c, k0) - lse[j];
      const bool part = k0 + R > least;
      const float near = (float)(row0 + c - k0 - 4 * g);
      // Block b of the tile: P (p) and dP less delta (dp), under a cap times its slope if `sloped`.
      auto block = [&](int b, bool sloped, f32x4(&p)[NB], f32x4(&dp)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
          p[j] = score.start(b);
          dp[j] = f32x4{-delta[j], -delta[j], -delta[j], -delta[j]};
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const Frag fk = Rows::row_frag(lk, b, ks, c, g), fv = Rows::row_frag(lv, b, ks, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            p[j] = attn_mfma<DT>(fk, q[j][ks], p[j]);
            dp[j] = attn_mfma<DT>(fv, go[j][ks], dp[j]);
          }
        }
        if constexpr (KIND == kAttnCap) {
          score.cap_all(p, [&](int j, int e, float slope) {
            if (sloped) dp[j][e] *= slope;
          });
        }
        if (score.single()) {
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) p[j][e] = score.biased(p[j][e], near + (float)(16 * j - 16 * b - e));
        }
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) p[j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[j][e], score.unit, ref[j]));
      };
      if (alone) {
        float all[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) all[j] = 0.f;
#pragma unroll
        for (int b = 0; b < R / 16; b++) {
          f32x4 p[NB], dp[NB];
          block(b, false, p, dp);
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) all[j] += k0 + 16 * b + 4 * g + e < sees[j] ? p[j][e] * dp[j][e] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < NB; j++) {
          delta[j] = cross_row_sum(all[j]);
          const int row = row0 + 16 * j + c;
          if (g == 0 && row < t.end) a.delta[(int64_t)head * a.T + row] = delta[j];
        }
      }
#pragma unroll
      for (int h = 0; h < R / 32; h++) {  // 32 keys at a time
        f32x4 s[2][NB];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          f32x4 dp[NB];
          block(2 * h + i, true, s[i], dp);
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[i][j][e] *= dp[j][e];
        }
        if (part) {
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
              for (int e = 0; e < 4; e++) s[i][j][e] = k0 + 32 * h + 16 * i + 4 * g + e < sees[j] ? s[i][j][e] : 0.f;
        }
        Frag ds[NB], rest[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) {
          if constexpr (DT == TMS_DTYPE_F16) range[j].follow(s[0][j], s[1][j], acc, j);
          ds[j] = attn_pack<DT>(s[0][j], s[1][j]);
          if constexpr (TWO) rest[j] = attn_rest<DT>(s[0][j], s[1][j]);
        }
#pragma unroll
        for (int d = 0; d < DB; d++) {
          const Frag f = Rows::col_frag(lk, h, d, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            acc[d][j] = attn_mfma<DT>(f, ds[j], acc[d][j]);
            if constexpr (TWO) acc[d][j] = attn_mfma<DT>(f, rest[j], acc[d][j]);
          }
        }
      }
    }
  }
  if (!a.dq) return;
  uint32_t odd[NB];
#pragma unroll
  for (int j = 0; j < NB; j++) {
    const int row = row0 + 16 * j + c;
    odd[j] = 0;
    if constexpr (MASK) {
      odd[j] = attn_odd(!attn_all_finite(acc, j) && row < t.end);
      if (odd[j] != 0) {
        __threadfence_block();  // delta is another lane's
        const int64_t at = (int64_t)head * a.T + row;
        odd[j] &= attn_odd(row < t.end && attn_finite(a.lse[at]) && attn_finite(a.delta[at]));
        const int unseen = row0 + 1 > t.prefix_end ? row0 + 1 : t.prefix_end, past = row0 + 16 * NB, end = (past > t.prefix_end ? past : t.prefix_end) + R;
        const E* k = (const E*)a.k + head / a.many * a.kh;
        if (odd[j] == 0 || attn_rows_finite<DT, D>(k, a.kt, unseen, end < t.end ? end : t.end)) {
          odd[j] = 0;
        } else {
          AttnColumns<D> bad;
          bad.template add<DT>(k, a.kt, t.begin, unseen);
          odd[j] &= attn_odd(row < t.end && attn_unexplained<DT, D>(acc, j, bad, k + row * a.kt, g));
        }
      }
    }
    if (row >= t.end || odd[j] >> c & 1) continue;
    const bool one = (row + 1 > t.prefix_end ? row + 1 : t.prefix_end) == t.begin + 1;  // the row sees one key: P = 1, dS = 0 (but for roundings)
    const float f = !t.real || one ? 0.f : (DT == TMS_DTYPE_F16 ? a.scale / range[j].held : a.scale) / AttnScore<DT, KIND, Rows::R>::kSlope;
    attn_store<DT>(a.dq, ((int64_t)row * a.H + head) * D, acc, j, f, g);
  }
#pragma unroll
  for (int j = 0; j < NB; j++) {
    for (uint32_t m = MASK ? odd[j] : 0; m != 0; m &= m - 1) {
      const int i = __builtin_ctz(m), row = row0 + 16 * j + i, kvh = head / a.many;
      const int ln = attn_lane();
      const float l = a.lse[(int64_t)head * a.T + row], dl = a.delta[(int64_t)head * a.T + row];
      const int sees = row + 1 > t.prefix_end ? row + 1 : t.prefix_end;
      const float f = sees == t.begin + 1 ? 0.f : a.scale;
      float x[(D + 63) / 64] = {};
      attn_alone<DT, D, KIND, kAttnDq>(a, head, row, t.begin, sees, (const E*)a.q + head * a.qh + row * a.qt,
                                       (const E*)a.grad + ((int64_t)row * a.H + head) * D, (const E*)a.k + kvh * a.kh, a.kt, (const E*)a.v + kvh * a.vh, a.vt, l, dl,
                                       x, x);
#pragma unroll
      for (int u = 0; u < (D + 63) / 64; u++)
        if (64 * u + ln < D) ((E*)a.dq)[((int64_t)row * a.H + head) * D + 64 * u + ln] = attn_round<DT>(x[u] * f);
    }
  }
}

// dk and dv: a workgroup has a tile of keys and goes over the queries that see them, head by head of
// those that share the keys. Both gradients' sums are as many registers as the keys and values: more than two
// workgroups a CU spill (heads of 128, a bound of three: 166 us, 118 with two).
template <int DT, int D, int NB, int KIND, bool SHORT, bool MASK>
__global__ __launch_bounds__(kAttnThreads, 2) void attn_dkv_kernel(AttnArgs a) {
  typedef AttnRows<DT, D, attn_rows<DT, D, NB>(kAttnDkv)> Rows;
  typedef typename AttnType<DT>::E E;
  typedef typename AttnType<DT>::Frag Frag;
  constexpr bool TWO = SHORT && DT != TMS_DTYPE_F32;
  constexpr int R = Rows::R, DB = D / 16, KS = D / 32, BK = 64 * NB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t attn_mem[];
  float* const stats = (float*)(attn_mem + 4 * Rows::kBytes);  // [buffer][lse, delta][R]
  int slot, kvh;
  if (!attn_place(a, a.KV * a.parts, slot, kvh)) return;
  const int part_of = kvh % a.parts;
  kvh /= a.parts;
  AttnTile t;
  t.find<BK>(a, slot);
  if (t.text < 0) return;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int key0 = t.first + wave * 16 * NB;
  const int head0 = kvh * a.many + part_of * a.many / a.parts, heads = kvh * a.many + (part_of + 1) * a.many / a.parts - head0;

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
    int rows = t.first < t.prefix_end ? t.begin : t.first, rows_end = t.end;
    const int mine = key0 >= t.end ? 0x7fffffff : key0 < t.prefix_end ? t.begin : key0;
    const int all = key0 + 16 * NB <= t.prefix_end || t.prefix_end == t.end ? t.begin : key0 + 16 * NB - 1;
    if constexpr (KIND == kAttnBias) {  // as far as the farthest of the heads reaches
      int reach = 0;
      for (int h = 0; h < heads; h++) {
        const int of = attn_reach(a, head0 + h);
        reach = of > reach ? of : reach;
      }
      const int last = t.first + BK < t.end ? t.first + BK : t.end;
      if (t.first - reach > rows) rows = t.first - reach;
      if (last + reach < rows_end) rows_end = last + reach;
    }
    const int tiles = (rows_end - rows + R - 1) / R, total = tiles * heads;

    Rows rq, rg;
    rq.init(a.qt);
    rg.init((int64_t)a.H * D);
    float st = 0.f;  // a thread's share of the tile's statistics: lse (the first R), delta (the next)
    auto load = [&](int n) {
      const int head = head0 + n / tiles, r0 = rows + n % tiles * R;
      rq.load((const E*)a.q + head * a.qh, a.qt, r0, rows_end);
      rg.load((const E*)a.grad + (int64_t)head * D, (int64_t)a.H * D, r0, rows_end);
      if ((int)threadIdx.x < 2 * R) {
        const int r = r0 + (int)threadIdx.x % R;
        const float* from_ = (int)threadIdx.x < R ? a.lse : a.delta;
        st = -(r < rows_end ? from_[(int64_t)head * a.T + r] : (int)threadIdx.x < R ? __builtin_inff() : 0.f);
      }
    };
    AttnScore<DT, KIND, R> score;
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
      if (n % tiles == 0) score.init(a, head0 + n / tiles);
      if (r0 + R <= mine) continue;  // uniform in the wave
      const bool part = r0 < all;
      const float near = (float)(r0 + 4 * g - key0 - c);
      score.tile(r0, key0, key0 + 16 * NB, g);
      float shift[NB];
#pragma unroll
      for (int j = 0; j < NB; j++) shift[j] = score.shift(key0 + 16 * j + c, r0);
#pragma unroll
      for (int h = 0; h < R / 32; h++) {  // 32 rows at a time
        f32x4 p[2][NB], s[2][NB];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int b = 2 * h + i;
          const f32x4 lse = *(const f32x4*)(ls + 16 * b + 4 * g), delta = *(const f32x4*)(ls + R + 16 * b + 4 * g);  // both negated
          f32x4 dp[NB];
#pragma unroll
          for (int j = 0; j < NB; j++) {
            s[i][j] = score.start(b);
            dp[j] = delta;
          }
#pragma unroll
          for (int ks = 0; ks < KS; ks++) {
            const Frag fq = Rows::row_frag(lq, b, ks, c, g), fg = Rows::row_frag(lg, b, ks, c, g);
#pragma unroll
            for (int j = 0; j < NB; j++) {
              s[i][j] = attn_mfma<DT>(fq, k[j][ks], s[i][j]);
              dp[j] = attn_mfma<DT>(fg, v[j][ks], dp[j]);
            }
          }
          if constexpr (KIND == kAttnCap) score.cap_all(s[i], [&](int j, int e, float slope) { dp[j][e] *= slope; });
          if (score.single()) {
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
              for (int e = 0; e < 4; e++) s[i][j][e] = score.biased(s[i][j][e], near + (float)(16 * b + e - 16 * j));
          }
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float ref = KIND == kAttnBias ? lse[e] + shift[j] : lse[e];
              const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j][e], score.unit, ref));
              s[i][j][e] = y * dp[j][e];
              p[i][j][e] = y * (float)(1 << attn_up<DT>());
            }
        }
        if (part) {
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const bool in = r0 + 32 * h + 16 * i + 4 * g + e >= from[j];
                p[i][j][e] = in ? p[i][j][e] : 0.f;
                s[i][j][e] = in ? s[i][j][e] : 0.f;
              }
        }
        Frag pf[NB], sf[NB], prest[NB], srest[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) {
          if constexpr (DT == TMS_DTYPE_F16) range[j].follow(s[0][j], s[1][j], dk, j);
          pf[j] = attn_pack<DT>(p[0][j], p[1][j]);
          sf[j] = attn_pack<DT>(s[0][j], s[1][j]);
          if constexpr (TWO) {
            prest[j] = attn_rest<DT>(p[0][j], p[1][j]);
            srest[j] = attn_rest<DT>(s[0][j], s[1][j]);
          }
        }
#pragma unroll
        for (int d = 0; d < DB; d++) {
          const Frag fg = Rows::col_frag(lg, h, d, c, g), fq = Rows::col_frag(lq, h, d, c, g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            dv[d][j] = attn_mfma<DT>(fg, pf[j], dv[d][j]);
            dk[d][j] = attn_mfma<DT>(fq, sf[j], dk[d][j]);
            if constexpr (TWO) {
              dv[d][j] = attn_mfma<DT>(fg, prest[j], dv[d][j]);
              dk[d][j] = attn_mfma<DT>(fq, srest[j], dk[d][j]);
            }
          }
        }
      }
    }
  }
  uint32_t odd[NB];
#pragma unroll
  for (int j = 0; j < NB; j++) {
    const int key = key0 + 16 * j + c;
    odd[j] = 0;
    if constexpr (MASK) {
      odd[j] = attn_odd(!(attn_all_finite(dk, j) && attn_all_finite(dv, j)) && key < t.end);
      if (odd[j] != 0) {
        const int from = key0 < t.prefix_end ? t.begin : key0 - R, last = key0 + 16 * NB - 1;
        const int begin = from > t.begin ? from : t.begin, end = last < t.end ? last : t.end;  // of rows that some key is not seen by
        const int64_t gt = (int64_t)a.H * D;
        bool all = true, dead = false, some_v = key < t.end;  // dead: dk of all columns, or of this key's
        AttnColumns<D> bad;
        for (int head = head0; head < head0 + heads; head++) {
          const E *q = (const E*)a.q + head * a.qh, *grad = (const E*)a.grad + (int64_t)head * D;
          const int64_t at = (int64_t)head * a.T;
          odd[j] &= attn_odd(key < t.end && attn_finite(a.lse[at + key]));
          if (odd[j] == 0) break;
          all = all && attn_rows_finite<DT, D>(q, a.qt, begin, end) && attn_rows_finite<DT, D>(grad, gt, begin, end);
          bool lost = false, none = false;  // rows that all keys are seen by: of no delta, and of no P
          for (int r = last + attn_lane(); r < t.end; r += 64) {
            none |= !attn_finite(a.lse[at + r]);
            lost |= !attn_finite(a.delta[at + r]);
          }
          if (__ballot(none) != 0ull) {
            odd[j] = 0;
            break;
          }
          dead |= __ballot(lost) != 0ull || (key < t.end && !attn_finite(a.delta[at + key]));
          bad.template add<DT>(grad, gt, last, t.end);
          some_v = some_v && attn_unexplained<DT, D>(dv, j, bad, grad + key * gt, g);
        }
        if (all) odd[j] = 0;
        odd[j] &= attn_odd(some_v || (key < t.end && !dead && !attn_all_finite(dk, j)));
      }
    }
    if (key >= t.end || odd[j] >> c & 1) continue;
    const int64_t at = ((int64_t)key * a.KV + kvh) * D;
    // of a text of one token dS is 0, but for roundings
    const float fk = !t.real || t.end - t.begin == 1 ? 0.f : (DT == TMS_DTYPE_F16 ? a.scale / range[j].held : a.scale) / AttnScore<DT, KIND, Rows::R>::kSlope;
    const float fv = !t.real ? 0.f : 1.f / (float)(1 << attn_up<DT>());
    if (a.parts > 1) {
      const int64_t one = a.T * a.KV * D;
      attn_store<TMS_DTYPE_F32>(a.sums + 2 * part_of * one, at, dk, j, fk, g);
      attn_store<TMS_DTYPE_F32>(a.sums + (2 * part_of + 1) * one, at, dv, j, fv, g);
      continue;
    }
    if (a.dk) attn_store<DT>(a.dk, at, dk, j, fk, g);
    if (a.dv) attn_store<DT>(a.dv, at, dv, j, fv, g);
  }
#pragma unroll
  for (int j = 0; j < NB; j++) {
    for (uint32_t m = MASK ? odd[j] : 0; m != 0; m &= m - 1) {
      const int key = key0 + 16 * j + __builtin_ctz(m);
      float x[(D + 63) / 64] = {}, y[(D + 63) / 64] = {};
      for (int head = head0; head < head0 + heads; head++)
        attn_alone<DT, D, KIND, kAttnDkv>(a, head, key, key < t.prefix_end ? t.begin : key, t.end, (const E*)a.k + kvh * a.kh + key * a.kt,
                                          (const E*)a.v + kvh * a.vh + key * a.vt, (const E*)a.q + head * a.qh, a.qt, (const E*)a.grad + (int64_t)head * D,
                                          (int64_t)a.H * D, 0.f, 0.f, x, y);
#pragma unroll
      for (int u = 0; u < (D + 63) / 64; u++) {
        const int64_t at = ((int64_t)key * a.KV + kvh) * D + 64 * u + attn_lane(), one = a.T * a.KV * D;
        if (64 * u + attn_lane() >= D) continue;
        if (a.parts > 1) {
          a.sums[2 * part_of * one + at] = x[u] * a.scale;
          a.sums[(2 * part_of + 1) * one + at] = y[u];
          continue;
        }
        if (a.dk) ((E*)a.dk)[at] = attn_round<DT>(x[u] * a.scale);
        if (a.dv) ((E*)a.dv)[at] = attn_round<DT>(y[u]);
      }
    }
  }
}

// dk and dv from the parts' sums, in their order: four elements a thread. Bound by reading them (two parts of 12,961
// tokens, 2 heads of 128: 53 MB in 11 us).
template <int DT>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(const float* sums, int parts, int64_t n, void* dk, void* dv) {
  typedef typename AttnType<DT>::E E;
  struct __attribute__((packed, aligned(4 * sizeof(E)))) Four { E x[4]; };
  for (int64_t i = (int64_t)blockIdx.x * kAttnThreads + threadIdx.x; i < n / 2; i += (int64_t)gridDim.x * kAttnThreads) {
    const bool second = i >= n / 4;
    E* to = (E*)(second ? dv : dk);
    if (to == nullptr) continue;
    const int64_t at = (second ? i - n / 4 : i) * 4;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; p++) {
      const f32x4 y = *(const f32x4*)(sums + (2 * p + second) * n + at);
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] += y[e];
    }
    Four o;
#pragma unroll
    for (int e = 0; e < 4; e++) o.x[e] = attn_round<DT>(x[e]);
    *(Four*)(to + at) = o;
  }
}

// ---------------------------------------------------------------- launches

template <int DT, int D, int NB, int KIND, AttnPass PASS, bool MASK>
static int attn_launch(AttnArgs a, hipStream_t st) {
  typedef AttnRows<DT, D, attn_rows<DT, D, NB>(PASS)> Rows;
  a.slots = (int32_t)attn_slots(a.T, a.B, 64 * NB);
  const dim3 grid((unsigned)attn_grid(a.slots, PASS == kAttnDkv ? a.KV * a.parts : a.H)), threads(kAttnThreads);  // below 2^23
  constexpr size_t lds = 4 * (size_t)Rows::kBytes;
  if constexpr (PASS == kAttnForward) {
    hipLaunchKernelGGL((attn_forward_kernel<DT, D, NB, KIND, MASK>), grid, threads, lds, st, a);
    return check_launch("attn_forward_kernel");
  } else if constexpr (PASS == kAttnDq) {
    if constexpr (NB == 1) {
      if (attn_short(a.T, a.B)) {
        hipLaunchKernelGGL((attn_dq_kernel<DT, D, NB, KIND, true, MASK>), grid, threads, lds, st, a);
        return check_launch("attn_dq_kernel");
      }
    }
    hipLaunchKernelGGL((attn_dq_kernel<DT, D, NB, KIND, false, MASK>), grid, threads, lds, st, a);
    return check_launch("attn_dq_kernel");
  } else {
    constexpr size_t both = lds + 4 * Rows::R * sizeof(float);
    bool few = false;
    if constexpr (NB == 1 && DT != TMS_DTYPE_F32) {
      few = attn_short(a.T, a.B);
      if (few) hipLaunchKernelGGL((attn_dkv_kernel<DT, D, NB, KIND, true, MASK>), grid, threads, both, st, a);
    }
    if (!few) hipLaunchKernelGGL((attn_dkv_kernel<DT, D, NB, KIND, false, MASK>), grid, threads, both, st, a);
    const int rc = check_launch("attn_dkv_kernel");
    if (rc || a.parts == 1) return rc;
    const int64_t n = a.T * a.KV * D, groups = (n / 2 + kAttnThreads - 1) / kAttnThreads;
    hipLaunchKernelGGL(attn_join_kernel<DT>, dim3((unsigned)(groups < 65536 ? groups : 65536)), threads, 0, st, a.sums, a.parts, n, a.dk, a.dv);
    return check_launch("attn_join_kernel");
  }
}

// One of these for each dtype, in a file of its own.
int attn_run_f16(const AttnArgs& a, int D, AttnPass pass, hipStream_t st);
int attn_run_bf16(const AttnArgs& a, int D, AttnPass pass, hipStream_t st);
int attn_run_f32(const AttnArgs& a, int D, AttnPass pass, hipStream_t st);

// Whether a pass has the registers for two blocks of 16 of its own rows: dk and dv need keys, values and both
// gradients (96 under a bias, with spills: 585 us, 320 with one block), dq queries, their gradients and sums.
template <int DT, int D, int KIND>
constexpr bool attn_two(AttnPass pass) {
  if (DT == TMS_DTYPE_F32) return false;
  if (pass == kAttnDkv) return D <= 64 || (D == 96 && KIND == kAttnPlain);
  return pass == kAttnForward || D < 128 || KIND == kAttnPlain;
}
template <int DT, int D, int KIND, AttnPass PASS, bool MASK>
static int attn_run_mask(const AttnArgs& a, hipStream_t st) {
  if constexpr (attn_two<DT, D, KIND>(PASS)) {
    if (attn_wide(a.T, a.B, PASS == kAttnDkv ? (int64_t)a.KV * a.parts : a.H)) return attn_launch<DT, D, 2, KIND, PASS, MASK>(a, st);
  }
  return attn_launch<DT, D, 1, KIND, PASS, MASK>(a, st);
}
template <int DT, int D, int KIND, AttnPass PASS>
static int attn_run_pass(const AttnArgs& a, hipStream_t st) {
  return a.prefix != nullptr ? attn_run_mask<DT, D, KIND, PASS, true>(a, st) : attn_run_mask<DT, D, KIND, PASS, false>(a, st);
}
template <int DT, int D, int KIND>
static int attn_run_kind(const AttnArgs& a, AttnPass pass, hipStream_t st) {
  if (pass == kAttnForward) return attn_run_pass<DT, D, KIND, kAttnForward>(a, st);
  if (pass == kAttnDq) return attn_run_pass<DT, D, KIND, kAttnDq>(a, st);
  return attn_run_pass<DT, D, KIND, kAttnDkv>(a, st);
}
template <int DT, int D>
static int attn_run_d(const AttnArgs& a, AttnPass pass, hipStream_t st) {
  if (a.norms && pass == kAttnForward) {
    hipLaunchKernelGGL((attn_norms_kernel<DT, D>), dim3((unsigned)((a.H + a.KV) * kAttnNorms)), dim3(kAttnThreads), 0, st, a);
    const int rc = check_launch("attn_norms_kernel");
    if (rc) return rc;
  }
  if (a.cap > 0.f) return attn_run_kind<DT, D, kAttnCap>(a, pass, st);
  if (a.slopes) return attn_run_kind<DT, D, kAttnBias>(a, pass, st);
  return attn_run_kind<DT, D, kAttnPlain>(a, pass, st);
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
