// What the expert products on microscaled and bfloat16 banks share: their arguments, the operands' places (Format), and
// the passes over ragged groups of rows.
//
// A product is out[p, n] = sum_k x[row(p), k] w[expert(p), n, k] for the pairs p of rows and experts, as
// v_mfma tiles of 16 weight rows x 16 pairs. K goes by in stages of two MFMA steps; every kernel adds a pair's stages
// and steps in the same order into one float32 accumulator, so a result depends on the pair's row and expert alone, not on
// the kernel, the tile or the rows beside it.
#pragma once
#include "mx.hpp"
#include "wide_tile.hpp"

namespace d3 {

struct ExpertProduct {
  const uint8_t* x;        // rows [x_rows, row_bytes]
  const uint8_t* x_scale;  // microscaled rows: [x_rows, 8 * stages]
  int x_rows;
  const int64_t* ids;      // gemv: [pairs]
  int per_row;             // gemv: pairs to a row of x
  const int32_t* groups;   // grouped: [n_groups, 5] (expert, ., ., first, rows)
  int n_groups;
  const int64_t* order;    // grouped: pair at each place, or null (the place's own row)
  int k;                   // pairs to a row of x, with order
  int pairs;
  const uint8_t* w;
  const uint8_t* w_scale;
  int E, N, stages;        // N rows an expert; stages of K
  void* out;               // [pairs, N] float32 or bf16; swiglu: [pairs, N / 2] bf16
};

// Where a format's operands lie. A (weights): a lane's 16 bytes of stage st, step s of tile t at
// a_base(t, lane) + st * A_STAGE + s * A_STEP. B (rows): ROW bytes of a row to a stage; a lane's operand of step s is the
// 16-byte pieces b_piece(s, q, 0 ..) of them.
template <int BITS_>
struct Mx {
  static constexpr bool SCALED = true;
  static constexpr int BITS = BITS_, ROW = 32 * BITS, PIECES = BITS / 4, SEG = 8;  // SEG: stages whose rows LDS holds
  static constexpr int A_STAGE = 2048, A_STEP = 1024;
  static D3_INLINE size_t a_base(size_t tile, int stages, int lane) { return tile * stages * 2048 + lane * 16; }
  static D3_INLINE int b_piece(int s, int q, int i) {
    return BITS == 4 ? 2 * q + s : 4 * (q >> 1) + 2 * s + (q & 1) + 8 * i;
  }
};
// bfloat16: a stage is 64 columns (128 bytes of a row), step s multiplies the pieces 4 s + q of 8 columns; the weights lie
// row by row
struct Bf16 {
  static constexpr bool SCALED = false;
  static constexpr int BITS = 16, ROW = 128, PIECES = 1, SEG = 32;
  static constexpr int A_STAGE = 128, A_STEP = 64;
  static D3_INLINE size_t a_base(size_t tile, int stages, int lane) {
    return (tile * 16 + (lane & 15)) * ((size_t)stages * 128) + 16 * (lane >> 4);
  }
  static D3_INLINE int b_piece(int s, int q, int) { return 4 * s + q; }
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A step's operand b of e4m3 rows in two parts, below 2 and from 2 on (zeros in between): b = low + high.
//
// Against e4m3, v_mfma_scale aligns a block's 32 products to the largest one's exponent and keeps 13 bits below it (measured:
// of 256 - 256 + 2^-n it gives 2^-5 and nothing smaller; e2m1 against e2m1 loses nothing). e4m3 spans 18 binades, so
// small elements beside a block's large ones are cut, each by up to 2^-13 of the block's largest product: 7e-6 of a result's
// norm on normally distributed rows with a few channels eight times as large, where float32 sums give 2e-7, and without a
// bound where large products cancel. Of each part every product keeps all its bits: e2m1 is a multiple
// of 1/2, high of 1/4 and low of 2^-9, so products are multiples of 2^-3 with exponents up to 8 + 2 = 10, and of 2^-10 with
// exponents up to 0 + 2 = 2 (4000 random blocks of each part came out exactly, with the border at 1 or 8 they did not).
D3_INLINE void split_e4m3(i32x8 b, i32x8& low, i32x8& high) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t v = (uint32_t)b[i], from2 = v & 0x40404040u;  // 2 is code 0x40, and every larger one has that bit
    const uint32_t part = v & ((from2 << 2) - (from2 >> 6));     // (0xFF in the bytes that have it)
    high[i] = (int)part;
    low[i] = (int)(v ^ part);
  }
}

// acc + a . b over a step. sa, sb: scale words, byte OA and OB of them. (The upper half of an e2m1 operand is not
// read.) e4m3 rows in two parts whatever becomes of the result: what the instruction cuts goes by a block's largest product,
// not by the sum, and where large products cancel, rounding the sum to bf16 does not hide it.
template <class F, int OA, int OB>
D3_INLINE f32x4 step_product(i32x4 a, const i32x4 (&b)[F::PIECES], f32x4 acc, uint32_t sa, uint32_t sb) {
  if constexpr (F::SCALED) {
    const i32x8 A = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
    if constexpr (F::BITS == 4) {
      const i32x8 B = __builtin_shufflevector(b[0], b[0], 0, 1, 2, 3, -1, -1, -1, -1);
      return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc, 4, 4, OA, (int)sa, OB, (int)sb);
    } else {
      const i32x8 B = __builtin_shufflevector(b[0], b[F::PIECES - 1], 0, 1, 2, 3, 4, 5, 6, 7);
      i32x8 low, high;
      split_e4m3(B, low, high);
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, high, acc, 4, 0, OA, (int)sa, OB, (int)sb);
      return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, low, acc, 4, 0, OA, (int)sa, OB, (int)sb);
    }
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b[0]), acc,
                                                   0, 0, 0);
  }
}

// four float32 sums rounded to bf16 (to nearest, ties to even, by the converter)
D3_INLINE i32x2 bf16_4(f32x4 v) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(i32x2, __builtin_convertvector(v, bf16x4));
}
// SiLU(gate) * up in float32, then rounded to bf16 as the rows that the next product reads. exp and the reciprocal are the
// hardware's, within 2 and 1 units of the last place, and exp takes a rounded gate / ln 2, |gate| 2^-23 of the value more: within
// (2^-21 + |gate| 2^-23) of it in all, 2^-16 at |gate| = 87, which the rounding's 2^-8 hides. (Below, SiLU is under 2^-118 and
// its reciprocal may come out as zero.)
D3_INLINE i32x2 swiglu_4(f32x4 gate, f32x4 up) {
  f32x4 h;
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = gate[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-gate[i])) * up[i];
  return bf16_4(h);
}

struct Pass {
  int expert, first, rows;
};

// group g's expert, first place and rows; no rows past the last group, and where the expert or the places lie outside the
// bank or the pairs
D3_INLINE void read_group(const ExpertProduct& a, int g, int& expert, int& first, int& rows) {
  expert = first = rows = 0;
  if (g >= a.n_groups) return;
  const int32_t* p = a.groups + 5 * (size_t)g;
  expert = p[0], first = p[3], rows = p[4];
  if (expert < 0 || expert >= a.E || first < 0 || rows < 0 || first > a.pairs || rows > a.pairs - first) rows = 0;
}

// the sum of n over the lanes up to this one
D3_INLINE int wave_scan_i32(int n) {
  n += __builtin_amdgcn_update_dpp(0, n, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8: within rows of 16 lanes
  n += __builtin_amdgcn_update_dpp(0, n, 0x112, 0xF, 0xF, true);
  n += __builtin_amdgcn_update_dpp(0, n, 0x114, 0xF, 0xF, true);
  n += __builtin_amdgcn_update_dpp(0, n, 0x118, 0xF, 0xF, true);
  n += __builtin_amdgcn_update_dpp(0, n, 0x142, 0xA, 0xF, false);  // row_bcast 15: the first row's sum to the second, ..
  n += __builtin_amdgcn_update_dpp(0, n, 0x143, 0xC, 0xF, false);  // row_bcast 31: the first half's to the second
  return n;
}

// The first lane with at < the sum of n over the lanes up to it, and in `before` the sum over those before it; -1 if
// there is none, with the sum over all. The whole wave calls.
D3_INLINE int find_lane(int n, int at, int& before) {
  const int incl = wave_scan_i32(n);
  const uint64_t past = __ballot(incl > at);
  if (!past) {
    before = __builtin_amdgcn_readlane(incl, 63);
    return -1;
  }
  const int l = __ffsll((unsigned long long)past) - 1;
  before = __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l);
  return l;
}

// Pass `at` of the groups' passes of at most `most` rows, in the groups' order: its expert, first place and rows (0: there
// is no such pass). The whole wave calls.
D3_INLINE Pass find_pass(const ExpertProduct& a, int most, int at) {
  const int lane = threadIdx.x & 63;
  for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
    int expert, first, rows, before;
    read_group(a, g0 + lane, expert, first, rows);
    const int l = find_lane((rows + most - 1) / most, at, before);
    if (l >= 0) {
      const int from = (at - before) * most;
      return Pass{__builtin_amdgcn_readlane(expert, l), __builtin_amdgcn_readlane(first, l) + from,
                  min(most, __builtin_amdgcn_readlane(rows, l) - from)};
    }
    at -= before;
  }
  return Pass{0, 0, 0};
}

// the pair at place p, and the row of x of a pair
D3_INLINE int64_t pair_at(const ExpertProduct& a, int p) { return a.order ? a.order[p] : p; }
D3_INLINE int pair_row(const ExpertProduct& a, int64_t pair) {
  const uint32_t at = (uint32_t)min<int64_t>(max<int64_t>(pair, 0), INT32_MAX);
  return min((int)(a.order ? at / (uint32_t)a.k : at), a.x_rows - 1);
}

// passes of at most `most` rows that groups of `pairs` rows in all can have
inline int most_passes(int pairs, int n_groups, int most) {
  const int64_t n = (int64_t)pairs / most + n_groups;
  return (int)(n < pairs ? n : pairs);
}

}  // namespace d3
