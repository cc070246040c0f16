// Dense products on the matrix cores: out[m, n] = sum_k x(m, k) w(n, k), bfloat16 operands, float32 sums, either operand stored
// with its k side by side (rows, as activations and weights lie) or with its m or n side by side (transposed: the same
// tensors where a gradient sums over their rows). A workgroup computes a tile of TM x TN, its waves WM x WN of them
// MT x NT MFMA tiles of 16 x 16 each; the weight side is the instruction's first operand, so a lane holds 4 results
// that follow each other in a row of out.
//
// Both operands of a stage of 64 k lie in LDS, copied there without passing through registers:
//   rows        128 bytes a row, in 16-byte pieces, piece j of row r at slot j ^ ((r >> 1) & 7) (wide_tile.hpp)
//   transposed  64 rows of k; a lane's operand is 4 k of one column, which the transposing LDS read gives from 4 rows of 16
//               columns; those 32-byte chunks of a row lie at chunk ^ t_turn(k), so that the 8 rows that 32 lanes read
//               meet 8 different groups of banks
// Columns past K read as zeros in both operands (each lane clears what it copied of them, in the last stage alone); rows past M
// and N read the last one, and are not stored.
#pragma once
#include "wide_tile.hpp"

#include <type_traits>

namespace d3 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// what becomes of a tile
enum DenseEnd {
  END_ROWS,     // out bf16
  END_SWIGLU,   // w holds `half` gate rows, then as many up rows: out [M, half] = SiLU(gate) * up, and pre where it is given
  END_DSWIGLU,  // the sums are the gradient of SiLU(gate) * up: out [M, 2 half] = the gradients of gate and up (from pre)
  END_INNER,    // out bf16 = alpha times the sums, of the tile's rows (up to 64) whose bit is set in `rows`
};

struct Dense {
  const uint16_t* x;
  const uint16_t* w;
  int64_t ldx, ldw, ldo;  // elements from row to row as they are stored (ldo: of out)
  uint16_t* out;
  float* pre;     // [M, 2 half]: gate and up before the activation
  int M, N, K, half;
  // adapters: out += p(m) . b[ids[m]](n), p [M, rank] of this row's own adapter; rows with an id outside have none
  const uint16_t* p;
  const uint16_t* b;  // [adapters, N, rank]
  const int64_t* ids;
  int rank, adapters;
  uint64_t rows;
  float alpha;
};

// dma16 as an instruction that the compiler may move other memory accesses past: its place among the barriers (which
// nothing passes) is what the LDS that it writes needs
D3_INLINE void copy16(uint32_t lds, const uint8_t* base, uint32_t off) {
  const uint64_t at = (uint64_t)base;
  const uint64_t sbase = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32;
  uint64_t from;
  asm volatile("s_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
               : "=&s"(from)
               : "{m0}"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(sbase));
}

template <int N>
D3_INLINE void loads_but() {
  static_assert(N < 64);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

D3_INLINE f32x4 mfma_bf16(i32x4 a, i32x4 b, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

// which turn row k's chunks take: bits of k that tell 8 rows 0 .. 3, 8 .. 11 apart (of 64 columns two rows share a group of banks)
template <int ROWS>
D3_INLINE int t_turn(int k) { return ROWS >= 128 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1; }
template <int ROWS> constexpr int t_turns = ROWS >= 128 ? 7 : 3;

// One operand's side of a tile: ROWS m or n. T: transposed. W waves copy it, PER kilobytes each.
template <int ROWS, bool T, int W>
struct Side {
  static constexpr int BYTES = ROWS * 128, PER = BYTES / 1024 / W;
  static_assert(BYTES % (1024 * W) == 0 && (!T || ROWS % 64 == 0));
  const uint8_t* base;  // of the next stage to copy
  uint32_t step;        // bytes from stage to stage
  uint32_t off[PER];
  // the row (T: the k) and the first column of the 16 bytes that this lane copies in copy i
  static D3_INLINE int row_of(int i, int w, int lane) { return T ? ((w * PER + i) * 1024 + lane * 16) / (2 * ROWS) : (w * PER + i) * 8 + (lane >> 3); }
  static D3_INLINE int col_of(int i, int w, int lane) {
    const int r = row_of(i, w, lane);
    if constexpr (!T) return 8 * wt_slot(r, lane & 7);
    const int at = (lane * 16) % (2 * ROWS), c = at >> 5;
    return 16 * ((c & ~t_turns<ROWS>) | ((c & t_turns<ROWS>) ^ t_turn<ROWS>(r))) + ((at >> 4) & 1) * 8;
  }
  // which of a stage's k that is
  static D3_INLINE int k_of(int i, int w, int lane) { return T ? row_of(i, w, lane) : col_of(i, w, lane); }
};

// Where a lane's operands of k-step s lie in a side's stage, those of MFMA tile 0: lane (q, c) holds k = 8 q .. 8 q + 7 of row c.
template <int ROWS, bool T>
D3_INLINE uint32_t operand_at(int s, int lane) {
  const int q = lane >> 4, c = lane & 15;
  if constexpr (!T) return c * 128 + wt_slot(c, 4 * s + q) * 16;
  const int k = 8 * q + (c >> 2);
  return k * (2 * ROWS) + t_turn<ROWS>(k) * 32 + (c & 3) * 8 + s * 64 * ROWS;
}
// the operand of tile t, `at` the place above in this stage's buffer (whose address, like a row of k's, ends in zeros where t's turn goes)
template <int ROWS, bool T>
D3_INLINE i32x4 operand(uint32_t at, int t) {
  typedef __attribute__((address_space(3))) const i32x4 lds_i32x4;
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  if constexpr (!T) {
    return *(lds_i32x4*)(uintptr_t)(at + t * 2048);
  } else {
    const uint32_t here = (at ^ ((t & t_turns<ROWS>) * 32)) + (t & ~t_turns<ROWS>) * 32;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)here);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)(here + 8 * ROWS));
    return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}
// v, of which the compiler forgets what it knows: what is computed from it here is neither kept from earlier nor made ahead of a loop
// (registers that the wide tile does not have: a reload from scratch memory would wait for all copies on their way)
D3_INLINE uint32_t anew(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// SiLU(g) u and its gradients from the float32 sums. The sigmoid's exponential and reciprocal are the hardware's
// (within 2^-21 + |g| 2^-23 of the value in all), which the rounding of the results to bf16 hides. At -g past 88 the exponential
// is infinite and the sigmoid 0, as in the limit.
D3_INLINE float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// four results rounded to bf16
D3_INLINE i32x2 round4(f32x4 v) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(i32x2, __builtin_convertvector(v, bf16x4));
}

// A row's results of two neighbouring MFMA tiles (of `tiles` whose columns are all there), lane (q, c) holding 4 of each, as 16-byte
// stores, 64 bytes a row in a row: the odd q's of the first tile change places with the even ones of the second, so
// that a lane holds 8 in a row of one tile. `at`: the row's first of the 32 columns; `stored`: columns from there on that
// there are (0: none, the whole wave calls all the same).
D3_INLINE void store_two(uint16_t* at, i32x2 v0, i32x2 v1, int stored) {
  const int q = (threadIdx.x & 63) >> 4, n = 16 * (q & 1) + 8 * (q >> 1);
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v0[0], (uint32_t)v1[0], false, false);
  const auto b = __builtin_amdgcn_permlane16_swap((uint32_t)v0[1], (uint32_t)v1[1], false, false);
  if (n < stored) *(i32x4*)(at + n) = i32x4{(int)a[0], (int)b[0], (int)a[1], (int)b[1]};
}

// The tile of a workgroup among nm x nn: those of an XCD (workgroup i runs on XCD i % 8) lie side by side, and go by
// groups of GROUP rows of tiles, column by column, so that what they read stays in its L2.
D3_INLINE void place(int at, int nm, int nn, int& tm, int& tn) {
  constexpr int GROUP = 8;
  const int all = nm * nn, xcd = at & 7, i = at >> 3, per = all >> 3, more = all & 7;
  int t = xcd * per + min(xcd, more) + i;
  const int rows = GROUP * nn, g = t / rows, first = g * GROUP, high = min(GROUP, nm - first);
  t -= g * rows;
  tm = first + t % high;
  tn = t / high;
}

template <int WM_, int WN_, int MT_, int NT_, int BUFS_, int DEPTH_ = 1>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, BUFS = BUFS_, DEPTH = DEPTH_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int TM = 16 * WM * MT, TN = 16 * WN * NT, LDS = BUFS * (TM + TN) * 128;
};

// The adapters of a wave's rows: the products of p and b, by steps of one adapter that the rows name and up to 64 ranks, DEPTH
// steps' operands on their way at once (decode lines name about as many adapters as rows); the first of them from before the
// last stage on, the ids from before the first. Past the last adapter a step reads adapter 0 again, whose sums no row takes: a
// branch a step costs more (500 rows of 24 adapters by turns, rank 32, 2048 x 2048, this product alone: 15.4 us, 14.6 without). 61 rows
// of 24 adapters of rank 64, 4096 x 2048, alone: 7.4 us without adapters, 16.7 with them by turns, 13.2 in runs.
template <class C>
struct RowAdapters {
  static constexpr int DEPTH = C::DEPTH, NONE = -2;
  int id[C::MT];         // of row c of tile t; -1: none
  uint32_t open[C::MT];  // rows whose adapter is still to come in this run of ranks
  int r0;                // the run's first rank
  bool two;              // the run has more than 32 ranks
  bool there[2];         // this lane's ranks of either half are ranks
  int who[DEPTH];        // the steps' adapters, or NONE
  uint32_t at[C::NT];    // this lane's rows of an adapter's b, in bytes
  i32x4 bv[DEPTH][2][C::NT], pv[2][C::MT];

  D3_INLINE void begin(const Dense& a, int m0, int lane) {
#pragma unroll
    for (int t = 0; t < C::MT; t++) {
      const int m = m0 + 16 * t + (lane & 15);
      const int64_t named = m < a.M ? a.ids[m] : -1;
      id[t] = named >= 0 && named < a.adapters ? (int)named : -1;
    }
  }
  // the next adapter that a row names
  D3_INLINE int next() {
    int now = NONE;
#pragma unroll
    for (int t = C::MT - 1; t >= 0; t--) {
      const int first = __builtin_amdgcn_readlane(id[t], (__ffs((int)open[t]) - 1) & 15);
      now = open[t] ? first : now;
    }
#pragma unroll
    for (int t = 0; t < C::MT; t++) open[t] &= ~(uint32_t)__ballot(id[t] == now);
    return now;
  }
  // sends the next step's loads (a lane without ranks: the adapter's first ones)
  D3_INLINE void load(const Dense& a, int i) {
    who[i] = next();
    const uint8_t* b = (const uint8_t*)(a.b + (size_t)max(who[i], 0) * a.N * a.rank + r0);
#pragma unroll
    for (int u = 0; u < C::NT; u++) bv[i][0][u] = *(const i32x4*)(b + (there[0] ? at[u] : 0u));
    if (two) {
#pragma unroll
      for (int u = 0; u < C::NT; u++) bv[i][1][u] = *(const i32x4*)(b + (there[1] ? at[u] + 64 : 0u));
    }
  }
  // the rows' inner products of ranks r0 .. r0 + 63 (where a row has an adapter: what the others hold is not used), and the first
  // steps with them
  D3_INLINE void ranks(const Dense& a, int m0, int lane) {
    two = r0 + 32 < a.rank;
#pragma unroll
    for (int t = 0; t < C::MT; t++) open[t] = (uint32_t)__ballot(id[t] >= 0) & 0xFFFFu;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = r0 + 32 * h + 8 * (lane >> 4);
      there[h] = r < a.rank;
#pragma unroll
      for (int t = 0; t < C::MT; t++) {
        pv[h][t] = i32x4{0, 0, 0, 0};
        if (id[t] >= 0 && there[h]) pv[h][t] = *(const i32x4*)(a.p + (size_t)(m0 + 16 * t + (lane & 15)) * a.rank + r);
      }
    }
#pragma unroll
    for (int i = 0; i < DEPTH; i++) load(a, i);
  }
  // n: this lane's rows of b
  D3_INLINE void first(const Dense& a, int m0, const int (&n)[C::NT], int lane) {
#pragma unroll
    for (int u = 0; u < C::NT; u++) at[u] = (uint32_t)(n[u] * a.rank + 8 * (lane >> 4)) * 2;
    r0 = 0;
    ranks(a, m0, lane);
  }
  D3_INLINE void multiply(f32x4 (&acc)[C::NT][C::MT], int i, int h) {
#pragma unroll
    for (int u = 0; u < C::NT; u++) {
      i32x4 b = bv[i][h][u];
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = there[h] ? b[j] : 0;
#pragma unroll
      for (int t = 0; t < C::MT; t++) {
        // (the other rows keep their sums, also where this adapter holds infinities or NaN)
        const f32x4 with = mfma_bf16(b, pv[h][t], acc[u][t]);
        acc[u][t] = id[t] == who[i] ? with : acc[u][t];
      }
    }
  }
  D3_INLINE void add(const Dense& a, f32x4 (&acc)[C::NT][C::MT], int m0, int lane) {
    while (true) {
      while (who[0] != NONE) {
#pragma unroll
        for (int i = 0; i < DEPTH; i++) {
          multiply(acc, i, 0);
          if (two) multiply(acc, i, 1);
          load(a, i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if ((r0 += 64) >= a.rank) return;
      ranks(a, m0, lane);
    }
  }
};

// The loop over the stages is one stream of MFMA groups (NT products of one row tile each). Beside each group go the LDS reads of
// the operands that the half stage after needs, into the registers that the group has just read, and, in a stage's second
// half, its share of the copies of the stage BUFS later: with all copies at the start of a stage the waves stood in line
// to send them, and copies and products took turns (256 x 256 on 4096 x 4096 x 11008, alone: 321 us so, 285 after that step, and
// 266 once its addresses no longer spilled; 2048 x 6144 x 4096 transposed twice 114, 90, 86). A stage's one barrier stands after
// group BAR of its second half, when the reads of its own operands are long done.
template <class C, bool XT, bool WT, int END, bool LORA>
D3_INLINE void dense_tile(const Dense& a, int tm, int tn, uint8_t* smem) {
  constexpr int TM = C::TM, TN = C::TN, W = C::WAVES, BUFS = C::BUFS;
  using SX = Side<TM, XT, W>;
  using SW = Side<TN, WT, W>;
  constexpr int STAGE = SX::BYTES + SW::BYTES;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, c = lane & 15, wn = w % C::WN, wm = w / C::WN;
  constexpr int UN = END == END_SWIGLU ? TN / 2 : TN;  // columns of out to a tile
  const int m0 = tm * TM, n0 = tn * UN, stages = (a.K + 63) / 64;
  const uint32_t lds = lds_address(smem);

  // the rows of w (n) of a tile's row r, gate and up rows by turns of the waves' tiles
  auto w_row = [&](int r) {
    if constexpr (END == END_SWIGLU) {
      const int t = r / 16 % C::NT, unit = n0 + r / (16 * C::NT) * (8 * C::NT) + t % (C::NT / 2) * 16 + r % 16;
      return min(unit, a.half - 1) + (t >= C::NT / 2 ? a.half : 0);
    } else {
      return min(n0 + r, a.N - 1);
    }
  };
  SX sx;
  SW sw;
  sx.step = XT ? (uint32_t)(128 * a.ldx) : 128u;
  sw.step = WT ? (uint32_t)(128 * a.ldw) : 128u;
  sx.base = (const uint8_t*)(a.x + (XT ? m0 : m0 * a.ldx));
  sw.base = (const uint8_t*)(a.w + (WT ? n0 : END == END_SWIGLU ? 0 : n0 * a.ldw));
#pragma unroll
  for (int i = 0; i < SX::PER; i++) {
    const int r = SX::row_of(i, w, lane), col = SX::col_of(i, w, lane);
    sx.off[i] = XT ? (uint32_t)(r * a.ldx + min(col, a.M - 8 - m0)) * 2 : (uint32_t)((min(m0 + r, a.M - 1) - m0) * a.ldx + col) * 2;
  }
#pragma unroll
  for (int i = 0; i < SW::PER; i++) {
    const int r = SW::row_of(i, w, lane), col = SW::col_of(i, w, lane);
    sw.off[i] = WT ? (uint32_t)(r * a.ldw + min(col, a.N - 8 - n0)) * 2
                   : (uint32_t)((w_row(r) - (END == END_SWIGLU ? 0 : n0)) * a.ldw + col) * 2;
  }
  constexpr int PIECES = SX::PER + SW::PER;
  auto piece = [&](int i, int buf) {
    const uint32_t at = lds + buf * STAGE;
    if (i < SX::PER) copy16(at + (w * SX::PER + i) * 1024, sx.base, sx.off[i]);
    else copy16(at + SX::BYTES + (w * SW::PER + i - SX::PER) * 1024, sw.base, sw.off[i - SX::PER]);
  };
  // before stage s is copied: where it ends past K (it is the last one then), the lanes of k past K read from its k 0
  auto ready = [&](int s) {
    const int left = a.K - s * 64;
    if (left >= 64) return;
    const int l = (int)anew(lane);
#pragma unroll
    for (int i = 0; i < SX::PER; i++) {
      const int k = SX::k_of(i, w, l);
      if (k >= left) sx.off[i] -= (uint32_t)(XT ? k * a.ldx : k) * 2;
    }
#pragma unroll
    for (int i = 0; i < SW::PER; i++) {
      const int k = SW::k_of(i, w, l);
      if (k >= left) sw.off[i] -= (uint32_t)(WT ? k * a.ldw : k) * 2;
    }
  };
  // and once it has come, each lane clears what it copied of them
  auto clear = [&](int s, int buf) {
    const int left = a.K - s * 64;
    if (left >= 64) return;
    typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
    const int l = (int)anew(lane);
    const uint32_t at = lds + buf * STAGE + w * (SX::PER * 1024) + l * 16;
    const uint32_t at_w = lds + buf * STAGE + SX::BYTES + w * (SW::PER * 1024) + l * 16;
#pragma unroll
    for (int i = 0; i < SX::PER; i++)
      if (SX::k_of(i, w, l) >= left) *(lds_i32x4*)(uintptr_t)(at + i * 1024) = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < SW::PER; i++)
      if (SW::k_of(i, w, l) >= left) *(lds_i32x4*)(uintptr_t)(at_w + i * 1024) = i32x4{0, 0, 0, 0};
  };

  f32x4 acc[C::NT][C::MT];
#pragma unroll
  for (int u = 0; u < C::NT; u++)
#pragma unroll
    for (int t = 0; t < C::MT; t++) acc[u][t] = f32x4{0, 0, 0, 0};

  const int mw = m0 + wm * C::MT * 16;  // this wave's first row
  [[maybe_unused]] RowAdapters<C> adapters;
  if constexpr (LORA) adapters.begin(a, mw, lane);
  for (int s = 0; s < BUFS && s < stages; s++) {
    ready(s);
#pragma unroll
    for (int i = 0; i < PIECES; i++) piece(i, s);
    sx.base += sx.step, sw.base += sw.step;
  }
  if (stages >= BUFS) loads_but<(BUFS - 1) * PIECES>();
  else loads_but<0>();
  clear(0, 0);
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  // this wave's operands of half stage k
  const uint32_t x_at[2] = {operand_at<TM, XT>(0, lane) + (XT ? 0 : wm * C::MT * 2048), operand_at<TM, XT>(1, lane) + (XT ? 0 : wm * C::MT * 2048)};
  const uint32_t w_at[2] = {operand_at<TN, WT>(0, lane) + (WT ? 0 : wn * C::NT * 2048), operand_at<TN, WT>(1, lane) + (WT ? 0 : wn * C::NT * 2048)};
  auto x_operand = [&](uint32_t at, int t) { return operand<TM, XT>(at, XT ? wm * C::MT + t : t); };
  auto w_operand = [&](uint32_t at, int u) { return operand<TN, WT>(at, WT ? wn * C::NT + u : u); };
  i32x4 xv[C::MT], wv[2][C::NT];
  {
    const uint32_t x0 = lds + x_at[0], w0 = lds + SX::BYTES + w_at[0];
#pragma unroll
    for (int u = 0; u < C::NT; u++) wv[0][u] = w_operand(w0, u);
#pragma unroll
    for (int t = 0; t < C::MT; t++) xv[t] = x_operand(x0, t);
  }
  int buf = 0;
  // stage s; COPY: stage s + BUFS is to be copied; NEXT: there is a stage s + 1
  auto stage = [&](int s, auto copy, auto next) {
    constexpr bool COPY = decltype(copy)::value, NEXT = decltype(next)::value;
    constexpr int MT = C::MT, NT = C::NT, BAR = MT > 4 ? 1 : 0;
    const int after = buf + 1 == BUFS ? 0 : buf + 1;
    const uint32_t x1 = anew(lds + buf * STAGE + x_at[1]), w1 = anew(lds + buf * STAGE + SX::BYTES + w_at[1]);
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
      for (int u = 0; u < NT; u++) acc[u][t] = mfma_bf16(wv[0][u], xv[t], acc[u][t]);
      xv[t] = x_operand(x1, t);
#pragma unroll
      for (int u = t * NT / MT; u < (t + 1) * NT / MT; u++) wv[1][u] = w_operand(w1, u);
      __builtin_amdgcn_sched_barrier(0);
    }
    const uint32_t x0 = anew(lds + after * STAGE + x_at[0]), w0 = anew(lds + after * STAGE + SX::BYTES + w_at[0]);
    if constexpr (COPY) ready(s + BUFS);
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
      for (int u = 0; u < NT; u++) acc[u][t] = mfma_bf16(wv[1][u], xv[t], acc[u][t]);
      if constexpr (NEXT) {
        if (t == BAR) {
          // stage s + 1 has come, of every wave, and stage s is read: its place is free
          if (COPY || s + BUFS == stages) loads_but<(BUFS - 2) * PIECES>();
          else loads_but<0>();
          if constexpr (!COPY) clear(s + 1, after);
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
          for (int v = 0; v < BAR; v++) xv[v] = x_operand(x0, v);
        }
        if (t >= BAR) {
#pragma unroll
          for (int u = t == BAR ? 0 : t * NT / MT; u < (t + 1) * NT / MT; u++) wv[0][u] = w_operand(w0, u);
          xv[t] = x_operand(x0, t);
          if constexpr (COPY) {
#pragma unroll
            for (int i = (t - BAR) * PIECES / (MT - BAR); i < (t - BAR + 1) * PIECES / (MT - BAR); i++) piece(i, buf);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (COPY) sx.base += sx.step, sw.base += sw.step;
    buf = after;
  };
  int s = 0;
  for (; s + BUFS < stages; s++) stage(s, std::true_type{}, std::true_type{});
  for (; s + 1 < stages; s++) stage(s, std::false_type{}, std::true_type{});
  if constexpr (LORA) {
    int n[C::NT];
#pragma unroll
    for (int u = 0; u < C::NT; u++) n[u] = w_row((wn * C::NT + u) * 16 + c);
    adapters.first(a, mw, n, lane);
    stage(s, std::false_type{}, std::false_type{});
    adapters.add(a, acc, mw, lane);
  } else {
    stage(s, std::false_type{}, std::false_type{});
  }

#pragma unroll
  for (int t = 0; t < C::MT; t++) {
    const int m = mw + 16 * t + c;
    const bool row = m < a.M;  // (every lane goes on: store_two exchanges between them)
    if constexpr (END == END_SWIGLU) {
#pragma unroll
      for (int u = 0; u < C::NT / 2; u += 2) {
        const int n = n0 + wn * (8 * C::NT) + 16 * u;  // of two tiles' units the first
        i32x2 h[2] = {};
#pragma unroll
        for (int v = 0; v < 2 && u + v < C::NT / 2; v++) {
          const f32x4 g = acc[u + v][t], up = acc[u + v + C::NT / 2][t];
          const int at = n + 16 * v + 4 * q;
          if (a.pre && row && at < a.half) {
            *(f32x4*)(a.pre + (size_t)m * 2 * a.half + at) = g;
            *(f32x4*)(a.pre + (size_t)m * 2 * a.half + a.half + at) = up;
          }
          f32x4 s;
#pragma unroll
          for (int i = 0; i < 4; i++) s[i] = g[i] * sigmoid(g[i]) * up[i];
          h[v] = round4(s);
        }
        store_two(a.out + m * a.ldo + n, h[0], h[1], row ? (C::NT / 2 > 1 ? a.half - n : min(16, a.half - n)) : 0);
      }
    } else {
#pragma unroll
      for (int u = 0; u < C::NT; u += 2) {
        const int n = n0 + (wn * C::NT + u) * 16;
        if constexpr (END == END_ROWS) {
          store_two(a.out + m * a.ldo + n, round4(acc[u][t]), round4(acc[u + 1][t]), row ? a.N - n : 0);
        } else if constexpr (END == END_INNER) {
          const bool mine = row && (a.rows >> (m - m0) & 1);
          store_two(a.out + m * a.ldo + n, round4(acc[u][t] * a.alpha), round4(acc[u + 1][t] * a.alpha), mine ? a.N - n : 0);
        } else {
          i32x2 dg[2], du[2];
#pragma unroll
          for (int v = 0; v < 2; v++) {
            const int at = n + 16 * v + 4 * q;
            f32x4 g{0, 0, 0, 0}, up{0, 0, 0, 0};
            if (row && at < a.N) {
              g = *(const f32x4*)(a.pre + (size_t)m * 2 * a.half + at);
              up = *(const f32x4*)(a.pre + (size_t)m * 2 * a.half + a.half + at);
            }
            f32x4 g1, u1;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float s = sigmoid(g[i]), silu = g[i] * s, d = acc[u + v][t][i];
              g1[i] = d * up[i] * (s + silu * (1.0f - s));
              u1[i] = d * silu;
            }
            dg[v] = round4(g1), du[v] = round4(u1);
          }
          store_two(a.out + m * a.ldo + n, dg[0], dg[1], row ? a.N - n : 0);
          store_two(a.out + m * a.ldo + a.half + n, du[0], du[1], row ? a.N - n : 0);
        }
      }
    }
  }
}

// the tiles of a's out, tile `at` of them (END_SWIGLU: half as many columns)
template <class C, int END>
D3_INLINE bool tile_at(const Dense& a, int at, int& tm, int& tn) {
  constexpr int UN = END == END_SWIGLU ? C::TN / 2 : C::TN;
  const int nm = (a.M + C::TM - 1) / C::TM, nn = ((END == END_SWIGLU ? a.half : a.N) + UN - 1) / UN;
  if (at >= nm * nn) return false;
  place(at, nm, nn, tm, tn);
  return true;
}

// (tiles along y: a grid's x has room for 2^32 threads)
template <class C, bool WT, int END, bool LORA>
__global__ void __launch_bounds__(C::THREADS, 2) dense_tile_kernel(Dense a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::LDS];
  int tm, tn;
  if (tile_at<C, END>(a, blockIdx.y, tm, tn)) dense_tile<C, false, WT, END, LORA>(a, tm, tn, smem);
}

// Up to three products that do not need each other in one launch, the longest first: rows with a transposed w (the gradient of
// rows), or both transposed (of weights). Their tiles fill the CUs together where each alone would leave some idle at its end.
struct DenseSet {
  Dense product[3];
  int tiles[3];  // rounded up to a multiple of 8, one for each XCD
  int count, rows;  // rows: which of them is a gradient of rows
};
template <class C>
__global__ void __launch_bounds__(C::THREADS, 2) dense_set_kernel(DenseSet set) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::LDS];
  int at = blockIdx.y, i = 0, tm, tn;
  while (i < set.count - 1 && at >= set.tiles[i]) at -= set.tiles[i++];
  const Dense& a = set.product[i];
  if (!tile_at<C, END_ROWS>(a, at, tm, tn)) return;
  if (i == set.rows) dense_tile<C, false, true, END_ROWS, false>(a, tm, tn, smem);
  else dense_tile<C, true, true, END_ROWS, false>(a, tm, tn, smem);
}

}  // namespace d3
