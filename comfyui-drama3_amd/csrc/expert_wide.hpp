// Expert products with many rows to an expert: 256 weight rows against up to 320 rows (160 e4m3 rows, which are twice as
// wide) at a time, both operands of a stage in LDS, copied there without passing through registers while the
// stage before is multiplied. 8 waves, 4 over the weight rows (64 each) and 2 over the rows' 16-row tiles (in turn).
//
// One workgroup a CU, which walks its share of the (pass, column) items as one stream of stages: the copies of the next
// item begin during the last stages of this. The rows, which other columns' workgroups read too, are copied a stage ahead;
// the weights come from HBM and are copied by halves of a stage (a step), three (bf16: four) ahead, so that there are always
// some on their way: with whole stages, one ahead, a stage of bf16 took 4200 clocks, of which the products take 2200.
//
// Bound by what comes from HBM and the memory-side cache (each XCD reads the rows of its experts for itself), the 7 us until
// a workgroup's first products and the epilogues (2 us an item) beside it. 4096 rows, top-8 of 128 experts, first bank (FFN 768)
// with SwiGLU: bf16 228 us, 0.97 GB read past the L2s and 50 MB written at 4.5 TB/s (12% less with the products left out; the
// matrix units work 51% of the time); e2m1 rows on e2m1 weights 80 us, 0.28 GB read and 50 MB written at 4.1 TB/s (29%; 35%).
// An e4m3 row takes two products a step (ragged.hpp), and its passes of 160 rows read the weights twice as often: 215 us,
// products before all (93 without them), 150 us on the second bank (124).
#pragma once
#include "expert_stream.hpp"

#include <algorithm>

namespace d3 {

constexpr int WX_N = 256, WX_THREADS = 512;
template <class F> constexpr int wx_tiles() { return 2560 / F::ROW; }  // of 16 rows a pass

// 4 bytes per lane from base + off (the lane's own) into LDS at lds + 4 * lane: dma16's rules (wide_tile.hpp)
D3_INLINE void dma4(uint32_t lds, const void* base, uint32_t off) {
  const uint64_t at = (uint64_t)base;
  const uint64_t sbase = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32;
  uint64_t from;
  asm volatile("s_mov_b64 %0, %3\n\tglobal_load_lds_dword %2, %0"
               : "=&s"(from)
               : "{m0}"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(sbase)
               : "memory");
}

// dma16; ONCE: nontemporal, for weights that no other workgroup reads (whole lines: what two copies take halves of would come
// from HBM twice)
template <bool ONCE>
D3_INLINE void dma16_weights(uint32_t lds, const void* base, uint32_t off) {
  if constexpr (!ONCE) {
    dma16(lds, base, off);
  } else {
    const uint64_t at = (uint64_t)base;
    const uint64_t sbase = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32;
    uint64_t from;
    asm volatile("s_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0 nt"
                 : "=&s"(from)
                 : "{m0}"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(sbase)
                 : "memory");
  }
}

// all but the N last of this wave's loads have come
template <int N>
D3_INLINE void wait_loads() {
  static_assert(N < 64);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// the place in LDS of piece j (16 bytes) of row r of a stage: 16 lanes that read one (s, q) of 16 rows, and the mixed
// groups of lanes that a 16-byte read takes together, meet 16 different groups of banks
template <class F>
D3_INLINE int wx_slot(int r, int j) {
  if constexpr (F::ROW != 128) return j ^ (r & 15);
  return (F::SCALED ? (j >> 1) | ((j & 1) << 2) : j) ^ ((r >> 1) & 7);
}
// the piece in place t of row r
template <class F>
D3_INLINE int wx_piece(int r, int t) {
  if constexpr (F::ROW != 128) return t ^ (r & 15);
  const int p = t ^ ((r >> 1) & 7);
  return F::SCALED ? ((p & 3) << 1) | (p >> 2) : p;
}// the same of bf16 weights by the step, 64 bytes a row: piece q of row r of 16
D3_INLINE int wx_step_slot(int r, int q) { return q ^ ((4 - (r >> 2)) & 3); }

// The passes go by what they cost: those of most tiles first (three classes of them), so that the items of a turn take
// about as long as each other. How many passes of class `k` an expert's rows have.
constexpr int WX_CLASSES = 3;
template <class F>
D3_INLINE int class_passes(int rows, int k) {
  const int tiles = 20 * wt_tiles(rows, wx_tiles<F>()) / wx_tiles<F>();
  return k == (tiles > 14 ? 0 : tiles > 7 ? 1 : 2) ? wt_passes(rows, wx_tiles<F>()) : 0;
}

// The passes of 64 items at once, one a lane: pass `at` (each lane's own) of the groups' passes in wx_tiles tiles or
// fewer, an expert's passes as long as each other but for the last.
template <class F>
D3_INLINE Pass wide_passes(const ExpertProduct& a, int at) {
  const int lane = threadIdx.x & 63;
  Pass mine{0, 0, 0};
  constexpr int AT_ONCE = 4;  // times 64 groups on their way together
  for (int k = 0; k < WX_CLASSES; k++) {
    for (int g0 = 0; g0 < a.n_groups; g0 += 64 * AT_ONCE) {
      int expert[AT_ONCE], first[AT_ONCE], rows[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++) read_group(a, g0 + 64 * i + lane, expert[i], first[i], rows[i]);
#pragma unroll
      for (int i = 0; i < AT_ONCE; i++) {
        if (g0 + 64 * i >= a.n_groups) break;
        const int np = class_passes<F>(rows[i], k), incl = wave_scan_i32(np), all = __builtin_amdgcn_readlane(incl, 63);
        if (__ballot(at >= 0 && at < all)) {
          int l = 0;  // the first lane whose sum is past `at`
#pragma unroll
          for (int d = 32; d > 0; d >>= 1)
            if (__shfl(incl, l + d - 1) <= at) l += d;
          l = min(l, 63);
          const int before = __shfl(incl - np, l), n = __shfl(rows[i], l), e = __shfl(expert[i], l), f = __shfl(first[i], l);
          if (at >= 0 && at < all) {
            const int step = 16 * wt_tiles(n, wx_tiles<F>()), from = (at - before) * step;
            mine = Pass{e, f + from, min(step, n - from)};
          }
        }
        at -= all;  // (below zero once found)
      }
    }
  }
  return mine;
}

// how many passes there are
template <class F>
D3_INLINE int count_passes(const ExpertProduct& a) {
  int n = 0;
#pragma unroll 4
  for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
    int expert, first, rows;
    read_group(a, g0 + (threadIdx.x & 63), expert, first, rows);
    n += wt_passes(rows, wx_tiles<F>());
  }
  return wave_sum_i32(n);
}

// A row's 16 results of two neighbouring tiles (of `tiles` that there are), lane (q, c) holding 4 of each, as two 16-byte
// stores a row and tile instead of four of 8: the odd q's of the first tile change places with the even ones of the second,
// so that a lane holds 8 in a row of one tile. The whole wave calls, also for rows that are not stored.
D3_INLINE void store_pair(uint16_t* row, i32x2 v0, i32x2 v1, bool stored, int tiles) {
  const int q = (threadIdx.x & 63) >> 4;
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v0[0], (uint32_t)v1[0], false, false);
  const auto b = __builtin_amdgcn_permlane16_swap((uint32_t)v0[1], (uint32_t)v1[1], false, false);
  if (stored && (q & 1) < tiles)
    *(i32x4*)(row + 16 * (q & 1) + 8 * (q >> 1)) = i32x4{(int)a[0], (int)b[0], (int)a[1], (int)b[1]};
}

template <class F, bool SWIGLU, bool OUT_BF16, bool ONCE>
__global__ void __launch_bounds__(WX_THREADS, 2) expert_wide_kernel(ExpertProduct a, int columns) {
  constexpr int TILES = wx_tiles<F>(), ROWS = 16 * TILES, STEP = WX_N * 64, STAGE = ROWS * F::ROW;
  constexpr int PER = 1024 / F::ROW, LANES = 64 / PER;  // rows of a 1 KB copy, lanes to a row of it
  constexpr int COPIES = ROWS / PER / 8;                // of the rows, per wave
  constexpr int SCOPIES = F::SCALED ? (ROWS + 255) / 256 : 0;  // of the rows' scale words, per wave
  // LDS: RING steps' weights, two stages' rows, and of microscaled ones the rows' scales of two stages and the weights' scale
  // words of two pairs of stages (tile, lane): all of a CU's 160 KB (e4m3: 156)
  constexpr int RING = F::SCALED ? 4 : 5, XSCALE = 2048 * SCOPIES, WSCALE = F::SCALED ? 16 * 256 : 0;
  constexpr int AT_ROWS = RING * STEP, AT_XSCALE = AT_ROWS + 2 * STAGE, AT_WSCALE = AT_XSCALE + 2 * XSCALE;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[AT_WSCALE + 2 * WSCALE];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, c = lane & 15, wn = w & 3, wm = w >> 2;
  const int S = a.stages, bank_tiles = a.N / 16, half = bank_tiles / 2;
  const uint32_t lds0 = lds_address(smem);
  // A step of bf16 weights is half lines of memory. LINES: a half of a stage is both steps of two of a wave's four tiles
  // instead of one step of all, which reads the rows' operands twice from LDS.
  constexpr bool LINES = ONCE && !F::SCALED;
  // a lane's place in a copy of 1 KB: a step of a tile; LINES, 8 rows of a stage of it
  uint32_t woff[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int r = LINES ? 8 * k + (lane >> 3) : lane >> 2;
    woff[k] = F::SCALED ? 16 * lane
                        : (uint32_t)(r * S * 128 + 16 * (LINES ? wx_piece<F>(r, lane & 7) : wx_step_slot(r, lane & 3)));
  }

  // The workgroup's items. Two passes that follow each other (mostly one expert's) go to one XCD with all columns of each, so
  // that their weights and rows are read once into its L2; its items are dealt to its workgroups in turn. Those that are left
  // for the last turn, if they are at most half as many as the workgroups, are shared by two each: such an item has every
  // other tile twice in LDS and stores one (its products cost as much as before, its weights from HBM half).
  const int xcd = blockIdx.x & 7, turn0 = blockIdx.x >> 3, per_turn = gridDim.x >> 3;
  const int passes = count_passes<F>(a), mine = passes / 16 * 2 + min(max(passes % 16 - 2 * xcd, 0), 2);
  const int items = mine * columns, turns = items / per_turn, rest = items % per_turn;
  const bool shared = 2 * rest <= per_turn;
  struct Item {
    int expert, first, rows, column, part;  // part: 0 or 1 of a shared item, -1 of a whole one
  };
  // item k of this workgroup, an index into the XCD's items (-1: none), with its part; the pass and column of an item
  auto item_at = [&](int k, int& part) __attribute__((always_inline)) {
    part = k == turns && shared ? turn0 & 1 : -1;
    if (k < turns) return turn0 + k * per_turn;
    const int at = shared ? turn0 >> 1 : turn0;
    return k == turns && at < rest ? turns * per_turn + at : -1;
  };
  auto place = [&](int i, int& at, int& column) __attribute__((always_inline)) {
    const int chunk = i / (2 * columns), in = i % (2 * columns), size = min(2, mine - 2 * chunk);
    at = 16 * chunk + 2 * xcd + in % size;
    column = in / size;
  };
  Pass table;  // of 64 items: lane l that of item 64 n + l
  int taken = 0;
  auto next_item = [&](Item& t) __attribute__((always_inline)) {
    t.rows = 0;
    const int i = item_at(taken, t.part);
    if (i < 0) return;
    int at, column;
    if ((taken & 63) == 0) {
      int part;
      const int own = item_at(taken + lane, part);
      place(max(own, 0), at, column);
      table = wide_passes<F>(a, at);
    }
    place(i, at, t.column);
    const int l = taken & 63;
    t.expert = __builtin_amdgcn_readlane(table.expert, l), t.first = __builtin_amdgcn_readlane(table.first, l);
    t.rows = __builtin_amdgcn_readlane(table.rows, l);
    taken++;
  };
  // where an item's weights lie: wave w copies the tiles in places 2 w and 2 w + 1, and their scales; LINES, one of the first
  // two and one of the last two of wave w / 2's tiles
  struct Weights {
    const uint8_t *src[2], *word[2];
  };
  auto find_weights = [&](const Item& t, Weights& at) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      // the expert's tile in the place of the 16 (a place past the expert's last tile repeats that)
      const int slot = !LINES ? 2 * w + i : 4 * (w >> 1) + 2 * i + (w & 1), part = max(t.part, 0);
      const int unit = t.part < 0 ? 2 * (slot >> 2) + (slot & 1) : 4 * part + (slot >> 2);
      const int tile = SWIGLU ? min(8 * t.column + unit, half - 1) + ((slot >> 1) & 1) * half
                              : min(16 * t.column + (t.part < 0 ? slot : 8 * part + (slot >> 1)), bank_tiles - 1);
      const size_t n = (size_t)t.expert * bank_tiles + tile;
      at.src[i] = a.w + n * ((size_t)S * 2048);
      at.word[i] = a.w_scale + n * (64 * (size_t)mx_lane_scales(S));
    }
  };
  // and its rows
  uint32_t xoff[COPIES], soff[2];  // the copies w, w + 8, .. and their scale words w, w + 8 of 64
  // the pairs whose rows those are: lane l that of copy l / PER, l % PER, and of scale words l / 32, l % 32
  int64_t pair_x = 0, pair_s = 0;
  auto find_pairs = [&](const Item& t) __attribute__((always_inline)) {
    pair_x = pair_at(a, t.first + min(PER * (w + 8 * (lane / PER)) + lane % PER, t.rows - 1));
    if constexpr (F::SCALED) pair_s = pair_at(a, t.first + min(32 * (w + 8 * (lane >> 5)) + (lane & 31), t.rows - 1));
  };
  auto find_rows = [&]() __attribute__((always_inline)) {
    const int row_x = pair_row(a, pair_x), row_s = F::SCALED ? pair_row(a, pair_s) : 0;
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
      const int r = PER * (w + 8 * i) + lane / LANES;
      xoff[i] = (uint32_t)__shfl(row_x, PER * i + lane / LANES) * (uint32_t)(S * F::ROW) + 16 * wx_piece<F>(r, lane % LANES);
    }
    if constexpr (F::SCALED) {
#pragma unroll
      for (int i = 0; i < 2; i++) soff[i] = (uint32_t)__shfl(row_s, 32 * i + (lane >> 1)) * (uint32_t)(8 * S) + 4 * (lane & 1);
    }
  };
  Item cur, nxt;
  Weights at, at_next;
  // the copies of half s of stage st (from the next item where this one ends) to buffer `to`: step s of every
  // tile; LINES, both steps of the first or the last two tiles of every wave
  auto load_weights = [&](int st, int s, int to) __attribute__((always_inline)) {
    const bool here = st < S || nxt.rows == 0;
    st = st < S ? st : nxt.rows ? st - S : S - 1;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int t = LINES ? s : i;
      dma16_weights<ONCE>(lds0 + to * STEP + (2 * w + i) * 1024, (here ? at.src[t] : at_next.src[t]) +
                          (size_t)st * F::A_STAGE + (LINES ? 0 : s * F::A_STEP), woff[i]);
    }
  };
  auto load_rows = [&](int k, int st, int buf) __attribute__((always_inline)) {
    dma16(lds0 + AT_ROWS + buf * STAGE + (uint32_t)(w + 8 * k) * 1024, a.x + (size_t)st * F::ROW, xoff[k]);
  };
  // (all waves as many copies, so that each knows how many of its loads are on their way: past the rows, the last one again)
  auto load_scales = [&](int st, int buf, int pair, const Weights& of) __attribute__((always_inline)) {
    if constexpr (F::SCALED) {
#pragma unroll
      for (int k = 0; k < SCOPIES; k++) dma4(lds0 + AT_XSCALE + buf * XSCALE + 256 * (w + 8 * k), a.x_scale + 8 * st, soff[k]);
#pragma unroll
      for (int k = 0; k < 2; k++)
        dma4(lds0 + AT_WSCALE + pair * WSCALE + 256 * (2 * w + k), of.word[k] + 4 * (st >> 1), lane * mx_lane_scales(S));
    }
  };

  next_item(cur);
  if (cur.rows == 0) return;
  find_pairs(cur);
  find_weights(cur, at);
  nxt.rows = 0;
  // the buffers of the step's weights, of the stage's rows and of the pair of stages' scale words
  int ring = 0, buf = 0, pair = 1;
#pragma unroll
  for (int h = 0; h < RING - 1; h++) load_weights(h >> 1, h & 1, h);
  find_rows();
#pragma unroll
  for (int k = 0; k < COPIES; k++)
    if (PER * (w + 8 * k) < cur.rows) load_rows(k, 0, 0);
  load_scales(0, 0, 0, at);
  next_item(nxt);
  if (nxt.rows) find_weights(nxt, at_next);

  // An item's products. A wave's tiles: rows 16 (wm + 2 j) .., j < NT (tiles past the pass's run on what lies there and
  // store nothing)
  auto run = [&]<int NT>() __attribute__((always_inline)) {
    f32x4 acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int n = 0; n < 4; n++) acc[j][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // (the copies of the first stage: the start's, or the last stage's before, which waited for them)
    for (int st = 0; st < S; st++, buf ^= 1) {
      if ((st & 1) == 0) pair ^= 1;
      const uint8_t* xlane[2][F::PIECES];  // this lane's operands of the wave's first tile
#pragma unroll
      for (int s = 0; s < 2; s++)
#pragma unroll
        for (int k = 0; k < F::PIECES; k++)
          xlane[s][k] = smem + AT_ROWS + buf * STAGE + (16 * wm + c) * F::ROW + 16 * wx_slot<F>(c, F::b_piece(s, q, k));
      const uint8_t* slane = smem + AT_XSCALE + buf * XSCALE + 8 * (16 * wm + c) + 2 * q;
      i32x4 wa[4], b[4][F::PIECES];
      uint32_t sw[4] = {0, 0, 0, 0}, sb[4] = {0, 0, 0, 0};
      auto read_w = [&](int s) __attribute__((always_inline)) {
        // step s of the wave's four tiles; LINES: steps 0 and 1 of two of them
        const uint8_t* from = smem + ring * STEP + 4 * wn * 1024;
#pragma unroll
        for (int n = 0; n < 4; n++)
          wa[n] = *(const i32x4*)(F::SCALED ? from + 1024 * n + 16 * lane
                                  : LINES   ? from + 2048 * (n >> 1) + 128 * c + 16 * wx_slot<F>(c, 4 * (n & 1) + q)
                                            : from + 1024 * n + 64 * c + 16 * wx_step_slot(c, q));
      };
      // operand i: tile i % NT, step i / NT; LINES: step i & 1 of tile i / 2, all again for the other weights
      auto read_x = [&](int i) __attribute__((always_inline)) {
        const int step = LINES ? i & 1 : i / NT, j = LINES ? i % (2 * NT) / 2 : i % NT;
#pragma unroll
        for (int k = 0; k < F::PIECES; k++) b[i & 3][k] = *(const i32x4*)(xlane[step][k] + j * 32 * F::ROW);
        if constexpr (F::SCALED) sb[i & 3] = *(const uint16_t*)(slane + (i % NT) * 256);
      };
      read_w(0);
      read_x(0);
      if constexpr (F::SCALED) {
#pragma unroll
        for (int n = 0; n < 4; n++)
          sw[n] = *(const uint32_t*)(smem + AT_WSCALE + pair * WSCALE + 256 * (4 * wn + n) + 4 * lane) >> (16 * (st & 1));
      }
      read_x(1);
      // The next stage's rows, of this item or the next, go out between the products: those that this item's rows need
      // without a branch (after the last item they copy what is there once more). Whatever branches stands before the
      // products, which the compiler would move past it, with all their operands waiting in registers.
      const bool last = st + 1 == S;
      if (nxt.rows && st + 2 == S) find_pairs(nxt);  // for the next stage
      if (last && nxt.rows) find_rows();
      const int st_next = last ? 0 : st + 1;
      constexpr int MINE = (32 * NT / PER + 7) / 8;
      if (last) {
#pragma unroll
        for (int k = MINE; k < COPIES; k++)
          if (PER * (w + 8 * k) < nxt.rows) load_rows(k, 0, buf ^ 1);
      }
      load_scales(st_next, buf ^ 1, st_next & 1 ? pair : pair ^ 1, last && nxt.rows ? at_next : at);
      auto products = [&]<int s>() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const int i = (LINES ? 2 : 1) * (s * NT + j);
          if constexpr (!LINES) {
            if (i + 2 < 2 * NT) read_x(i + 2);
            __builtin_amdgcn_sched_barrier(0);  // the reads first
#pragma unroll
            for (int n = 0; n < 4; n++)
              acc[j][n] = step_product<F, s, s>(wa[n], b[i & 3], acc[j][n], sw[n], sb[i & 3]);
          } else {
            if (i + 2 < 4 * NT) read_x(i + 2), read_x(i + 3);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
              for (int n = 0; n < 2; n++)
                acc[j][2 * s + n] = step_product<F, 0, 0>(wa[2 * n + k], b[(i + k) & 3], acc[j][2 * s + n], 0, 0);
          }
          if (s == 0) {
            constexpr int SPREAD = (MINE + NT - 1) / NT;
#pragma unroll
            for (int k = SPREAD * j; k < SPREAD * (j + 1) && k < MINE; k++) load_rows(k, st_next, buf ^ 1);
          }
        }
      };
      // A step's weights go to the buffer of the step before. They come in the order in which they were asked for: with the
      // next stage's rows, those of its steps that went out before have come too.
      auto next_step = [&](int s) __attribute__((always_inline)) {  // RING - 1 steps on
        load_weights(st + (s + RING - 1) / 2, (s + RING - 1) & 1, ring ? ring - 1 : RING - 1);
      };
      auto turn = [&]() __attribute__((always_inline)) { ring = ring + 1 < RING ? ring + 1 : 0; };
      products.template operator()<0>();
      next_step(0);
      if constexpr (RING == 4) wait_loads<2 + SCOPIES + 2 + MINE + 2>();  // all but the step after the next and this step's copies
      __syncthreads();
      turn();
      read_w(1);
      next_step(1);
      products.template operator()<1>();
      wait_loads<4>();  // all but this stage's two steps of weights
      __syncthreads();
      turn();
    }

    // lane l holds weight rows 4 q .. + 3 of its tiles of the pass's row 16 (wm + 2 j) + c
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int r = 16 * (wm + 2 * j) + c;
      const size_t p = (size_t)(cur.first + r);
      const bool whole = cur.part < 0, stored = r < cur.rows;
      if constexpr (SWIGLU) {
        const int unit = 8 * cur.column + (whole ? 2 * wn : 4 * cur.part + wn);  // the wave's two, or one
        store_pair((uint16_t*)a.out + p * (a.N / 2) + 16 * unit, swiglu_4(acc[j][0], acc[j][2]),
                   swiglu_4(acc[j][1], acc[j][3]), stored, min(half - unit, whole ? 2 : 1));
      } else {
        const int tile0 = 16 * cur.column + (whole ? 4 * wn : 8 * cur.part + 2 * wn);
        if constexpr (OUT_BF16) {
#pragma unroll
          for (int n = 0; n < 4; n += 2) {
            const int tile = tile0 + (whole ? n : n >> 1);
            store_pair((uint16_t*)a.out + p * a.N + 16 * tile, bf16_4(acc[j][n]), bf16_4(acc[j][n + 1]), stored,
                       min(bank_tiles - tile, whole ? 2 : 1));
          }
        } else {
#pragma unroll
          for (int n = 0; n < 4; n++) {
            const int tile = tile0 + (whole ? n : n >> 1);
            if (stored && tile < bank_tiles && (whole || !(n & 1)))
              *(f32x4*)((float*)a.out + p * a.N + 16 * tile + 4 * q) = acc[j][n];
          }
        }
      }
    }
  };
  wait_loads<0>();
  __syncthreads();
  while (true) {
    const int most = ((cur.rows + 15) / 16 + 1) / 2;  // tiles of a wave
    if constexpr (TILES > 10) {
      if (most > 9) run.template operator()<10>();
      else if (most > 8) run.template operator()<9>();
      else if (most > 7) run.template operator()<8>();
      else if (most > 6) run.template operator()<7>();
      else if (most > 5) run.template operator()<6>();
    }
    if (TILES <= 10 || most <= 5) {
      if (most > 4) run.template operator()<5>();
      else if (most > 3) run.template operator()<4>();
      else if (most > 2) run.template operator()<3>();
      else run.template operator()<2>();
    }
    if (nxt.rows == 0) break;
    cur = nxt;
    at = at_next;
    next_item(nxt);
    if (nxt.rows) find_weights(nxt, at_next);
  }
  wait_loads<0>();  // no copy is on its way to an LDS that is another workgroup's
}

// compute units of the current device
inline int device_cus() {
  int device = 0, n = 0;
  if (hipGetDevice(&device) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1)
    return 256;
  return n;
}

template <class F, bool ONCE>
void launch_wide_of(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  const int columns = (a.N + WX_N - 1) / WX_N, passes = most_passes(a.pairs, a.n_groups, 16 * wx_tiles<F>());
  const int64_t items = (int64_t)2 * passes * columns;  // shared ones twice
  const int cus = std::max(device_cus() & ~7, 8);       // as many for each XCD
  const dim3 grid((unsigned)std::min<int64_t>((items + 7) & ~7, cus)), block(WX_THREADS);
  if (swiglu) hipLaunchKernelGGL((expert_wide_kernel<F, true, true, ONCE>), grid, block, 0, s, a, columns);
  else if (out_bf16) hipLaunchKernelGGL((expert_wide_kernel<F, false, true, ONCE>), grid, block, 0, s, a, columns);
  else hipLaunchKernelGGL((expert_wide_kernel<F, false, false, ONCE>), grid, block, 0, s, a, columns);
}

// Where an expert's rows are one pass, mostly, its weights are read once: nontemporal. us without / with (first bank,
// 128 experts): bf16 512 rows 191 / 182, 1024 197 / 193, 4096 247 / 242 and on the second bank 183 / 175; e4m3 1024 rows
// 84 / 83; e2m1 4096 rows the same; bf16 rows of 13 passes an expert 193 / 201.
template <class F>
void launch_wide(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  if ((int64_t)a.pairs <= (int64_t)16 * wx_tiles<F>() * a.n_groups) launch_wide_of<F, true>(a, swiglu, out_bf16, s);
  else launch_wide_of<F, false>(a, swiglu, out_bf16, s);
}

// Whether a grouped product runs in wide passes: by the rows an expert has on average. (The copies to LDS take 32-bit
// offsets.)
template <class F>
bool wide_fits(const ExpertProduct& a) {
  return (int64_t)a.pairs >= (int64_t)32 * a.n_groups && a.stages >= 2 && (int64_t)a.x_rows * a.stages * F::ROW <= UINT32_MAX;
}

// Wide passes, or streamed ones of 32 rows, or of 16, by the rows an expert has on average. Top-8 of 128 experts (FFN 768),
// us with 16 / 32 / wide: first bank, e4m3 rows, 150 rows (9 to an expert) 43 / 56 / 71, 256 rows 57 / 59 / 72 (Zipf 59 / 64
// / 83), 300 rows 69 / 61 / 70, 400 rows 77 / 65 / 69, 500 rows 89 / 74 / 72, 1024 rows 139 / 114 / 83; second bank 16 to an
// expert 31 / 36 / 43 (few stages: a 32-row pass has less to stream than it takes to set up), 25 to an expert 40 / 41 / 42,
// 44 to an expert 60 streamed, 47 wide; bf16 first bank 16 to an expert 196 / 164 / 190, 25: 238 / 174 / 192; second bank 16:
// 100 / 89 / 102.
template <class F>
void launch_grouped(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  if (wide_fits<F>(a)) return launch_wide<F>(a, swiglu, out_bf16, s);
  const bool small = a.stages <= F::SEG / 2;  // half the LDS holds the rows
  const bool two = (int64_t)a.pairs >= (int64_t)(F::SCALED && small ? 24 : 12) * a.n_groups;
  if (two && small) launch_stream<F, 2, F::SEG / 2>(a, swiglu, out_bf16, s);
  else if (two) launch_stream<F, 2, F::SEG>(a, swiglu, out_bf16, s);
  else if (small) launch_stream<F, 1, F::SEG / 2>(a, swiglu, out_bf16, s);
  else launch_stream<F, 1, F::SEG>(a, swiglu, out_bf16, s);
}

}  // namespace d3
