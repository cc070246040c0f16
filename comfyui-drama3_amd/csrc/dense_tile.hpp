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

namespace d3 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// what becomes of a tile
enum DenseEnd {
  END_ROWS,     // out bf16
  END_SWIGLU,   // w holds `half` gate rows, then as many up rows: out [M, half] = SiLU(gate) * up, and pre where it is given
  END_DSWIGLU,  // the sums are the gradient of SiLU(gate) * up: out [M, 2 half] = the gradients of gate and up (from pre)
  END_PART,     // float32 sums of a part of K, part `split` of the workspace
};

struct Dense {
  const uint16_t* x;
  const uint16_t* w;
  int64_t ldx, ldw, ldo;  // elements from row to row as they are stored (ldo: of out)
  uint16_t* out;
  float* pre;     // [M, 2 half]: gate and up before the activation
  float* parts;   // [splits, M, N]
  int M, N, K, half;
  int splits, split_stages;  // K in `splits` runs of split_stages stages
  // adapters: out += p(m) . b[ids[m]](n), p [M, rank] of this row's own adapter; rows with an id outside have none
  const uint16_t* p;
  const uint16_t* b;  // [adapters, N, rank]
  const int64_t* ids;
  int rank, adapters;
};

// 16 bytes a lane from base + off into LDS at lds + 16 * lane (dma16's rules), base a scalar already
D3_INLINE void copy16(uint32_t lds, const uint8_t* base, uint32_t off) { dma16(lds, base, off); }

template <int N>
D3_INLINE void loads_but() {
  static_assert(N < 64);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

D3_INLINE f32x4 mfma_bf16(i32x4 a, i32x4 b, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

// which turn row k's chunks take
D3_INLINE int t_turn(int k) { return (k & 3) | ((k >> 3) & 1) << 2; }

// One operand's side of a tile: ROWS m or n. T: transposed. W waves copy it, PER kilobytes each.
template <int ROWS, bool T, int W>
struct Side {
  static constexpr int BYTES = ROWS * 128, PER = BYTES / 1024 / W;
  static_assert(BYTES % (1024 * W) == 0 && ROWS % 128 == 0);
  const uint8_t* base;  // of the next stage to copy
  uint32_t step;        // bytes from stage to stage
  uint32_t off[PER];
  // the row (T: the k) and the first column of the 16 bytes that this lane copies in copy i
  static D3_INLINE int row_of(int i, int w, int lane) { return T ? ((w * PER + i) * 1024 + lane * 16) / (2 * ROWS) : (w * PER + i) * 8 + (lane >> 3); }
  static D3_INLINE int col_of(int i, int w, int lane) {
    const int r = row_of(i, w, lane);
    if constexpr (!T) return 8 * ((lane & 7) ^ ((r >> 1) & 7));
    const int at = (lane * 16) % (2 * ROWS), c = at >> 5;  // (a copy holds whole rows of k, or half a row of 256 m)
    return 16 * ((c & ~7) | ((c & 7) ^ t_turn(r))) + ((at >> 4) & 1) * 8;
  }
};

// MFMA operand `t` (16 m or n) of k-step s: lane (q, c) holds k = 8 q .. 8 q + 7 of row c
template <int ROWS, bool T>
D3_INLINE i32x4 operand(uint32_t side, int t, int s, int lane) {
  typedef __attribute__((address_space(3))) const i32x4 lds_i32x4;
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  const int q = lane >> 4, c = lane & 15;
  if constexpr (!T) {
    const uint32_t at = side + (t * 16 + c) * 128 + ((4 * s + q) ^ ((c >> 1) & 7)) * 16;
    return *(lds_i32x4*)(uintptr_t)at;
  } else {
    const int k = 8 * q + (c >> 2);
    const uint32_t at = (side + k * (2 * ROWS) + (t & ~7) * 32 + (t_turn(k) ^ (t & 7)) * 32 + (c & 3) * 8) + s * 64 * ROWS;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)at);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)(at + 8 * ROWS));
    return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// SiLU(g) u and its gradients from the float32 sums. The sigmoid's exponential and reciprocal are the hardware's
// (within 2^-21 + |g| 2^-23 of the value in all), which the rounding of the results to bf16 hides. At -g past 88 the exponential
// is infinite and the sigmoid 0, as in the limit.
D3_INLINE float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// Four results of a row, rounded to bf16 and stored; n a multiple of 4, N of 8.
D3_INLINE i32x2 round4(f32x4 v) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(i32x2, __builtin_convertvector(v, bf16x4));
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

template <int WM_, int WN_, int MT_, int NT_, int BUFS_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, BUFS = BUFS_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int TM = 16 * WM * MT, TN = 16 * WN * NT;
};

// A row of m's adapters: the products of p and b, added for one adapter after the other that the wave's rows name.
template <class C>
D3_INLINE void add_adapters(const Dense& a, f32x4 (&acc)[C::NT][C::MT], int m0, const int (&n)[C::NT], int lane) {
  const int q = lane >> 4, c = lane & 15;
  int id[C::MT];        // -1: none
  uint32_t open[C::MT];  // rows whose adapter is still to come
#pragma unroll
  for (int t = 0; t < C::MT; t++) {
    const int m = m0 + 16 * t + c;
    const int64_t named = m < a.M ? a.ids[m] : -1;
    id[t] = named >= 0 && named < a.adapters ? (int)named : -1;
    open[t] = (uint32_t)__ballot(id[t] >= 0) & 0xFFFFu;
  }
  while (true) {
    int now = -1;
#pragma unroll
    for (int t = C::MT - 1; t >= 0; t--)
      if (open[t]) now = __builtin_amdgcn_readlane(id[t], __ffs((int)open[t]) - 1);
    if (now < 0) break;
    const uint16_t* b = a.b + (size_t)now * a.N * a.rank;
    uint32_t some = 0;  // which of the wave's tiles have rows of it
#pragma unroll
    for (int t = 0; t < C::MT; t++) {
      const uint32_t rows = (uint32_t)__ballot(id[t] == now) & 0xFFFFu;
      open[t] &= ~rows;
      some |= (rows ? 1u : 0u) << t;
    }
    for (int r0 = 0; r0 < a.rank; r0 += 32) {
      const int r = r0 + 8 * q;
      i32x4 bv[C::NT];
#pragma unroll
      for (int u = 0; u < C::NT; u++) {
        bv[u] = i32x4{0, 0, 0, 0};
        if (r < a.rank) bv[u] = *(const i32x4*)(b + (size_t)n[u] * a.rank + r);
      }
#pragma unroll
      for (int t = 0; t < C::MT; t++) {
        if (!(some >> t & 1)) continue;
        const bool mine = id[t] == now;
        i32x4 pv{0, 0, 0, 0};
        if (mine && r < a.rank) pv = *(const i32x4*)(a.p + (size_t)(m0 + 16 * t + c) * a.rank + r);
#pragma unroll
        for (int u = 0; u < C::NT; u++) {
          // (the other rows keep their sums, also where this adapter holds infinities or NaN)
          const f32x4 with = mfma_bf16(bv[u], pv, acc[u][t]);
          acc[u][t] = mine ? with : acc[u][t];
        }
      }
    }
  }
}

template <class C, bool XT, bool WT, int END, bool LORA>
__global__ void __launch_bounds__(C::THREADS, 2) dense_tile_kernel(Dense one, Dense two, int tiles_one) {
  constexpr int TM = C::TM, TN = C::TN, W = C::WAVES, BUFS = C::BUFS;
  using SX = Side<TM, XT, W>;
  using SW = Side<TN, WT, W>;
  constexpr int STAGE = SX::BYTES + SW::BYTES;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[BUFS * STAGE];
  const bool second = (int)blockIdx.x >= tiles_one;
  const Dense& a = second ? two : one;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, c = lane & 15, wn = w % C::WN, wm = w / C::WN;
  constexpr int UN = END == END_SWIGLU ? TN / 2 : TN;  // columns of out to a tile
  const int columns = END == END_SWIGLU ? a.half : a.N, nm = (a.M + TM - 1) / TM, nn = (columns + UN - 1) / UN;
  int tm, tn;
  place((int)blockIdx.x - (second ? tiles_one : 0), nm, nn, tm, tn);
  const int m0 = tm * TM, n0 = tn * UN, split = blockIdx.y;
  const int all_stages = (a.K + 63) / 64, first = split * a.split_stages, stages = min(a.split_stages, all_stages - first);
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
  sx.base = (const uint8_t*)(a.x + (XT ? (int64_t)first * 64 * a.ldx + m0 : m0 * a.ldx + (int64_t)first * 64));
  sw.base = (const uint8_t*)(a.w + (WT ? (int64_t)first * 64 * a.ldw + n0 : (END == END_SWIGLU ? 0 : n0 * a.ldw) + (int64_t)first * 64));
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
  // how many k of stage s there are, and its copies: the lanes of k past K read from k 0 of the stage instead (cleared later)
  auto copy = [&](int s) {
    const int left = a.K - (first + s) * 64;
    const uint32_t at = lds + (s % BUFS) * STAGE + w * (SX::PER * 1024);
    const uint32_t at_w = lds + (s % BUFS) * STAGE + SX::BYTES + w * (SW::PER * 1024);
    if (left >= 64) {
#pragma unroll
      for (int i = 0; i < SX::PER; i++) copy16(at + i * 1024, sx.base, sx.off[i]);
#pragma unroll
      for (int i = 0; i < SW::PER; i++) copy16(at_w + i * 1024, sw.base, sw.off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < SX::PER; i++) {
        const int k = XT ? SX::row_of(i, w, lane) : SX::col_of(i, w, lane);
        copy16(at + i * 1024, sx.base, k < left ? sx.off[i] : sx.off[i] - (uint32_t)(XT ? k * a.ldx : k) * 2);
      }
#pragma unroll
      for (int i = 0; i < SW::PER; i++) {
        const int k = WT ? SW::row_of(i, w, lane) : SW::col_of(i, w, lane);
        copy16(at_w + i * 1024, sw.base, k < left ? sw.off[i] : sw.off[i] - (uint32_t)(WT ? k * a.ldw : k) * 2);
      }
    }
    sx.base += sx.step;
    sw.base += sw.step;
  };
  auto clear = [&](int s) {
    const int left = a.K - (first + s) * 64;
    if (left >= 64) return;
    typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
    const uint32_t at = lds + (s % BUFS) * STAGE + w * (SX::PER * 1024) + lane * 16;
    const uint32_t at_w = lds + (s % BUFS) * STAGE + SX::BYTES + w * (SW::PER * 1024) + lane * 16;
#pragma unroll
    for (int i = 0; i < SX::PER; i++)
      if ((XT ? SX::row_of(i, w, lane) : SX::col_of(i, w, lane)) >= left) *(lds_i32x4*)(uintptr_t)(at + i * 1024) = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < SW::PER; i++)
      if ((WT ? SW::row_of(i, w, lane) : SW::col_of(i, w, lane)) >= left) *(lds_i32x4*)(uintptr_t)(at_w + i * 1024) = i32x4{0, 0, 0, 0};
  };

  f32x4 acc[C::NT][C::MT];
#pragma unroll
  for (int u = 0; u < C::NT; u++)
#pragma unroll
    for (int t = 0; t < C::MT; t++) acc[u][t] = f32x4{0, 0, 0, 0};

#pragma unroll
  for (int s = 0; s < BUFS - 1; s++)
    if (s < stages) copy(s);
  for (int s = 0; s < stages; s++) {
    // stage s has come, of every wave, and stage s - 1 is read: its place may be overwritten
    if (s + BUFS - 2 < stages) loads_but<(BUFS - 2) * (SX::PER + SW::PER)>();
    else loads_but<0>();
    clear(s);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + BUFS - 1 < stages) copy(s + BUFS - 1);
    const uint32_t at = lds + (s % BUFS) * STAGE;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      i32x4 xv[C::MT], wv[C::NT];
#pragma unroll
      for (int u = 0; u < C::NT; u++) wv[u] = operand<TN, WT>(at + SX::BYTES, wn * C::NT + u, k, lane);
#pragma unroll
      for (int t = 0; t < C::MT; t++) xv[t] = operand<TM, XT>(at, wm * C::MT + t, k, lane);
#pragma unroll
      for (int t = 0; t < C::MT; t++)
#pragma unroll
        for (int u = 0; u < C::NT; u++) acc[u][t] = mfma_bf16(wv[u], xv[t], acc[u][t]);
    }
  }

  const int mw = m0 + wm * C::MT * 16;  // this wave's first row
  if constexpr (LORA) {
    int n[C::NT];
#pragma unroll
    for (int u = 0; u < C::NT; u++) n[u] = w_row((wn * C::NT + u) * 16 + c);
    add_adapters<C>(a, acc, mw, n, lane);
  }
#pragma unroll
  for (int t = 0; t < C::MT; t++) {
    const int m = mw + 16 * t + c;
    if (m >= a.M) continue;
    if constexpr (END == END_SWIGLU) {
#pragma unroll
      for (int u = 0; u < C::NT / 2; u++) {
        const int n = n0 + wn * (8 * C::NT) + 16 * u + 4 * q;
        if (n >= a.half) continue;
        const f32x4 g = acc[u][t], up = acc[u + C::NT / 2][t];
        if (a.pre) {
          *(f32x4*)(a.pre + (size_t)m * 2 * a.half + n) = g;
          *(f32x4*)(a.pre + (size_t)m * 2 * a.half + a.half + n) = up;
        }
        f32x4 h;
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = g[i] * sigmoid(g[i]) * up[i];
        *(i32x2*)(a.out + m * a.ldo + n) = round4(h);
      }
    } else {
#pragma unroll
      for (int u = 0; u < C::NT; u++) {
        const int n = n0 + (wn * C::NT + u) * 16 + 4 * q;
        if (n >= a.N) continue;
        if constexpr (END == END_ROWS) {
          *(i32x2*)(a.out + m * a.ldo + n) = round4(acc[u][t]);
        } else if constexpr (END == END_PART) {
          *(f32x4*)(a.parts + ((size_t)split * a.M + m) * a.N + n) = acc[u][t];
        } else {
          const f32x4 g = *(const f32x4*)(a.pre + (size_t)m * 2 * a.half + n), up = *(const f32x4*)(a.pre + (size_t)m * 2 * a.half + a.half + n);
          f32x4 dg, du;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float s = sigmoid(g[i]), silu = g[i] * s;
            dg[i] = acc[u][t][i] * up[i] * (s + silu * (1.0f - s));
            du[i] = acc[u][t][i] * silu;
          }
          *(i32x2*)(a.out + m * a.ldo + n) = round4(dg);
          *(i32x2*)(a.out + m * a.ldo + a.half + n) = round4(du);
        }
      }
    }
  }
}

}  // namespace d3
