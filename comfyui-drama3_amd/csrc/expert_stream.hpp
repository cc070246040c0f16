// Expert products with few rows to an expert: a decode line's experts (gemv: a pass is one pair) and a short prompt's
// groups in passes of up to 16 MT rows. HBM-bound: the experts' weights go by once, so what counts is how many bytes are
// on their way. A wave streams its tiles of 16 weight rows from memory straight into the MFMA operands, DEPTH stages
// ahead; nothing but the accumulators is shared along K, so there is no barrier in the loop. The pass's rows lie whole in
// LDS (SEG stages at a time), read by all waves.
//
// Short prompts run near what memory gives: 77 rows of top-8 of 256 experts (FFN 512) on e4m3 rows, first bank, 46 us (260 MB of
// weights at 5.6 TB/s; 44 with one product a step, ragged.hpp); of 128 experts, bf16, second bank, 65 us (400 MB at 6.1). A
// line's experts are few bytes, and its time a launch and one round trip of loads: 8 pairs of the first bank 6.0 us (e2m1
// weights, 13 MB, e4m3 rows; 4.4 with one product a step) and 11 us (bf16, 50 MB at 4.6 TB/s).
#pragma once
#include "ragged.hpp"

namespace d3 {

constexpr int ST_THREADS = 256;

// LDS bytes of a row of the stages, and where its 16-byte piece j lies: pieces of 256 bytes swapped by the row, so that
// 16 rows' pieces j are in 16 different groups of banks
template <class F, int SEG> constexpr int st_pitch() { return (SEG * F::ROW + 255) / 256 * 256; }
// waves of a SIMD that LDS has room for, up to two
template <class F, int SEG, int MT> constexpr int st_waves() { return 16 * MT * st_pitch<F, SEG>() > 80000 ? 1 : 2; }
D3_INLINE int st_piece(int r, int j) { return 16 * (j ^ (r & 15)); }

// 16 bytes of weights; ONCE: nontemporal, for weights that hardly another workgroup reads. (Only where a load takes whole lines:
// with the hint, a line that two loads take halves of comes from HBM twice, 10.6 -> 14.8 us for a bf16 decode line.)
template <bool ONCE>
D3_INLINE i32x4 weights_16(const uint8_t* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load((const i32x4*)p);
  else return *(const i32x4*)p;
}

// bf16 rows are loaded by whole lines in the grouped products: the first load of a stage takes rows 0 - 7 of the tile, lane (q, c)
// piece 4 (c >> 3) + q of row c & 7, the second rows 8 - 15, piece 4 (1 - (c >> 3)) + q of row 8 + (c & 7). (A decode line is
// latency, and takes the operands as they are: 10.8 us, 12.1 by lines.)
template <class F, bool LINES>
D3_INLINE size_t st_base(size_t tile, int stages, int lane) {
  if constexpr (!LINES) return F::a_base(tile, stages, lane);
  else return (tile * 16 + (lane & 7)) * ((size_t)stages * F::A_STAGE) + 64 * ((lane >> 3) & 1) + 16 * (lane >> 4);
}
// from a stage's first load to its second
template <class F, bool LINES>
D3_INLINE int64_t st_second(int stages, int lane) {
  if constexpr (!LINES) return F::A_STEP;
  else return (int64_t)8 * stages * F::A_STAGE + (lane & 8 ? -64 : 64);
}
// what the lines' loads brought, as the operands of the stage's steps: of 16 lanes the first 8 of the first load and the last
// 8 of the second are step 0's, in their places, the others step 1's, 8 lanes on
D3_INLINE void steps_of_lines(i32x4& first, i32x4& second) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int a = first[i], b = second[i], turned = __builtin_amdgcn_update_dpp(0, a, 0x128, 0xF, 0x3, false);  // row_ror 8
    first[i] = __builtin_amdgcn_update_dpp(a, b, 0xE4, 0xF, 0xC, false);
    second[i] = __builtin_amdgcn_update_dpp(turned, b, 0x128, 0xF, 0xC, false);
  }
}

// NT tiles of weight rows a wave; SWIGLU with NT 2: a gate tile and its up tile, with NT 1 (gemv): those of two
// neighbouring waves
template <class F, bool GEMV, bool SWIGLU, bool OUT_BF16, int NT, int MT, int DEPTH, int SEG, bool ONCE>
__global__ void __launch_bounds__(ST_THREADS, (st_waves<F, SEG, MT>()))
    expert_stream_kernel(ExpertProduct a, int columns, int per) {
  constexpr bool LINES = !GEMV && !F::SCALED;
  constexpr int ROWS = GEMV ? 1 : 16 * MT, PITCH = st_pitch<F, SEG>(), SPITCH = 8 * SEG + 4;
  __shared__ __attribute__((aligned(1024))) uint8_t xs[ROWS * PITCH];
  __shared__ __attribute__((aligned(16))) uint8_t ss[F::SCALED ? ROWS * SPITCH : 16];
  __shared__ f32x4 other[2][GEMV && SWIGLU ? ST_THREADS / 64 : 1][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, c = lane & 15;
  const int at = blockIdx.y, column0 = blockIdx.x * per;
  Pass pass;
  int my_row;  // lane r: row r of the pass
  if constexpr (GEMV) {
    const int64_t id = a.ids[at];
    const bool valid = id >= 0 && id < a.E;
    pass = Pass{valid ? (int)id : -1, at, 1};
    my_row = at / a.per_row;
  } else {
    pass = find_pass(a, ROWS, at);
    if (pass.rows == 0) return;
    my_row = pair_row(a, pair_at(a, pass.first + min(lane, pass.rows - 1)));
  }
  const int tiles = a.N / 16, half = tiles / 2;
  for (int column = column0; column < (GEMV ? column0 + 1 : min(column0 + per, columns)); column++) {
  // the wave's tiles of an expert's N / 16
  int tile[NT];
  bool mine;  // the wave has a tile of its own (a column past the last one repeats it and stores nothing)
  if constexpr (SWIGLU && NT == 1) {
    const int unit = column * 2 + (w >> 1);
    mine = unit < half;
    tile[0] = min(unit, half - 1) + (w & 1) * half;
  } else if constexpr (SWIGLU) {
    const int unit = column * 4 + w;
    mine = unit < half;
    tile[0] = min(unit, half - 1);
    tile[NT - 1] = tile[0] + half;
  } else {
    const int first = (column * 4 + w) * NT;
    mine = first < tiles;
#pragma unroll
    for (int n = 0; n < NT; n++) tile[n] = min(first + n, tiles - 1);
  }
  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int m = 0; m < MT; m++) acc[n][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  if (!GEMV || pass.expert >= 0) {
    const int S = a.stages;
    const uint8_t* wp[NT];
    const uint8_t* sp[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const size_t t = (size_t)pass.expert * tiles + tile[n];
      wp[n] = a.w + st_base<F, LINES>(t, S, lane);
      sp[n] = F::SCALED ? a.w_scale + (t * 64 + lane) * mx_lane_scales(S) : nullptr;
    }
    const size_t row_bytes = (size_t)S * F::ROW;
    const int64_t second = st_second<F, LINES>(S, lane);
    for (int s0 = 0; s0 < S; s0 += SEG) {
      const int n_st = min(SEG, S - s0);
      i32x4 buf[DEPTH][NT][2];
      uint32_t sa[NT][F::SCALED ? SEG / 2 : 1];
      auto load = [&](int d, int st) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int s = 0; s < 2; s++)
            buf[d][n][s] = weights_16<ONCE>(wp[n] + (size_t)(s0 + st) * F::A_STAGE + (s ? second : 0));
      };
#pragma unroll
      for (int d = 0; d < DEPTH; d++) load(d, min(d, n_st - 1));
      if constexpr (F::SCALED) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < SEG / 2; i++) sa[n][i] = ((const uint32_t*)(sp[n] + 2 * s0))[min(i, (n_st - 1) / 2)];
      }
      // the rows: wave w copies rows w, w + 4, .. to LDS, lane by lane into place (once for all columns if they fit)
      if (S > SEG || column == column0) {
      if (s0 || column != column0) __syncthreads();
      for (int r = w; r < pass.rows; r += ST_THREADS / 64) {
        const uint8_t* src = a.x + (size_t)__builtin_amdgcn_readlane(my_row, r) * row_bytes + (size_t)s0 * F::ROW;
        for (int j = 0; j < n_st * F::ROW / 16; j += 64) {
          const int slot = j + lane, piece = (slot & ~15) | ((slot ^ r) & 15);
          if (16 * piece < n_st * F::ROW) dma16(lds_address(xs + r * PITCH + 16 * j), src, 16 * piece);
        }
      }
      if constexpr (F::SCALED) {
#pragma unroll
        for (int r0 = 0; r0 < ROWS; r0 += ST_THREADS / 16) {
          const int r = r0 + (tid >> 4), row = GEMV ? my_row : __shfl(my_row, r);  // (all lanes: each may be read)
          if (r < pass.rows && (tid & 15) < 2 * n_st)
            *(uint32_t*)(ss + r * SPITCH + 4 * (tid & 15)) =
                ((const uint32_t*)(a.x_scale + ((size_t)row * S + s0) * 8))[tid & 15];
        }
      }
      dma_wait();
      __syncthreads();
      }
      // lane's rows of the MT tiles (a row past the pass's repeats its last: its results are not stored)
      int xr[MT];
#pragma unroll
      for (int m = 0; m < MT; m++) xr[m] = min(16 * m + c, pass.rows - 1);
      auto products = [&]<int ODD>(int d, int st, uint32_t (&sw)[NT]) __attribute__((always_inline)) {
        uint32_t sb[MT];
        i32x4 b[MT][2][F::PIECES];
#pragma unroll
        for (int m = 0; m < MT; m++) {
          sb[m] = F::SCALED ? *(const uint16_t*)(ss + xr[m] * SPITCH + 8 * st + 2 * q) : 0u;
#pragma unroll
          for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < F::PIECES; i++) {
              const int j = st * (F::ROW / 16) + F::b_piece(s, q, i);
              b[m][s][i] = *(const i32x4*)(xs + xr[m] * PITCH + 16 * (j & ~15) + st_piece(xr[m], j & 15));
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          i32x4 w[2] = {buf[d][n][0], buf[d][n][1]};
          if constexpr (LINES) steps_of_lines(w[0], w[1]);
#pragma unroll
          for (int m = 0; m < MT; m++) {
            acc[n][m] = step_product<F, 2 * ODD, 0>(w[0], b[m][0], acc[n][m], sw[n], sb[m]);
            acc[n][m] = step_product<F, 2 * ODD + 1, 1>(w[1], b[m][1], acc[n][m], sw[n], sb[m]);
          }
        }
      };
      auto run = [&](int d, int st) __attribute__((always_inline)) {
        uint32_t sw[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) sw[n] = F::SCALED ? sa[n][st / 2] : 0u;
        if (st & 1) products.template operator()<1>(d, st, sw);
        else products.template operator()<0>(d, st, sw);
      };
      if constexpr (F::SCALED) {  // at most SEG / DEPTH turns, unrolled: the scale words stay in registers
#pragma unroll
        for (int base = 0; base < SEG; base += DEPTH) {
          if (base + DEPTH < n_st) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
              run(d, base + d);
              load(d, min(base + d + DEPTH, n_st - 1));
            }
          } else if (base < n_st) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++)
              if (base + d < n_st) run(d, base + d);
          }
        }
      } else {
        int st = 0;
        for (; st + DEPTH < n_st; st += DEPTH) {
#pragma unroll
          for (int d = 0; d < DEPTH; d++) {
            run(d, st + d);
            load(d, min(st + d + DEPTH, n_st - 1));
          }
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
          if (st + d < n_st) run(d, st + d);
      }
    }
  }

  // lane (q, c) holds weight rows 16 tile + 4 q .. + 3 of the pass's row 16 m + c
  if constexpr (GEMV && SWIGLU) {
    if (c == 0) other[column & 1][w][q] = acc[0][0];
    __syncthreads();
    if (mine && !(w & 1) && c == 0) {
      *(i32x2*)((uint16_t*)a.out + (size_t)pass.first * (a.N / 2) + tile[0] * 16 + 4 * q) =
          swiglu_4(acc[0][0], other[column & 1][w | 1][q]);
    }
  } else if (mine) {
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const int r = 16 * m + c;
      if (r >= pass.rows) continue;
      const size_t p = (size_t)(pass.first + r);
      if constexpr (SWIGLU) {
        *(i32x2*)((uint16_t*)a.out + p * (a.N / 2) + tile[0] * 16 + 4 * q) = swiglu_4(acc[0][m], acc[NT - 1][m]);
      } else {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          if ((column * 4 + w) * NT + n >= tiles) continue;
          const size_t o = p * a.N + tile[n] * 16 + 4 * q;
          if constexpr (OUT_BF16) *(i32x2*)((uint16_t*)a.out + o) = bf16_4(acc[n][m]);
          else *(f32x4*)((float*)a.out + o) = acc[n][m];
        }
      }
    }
  }
  }
}

// workgroups to a pass
template <bool GEMV, bool SWIGLU, int NT>
int st_columns(int N) {
  const int per = SWIGLU && NT == 1 ? 4 : SWIGLU ? 8 : 4 * NT;  // tiles of a workgroup
  return (N / 16 + per - 1) / per;
}

// (the passes along y: HIP launches nothing, without an error, where a dimension of the grid has 2^32 threads)
template <class F, bool GEMV, bool SWIGLU, bool OUT_BF16, int NT, int MT, int DEPTH, int SEG, bool ONCE>
void launch_stream_of(const ExpertProduct& a, int passes, int per, hipStream_t s) {
  const int columns = st_columns<GEMV, SWIGLU, NT>(a.N);
  per = per < columns ? per : columns;
  hipLaunchKernelGGL((expert_stream_kernel<F, GEMV, SWIGLU, OUT_BF16, NT, MT, DEPTH, SEG, ONCE>),
                     dim3((unsigned)((columns + per - 1) / per), (unsigned)passes), dim3(ST_THREADS), 0, s, a, columns, per);
}

template <class F, bool GEMV, int MT, int DEPTH, int SEG, bool ONCE>
void launch_stream_out(const ExpertProduct& a, bool swiglu, bool out_bf16, int passes, int per, hipStream_t s) {
  constexpr int NT = GEMV ? 1 : 2;
  if (swiglu) launch_stream_of<F, GEMV, true, true, NT, MT, DEPTH, SEG, ONCE>(a, passes, per, s);
  else if (out_bf16) launch_stream_of<F, GEMV, false, true, NT, MT, DEPTH, SEG, ONCE>(a, passes, per, s);
  else launch_stream_of<F, GEMV, false, false, NT, MT, DEPTH, SEG, ONCE>(a, passes, per, s);
}

// DEPTH for microscaled rows of fewer than 8 stages: no more loads than there are stages
template <class F>
void launch_gemv(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  // Few pairs, of which hardly two meet in an expert, read its weights once. Of 128 experts (e4m3 rows), us without / with:
  // first bank 8 pairs 6.7 / 6.0, 16 9.4 / 8.9, 32 12.6 / 12.5, 64 20.0 / 21.4, 128 37.5 / 40.2; second bank 16 pairs 5.5 /
  // 5.0, 32 7.8 / 8.3; 40 of 256 experts, second bank: 6.1 / 5.0.
  if constexpr (F::SCALED) {
    if ((int64_t)6 * a.pairs <= a.E) {
      if (a.stages >= 8) launch_stream_out<F, true, 1, 8, F::SEG, true>(a, swiglu, out_bf16, a.pairs, 1, s);
      else if (a.stages >= 4) launch_stream_out<F, true, 1, 4, F::SEG, true>(a, swiglu, out_bf16, a.pairs, 1, s);
      else if (a.stages == 3) launch_stream_out<F, true, 1, 3, F::SEG, true>(a, swiglu, out_bf16, a.pairs, 1, s);
      else launch_stream_out<F, true, 1, 2, F::SEG, true>(a, swiglu, out_bf16, a.pairs, 1, s);
      return;
    }
  }
  launch_stream_out<F, true, 1, 8, F::SEG, false>(a, swiglu, out_bf16, a.pairs, 1, s);
}

template <class F, int MT, int SEG>
void launch_stream(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  const int passes = most_passes(a.pairs, a.n_groups, 16 * MT);
  // A workgroup finds its pass and copies the rows before it streams anything: with few stages to a column it takes some
  // columns in turn. Second bank of 128 experts (2048 x 768, e4m3), 256 rows: 32 us with two, 38 with one; first bank
  // (8 stages): 58 with one, 59 with two.
  const int per = F::SCALED && a.stages < 6 ? 6 / a.stages : 1;
  // Up to 16 rows an expert its weights go by in one pass, mostly: nontemporal, e2m1 where a column is long (first bank, e4m3
  // rows, 77 of 256 experts 53.8 -> 48.6 us, 100 of 128 42.8 -> 40.0; second bank, 256 rows, Zipf: 32.0 -> 33.5, so not
  // there), bf16 (16 rows of 128 experts 103 -> 91 and 51 -> 43 us, 77 rows on the second bank 79 -> 68), and up to 32 rows
  // bf16's long columns (256 rows of 128 experts 184 -> 163 us, Zipf 186 either way; second bank, 700 rows of 256 experts 134
  // -> 141).
  constexpr bool LONG = SEG == F::SEG, ONCE = F::SCALED ? MT == 1 && LONG : MT == 1 || LONG;
  if constexpr (F::SCALED && SEG < F::SEG) {  // (second bank, 256 rows of 128 experts: 31.3 -> 29.2 us)
    if (a.stages == 3) return launch_stream_out<F, false, MT, 3, SEG, ONCE>(a, swiglu, out_bf16, passes, per, s);
    if (a.stages < 3) return launch_stream_out<F, false, MT, 2, SEG, ONCE>(a, swiglu, out_bf16, passes, per, s);
  }
  launch_stream_out<F, false, MT, 4, SEG, ONCE>(a, swiglu, out_bf16, passes, per, s);
}

}  // namespace d3
