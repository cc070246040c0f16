// Expert products with many rows to an expert: 256 weight rows against up to 256 rows (128 e4m3 rows, which are twice as
// wide) a workgroup, both operands of a stage in LDS, copied there without passing through registers while the
// stage before is multiplied. 8 waves, 4 over the weight rows (64 each) and 2 over the rows' 16-row tiles (in turn).
#pragma once
#include "expert_stream.hpp"

namespace d3 {

constexpr int WX_N = 256, WX_THREADS = 512;
template <class F> constexpr int wx_tiles() { return 2048 / F::ROW; }  // of 16 rows a pass

// Pass `at` of the groups' passes in wx_tiles tiles or fewer, an expert's passes as long as each other but for the last
template <class F>
D3_INLINE Pass find_wide_pass(const ExpertProduct& a, int at) {
  const int lane = threadIdx.x & 63;
  for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
    int expert, first, rows;
    read_group(a, g0 + lane, expert, first, rows);
    const int np = wt_passes(rows, wx_tiles<F>());
    int before;
    const int l = find_lane(np, at, before);
    if (l >= 0) {
      const int all = __builtin_amdgcn_readlane(rows, l), step = 16 * wt_tiles(all, wx_tiles<F>()), from = (at - before) * step;
      return Pass{__builtin_amdgcn_readlane(expert, l), __builtin_amdgcn_readlane(first, l) + from, min(step, all - from)};
    }
    at -= before;
  }
  return Pass{0, 0, 0};
}

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

// the place in LDS of piece j (16 bytes) of row r of a stage, and where it comes from (the same swap)
template <class F>
D3_INLINE int wx_slot(int r, int j) {
  return F::ROW == 128 ? wt_slot(r, j) : j ^ (r & 15);
}

template <class F, bool SWIGLU, bool OUT_BF16>
__global__ void __launch_bounds__(WX_THREADS, 2) expert_wide_kernel(ExpertProduct a, int columns) {
  constexpr int TILES = wx_tiles<F>(), ROWS = 16 * TILES, A_BYTES = WX_N * 128, STAGE = A_BYTES + ROWS * F::ROW;
  constexpr int PER = 1024 / F::ROW;            // rows of a 1 KB copy
  constexpr int COPIES = ROWS / PER / 8;        // of the rows, per wave
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t xscale[2][F::SCALED ? 8 * ROWS : 16];
  int at, column;
  wt_place(blockIdx.x, columns, at, column);
  const Pass pass = find_wide_pass<F>(a, at);
  if (pass.rows == 0) return;
  const int expert = __builtin_amdgcn_readfirstlane(pass.expert), first = __builtin_amdgcn_readfirstlane(pass.first),
            rows = __builtin_amdgcn_readfirstlane(pass.rows), tiles = (rows + 15) / 16;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, c = lane & 15, wn = w & 3, wm = w >> 2;
  const int S = a.stages, bank_tiles = a.N / 16, half = bank_tiles / 2;
  const uint32_t lds0 = lds_address(smem);
  // the expert's tile in place `slot` of the workgroup's 16 (a place past the expert's last repeats that)
  auto tile_of = [&](int slot) __attribute__((always_inline)) {
    if constexpr (SWIGLU) return min(8 * column + 2 * (slot >> 2) + (slot & 1), half - 1) + ((slot >> 1) & 1) * half;
    else return min(16 * column + slot, bank_tiles - 1);
  };

  // weights: wave w copies the places 2 w and 2 w + 1, two copies of 1 KB each
  const uint8_t* src[2];
#pragma unroll
  for (int i = 0; i < 2; i++)
    src[i] = a.w + ((size_t)expert * bank_tiles + tile_of(2 * w + i)) * ((size_t)S * 2048);
  uint32_t woff[2];  // from a stage's start, for the two copies
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = 8 * i + (lane >> 3);
    woff[i] = F::SCALED ? 1024 * i + 16 * lane : (uint32_t)(r * S * 128 + 16 * wt_slot(r, lane & 7));
  }
  // rows: wave w takes the copies w, w + 8, ..
  uint32_t xoff[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; i++) {
    const int r = PER * (w + 8 * i) + lane / (64 / PER);
    xoff[i] = (uint32_t)row_at(a, first + min(r, rows - 1)) * (uint32_t)(S * F::ROW) +
              16 * wx_slot<F>(r, lane % (64 / PER));
  }
  uint32_t soff = 0;  // scales: lane's word of the stage's 8 bytes a row
  if constexpr (F::SCALED) soff = (uint32_t)row_at(a, first + min(tid >> 1, rows - 1)) * (uint32_t)(8 * S) + 4 * (tid & 1);
  auto load = [&](int st, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++)
        dma16(lds0 + buf * STAGE + (2 * w + i) * 2048 + 1024 * j, src[i] + (size_t)st * F::A_STAGE, woff[j]);
#pragma unroll
    for (int i = 0; i < COPIES; i++)
      if (PER * (w + 8 * i) < 16 * tiles)
        dma16(lds0 + buf * STAGE + A_BYTES + (uint32_t)(w + 8 * i) * 1024, a.x + (size_t)st * F::ROW, xoff[i]);
    if constexpr (F::SCALED)
      if (w * 32 < 16 * tiles) dma4(lds_address(xscale[buf]) + 256 * w, a.x_scale + 8 * st, soff);
  };
  const uint32_t* wscale[4];  // a lane's scale words of its wave's tiles
#pragma unroll
  for (int n = 0; n < 4; n++)
    wscale[n] = (const uint32_t*)(a.w_scale + (((size_t)expert * bank_tiles + tile_of(4 * wn + n)) * 64 + lane) *
                                                  mx_lane_scales(S));
  load(0, 0);

  // A wave's tiles: rows 16 (wm + 2 j) .., j < NT (tiles past the pass's run on what lies there and store nothing)
  auto run = [&]<int NT>() __attribute__((always_inline)) {
    f32x4 acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int n = 0; n < 4; n++) acc[j][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t sw[4] = {0, 0, 0, 0}, sw_next[4] = {0, 0, 0, 0};
    if constexpr (F::SCALED) {
#pragma unroll
      for (int n = 0; n < 4; n++) sw_next[n] = wscale[n][0];
    }
    dma_wait();
    __syncthreads();
    for (int st = 0; st < S; st++) {
      const int buf = st & 1;
      const uint8_t* wbase = smem + buf * STAGE;
      const uint8_t* xbase = wbase + A_BYTES;
      i32x4 wa[4][2], b[2][2][F::PIECES];
      uint32_t sb[2];
      auto read_x = [&](int j) __attribute__((always_inline)) {
        const int r = 16 * (wm + 2 * j) + c;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
          for (int i = 0; i < F::PIECES; i++)
            b[j & 1][s][i] = *(const i32x4*)(xbase + r * F::ROW + 16 * wx_slot<F>(c, F::b_piece(s, q, i)));
        sb[j & 1] = F::SCALED ? *(const uint16_t*)(xscale[buf] + 8 * r + 2 * q) : 0u;
      };
#pragma unroll
      for (int n = 0; n < 4; n++)
#pragma unroll
        for (int s = 0; s < 2; s++)
          wa[n][s] = *(const i32x4*)(wbase + (4 * wn + n) * 2048 +
                                     (F::SCALED ? 1024 * s + 16 * lane : c * 128 + 16 * wt_slot(c, 2 * q + s)));
      read_x(0);
      if constexpr (F::SCALED) {
#pragma unroll
        for (int n = 0; n < 4; n++) {
          if (st & 1) sw[n] >>= 16;
          else sw[n] = sw_next[n];
        }
      }
      if (st + 1 < S) {
        load(st + 1, buf ^ 1);
        if constexpr (F::SCALED) {
          if (st & 1) {
#pragma unroll
            for (int n = 0; n < 4; n++) sw_next[n] = wscale[n][(st + 1) / 2];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        if (j + 1 < NT) read_x(j + 1);
        __builtin_amdgcn_sched_barrier(0);  // the reads first
#pragma unroll
        for (int n = 0; n < 4; n++) acc[j][n] = step_product<F, !OUT_BF16, 0, 0>(wa[n][0], b[j & 1][0], acc[j][n], sw[n], sb[j & 1]);
#pragma unroll
        for (int n = 0; n < 4; n++) acc[j][n] = step_product<F, !OUT_BF16, 1, 1>(wa[n][1], b[j & 1][1], acc[j][n], sw[n], sb[j & 1]);
      }
      dma_wait();
      __syncthreads();
    }

    // lane l holds weight rows 4 q .. + 3 of its tiles of the pass's row 16 (wm + 2 j) + c
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int r = 16 * (wm + 2 * j) + c;
      if (r >= rows) continue;
      const size_t p = (size_t)(first + r);
      if constexpr (SWIGLU) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const int unit = 8 * column + 2 * wn + n;
          if (unit >= half) continue;
          const f32x4 g = acc[j][n], u = acc[j][n + 2];
          *(i32x2*)((uint16_t*)a.out + p * (a.N / 2) + 16 * unit + 4 * q) =
              i32x2{(int)(swiglu_bf16(g[0], u[0]) | swiglu_bf16(g[1], u[1]) << 16),
                    (int)(swiglu_bf16(g[2], u[2]) | swiglu_bf16(g[3], u[3]) << 16)};
        }
      } else {
#pragma unroll
        for (int n = 0; n < 4; n++) {
          const int tile = 16 * column + 4 * wn + n;
          if (tile >= bank_tiles) continue;
          const f32x4 v = acc[j][n];
          const size_t o = p * a.N + 16 * tile + 4 * q;
          if constexpr (OUT_BF16)
            *(i32x2*)((uint16_t*)a.out + o) = i32x2{(int)(f32_to_bf16(v[0]) | f32_to_bf16(v[1]) << 16),
                                                    (int)(f32_to_bf16(v[2]) | f32_to_bf16(v[3]) << 16)};
          else
            *(f32x4*)((float*)a.out + o) = v;
        }
      }
    }
  };
  if constexpr (TILES > 8) {
    if (tiles > 12) return run.template operator()<8>();
    if (tiles > 8) return run.template operator()<6>();
  }
  if (tiles > 4) run.template operator()<4>();
  else run.template operator()<2>();
}

template <class F>
void launch_wide(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  const int columns = (a.N + WX_N - 1) / WX_N, passes = most_passes(a.pairs, a.n_groups, 16 * wx_tiles<F>());
  const dim3 grid((unsigned)(wt_places(passes) * columns)), block(WX_THREADS);
  if (swiglu) hipLaunchKernelGGL((expert_wide_kernel<F, true, true>), grid, block, 0, s, a, columns);
  else if (out_bf16) hipLaunchKernelGGL((expert_wide_kernel<F, false, true>), grid, block, 0, s, a, columns);
  else hipLaunchKernelGGL((expert_wide_kernel<F, false, false>), grid, block, 0, s, a, columns);
}

// Whether a grouped product runs in wide passes: by the rows an expert has on average. (The copies to LDS take 32-bit
// offsets.)
template <class F>
bool wide_fits(const ExpertProduct& a) {
  return (int64_t)a.pairs >= (int64_t)32 * a.n_groups && (int64_t)a.x_rows * a.stages * F::ROW <= UINT32_MAX;
}

template <class F>
void launch_grouped(const ExpertProduct& a, bool swiglu, bool out_bf16, hipStream_t s) {
  if (wide_fits<F>(a)) launch_wide<F>(a, swiglu, out_bf16, s);
  else launch_stream<F, 1>(a, swiglu, out_bf16, s);
}

}  // namespace d3
