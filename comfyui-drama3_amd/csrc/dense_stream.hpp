// Dense products of up to 16 rows: the weights stream from memory straight into the matrix instruction's operands. A workgroup
// takes 16 weight rows (with SwiGLU 8 units, gate and up rows by turns); its 8 waves each take an eighth of K and the sums
// are added in LDS, so that even the narrow weights of one shared expert (64 workgroups) come in one round of loads a
// wave. One row through a shared expert of FFN 512: 4.9 us and 3.4 us on the GPU.
#pragma once
#include "dense_tile.hpp"

namespace d3 {

constexpr int ST_WAVES = 8, ST_THREADS = 64 * ST_WAVES;

// this wave's part of the sums of 16 rows (lane's own at w) with RT times 16 others (lane's own at x[t]), AT_ONCE stages of 64 k whose
// loads it sends together
template <int RT, int AT_ONCE>
D3_INLINE void stream_sums(const uint16_t* w, const uint16_t* const (&x)[RT], int K, int wave, f32x4 (&acc)[RT]) {
  const int q = (threadIdx.x & 63) >> 4, stages = (K + 63) / 64;
  const int first = stages * wave / ST_WAVES, last = stages * (wave + 1) / ST_WAVES;
#pragma unroll
  for (int t = 0; t < RT; t++) acc[t] = f32x4{0, 0, 0, 0};
  int s = first;
  for (; s + AT_ONCE <= last && (s + AT_ONCE) * 64 <= K; s += AT_ONCE) {
    i32x4 wv[2 * AT_ONCE], xv[RT][2 * AT_ONCE];
#pragma unroll
    for (int i = 0; i < 2 * AT_ONCE; i++) wv[i] = *(const i32x4*)(w + s * 64 + i * 32 + 8 * q);
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int i = 0; i < 2 * AT_ONCE; i++) xv[t][i] = *(const i32x4*)(x[t] + s * 64 + i * 32 + 8 * q);
    __builtin_amdgcn_sched_barrier(0);  // (all loads on their way before the first product)
#pragma unroll
    for (int i = 0; i < 2 * AT_ONCE; i++)
#pragma unroll
      for (int t = 0; t < RT; t++) acc[t] = mfma_bf16(wv[i], xv[t][i], acc[t]);
  }
  for (; s < last; s++) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int k = s * 64 + i * 32 + 8 * q;
      i32x4 wv{0, 0, 0, 0}, xv[RT];
      if (k < K) wv = *(const i32x4*)(w + k);
#pragma unroll
      for (int t = 0; t < RT; t++) {
        xv[t] = i32x4{0, 0, 0, 0};
        if (k < K) xv[t] = *(const i32x4*)(x[t] + k);
      }
#pragma unroll
      for (int t = 0; t < RT; t++) acc[t] = mfma_bf16(wv, xv[t], acc[t]);
    }
  }
}

// the waves' parts added up, in their order: wave t < RT returns tile t's
template <int RT>
D3_INLINE f32x4 join_waves(f32x4 (*part)[RT][64], const f32x4 (&acc)[RT], int wave) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int t = 0; t < RT; t++) part[wave][t][lane] = acc[t];
  __syncthreads();
  f32x4 sum{0, 0, 0, 0};
  if (wave < RT) {
    sum = part[0][wave][lane];
#pragma unroll
    for (int i = 1; i < ST_WAVES; i++) sum += part[i][wave][lane];
  }
  return sum;
}

template <int END, bool LORA>
__global__ void __launch_bounds__(ST_THREADS) dense_stream_kernel(Dense a) {
  __shared__ f32x4 part[ST_WAVES][1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.x * (END == END_SWIGLU ? 8 : 16), n = END == END_SWIGLU ? n0 + (c >> 1) + (c & 1) * a.half : min(n0 + c, a.N - 1);
  const uint16_t* x[1] = {a.x + min(c, a.M - 1) * a.ldx};
  f32x4 acc[1];
  stream_sums<1, 4>(a.w + n * a.ldw, x, a.K, wave, acc);
  if constexpr (LORA) {
    // the rows' adapters, an eighth of them to each wave: lane l has row l's
    const int64_t id = lane < a.M ? a.ids[lane] : -1;
    uint64_t open = __ballot(id >= 0 && id < a.adapters);
    for (int i = 0; open; i++) {
      const int64_t now = __shfl(id, __ffsll((unsigned long long)open) - 1);
      const uint64_t rows = __ballot(id == now);
      open &= ~rows;
      if (i % ST_WAVES != wave) continue;
      const bool mine = rows >> c & 1;
      const uint16_t *b = a.b + ((size_t)now * a.N + n) * a.rank, *p = a.p + (size_t)c * a.rank;
      for (int r0 = 0; r0 < a.rank; r0 += 64) {
        i32x4 bv[2], pv[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = r0 + 32 * h + 8 * q;
          bv[h] = pv[h] = i32x4{0, 0, 0, 0};
          if (r < a.rank) bv[h] = *(const i32x4*)(b + r);
          if (r < a.rank && mine) pv[h] = *(const i32x4*)(p + r);
        }
        // (the other rows keep their sums, also where this adapter holds infinities or NaN)
        const f32x4 with = mfma_bf16(bv[1], pv[1], mfma_bf16(bv[0], pv[0], acc[0]));
        acc[0] = mine ? with : acc[0];
      }
    }
  }
  const f32x4 v = join_waves<1>(part, acc, wave);
  if (wave > 0 || c >= a.M) return;
  if constexpr (END == END_SWIGLU) {
    // results 4 q .. 4 q + 3: gate and up of units n0 + 2 q and n0 + 2 q + 1
    const int u = n0 + 2 * q;
    if (a.pre) {
      *(f32x2*)(a.pre + (size_t)c * 2 * a.half + u) = f32x2{v[0], v[2]};
      *(f32x2*)(a.pre + (size_t)c * 2 * a.half + a.half + u) = f32x2{v[1], v[3]};
    }
    const f32x4 h{v[0] * sigmoid(v[0]) * v[1], v[2] * sigmoid(v[2]) * v[3], 0, 0};
    *(int*)(a.out + c * a.ldo + u) = round4(h)[0];
  } else {
    if (n0 + 4 * q < a.N) *(i32x2*)(a.out + c * a.ldo + n0 + 4 * q) = round4(v);
  }
}

}  // namespace d3
