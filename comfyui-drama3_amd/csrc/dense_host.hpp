// How the dense products' C entries check and launch.
#pragma once
#include "dense_stream.hpp"

#include <algorithm>
#include <string>

namespace d3 {
int fail(const std::string& msg);
int hip_fail(hipError_t err, const char* what);

using Wide = Tile<2, 4, 8, 4, 2>;        // 256 x 256, 8 waves, one workgroup a CU
using Long = Tile<2, 4, 4, 4, 3, 1>;     // 128 x 256, the same
using Square = Tile<2, 4, 4, 2, 4, 1>;   // 128 x 128, the same
using Small = Tile<2, 2, 2, 2, 4, 4>;    // 64 x 64, 4 waves, two workgroups a CU
using Thin = Tile<4, 1, 1, 2, 6, 4>;     // 64 x 32, 4 waves, two workgroups a CU
using Flat = Tile<2, 2, 1, 2, 6>;        // 32 x 64, the same for a transposed w, of which LDS holds 64 columns at least

constexpr int64_t MAX_LD = 1 << 23;  // (a tile's rows within 32-bit byte offsets)
constexpr int MAX_ROWS = 1 << 30;

inline bool bad_rows(const void* p, int64_t ld, int64_t cols) { return !p || ((uintptr_t)p & 15u) || ld % 8 || ld < cols || ld > MAX_LD; }

template <class C>
inline int dense_tiles(const Dense& a, bool swiglu) {
  const int un = swiglu ? C::TN / 2 : C::TN;
  return ((a.M + C::TM - 1) / C::TM) * (((swiglu ? a.half : a.N) + un - 1) / un);
}

template <class C, bool WT, int END, bool LORA>
inline void launch_tile(const Dense& a, hipStream_t stream) {
  const int tiles = dense_tiles<C>(a, END == END_SWIGLU);
  dense_tile_kernel<C, WT, END, LORA><<<dim3(1, tiles), C::THREADS, 0, stream>>>(a);
}

enum TileSize { WIDE, LONG, SQUARE, SMALL, LEAST };
struct TilePlan {
  TileSize size;
  float cost;
};
constexpr float LONG_COST = 0.82f;

// The tile's size by what a stage of each takes, us, times the turns in which the 256 CUs take the tiles: 1.5 (256 x 256),
// 0.82 (128 x 256), 0.45 (128 x 128; 0.5 in several turns), 0.17 (64 x 64), 0.155 (64 x 32), measured with the CUs at work.
// So the large ones, which read least, where they come out even, and small ones for few rows. Measured, us, each product alone, in this
// order (t: a transposed operand; tt: both, as in launch_dense_set):
//   4096 x 4096 x 11008    266 276 317   -   -     4096 x 2048 x 6144    115  80  91   -   -     4096 x 12288 x 2048  154 170 200  -  -
//   12288 x 2048 x 4096 tt 177 177 211   -   -     2048 x 6144 x 4096 tt  86 107 106   -   -     1391 x 1536 x 2048    -   -  16  19  -
//    509 x 1024 x 2048       -   -   - 8.1 7.4       61 x 4096 x 2048      -   -   - 7.9 7.1     1391 x 2048 x 1536 t   -   -  13  16  -
template <bool WT, int END, bool LORA>
inline TilePlan plan_tiles(const Dense& a) {
  constexpr bool SWIGLU = END == END_SWIGLU;
  using Least = std::conditional_t<WT, Flat, Thin>;
  auto turns = [](int tiles) { return (float)((tiles + 255) / 256); };
  TilePlan best{LONG, LONG_COST * turns(dense_tiles<Long>(a, SWIGLU))};
  auto try_size = [&](TileSize size, float cost) {
    if (cost < best.cost) best = TilePlan{size, cost};
  };
  if (!LORA) try_size(WIDE, 1.5f * turns(dense_tiles<Wide>(a, SWIGLU)));  // (with adapters its sums do not stay in registers)
  const float square = turns(dense_tiles<Square>(a, SWIGLU));
  try_size(SQUARE, (square > 1 ? 0.5f : 0.45f) * square);
  try_size(SMALL, 0.17f * turns(dense_tiles<Small>(a, SWIGLU)));
  try_size(LEAST, 0.155f * turns(dense_tiles<Least>(a, SWIGLU)));
  return best;
}

template <bool WT, int END, bool LORA>
inline void launch_plan(TileSize size, const Dense& a, hipStream_t stream) {
  if constexpr (!LORA) {
    if (size == WIDE) return launch_tile<Wide, WT, END, LORA>(a, stream);
  }
  if (size == LONG) launch_tile<Long, WT, END, LORA>(a, stream);
  else if (size == SQUARE) launch_tile<Square, WT, END, LORA>(a, stream);
  else if (size == SMALL) launch_tile<Small, WT, END, LORA>(a, stream);
  else launch_tile<std::conditional_t<WT, Flat, Thin>, WT, END, LORA>(a, stream);
}

// a's rows from m on
inline Dense rows_from(Dense a, int m, int rows) {
  a.x += m * a.ldx;
  a.out += m * a.ldo;
  if (a.pre) a.pre += (int64_t)m * 2 * a.half;
  if (a.ids) a.ids += m, a.p += (int64_t)m * a.rank;
  a.M = rows;
  return a;
}

// The whole product by one size of tile, or the rows that fill whole turns of 128 x 256 tiles by those and the rest by
// what suits it, where that is 8% less (the second launch takes 3 us): 5000 x 4096 x 2048 is 2.5 turns.
template <bool WT, int END, bool LORA = false>
inline void launch_tiles(const Dense& a, hipStream_t stream) {
  const TilePlan whole = plan_tiles<WT, END, LORA>(a);
  const int columns = dense_tiles<Long>(Dense{.M = 1, .N = a.N, .K = a.K, .half = a.half}, END == END_SWIGLU);
  const int full = dense_tiles<Long>(a, END == END_SWIGLU) / 256, rows = 256 * full / columns * Long::TM;
  if (full >= 1 && rows > 0 && rows < a.M) {
    const Dense rest = rows_from(a, rows, a.M - rows);
    const TilePlan left = plan_tiles<WT, END, LORA>(rest);
    if (LONG_COST * full + left.cost < 0.92f * whole.cost) {
      launch_tile<Long, WT, END, LORA>(rows_from(a, 0, rows), stream);
      return launch_plan<WT, END, LORA>(left.size, rest, stream);
    }
  }
  launch_plan<WT, END, LORA>(whole.size, a, stream);
}

// A set of products in one launch. The size of tile, one for all of them, by the same costs of a stage: its share of all tiles'
// stages, or the longest tile's, and half of the shortest's for the end.
template <class C>
inline void launch_set(DenseSet set, hipStream_t stream) {
  int all = 0;
  for (int i = 0; i < set.count; i++) all += set.tiles[i] = (dense_tiles<C>(set.product[i], false) + 7) / 8 * 8;
  dense_set_kernel<C><<<dim3(1, all), C::THREADS, 0, stream>>>(set);
}
template <class C>
inline float set_cost(const DenseSet& set, float stage) {
  float all = 0.0f, most = 0.0f, least = 1e30f;
  for (int i = 0; i < set.count; i++) {
    const float stages = (float)((set.product[i].K + 63) / 64);
    all += dense_tiles<C>(set.product[i], false) * stages;
    most = std::max(most, stages), least = std::min(least, stages);
  }
  return stage * std::max(all / 256.0f + 0.5f * least, most);
}
inline void launch_dense_set(DenseSet set, hipStream_t stream) {
  // the longest first
  for (int i = 1; i < set.count; i++)
    for (int j = i; j > 0 && set.product[j].K > set.product[j - 1].K; j--) {
      std::swap(set.product[j], set.product[j - 1]);
      if (set.rows == j) set.rows = j - 1;
      else if (set.rows == j - 1) set.rows = j;
    }
  const float wide = set_cost<Wide>(set, 1.5f), tall = set_cost<Long>(set, LONG_COST), square = set_cost<Square>(set, 0.45f);
  const float small = set_cost<Small>(set, 0.17f);
  if (wide <= std::min({tall, square, small})) launch_set<Wide>(set, stream);
  else if (tall <= std::min(square, small)) launch_set<Long>(set, stream);
  else if (square <= small) launch_set<Square>(set, stream);
  else launch_set<Small>(set, stream);
}

// Products of rows with rows (both operands with their k side by side): up to 16 rows by streaming the weights, where a CU has
// no more than one of their 16-row columns, else by tiles. Both, us: 5 x 1024 x 2048 (SwiGLU) 5.1 and 6.9, 16 rows 6.1 and
// 6.9; 4 x 4096 x 4096 8.3 and 11.1, 16 rows 10.1 and 10.9; 4 x 6144 x 4096 12.9 and 11.1, 16 rows 16.8 and 11.3.
template <int END, bool LORA>
inline void launch_dense(const Dense& a, hipStream_t stream) {
  const int columns = END == END_SWIGLU ? (a.half + 7) / 8 : (a.N + 15) / 16;
  if (a.M <= 16 && columns <= 256) dense_stream_kernel<END, LORA><<<columns, ST_THREADS, 0, stream>>>(a);
  else launch_tiles<false, END, LORA>(a, stream);
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, what);
}

}  // namespace d3
