// How the dense products' C entries check and launch.
#pragma once
#include "dense_stream.hpp"

#include <string>

namespace d3 {
int fail(const std::string& msg);
int hip_fail(hipError_t err, const char* what);

using Wide = Tile<2, 4, 8, 4, 2>;    // 256 x 256, 8 waves, one workgroup a CU
using Narrow = Tile<2, 2, 4, 4, 2>;  // 128 x 128, 4 waves, two workgroups a CU

constexpr int64_t MAX_LD = 1 << 23;  // (a tile's rows within 32-bit byte offsets)

inline bool bad_rows(const void* p, int64_t ld, int64_t cols) { return !p || ((uintptr_t)p & 15u) || ld % 8 || ld < cols || ld > MAX_LD; }

template <class C>
inline int dense_tiles(const Dense& a, bool swiglu) {
  const int un = swiglu ? C::TN / 2 : C::TN;
  return ((a.M + C::TM - 1) / C::TM) * (((swiglu ? a.half : a.N) + un - 1) / un);
}

template <class C, bool XT, bool WT, int END, bool LORA = false>
inline void launch_tile(Dense a, hipStream_t stream) {
  a.splits = 1, a.split_stages = (a.K + 63) / 64;
  const int tiles = dense_tiles<C>(a, END == END_SWIGLU);
  dense_tile_kernel<C, XT, WT, END, LORA><<<tiles, C::THREADS, 0, stream>>>(a, a, tiles);
}

// the tile's size: 256 x 256 where that still gives every CU one
template <bool XT, bool WT, int END, bool LORA = false>
inline void launch_tiles(const Dense& a, hipStream_t stream) {
  if constexpr (!LORA) {  // (with adapters the wide tile's sums do not stay in registers)
    if (dense_tiles<Wide>(a, END == END_SWIGLU) >= 256) return launch_tile<Wide, XT, WT, END, LORA>(a, stream);
  }
  launch_tile<Narrow, XT, WT, END, LORA>(a, stream);
}

template <int RT, int END, bool LORA>
inline void launch_stream(const Dense& a, hipStream_t stream) {
  const int columns = END == END_SWIGLU ? (a.half + 7) / 8 : (a.N + 15) / 16;
  dense_stream_kernel<RT, END, LORA><<<dim3(columns, (a.M + 16 * RT - 1) / (16 * RT)), ST_THREADS, 0, stream>>>(a);
}

// products of rows with rows (both operands with their k side by side)
template <int END, bool LORA>
inline void launch_dense(const Dense& a, hipStream_t stream) {
  if (a.M <= 16) launch_stream<1, END, LORA>(a, stream);
  else if (a.M <= 32) launch_stream<2, END, LORA>(a, stream);
  else if (a.M <= 64) launch_stream<4, END, LORA>(a, stream);
  else launch_tiles<false, false, END, LORA>(a, stream);
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, what);
}

}  // namespace d3
