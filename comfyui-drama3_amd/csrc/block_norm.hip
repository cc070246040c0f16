// The end of one block and the start of the next, in one pass over the rows, and its backward pass:
//
//   v = y                            h = residual + scale gate v
//   v = y rstd(y) post  (post given) n = h rstd(h) weight            rstd(z) = 1 / sqrt(mean(z^2) + eps)
//
// with post and weight read as 1 + w where they are kept as offsets. Sums, h inside the pass and all products are float32; h and
// n are each rounded once, to the stream's and the block's type (n comes from h before its rounding).
//
// HBM-bound: a row is read once, held in registers through its sums, and written once: 8192 rows of 2048, a float32 stream
// and a bfloat16 block output, 42 us (4.8 TB/s); 4096 bfloat16 rows 14.2 us forward (4.7 TB/s), 21.0 backward (4.8 TB/s). A lane
// takes 8 columns at a time, 8 to 32 in all: a wave a row up to 1024 columns (four rows a workgroup), a workgroup a row above.
//
// Backward, for dh and dn (gradients of h and n), with z^ = z rstd(z) and m(z) the mean over a row:
//   a = dn weight        dresidual = dh + rstd(h) (a - h^ m(a h^))        dv = scale dresidual
//   dgate = dv v         b = dv gate post        dy = rstd(y) (b - y^ m(b y^))
//   dweight = sum_t dn h^,  dpost = sum_t dv gate y^,  dgate summed over the columns (a gate per row) or rows (per channel)
// Sums over the rows: a workgroup's lanes keep their columns' over the rows that it walks, and a second launch adds the
// workgroups' in a fixed order, so they are the same bits from call to call.
#include "common.hpp"
#include "../../include/drama3_moe.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace d3 {
int fail(const std::string& msg);
int hip_fail(hipError_t err, const char* what);

namespace {

typedef d3_add_norm_desc Desc;
struct bf16_t {
  uint16_t bits;
};
// (rows may start at any element)
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

// columns col .. col + 7 of a row as they are stored (zeros past H)
template <class T>
struct Eight;
template <>
struct Eight<bf16_t> {
  u32x4_at2 w;
  D3_INLINE void get(const bf16_t* row, int col, int H) {
    if (col + 8 <= H) {
      w = *(const u32x4_at2*)(row + col);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        w[i] = col + 2 * i < H ? row[col + 2 * i].bits : 0u;
        if (col + 2 * i + 1 < H) w[i] |= (uint32_t)row[col + 2 * i + 1].bits << 16;
      }
    }
  }
  D3_INLINE float operator[](int i) const { return i & 1 ? __uint_as_float(w[i / 2] & 0xFFFF0000u) : __uint_as_float(w[i / 2] << 16); }
};
template <>
struct Eight<float> {
  f32x4_at4 a, b;
  D3_INLINE void get(const float* row, int col, int H) {
    if (col + 8 <= H) {
      a = *(const f32x4_at4*)(row + col), b = *(const f32x4_at4*)(row + col + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        a[i] = col + i < H ? row[col + i] : 0.0f;
        b[i] = col + 4 + i < H ? row[col + 4 + i] : 0.0f;
      }
    }
  }
  D3_INLINE float operator[](int i) const { return i < 4 ? a[i] : b[i - 4]; }
};
template <class T>
D3_INLINE void load8(const T* row, int col, int H, float (&v)[8]) {
  Eight<T> e;
  e.get(row, col, H);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = e[i];
}
template <class T>
D3_INLINE void store8(T* row, int col, int H, const float (&v)[8]) {
  if (col + 8 <= H) {
    if constexpr (std::is_same_v<T, bf16_t>) {
      u32x4_at2 w;
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = f32_to_bf16(v[2 * i]) | f32_to_bf16(v[2 * i + 1]) << 16;
      *(u32x4_at2*)(row + col) = w;
    } else {
      *(f32x4_at4*)(row + col) = f32x4_at4{v[0], v[1], v[2], v[3]};
      *(f32x4_at4*)(row + col + 4) = f32x4_at4{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (col + i < H) {
        if constexpr (std::is_same_v<T, bf16_t>) row[col + i].bits = (uint16_t)f32_to_bf16(v[i]);
        else row[col + i] = v[i];
      }
    }
  }
}
// the same of a norm's weight or a gate, whose type goes by the call (1: bf16, 0: float32)
D3_INLINE void load8_of(const void* row, int type, int col, int H, float (&v)[8]) {
  if (type) load8((const bf16_t*)row, col, H, v);
  else load8((const float*)row, col, H, v);
}
D3_INLINE float load1_of(const void* p, int type, int64_t i) {
  return type ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}

// A row's sum over its lanes, the same in all of them: a wave's (WAVE) or the workgroup's, whose `slot` is LDS of this sum alone
// until two barriers later.
template <bool WAVE>
D3_INLINE float row_sum(float v, float* slot) {
  v = wave_sum_f32(v);
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
    for (int i = 1; i < (int)blockDim.x / 64; i++) v += slot[i];
  }
  return v;
}

constexpr int GATE_ROW = 1, GATE_CHANNEL = 2, GATE_FULL = 3;  // gate_kind; 0: none

// the gate's values at a row's columns
D3_INLINE void gate8(const Desc& d, int row, int col, float (&g)[8]) {
  const int64_t at = d.gate_kind == GATE_CHANNEL ? 0 : (int64_t)row * d.gate_stride;
  if (d.gate_kind == GATE_ROW) {
    const float one = load1_of(d.gate, d.gate_type, at);
#pragma unroll
    for (int i = 0; i < 8; i++) g[i] = one;
  } else {
    load8_of((const uint8_t*)d.gate + at * (d.gate_type ? 2 : 4), d.gate_type, col, d.H, g);
  }
}

// a norm's weight, as it multiplies
D3_INLINE void weight8(const void* w, int type, int offset, int col, int H, float (&v)[8]) {
  load8_of(w, type, col, H, v);
  if (offset) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += 1.0f;
  }
}

// Lanes: WAVE a wave a row and four rows a workgroup, else a row a workgroup, of which lane l has the 8 columns from 8 l and CH - 1
// times as many lanes further on.
template <bool WAVE>
D3_INLINE int lane_of() { return WAVE ? (int)threadIdx.x & 63 : (int)threadIdx.x; }
template <bool WAVE>
D3_INLINE int lanes_of() { return WAVE ? 64 : (int)blockDim.x; }

template <class TY, class TS, bool WAVE, int CH, int MOST>
__global__ void __launch_bounds__(MOST) add_norm_kernel(Desc d) {
  __shared__ float slots[2][16];
  const int lane = lane_of<WAVE>(), lanes = lanes_of<WAVE>();
  const int64_t row = WAVE ? (int64_t)blockIdx.y * 4 + threadIdx.x / 64 : blockIdx.y;
  if (row >= d.T) return;  // (whole waves, and then without barriers)
  float h[CH][8], w[CH][8];
#pragma unroll
  for (int j = 0; j < CH; j++) load8((const TS*)d.residual + row * d.residual_stride, 8 * (lane + lanes * j), d.H, h[j]);
  if (d.weight) {  // (on its way during the sums)
#pragma unroll
    for (int j = 0; j < CH; j++) weight8(d.weight, d.weight_type, d.unit_offset, 8 * (lane + lanes * j), d.H, w[j]);
  }
  if (d.y) {
    float v[CH][8];
#pragma unroll
    for (int j = 0; j < CH; j++) load8((const TY*)d.y + row * d.y_stride, 8 * (lane + lanes * j), d.H, v[j]);
    if (d.post) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < CH; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) sum += v[j][i] * v[j][i];
      const float rstd = rsqrtf(row_sum<WAVE>(sum, slots[0]) / (float)d.H + d.eps);
      if (d.rstd && lane == 0) d.rstd[d.T + row] = rstd;
#pragma unroll
      for (int j = 0; j < CH; j++) {
        float p[8];
        weight8(d.post, d.post_type, d.unit_offset, 8 * (lane + lanes * j), d.H, p);
#pragma unroll
        for (int i = 0; i < 8; i++) v[j][i] *= rstd * p[i];
      }
    }
#pragma unroll
    for (int j = 0; j < CH; j++) {
      float g[8] = {1, 1, 1, 1, 1, 1, 1, 1};
      if (d.gate_kind) gate8(d, (int)row, 8 * (lane + lanes * j), g);
#pragma unroll
      for (int i = 0; i < 8; i++) h[j][i] += d.scale * (g[i] * v[j][i]);
      if (d.h) store8((TS*)d.h + row * d.H, 8 * (lane + lanes * j), d.H, h[j]);
    }
  }
  if (!d.weight) return;
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < CH; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) sum += h[j][i] * h[j][i];
  const float rstd = rsqrtf(row_sum<WAVE>(sum, slots[1]) / (float)d.H + d.eps);
  if (d.rstd && lane == 0) d.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < CH; j++) {
#pragma unroll
    for (int i = 0; i < 8; i++) w[j][i] *= h[j][i] * rstd;
    store8((TY*)d.n + row * d.H, 8 * (lane + lanes * j), d.H, w[j]);
  }
}

// SIDE: there is a post norm or a gate; without them dy = scale dresidual. AGAIN: h is made again from y and residual, in float32 as
// the forward pass made it, and not read as it is stored: its rounding to bf16 would add to dweight as much error as that's
// own (4096 x 2048 without post and gate 20.8 us so, 18.5 from the stored h: one row less to read; with them y is read
// anyway). The next row's loads are on their way during a row's sums. What all rows share (weight, post, a gate per channel)
// stays in registers: loads come back in order, so one that a row waits for would wait for the next row's as well.
template <class TY, class TS, bool SIDE, bool AGAIN, bool WAVE, int CH, int MOST>
__global__ void __launch_bounds__(MOST) add_norm_backward_kernel(Desc d, int groups) {
  __shared__ float slots[2][3][16];
  const int lane = lane_of<WAVE>(), lanes = lanes_of<WAVE>(), group = WAVE ? (int)(blockIdx.x * 4 + threadIdx.x / 64) : (int)blockIdx.x;
  if (group >= groups) return;  // (whole waves, and then without barriers)
  constexpr int SC = SIDE ? CH : 1, YC = SIDE || AGAIN ? CH : 1;
  float sum_w[CH][8] = {}, sum_p[SC][8] = {}, sum_g[SC][8] = {}, w[CH][8] = {}, p[SC][8], g[SC][8];
  float next_g[SC][8], next_rstd = 0.0f, next_rstd_y = 1.0f;
  Eight<TS> next_dh[CH], next_h[CH];
  Eight<TY> next_dn[CH], next_y[YC];
#pragma unroll
  for (int j = 0; j < CH; j++) {
    const int col = 8 * (lane + lanes * j);
    if (d.weight) weight8(d.weight, d.weight_type, d.unit_offset, col, d.H, w[j]);
    if constexpr (SIDE) {
#pragma unroll
      for (int i = 0; i < 8; i++) p[j][i] = g[j][i] = next_g[j][i] = 1.0f;
      if (d.post) weight8(d.post, d.post_type, d.unit_offset, col, d.H, p[j]);
      if (d.gate_kind == GATE_CHANNEL) gate8(d, 0, col, g[j]);
    }
  }
  auto get = [&](int64_t row) {
    if (d.dn) next_rstd = d.rstd[row];
    if (SIDE && d.post) next_rstd_y = d.rstd[d.T + row];
#pragma unroll
    for (int j = 0; j < CH; j++) {
      const int col = 8 * (lane + lanes * j);
      if (d.dh) next_dh[j].get((const TS*)d.dh + row * d.H, col, d.H);
      if (d.dn) {
        next_dn[j].get((const TY*)d.dn + row * d.H, col, d.H);
        next_h[j].get((const TS*)(AGAIN ? d.residual : d.h) + row * d.residual_stride, col, d.H);
      }
      if constexpr (SIDE || AGAIN) next_y[j].get((const TY*)d.y + row * d.y_stride, col, d.H);
      if constexpr (SIDE) {
        if (d.gate_kind == GATE_ROW || d.gate_kind == GATE_FULL) gate8(d, (int)row, col, next_g[j]);
      }
    }
  };
  get(group);  // (there are no more groups than rows)
  int turn = 0;
  for (int64_t row = group; row < d.T; row += groups, turn ^= 1) {
    float dr[CH][8], a[CH][8], hat[CH][8], v[SC][8];
    const float rstd = next_rstd, rstd_y = next_rstd_y;
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        dr[j][i] = d.dh ? next_dh[j][i] : 0.0f;
        float side = 0.0f;
        if constexpr (SIDE) {
          if (d.gate_kind != GATE_CHANNEL) g[j][i] = next_g[j][i];
          v[j][i] = next_y[j][i] * rstd_y;  // y^
          side = g[j][i] * (v[j][i] * p[j][i]);
        } else if constexpr (AGAIN) {
          side = next_y[j][i];
        }
        if (d.dn) {
          a[j][i] = next_dn[j][i];
          hat[j][i] = (AGAIN ? next_h[j][i] + d.scale * side : next_h[j][i]) * rstd;
        }
      }
    if (row + groups < d.T) get(row + groups);
    if (d.dn) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < CH; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          sum_w[j][i] += a[j][i] * hat[j][i];
          a[j][i] *= w[j][i];
          sum += a[j][i] * hat[j][i];
        }
      const float mean = row_sum<WAVE>(sum, slots[turn][0]) / (float)d.H;
#pragma unroll
      for (int j = 0; j < CH; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) dr[j][i] += rstd * (a[j][i] - hat[j][i] * mean);
    }
    if (d.dresidual) {
#pragma unroll
      for (int j = 0; j < CH; j++) store8((TS*)d.dresidual + row * d.H, 8 * (lane + lanes * j), d.H, dr[j]);
    }
    if constexpr (!SIDE) {
      if (d.dy) {
#pragma unroll
        for (int j = 0; j < CH; j++) {
#pragma unroll
          for (int i = 0; i < 8; i++) dr[j][i] *= d.scale;
          store8((TY*)d.dy + row * d.H, 8 * (lane + lanes * j), d.H, dr[j]);
        }
      }
    } else {
      float sum_row = 0.0f, sum_b = 0.0f;
#pragma unroll
      for (int j = 0; j < CH; j++) {
        const int col = 8 * (lane + lanes * j);
        float full[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float dv = d.scale * dr[j][i];
          full[i] = dv * (v[j][i] * p[j][i]);
          sum_g[j][i] += full[i];
          sum_row += full[i];
          const float dnormed = dv * g[j][i];
          sum_p[j][i] += dnormed * v[j][i];
          dr[j][i] = dnormed * p[j][i];  // b
          sum_b += dr[j][i] * v[j][i];
        }
        if (d.dgate && d.gate_kind == GATE_FULL) {
          if (d.gate_type) store8((bf16_t*)d.dgate + row * d.H, col, d.H, full);
          else store8((float*)d.dgate + row * d.H, col, d.H, full);
        }
      }
      if (d.dgate && d.gate_kind == GATE_ROW) {
        sum_row = row_sum<WAVE>(sum_row, slots[turn][1]);
        if (lane == 0) {
          if (d.gate_type) ((uint16_t*)d.dgate)[row] = (uint16_t)f32_to_bf16(sum_row);
          else ((float*)d.dgate)[row] = sum_row;
        }
      }
      if (d.dy) {
        if (d.post) {
          const float mean = row_sum<WAVE>(sum_b, slots[turn][2]) / (float)d.H;
#pragma unroll
          for (int j = 0; j < CH; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) dr[j][i] = rstd_y * (dr[j][i] - v[j][i] * mean);
        }
#pragma unroll
        for (int j = 0; j < CH; j++) store8((TY*)d.dy + row * d.H, 8 * (lane + lanes * j), d.H, dr[j]);
      }
    }
  }
  float* part = d.partials + (int64_t)group * d.H;
  const int64_t step = (int64_t)groups * d.H;
#pragma unroll
  for (int j = 0; j < CH; j++) {
    const int col = 8 * (lane + lanes * j);
    float* to = part;
    if (d.dweight) store8(to, col, d.H, sum_w[j]), to += step;
    if constexpr (SIDE) {
      if (d.dpost) store8(to, col, d.H, sum_p[j]), to += step;
      if (d.dgate && d.gate_kind == GATE_CHANNEL) store8(to, col, d.H, sum_g[j]);
    }
  }
}

// the groups' sums over the rows added up: 32 columns a workgroup, 4 a lane, so that its 1024 lanes each add every 128th
// group, whose sums are then added in LDS
struct Sums {
  void* out[3];
  int type[3];
};
__global__ void __launch_bounds__(1024) add_groups_kernel(const float* partials, int groups, int H, Sums s) {
  __shared__ float part[128][32];
  const int lane = threadIdx.x & 7, slice = threadIdx.x >> 3, col = blockIdx.x * 32 + 4 * lane;
  const float* from = partials + (int64_t)blockIdx.y * groups * H;
  f32x4 sum{0, 0, 0, 0};
  if (col + 4 <= H) {
#pragma unroll 8
    for (int g = slice; g < groups; g += 128) sum += *(const f32x4_at4*)(from + (int64_t)g * H + col);
  } else {
    for (int g = slice; g < groups; g += 128)
      for (int i = 0; i < 4; i++)
        if (col + i < H) sum[i] += from[(int64_t)g * H + col + i];
  }
  *(f32x4*)&part[slice][4 * lane] = sum;
  __syncthreads();
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, out = blockIdx.x * 32 + c;
  float all = (part[r][c] + part[r + 32][c]) + (part[r + 64][c] + part[r + 96][c]);
  part[r][c] = all;  // (no other lane reads or writes these four)
  __syncthreads();
  if (r || out >= H) return;
#pragma unroll
  for (int i = 1; i < 32; i++) all += part[i][c];
  if (s.type[blockIdx.y]) ((uint16_t*)s.out[blockIdx.y])[out] = (uint16_t)f32_to_bf16(all);
  else ((float*)s.out[blockIdx.y])[out] = all;
}

constexpr int MAX_H = 16384;

// f(WAVE, CH, MOST, lanes) for rows of H columns: MOST lanes at 8 columns each, then 512 at more. 1391 rows of 5120, 640 lanes
// against 320: forward 17.2 us and 15.5, backward 28 and 48 (of which a CU holds one row at a time either way).
template <int MOST, class F>
void by_width(int H, F f) {
  const int units = (H + 7) / 8;
  auto lanes = [&](int ch) { return ((units + ch - 1) / ch + 63) / 64 * 64; };
  using std::bool_constant, std::integral_constant;
  if (units <= 64) f(bool_constant<true>{}, integral_constant<int, 1>{}, integral_constant<int, 256>{}, 256);
  else if (units <= 128) f(bool_constant<true>{}, integral_constant<int, 2>{}, integral_constant<int, 256>{}, 256);
  else if (units <= MOST) f(bool_constant<false>{}, integral_constant<int, 1>{}, integral_constant<int, MOST>{}, lanes(1));
  else if (units <= 1024) f(bool_constant<false>{}, integral_constant<int, 2>{}, integral_constant<int, 512>{}, lanes(2));
  else f(bool_constant<false>{}, integral_constant<int, 4>{}, integral_constant<int, 512>{}, lanes(4));
}
template <class F>
void by_types(const Desc& d, F f) {
  if (d.y_type) {
    if (d.stream_type) f(bf16_t{}, bf16_t{});
    else f(bf16_t{}, float{});
  } else {
    if (d.stream_type) f(float{}, bf16_t{});
    else f(float{}, float{});
  }
}

// Groups of rows whose sums over the rows a backward pass keeps apart: as many as the CUs hold at once (12 waves each), since
// each writes float32 sums of H columns that the second launch reads.
int groups_of(int T, int H) {
  const int units = (H + 7) / 8, most = units <= 128 ? 256 * 8 : 256 * std::max(1, 12 / ((units + 63) / 64));
  return std::min(T, most);
}

int check(const char* what, const Desc* d) {
  const std::string at = what;
  if (!d) return fail(at + ": null descriptor");
  if (d->T < 0 || d->H < 1 || d->H > MAX_H) return fail(at + ": H must be 1 to 16384, T not negative");
  if ((d->y_type | d->stream_type | d->weight_type | d->post_type | d->gate_type) & ~1) return fail(at + ": types are 0 (float32) or 1 (bf16)");
  if (d->gate_kind < 0 || d->gate_kind > 3 || (d->gate_kind && !d->gate)) return fail(at + ": gate_kind is 0 to 3, with a gate from 1 on");
  if (d->T > 0 && (d->post || d->gate_kind) && !d->y) return fail(at + ": post and gate go with y");
  if (d->T > 1 && ((d->y && d->y_stride < d->H) || d->residual_stride < d->H || (d->gate_kind == GATE_FULL && d->gate_stride < d->H) ||
                   (d->gate_kind == GATE_ROW && d->gate_stride < 1)))
    return fail(at + ": rows that lie less than their columns apart");
  return 0;
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int64_t d3_add_norm_partials(int32_t T, int32_t H) {
  if (T < 0 || H < 1) return 0;
  return (int64_t)groups_of(T, H) * H;
}

extern "C" int d3_add_norm(const d3_add_norm_desc* desc, void* stream) {
  if (const int rc = check("d3_add_norm", desc)) return rc;
  const Desc& d = *desc;
  if (d.T == 0) return 0;
  if (!d.residual || (d.y && !d.h) || (d.weight && !d.n) || !(d.y || d.weight)) return fail("d3_add_norm: null pointer");
  // (rows along y: a grid's x has room for 2^32 threads)
  by_types(d, [&](auto y, auto s) {
    by_width<512>(d.H, [&](auto wave, auto chunks, auto most, int lanes) {
      constexpr bool W = decltype(wave)::value;
      add_norm_kernel<decltype(y), decltype(s), W, decltype(chunks)::value, decltype(most)::value>
          <<<dim3(1, W ? (unsigned)(((int64_t)d.T + 3) / 4) : (unsigned)d.T), lanes, 0, (hipStream_t)stream>>>(d);
    });
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_add_norm launch");
}

extern "C" int d3_add_norm_backward(const d3_add_norm_desc* desc, void* stream) {
  if (const int rc = check("d3_add_norm_backward", desc)) return rc;
  const Desc& d = *desc;
  if ((d.dn || d.dweight) && !d.weight) return fail("d3_add_norm_backward: dn and dweight go with weight");
  if ((d.dpost && !d.post) || (d.dgate && !d.gate_kind) || (d.dy && !d.y))
    return fail("d3_add_norm_backward: dpost, dgate and dy go with post, gate and y");
  const int parts = !!d.dweight + !!d.dpost + (d.dgate && d.gate_kind == GATE_CHANNEL);
  const int groups = groups_of(d.T, d.H);
  if (d.T > 0) {
    if (!(d.dh || d.dn) || (d.dn && (!d.rstd || !(d.stream_type && d.y ? d.residual : d.h))) || (d.post && !d.rstd))
      return fail("d3_add_norm_backward: null pointer");
    if (parts && (!d.partials || d.partials_floats < (int64_t)parts * groups * d.H))
      return fail("d3_add_norm_backward: partials too small (d3_add_norm_partials)");
    by_types(d, [&](auto y, auto s) {
      by_width<768>(d.H, [&](auto wave, auto chunks, auto most, int lanes) {
        constexpr bool W = decltype(wave)::value;
        constexpr int CH = decltype(chunks)::value, MOST = decltype(most)::value;
        const int grid = W ? (groups + 3) / 4 : groups;
        // (a float32 stream holds h as it was)
        constexpr bool STORED_SHORT = std::is_same_v<decltype(s), bf16_t>;
        const bool again = STORED_SHORT && d.y && d.dn;
        auto launch = [&](auto side, auto again) {
          add_norm_backward_kernel<decltype(y), decltype(s), decltype(side)::value, decltype(again)::value, W, CH, MOST>
              <<<grid, lanes, 0, (hipStream_t)stream>>>(d, groups);
        };
        if (d.y && (d.post || d.gate_kind)) {
          if (again) launch(std::true_type{}, std::bool_constant<STORED_SHORT>{});
          else launch(std::true_type{}, std::false_type{});
        } else {
          if (again) launch(std::false_type{}, std::bool_constant<STORED_SHORT>{});
          else launch(std::false_type{}, std::false_type{});
        }
      });
    });
  }
  if (parts) {
    Sums sums{};
    int i = 0;
    if (d.dweight) sums.out[i] = d.dweight, sums.type[i++] = d.weight_type;
    if (d.dpost) sums.out[i] = d.dpost, sums.type[i++] = d.post_type;
    if (d.dgate && d.gate_kind == GATE_CHANNEL) sums.out[i] = d.dgate, sums.type[i++] = d.gate_type;
    add_groups_kernel<<<dim3((d.H + 31) / 32, parts), 1024, 0, (hipStream_t)stream>>>(d.partials, groups, d.H, sums);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_add_norm_backward launch");
}
