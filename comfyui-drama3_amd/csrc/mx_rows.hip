// Rows to the microscaled formats and back (mx.hpp): per block of 32 columns the scale is the power of two
// 2^(floor(log2 max|v|) - m), m = 2 for e2m1 and 8 for e4m3, so that the largest magnitude falls into the binade of the
// format's largest element; the elements are v / scale to nearest, ties to even, saturated at +-6 or +-448. Dividing by
// a power of two is exact, so the codes are those of the definition bit for bit. A block of zeros has scale code 0, a block with an
// infinity or NaN has 255 (NaN: all its values read as NaN).
//
// HBM-bound. A lane takes 8 columns (one 16-byte load of bf16, two of float32), four lanes a block, whose maximum
// goes round by DPP; consecutive lanes read and write consecutive bytes. A bank of 196608 x 2048 bf16 weights to e2m1 takes 167 us
// (805 MB read, 214 MB written: 6.1 TB/s), back 140 us (7.3 TB/s).
#include "mx.hpp"
#include "../../include/drama3_moe.h"

#include <string>
#include <type_traits>

namespace d3 {
int fail(const std::string& msg);
int hip_fail(hipError_t err, const char* what);

namespace {

// Units of a lane, 256 apart, whose loads go out together. A bank of bf16 weights to e2m1, us by units: 180, 172, 181 (4),
// with nontemporal loads (the input is read once; the codes that the products read next stay in the caches) 172, 167, 163, and
// with dequantize behind it 303 (2) and 306 (4). float32 rows: 158 with one, 166 with two; its loads are halves of a line each,
// which the hint would read twice.
template <bool BF16> constexpr int Q_UNITS = BF16 ? 2 : 1;

// columns 8 u .. 8 u + 7 of a row as float
template <bool BF16>
D3_INLINE void load8(const void* row, int u, float (&v)[8]) {
  if constexpr (BF16) {
    const i32x4 w = __builtin_nontemporal_load((const i32x4*)row + u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float((uint32_t)w[i] << 16);
      v[2 * i + 1] = __uint_as_float((uint32_t)w[i] & 0xFFFF0000u);
    }
  } else {
    const f32x4 a = *((const f32x4*)row + 2 * u), b = *((const f32x4*)row + 2 * u + 1);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
  }
}

template <int BITS, bool BF16>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const uint8_t* x, int64_t stride, uint32_t units, int cols,
                                                          int per, uint8_t* codes, uint8_t* scale) {
  constexpr int UNITS = Q_UNITS<BF16>;
  const uint32_t i0 = blockIdx.x * (256u * UNITS) + threadIdx.x;
  float all[UNITS][8] = {};
#pragma unroll
  for (int n = 0; n < UNITS; n++) {
    const uint32_t i = min(i0 + 256u * n, units - 1u), r = i / (uint32_t)per;
    const int u = (int)(i - r * (uint32_t)per);
    if (8 * u < cols) load8<BF16>(x + (int64_t)r * stride, u, all[n]);
  }
#pragma unroll
  for (int n = 0; n < UNITS; n++) {
    const uint32_t i = i0 + 256u * n;
    if (i >= units) return;  // (whole blocks of lanes: a row's units are a multiple of 32)
    float(&v)[8] = all[n];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    top = max(top, (uint32_t)dpp_i32((int)top, 0xB1));
    top = max(top, (uint32_t)dpp_i32((int)top, 0x4E));
    const uint32_t e = top >> 23;
    constexpr uint32_t M = BITS == 4 ? 2 : 8;
    const uint32_t code = e == 255u ? 255u : e > M ? e - M : 0u;
    const float inv = __uint_as_float((254u - min(code, 253u)) << 23);  // 2^(127 - code)
    if constexpr (BITS == 4) {
      uint32_t w = 0;
#define D3_PAIR(b) w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2 * b] * inv, v[2 * b + 1] * inv, 1.0f, b)
      D3_PAIR(0);
      D3_PAIR(1);
      D3_PAIR(2);
      D3_PAIR(3);
#undef D3_PAIR
      ((uint32_t*)codes)[i] = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = __builtin_amdgcn_fmed3f(v[j] * inv, -448.0f, 448.0f);
      ((i32x2*)codes)[i] =
          i32x2{(int)f32x4_to_fp8x4(v[0], v[1], v[2], v[3]), (int)f32x4_to_fp8x4(v[4], v[5], v[6], v[7])};
    }
    if ((i & 3u) == 0u) scale[i >> 2] = (uint8_t)code;
  }
}

// Back: mostly writes. A lane holds 16 bytes of the result (8 columns of bf16, 4 of float32), so that a wave's store is one
// run, four times 256 of them a workgroup, whose loads go out together; what is written is not read back soon (nontemporal).
// A bank's e2m1 codes to bf16: 140 us; 240 with one store a lane, 172 without the hint.
constexpr int DQ_STORES = 4;

template <int BITS, bool BF16>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* codes, const uint8_t* scale, uint32_t units,
                                                            int cols, int per, uint8_t* out) {
  constexpr int COLS = BF16 ? 8 : 4, BYTES = COLS * BITS / 8;
  using Codes = std::conditional_t<BYTES == 8, i32x2, std::conditional_t<BYTES == 4, uint32_t, uint16_t>>;
  const uint32_t i0 = blockIdx.x * (256u * DQ_STORES) + threadIdx.x, row_units = (uint32_t)cols / COLS;
  Codes word[DQ_STORES];
  uint32_t code[DQ_STORES];
#pragma unroll
  for (int n = 0; n < DQ_STORES; n++) {
    const uint32_t i = min(i0 + 256u * n, units - 1u), r = i / row_units;
    const int64_t at = (int64_t)r * per * (8 / COLS) + (i - r * row_units);  // the row's stored units reach to the next stage
    word[n] = ((const Codes*)codes)[at];
    code[n] = scale[at / (MX_BLOCK / COLS)];
  }
#pragma unroll
  for (int n = 0; n < DQ_STORES; n++) {
    const uint32_t i = i0 + 256u * n;
    if (i >= units) return;
    const float s = mx_scale(code[n]);
    float v[COLS];
#pragma unroll
    for (int j = 0; j < COLS / 4; j++) {  // four columns each
      f32x2 a, b;
      if constexpr (BITS == 4) {
        const uint32_t w = (uint32_t)word[n] >> (16 * j);
        a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
        b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
      } else {
        uint32_t w;
        if constexpr (BYTES == 8) w = (uint32_t)word[n][j];
        else w = word[n];
        a = fp8x2_to_f32<false>(w);
        b = fp8x2_to_f32<true>(w);
      }
      v[4 * j] = a.x * s, v[4 * j + 1] = a.y * s, v[4 * j + 2] = b.x * s, v[4 * j + 3] = b.y * s;
    }
    if constexpr (BF16) {
      i32x4 o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = (int)(f32_to_bf16(v[2 * j]) | f32_to_bf16(v[2 * j + 1]) << 16);
      __builtin_nontemporal_store(o, (i32x4*)out + i);
    } else {
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, (f32x4*)out + i);
    }
  }
}

bool misaligned(const void* p) { return (uintptr_t)p & 15u; }

// a row's units of 8 columns, those of its last stage whole (in 64 bits: of any int32)
int64_t row_units(int32_t cols) { return ((int64_t)cols + MX_STAGE - 1) / MX_STAGE * (MX_STAGE / 8); }

// the common checks of rows [rows, cols] in `bits`, `per` units to a row
int check_rows(const char* what, int32_t rows, int32_t cols, int32_t bits, int32_t type, int64_t per) {
  if (bits != 4 && bits != 8) return fail(std::string(what) + ": bits must be 4 or 8");
  if (type != 0 && type != 1) return fail(std::string(what) + ": type must be 0 (float32) or 1 (bfloat16)");
  if (rows < 0 || cols < 1 || cols % MX_BLOCK) return fail(std::string(what) + ": cols must be a positive multiple of 32");
  if (8 * per > INT32_MAX) return fail(std::string(what) + ": cols must be below 2^31 - 255");
  // (the last workgroup's units, of 4 columns where that is more, still in 32 bits)
  if ((int64_t)rows * per > INT32_MAX - 2048) return fail(std::string(what) + ": 2^31 units of 8 columns or more");
  return 0;
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_mx_quantize(const void* x, int32_t type, int64_t stride, int32_t rows, int32_t cols, int32_t bits,
                              void* codes, void* scale, void* stream) {
  const int64_t per = row_units(cols);
  if (const int rc = check_rows("d3_mx_quantize", rows, cols, bits, type, per)) return rc;
  const int64_t bytes = stride * (type ? 2 : 4);
  if (stride < 0 || bytes % 16) return fail("d3_mx_quantize: the row stride must be a multiple of 16 bytes");
  if (rows == 0) return 0;
  if (!x || !codes || !scale) return fail("d3_mx_quantize: null pointer");
  if (misaligned(x) || misaligned(codes)) return fail("d3_mx_quantize: x and codes must be 16-byte aligned");
  const uint32_t units = (uint32_t)rows * (uint32_t)per, each = 256u * (type ? Q_UNITS<true> : Q_UNITS<false>);
  const dim3 grid((units + each - 1u) / each), block(256);
  const hipStream_t s = (hipStream_t)stream;
#define D3_QUANTIZE(B, T)                                                                                           \
  hipLaunchKernelGGL((mx_quantize_kernel<B, T>), grid, block, 0, s, (const uint8_t*)x, bytes, units, cols, (int)per, \
                     (uint8_t*)codes, (uint8_t*)scale)
  if (bits == 4 && type) D3_QUANTIZE(4, true);
  else if (bits == 4) D3_QUANTIZE(4, false);
  else if (type) D3_QUANTIZE(8, true);
  else D3_QUANTIZE(8, false);
#undef D3_QUANTIZE
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_mx_quantize launch");
}

extern "C" int d3_mx_dequantize(const void* codes, const void* scale, int32_t rows, int32_t cols, int32_t bits,
                                int32_t type, void* out, void* stream) {
  const int64_t per = row_units(cols);
  if (const int rc = check_rows("d3_mx_dequantize", rows, cols, bits, type, per)) return rc;
  if (rows == 0) return 0;
  if (!codes || !scale || !out) return fail("d3_mx_dequantize: null pointer");
  if (misaligned(codes) || misaligned(out)) return fail("d3_mx_dequantize: codes and out must be 16-byte aligned");
  const uint32_t units = (uint32_t)rows * (uint32_t)(cols / (type ? 8 : 4));
  const dim3 grid((units + 256u * DQ_STORES - 1u) / (256u * DQ_STORES)), block(256);
  const hipStream_t s = (hipStream_t)stream;
#define D3_DEQUANTIZE(B, T)                                                                                         \
  hipLaunchKernelGGL((mx_dequantize_kernel<B, T>), grid, block, 0, s, (const uint8_t*)codes, (const uint8_t*)scale,  \
                     units, cols, (int)per, (uint8_t*)out)
  if (bits == 4 && type) D3_DEQUANTIZE(4, true);
  else if (bits == 4) D3_DEQUANTIZE(4, false);
  else if (type) D3_DEQUANTIZE(8, true);
  else D3_DEQUANTIZE(8, false);
#undef D3_DEQUANTIZE
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_mx_dequantize launch");
}
