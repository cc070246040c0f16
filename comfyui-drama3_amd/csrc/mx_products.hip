// Expert products on microscaled banks (mx.hpp): e2m1 weights against e4m3 or e2m1 rows on the scaled matrix
// instruction, both operands as they are stored.
#include "expert_stream.hpp"
#include "expert_wide.hpp"
#include "products_host.hpp"
#include "../../include/drama3_moe.h"

using namespace d3;

namespace {
int check_bits(const std::string& what, int32_t bits) {
  return bits == 4 || bits == 8 ? 0 : fail(what + ": bits must be 4 or 8");
}
}  // namespace

extern "C" int d3_mx_gemv(const void* codes, const void* scale, int32_t bits, int32_t rows, const int64_t* ids,
                          int32_t pairs, const void* w, const void* w_scale, int32_t E, int32_t N, int32_t K,
                          int32_t swiglu, int32_t out_bf16, void* out, void* stream) {
  ExpertProduct a{};
  a.x = (const uint8_t*)codes, a.x_scale = (const uint8_t*)scale, a.x_rows = rows, a.ids = ids, a.pairs = pairs;
  a.w = (const uint8_t*)w, a.w_scale = (const uint8_t*)w_scale, a.E = E, a.N = N, a.out = out;
  if (const int rc = check_bits("d3_mx_gemv", bits)) return rc;
  if (const int rc = check_product("d3_mx_gemv", a, K, MX_BLOCK, true, swiglu, false)) return rc;
  if (pairs == 0) return 0;
  a.stages = mx_stages(K), a.per_row = pairs / rows;
  if (bits == 4) launch_gemv<Mx<4>>(a, swiglu, out_bf16, (hipStream_t)stream);
  else launch_gemv<Mx<8>>(a, swiglu, out_bf16, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_mx_gemv launch");
}

extern "C" int d3_mx_grouped(const void* codes, const void* scale, int32_t bits, int32_t rows, const int64_t* order,
                             int32_t k, int32_t pairs, const int32_t* groups, int32_t n_groups, const void* w,
                             const void* w_scale, int32_t E, int32_t N, int32_t K, int32_t swiglu, int32_t out_bf16,
                             void* out, void* stream) {
  ExpertProduct a{};
  a.x = (const uint8_t*)codes, a.x_scale = (const uint8_t*)scale, a.x_rows = rows, a.order = order, a.k = k;
  a.pairs = pairs, a.groups = groups, a.n_groups = n_groups;
  a.w = (const uint8_t*)w, a.w_scale = (const uint8_t*)w_scale, a.E = E, a.N = N, a.out = out;
  if (const int rc = check_bits("d3_mx_grouped", bits)) return rc;
  if (const int rc = check_product("d3_mx_grouped", a, K, MX_BLOCK, true, swiglu, true)) return rc;
  if (pairs == 0) return 0;
  a.stages = mx_stages(K);
  if (bits == 4) launch_grouped<Mx<4>>(a, swiglu, out_bf16, (hipStream_t)stream);
  else launch_grouped<Mx<8>>(a, swiglu, out_bf16, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_mx_grouped launch");
}
