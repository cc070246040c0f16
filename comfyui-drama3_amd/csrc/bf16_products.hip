// Expert products on banks of bfloat16 weights, as a checkpoint holds them before conversion: [E * N, K] row by row,
// bfloat16 rows, float32 sums on the matrix cores.
#include "expert_stream.hpp"
#include "expert_wide.hpp"
#include "products_host.hpp"
#include "../../include/drama3_moe.h"

using namespace d3;

extern "C" int d3_bf16_gemv(const void* x, int32_t rows, const int64_t* ids, int32_t pairs, const void* w, int32_t E,
                            int32_t N, int32_t K, int32_t swiglu, int32_t out_bf16, void* out, void* stream) {
  ExpertProduct a{};
  a.x = (const uint8_t*)x, a.x_rows = rows, a.ids = ids, a.pairs = pairs;
  a.w = (const uint8_t*)w, a.E = E, a.N = N, a.stages = K / 64, a.out = out;
  if (const int rc = check_product("d3_bf16_gemv", a, K, 64, false, swiglu, false)) return rc;
  if (pairs == 0) return 0;
  a.per_row = pairs / rows;
  launch_gemv<Bf16>(a, swiglu, out_bf16, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_bf16_gemv launch");
}

extern "C" int d3_bf16_grouped(const void* x, int32_t rows, const int64_t* order, int32_t k, int32_t pairs,
                               const int32_t* groups, int32_t n_groups, const void* w, int32_t E, int32_t N, int32_t K,
                               int32_t swiglu, int32_t out_bf16, void* out, void* stream) {
  ExpertProduct a{};
  a.x = (const uint8_t*)x, a.x_rows = rows, a.order = order, a.k = k, a.pairs = pairs;
  a.groups = groups, a.n_groups = n_groups;
  a.w = (const uint8_t*)w, a.E = E, a.N = N, a.stages = K / 64, a.out = out;
  if (const int rc = check_product("d3_bf16_grouped", a, K, 64, false, swiglu, true)) return rc;
  if (pairs == 0) return 0;
  launch_grouped<Bf16>(a, swiglu, out_bf16, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, "d3_bf16_grouped launch");
}
