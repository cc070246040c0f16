// The checks that the expert products' C entries make before a launch.
#pragma once
#include "ragged.hpp"

#include <string>

namespace d3 {
int fail(const std::string& msg);
int hip_fail(hipError_t err, const char* what);

inline bool off16(const void* p) { return (uintptr_t)p & 15u; }

// sizes and pointers of a product over `pairs` rows; K % k_step == 0. 0: fine, and there is something to do unless
// a.pairs is 0.
inline int check_product(const std::string& what, const ExpertProduct& a, int K, int k_step, bool scaled, bool swiglu,
                         bool grouped) {
  if (a.pairs < 0 || a.x_rows < 0 || a.E < 0) return fail(what + ": negative sizes");
  if (K < 1 || K % k_step) return fail(what + ": K must be a positive multiple of " + std::to_string(k_step));
  if (a.N < 1 || a.N % (swiglu ? 32 : 16)) return fail(what + ": N must be a positive multiple of " + (swiglu ? "32" : "16"));
  if ((int64_t)a.N * K > INT32_MAX) return fail(what + ": an expert of more than 2^31 weights");
  if (a.pairs == 0) return 0;
  if (a.x_rows < 1 || a.E < 1) return fail(what + ": pairs without rows or experts");
  if (!a.x || !a.w || !a.out || (scaled && (!a.x_scale || !a.w_scale))) return fail(what + ": null pointer");
  if (off16(a.x) || off16(a.w) || off16(a.out) || (scaled && (((uintptr_t)a.x_scale & 7u) || ((uintptr_t)a.w_scale & 3u))))
    return fail(what + ": rows, weights and out must be 16-byte aligned (scales 8 and 4)");
  if (grouped) {
    if (!a.groups || a.n_groups < 1) return fail(what + ": pairs without groups");
    if (a.k < 1) return fail(what + ": k must be positive");
    // (groups may overlap: what the passes are counted in)
    if (((int64_t)a.pairs / 16 + 1) * a.n_groups > INT32_MAX) return fail(what + ": too many pairs and groups for one launch");
    if (!a.order && a.x_rows < a.pairs) return fail(what + ": fewer rows than pairs, and no order");
  } else {
    if (!a.ids) return fail(what + ": null pointer");
    if (a.pairs % a.x_rows) return fail(what + ": pairs must be a multiple of the rows");
  }
  // workgroups: at most one column of 32 weight rows a pass, at most one pass a pair
  if ((int64_t)(a.N / 32 + 1) * a.pairs > INT32_MAX) return fail(what + ": too many pairs for one launch");
  return 0;
}

}  // namespace d3
