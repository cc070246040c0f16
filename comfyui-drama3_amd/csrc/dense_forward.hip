// The gated feed-forward on bfloat16 weights, and a projection beside its rows' adapters: C entries.
#include "dense_host.hpp"
#include "../../include/drama3_moe.h"

using namespace d3;

namespace {

int check_dense(const std::string& what, const Dense& a) {
  if (a.M < 0) return fail(what + ": negative sizes");
  if (a.K < 8 || a.K % 8 || a.N < 8 || a.N % 8) return fail(what + ": widths must be positive multiples of 8");
  if ((int64_t)a.N * a.K > INT32_MAX) return fail(what + ": a weight of more than 2^31 elements");
  if (a.M == 0) return 0;
  if (bad_rows(a.x, a.ldx, a.K) || bad_rows(a.w, a.ldw, a.K) || bad_rows(a.out, a.ldo, a.half ? a.half : a.N))
    return fail(what + ": null pointer, or rows that are not 16-byte aligned or more than 2^23 apart");
  if ((int64_t)(a.N / 8) * ((a.M + 15) / 16) > INT32_MAX) return fail(what + ": too many rows for one launch");
  return 0;
}

int check_lora(const std::string& what, const Dense& a, const void* A, const float* alpha) {
  if (a.rank < 8 || a.rank % 8 || a.adapters < 0) return fail(what + ": rank must be a positive multiple of 8");
  if (a.M == 0) return 0;
  if (!a.ids || !a.p || (a.adapters && (!A || !a.b || !alpha))) return fail(what + ": null pointer");
  if (((uintptr_t)A | (uintptr_t)a.b | (uintptr_t)a.p) & 15u) return fail(what + ": adapters must be 16-byte aligned");
  if ((int64_t)a.rank * a.K > INT32_MAX || (int64_t)a.N * a.rank > INT32_MAX) return fail(what + ": an adapter of more than 2^31 elements");
  return 0;
}

void launch_inner(const Dense& a, const void* A, const float* alpha, hipStream_t stream) {
  const int ranks = (a.rank + 15) / 16;
  if (a.M <= 256) {
    lora_inner_kernel<1><<<dim3(ranks, (a.M + 15) / 16, 16), ST_THREADS, 0, stream>>>(
        a.x, a.ldx, (const uint16_t*)A, alpha, a.ids, a.M, a.K, a.rank, a.adapters, (uint16_t*)a.p);
  } else {
    lora_inner_kernel<4><<<dim3(ranks, (a.M + 63) / 64, 2), ST_THREADS, 0, stream>>>(
        a.x, a.ldx, (const uint16_t*)A, alpha, a.ids, a.M, a.K, a.rank, a.adapters, (uint16_t*)a.p);
  }
}

}  // namespace

extern "C" int d3_dense(const d3_dense_desc* d, void* stream) {
  if (!d) return fail("d3_dense: null descriptor");
  Dense a{};
  a.x = (const uint16_t*)d->x, a.ldx = d->x_stride, a.w = (const uint16_t*)d->w, a.ldw = d->K;
  a.M = d->T, a.N = d->N, a.K = d->K, a.out = (uint16_t*)d->out, a.pre = d->pre;
  if (d->swiglu) {
    if (d->N % 16) return fail("d3_dense: gate and up rows are multiples of 8 each");
    a.half = d->N / 2;
  }
  a.ldo = d->swiglu ? a.half : a.N;
  if (const int rc = check_dense("d3_dense", a)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  const bool lora = d->adapters > 0;
  if (lora) {
    a.p = (const uint16_t*)d->inner, a.b = (const uint16_t*)d->b, a.ids = d->ids, a.rank = d->rank, a.adapters = d->adapters;
    if (const int rc = check_lora("d3_dense", a, d->a, d->alpha)) return rc;
  }
  if (a.M == 0) return 0;
  if (lora) launch_inner(a, d->a, d->alpha, s);
  if (d->swiglu) {
    if (lora) launch_dense<END_SWIGLU, true>(a, s);
    else launch_dense<END_SWIGLU, false>(a, s);
  } else {
    if (lora) launch_dense<END_ROWS, true>(a, s);
    else launch_dense<END_ROWS, false>(a, s);
  }
  return launched("d3_dense launch");
}
