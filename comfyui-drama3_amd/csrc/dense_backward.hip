// The gradients of the gated feed-forward: C entries.
#include "dense_host.hpp"
#include "../../include/drama3_moe.h"

using namespace d3;

extern "C" int d3_gated_ffn_backward(const d3_gated_ffn_backward_desc* d, void* stream) {
  const std::string what = "d3_gated_ffn_backward";
  if (!d) return fail(what + ": null descriptor");
  const int T = d->T, H = d->H, I = d->I, O = d->O;
  if (T < 0 || T > MAX_ROWS) return fail(what + ": 0 to 2^30 rows");
  if (H < 8 || H % 8 || I < 8 || I % 8 || O < 8 || O % 8) return fail(what + ": widths must be positive multiples of 8");
  if (2 * (int64_t)I * H > INT32_MAX || (int64_t)O * I > INT32_MAX) return fail(what + ": a weight of more than 2^31 elements");
  if (2 * (int64_t)I > MAX_LD || H > MAX_LD || O > MAX_LD) return fail(what + ": widths of more than 2^23");
  if ((int64_t)((T + 15) / 16) * (std::max({2 * I, H, O}) / 8) > INT32_MAX) return fail(what + ": too many rows for one launch");
  if (T == 0) return 0;
  const hipStream_t s = (hipStream_t)stream;
  if (bad_rows(d->dout, O, O) || bad_rows(d->dgate_up_rows, 2 * (int64_t)I, I) || bad_rows(d->down, I, I) || bad_rows(d->pre, 2 * (int64_t)I, I))
    return fail(what + ": null pointer, or one that is not 16-byte aligned");
  if ((d->dx && (bad_rows(d->dx, H, H) || bad_rows(d->gate_up, H, H))) ||
      (d->dgate_up && (bad_rows(d->dgate_up, H, H) || bad_rows(d->x, d->x_stride, H))) ||
      (d->ddown && (bad_rows(d->ddown, I, I) || bad_rows(d->hidden, I, I))))
    return fail(what + ": null pointer, or rows that are not 16-byte aligned or more than 2^23 apart");
  if (d->dx || d->dgate_up) {
    // gradients of gate and up from dhidden = dout . down
    Dense a{};
    a.x = (const uint16_t*)d->dout, a.ldx = O, a.w = (const uint16_t*)d->down, a.ldw = I, a.M = T, a.N = I, a.K = O, a.half = I;
    a.out = (uint16_t*)d->dgate_up_rows, a.ldo = 2 * (int64_t)I, a.pre = (float*)d->pre;
    launch_tiles<true, END_DSWIGLU>(a, s);
  }
  DenseSet set{};
  set.rows = -1;
  if (d->dx) {
    Dense& a = set.product[set.rows = set.count++];
    a.x = (const uint16_t*)d->dgate_up_rows, a.ldx = 2 * (int64_t)I, a.w = (const uint16_t*)d->gate_up, a.ldw = H, a.M = T, a.N = H, a.K = 2 * I;
    a.out = (uint16_t*)d->dx, a.ldo = H;
  }
  if (d->dgate_up) {
    Dense& a = set.product[set.count++];
    a.x = (const uint16_t*)d->dgate_up_rows, a.ldx = 2 * (int64_t)I, a.w = (const uint16_t*)d->x, a.ldw = d->x_stride, a.M = 2 * I, a.N = H, a.K = T;
    a.out = (uint16_t*)d->dgate_up, a.ldo = H;
  }
  if (d->ddown) {
    Dense& a = set.product[set.count++];
    a.x = (const uint16_t*)d->dout, a.ldx = O, a.w = (const uint16_t*)d->hidden, a.ldw = I, a.M = O, a.N = I, a.K = T;
    a.out = (uint16_t*)d->ddown, a.ldo = I;
  }
  if (set.count) launch_dense_set(set, s);
  return launched("d3_gated_ffn_backward launch");
}
