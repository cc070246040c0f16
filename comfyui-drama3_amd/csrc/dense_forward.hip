// The gated feed-forward on bfloat16 weights, and a projection beside its rows' adapters: C entries.
#include "dense_host.hpp"
#include "../../include/drama3_moe.h"

using namespace d3;

namespace {

int check_dense(const std::string& what, const Dense& a) {
  if (a.M < 0 || a.M > MAX_ROWS) return fail(what + ": 0 to 2^30 rows");
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

// p[m, r] = alpha[a] sum_k x[m, k] A[a, r, k] for the adapter a of each row m, rounded to bf16 (the operand of the second product:
// a relative 2^-9 of what the adapter adds). A workgroup takes 32 ranks and 16 rows, one adapter that they name after the
// other (blockIdx.z of them at the start, gridDim.z apart), so that prompts' rows are read once up to rank 32; its 8 waves
// each take an eighth of K. Rows without an adapter are not written, nor read later.
__global__ void __launch_bounds__(ST_THREADS) lora_inner_kernel(const uint16_t* x, int64_t ldx, const uint16_t* A, const float* alpha,
                                                                const int64_t* ids, int M, int K, int rank, int adapters, uint16_t* p) {
  __shared__ f32x4 part[ST_WAVES][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, c = lane & 15;
  const int m0 = blockIdx.y * 16, r0 = blockIdx.x * 32;
  const int64_t id = lane < 16 && m0 + lane < M ? ids[m0 + lane] : -1;
  uint64_t open = __ballot(id >= 0 && id < adapters);
  const uint16_t* row = x + min(m0 + c, M - 1) * ldx;
  for (int i = 0; open; i++) {
    const int64_t now = __shfl(id, __ffsll((unsigned long long)open) - 1);
    const uint64_t rows = __ballot(id == now);
    open &= ~rows;
    if (i % (int)gridDim.z != (int)blockIdx.z) continue;
    // (here the adapter's two tiles of ranks are the operand that differs from tile to tile, and the rows the one that all share)
    const uint16_t* ranks[2];
#pragma unroll
    for (int t = 0; t < 2; t++) ranks[t] = A + ((size_t)now * rank + min(r0 + 16 * t + c, rank - 1)) * K;
    f32x4 acc[2];
    stream_sums<2>(row, ranks, K, wave, acc);
    // lane (q, c): rows 4 q .. 4 q + 3, rank c
    const f32x4 v = join_waves<2>(part, acc, wave) * alpha[now];
    const int r = r0 + 16 * wave + c;
    if (wave < 2 && r < rank) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (rows >> (4 * q + j) & 1) p[(size_t)(m0 + 4 * q + j) * rank + r] = (uint16_t)f32_to_bf16(v[j]);
    }
    __syncthreads();  // (the sums are read: the next adapter's may take their place)
  }
}

// few rows: a workgroup for every adapter that 16 rows can name; many: two, which is enough where requests' rows follow each other
void launch_inner(const Dense& a, const void* A, const float* alpha, hipStream_t stream) {
  lora_inner_kernel<<<dim3((a.rank + 31) / 32, (a.M + 15) / 16, a.M <= 256 ? 16 : 2), ST_THREADS, 0, stream>>>(
      a.x, a.ldx, (const uint16_t*)A, alpha, a.ids, a.M, a.K, a.rank, a.adapters, (uint16_t*)a.p);
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
