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
  if (a.pre && a.half && ((uintptr_t)a.pre & 15u)) return fail(what + ": pre must be 16-byte aligned");
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
// within 2^-8 of each value's size). Rows without an adapter are not written, nor read later. Two kernels:

// Up to 16 rows: a workgroup takes 16 ranks and an adapter that the rows name (blockIdx.y of them), its 8 waves an eighth of K each.
__global__ void __launch_bounds__(ST_THREADS) lora_inner_stream_kernel(Dense a, const uint16_t* A, const float* alpha) {
  __shared__ f32x4 part[ST_WAVES][1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, c = lane & 15;
  const int r0 = blockIdx.x * 16;
  const int64_t id = lane < a.M ? a.ids[lane] : -1;
  uint64_t open = __ballot(id >= 0 && id < a.adapters), rows = 0;
  int64_t now = 0;
  for (int i = 0; i <= (int)blockIdx.y; i++) {
    if (!open) return;
    now = __shfl(id, __ffsll((unsigned long long)open) - 1);
    rows = __ballot(id == now);
    open &= ~rows;
  }
  const uint16_t* x[1] = {a.x + min(c, a.M - 1) * a.ldx};
  const float scale = alpha[now];
  f32x4 acc[1];
  stream_sums<1, 4>(A + ((size_t)now * a.rank + min(r0 + c, a.rank - 1)) * a.K, x, a.K, wave, acc);
  const f32x4 v = join_waves<1>(part, acc, wave) * scale;
  if (wave == 0 && (rows >> c & 1) && r0 + 4 * q < a.rank) *(i32x2*)(a.out + (size_t)c * a.rank + r0 + 4 * q) = round4(v);
}

// More: tiles of 64 rows and 32 ranks, one adapter that the rows name after the other (blockIdx.z of them at the start, gridDim.z
// apart), all 64 rows multiplied and those of the adapter kept: rows of as many adapters by turns take as many times the work.
// 5000 rows of 12 requests, rank 32, K 2048: 8.0 us; with two workgroups a tile 12.4, and 20.3 with the rows and adapters read
// straight into operands.
__global__ void __launch_bounds__(Thin::THREADS, 2) lora_inner_tile_kernel(Dense a, const uint16_t* A, const float* alpha) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[Thin::LDS];
  static_assert(Thin::TM == 64);
  const int lane = threadIdx.x & 63, m = blockIdx.y * 64 + lane;
  const int64_t id = m < a.M ? a.ids[m] : -1;
  uint64_t open = __ballot(id >= 0 && id < a.adapters);
  for (int i = 0; open; i++) {
    const int64_t now = __shfl(id, __ffsll((unsigned long long)open) - 1);
    a.rows = __ballot(id == now);
    open &= ~a.rows;
    if (i % (int)gridDim.z != (int)blockIdx.z) continue;
    a.w = A + (size_t)now * a.rank * a.K;
    a.alpha = alpha[now];
    __syncthreads();  // (the last adapter's stages are read)
    dense_tile<Thin, false, false, END_INNER, false>(a, blockIdx.y, blockIdx.x, smem);
  }
}

void launch_inner(const Dense& of, const void* A, const float* alpha, hipStream_t stream) {
  Dense a = of;
  a.out = (uint16_t*)of.p, a.ldo = a.N = a.rank, a.ldw = a.K;
  if (a.M <= 16) {
    lora_inner_stream_kernel<<<dim3((a.rank + 15) / 16, a.M), ST_THREADS, 0, stream>>>(a, (const uint16_t*)A, alpha);
  } else {
    // Which adapters a tile of rows names only the device knows: as many workgroups a tile as it may name (64 rows, `adapters`), while
    // they fit the CUs at once (two each), at least two; those without an adapter end at once. A whole call, N 1024, rank 32, 32
    // adapters, by turns and in runs, us: 256 rows 19.7 and 16.2, 300 19.9 and 16.3, 1000 29.4 and 17.5, 5000 148 and 37; two
    // workgroups a tile: 300 rows 98 and 32, 1000 104 and 23, 5000 159 and 37.
    const int ranks = (a.rank + 31) / 32, tiles = (a.M + 63) / 64;
    const int z = std::clamp(512 / std::max<int64_t>((int64_t)ranks * tiles, 1), (int64_t)2, (int64_t)std::max(2, std::min(a.adapters, 64)));
    lora_inner_tile_kernel<<<dim3(ranks, tiles, z), Thin::THREADS, 0, stream>>>(a, (const uint16_t*)A, alpha);
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
