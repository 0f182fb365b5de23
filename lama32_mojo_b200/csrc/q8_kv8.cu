// 8-bit paged KV cache: append and read back.  Layout and packing of a call's
// rows: q8_kv8.cuh.  The f32 cache's append is k_rope_kv (q8_ops.cu).
#include "q8_kernels.h"
#include "q8_kv8.cuh"

#include <math.h>

namespace q8 {

int kv8_check(const char* what, const q8_kv8_pages* kv, const int32_t* seq_start, const int32_t* ctx, int64_t S,
              int64_t rows, const int32_t* block_table, int max_pages) {
  const bool any = S > 0 && rows > 0;  // an empty tensor's address is null
  Q8_CHECK_ARG(kv && kv->k && kv->v && kv->k_scale && kv->v_scale && (!any || (seq_start && ctx && block_table)),
               "%s: null pointer", what);
  Q8_CHECK_ARG(kv->head_dim == 64 || kv->head_dim == 128, "%s: head_dim %d unsupported (64/128)", what,
               kv->head_dim);
  Q8_CHECK_ARG(kv->page > 0 && kv->page % KV8_BLOCK == 0 && kv->page <= (1 << 20),
               "%s: page size %d is not a multiple of %d", what, kv->page, KV8_BLOCK);
  Q8_CHECK_ARG(kv->num_pages > 0 && kv->num_pages < ((int64_t)1 << 31) && kv->n_kv > 0 && kv->n_kv <= 65535,
               "%s: bad pages (%lld pages, %d kv heads)", what, (long long)kv->num_pages, kv->n_kv);
  Q8_CHECK_ARG(kv->num_pages * kv->n_kv * (kv->page / KV8_BLOCK) < ((int64_t)1 << 31), "%s: 2^31 blocks or more",
               what);
  Q8_CHECK_ARG((((uintptr_t)kv->k | (uintptr_t)kv->v) & 31) == 0, "%s: codes must be 32-byte aligned", what);
  Q8_CHECK_ARG(S >= 0 && S <= (1 << 20) && rows >= 0 && rows <= (1 << 24) && max_pages > 0,
               "%s: bad shape (%lld sequences, %lld rows, %d table columns)", what, (long long)S, (long long)rows,
               max_pages);
  return Q8_OK;
}

// round(x / s), ties to even, within +-127: the quotient of the real numbers,
// not of their f32 rounding.  r - |x - r s| stays exact: x - r s is a multiple
// of the smaller ulp of x and s and at most about s, so the FMA does not round.
// s > 0; x finite.
__device__ __forceinline__ int kv8_code(float x, float s) {
  float r = rintf(__fdiv_rn(x, s));
  if (!(fabsf(r) <= 127.f)) return x < 0.f ? -127 : 127;  // a scale below the normal range
  const float d = fmaf(-r, s, x);
  const float two = 2.f * fabsf(d);
  if (two > s || (two == s && ((int)r & 1))) r += d > 0.f ? 1.f : -1.f;
  return max(-127, min(127, (int)r));
}

// round(c s0 / s1) for a code that stays while its block's scale grows; the
// products fit 64-bit floats exactly.
__device__ __forceinline__ int kv8_rescale(int c, float s0, float s1) {
  int r = (int)rintf((float)c * __fdiv_rn(s0, s1));
  const double d = (double)c * (double)s0 - (double)r * (double)s1;
  const double two = 2.0 * fabs(d);
  if (two > (double)s1 || (two == (double)s1 && (r & 1))) r += d > 0.0 ? 1 : -1;
  return r;
}

// k or v rows of one call
struct Kv8Rows {
  const void* x;
  int64_t ld;
};

// One warp per (block of 16 positions, kv head, k or v); lane l holds dims
// l*HD/32 .. of every new token of the block.  Slots number the touched
// blocks: sequence b's start at starts[b]/16 + 2b, which leaves room for the
// n/16 + 2 blocks that n rows can touch.
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_kv8_append(Kv8Rows kr, Kv8Rows vr, int rows, const int32_t* __restrict__ starts,
                                                    const int32_t* __restrict__ ctx, int S, q8_kv8_pages kv,
                                                    const int32_t* __restrict__ table, int max_pages) {
  constexpr int E = HD / 32;
  const int slot = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int b = threadIdx.x; b < S; b += blockDim.x) before += min(max(starts[b], 0), rows) / KV8_BLOCK + 2 * b <= slot;
  __shared__ int s_cnt;
  if (threadIdx.x == 0) s_cnt = 0;
  __syncthreads();
  if (before) atomicAdd(&s_cnt, before);
  __syncthreads();
  const int b = s_cnt - 1;
  if (b < 0) return;
  const Kv8Seq sq = kv8_seq(starts, ctx, b, rows);
  if (sq.n <= 0) return;
  const int64_t first = max(sq.pos0, (int64_t)0);
  const int64_t blk = first / KV8_BLOCK + (slot - (sq.row0 / KV8_BLOCK + 2 * b));
  const int64_t lo = max(blk * KV8_BLOCK, first);
  const int64_t hi = min((blk + 1) * KV8_BLOCK, sq.pos0 + sq.n);
  if (lo >= hi) return;
  const int pg = kv8_page(table + (int64_t)b * max_pages, max_pages, kv.num_pages, kv.page, lo);
  if (pg < 0) return;
  const int in = (int)(lo % KV8_BLOCK), cnt = (int)(hi - lo);
  const int row = sq.row0 + (int)(lo - sq.pos0);
  const int unit = blockIdx.y * (blockDim.x >> 5) + warp;
  if (unit >= 2 * kv.n_kv) return;
  const int h = unit >> 1;
  const bool isv = unit & 1;
  const Kv8Rows src = isv ? vr : kr;
  const int64_t cell = (int64_t)pg * kv.n_kv + h;
  const int tok0 = (int)((blk * KV8_BLOCK) % kv.page);
  int8_t* codes = (isv ? kv.v : kv.k) + (cell * kv.page + tok0) * HD + lane * E;
  float* scale = (isv ? kv.v_scale : kv.k_scale) + cell * (kv.page / KV8_BLOCK) + tok0 / KV8_BLOCK;
  const T* x = (const T*)src.x + (int64_t)row * src.ld + h * HD + lane * E;
  float v[KV8_BLOCK][E];
  float high = 0.f;
#pragma unroll
  for (int i = 0; i < KV8_BLOCK; ++i) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[i][e] = i < cnt ? kv8_load(x + (int64_t)i * src.ld + e) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < KV8_BLOCK; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (v[i][e] != v[i][e]) v[i][e] = 0.f;  // NaN
      const float a = fabsf(v[i][e]);
      if (a != INFINITY) high = fmaxf(high, a);
    }
  high = warp_max(high);
  const float old = in > 0 ? *scale : 0.f;
  const float s = fmaxf(old, __fdiv_rn(high, 127.f));
  __syncwarp();
  if (s != old && in > 0) {
    for (int i = 0; i < in; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e)
        codes[i * HD + e] = old > 0.f ? (int8_t)kv8_rescale(codes[i * HD + e], old, s) : (int8_t)0;
  }
  if (lane == 0) *scale = s;
#pragma unroll
  for (int i = 0; i < KV8_BLOCK; ++i) {
    if (i >= cnt) break;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float a = v[i][e];
      int c = 0;
      if (fabsf(a) == INFINITY) c = a < 0.f ? -127 : 127;
      else if (s > 0.f) c = kv8_code(a, s);
      codes[(in + i) * HD + e] = (int8_t)c;
    }
  }
}

// One CTA per row of the call; rows without a page read as zeros.
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_read(int rows, const int32_t* __restrict__ starts,
                                                  const int32_t* __restrict__ ctx, int S, q8_kv8_pages kv,
                                                  const int32_t* __restrict__ table, int max_pages,
                                                  float* __restrict__ ko, float* __restrict__ vo) {
  const int t = blockIdx.x;
  int before = 0;
  for (int b = threadIdx.x; b < S; b += blockDim.x) before += min(max(starts[b], 0), rows) <= t;
  __shared__ int s_cnt;
  if (threadIdx.x == 0) s_cnt = 0;
  __syncthreads();
  if (before) atomicAdd(&s_cnt, before);
  __syncthreads();
  const int b = s_cnt - 1;
  if (b < 0) return;
  const Kv8Seq sq = kv8_seq(starts, ctx, b, rows);
  if (t >= sq.row0 + sq.n) return;  // behind the last sequence
  const int64_t p = sq.pos0 + (t - sq.row0);
  const int pg = kv8_page(table + (int64_t)b * max_pages, max_pages, kv.num_pages, kv.page, p);
  const int tok = pg < 0 ? 0 : (int)(p % kv.page);
  for (int i = threadIdx.x; i < 2 * kv.n_kv * HD; i += blockDim.x) {
    const bool isv = i >= kv.n_kv * HD;
    const int j = isv ? i - kv.n_kv * HD : i;
    const int h = j / HD, d = j % HD;
    float r = 0.f;
    if (pg >= 0) {
      const int64_t cell = (int64_t)pg * kv.n_kv + h;
      r = (float)(isv ? kv.v : kv.k)[(cell * kv.page + tok) * HD + d] *
          (isv ? kv.v_scale : kv.k_scale)[cell * (kv.page / KV8_BLOCK) + tok / KV8_BLOCK];
    }
    (isv ? vo : ko)[(int64_t)t * kv.n_kv * HD + j] = r;
  }
}

template <typename T>
static int append_run(const Kv8Rows& k, const Kv8Rows& v, int rows, const int32_t* starts, const int32_t* ctx, int S,
                      const q8_kv8_pages& kv, const int32_t* table, int max_pages, cudaStream_t st) {
  const dim3 grid(rows / KV8_BLOCK + 2 * S, ceil_div(2 * kv.n_kv, 8));
  if (kv.head_dim == 64) k_kv8_append<T, 64><<<grid, 256, 0, st>>>(k, v, rows, starts, ctx, S, kv, table, max_pages);
  else k_kv8_append<T, 128><<<grid, 256, 0, st>>>(k, v, rows, starts, ctx, S, kv, table, max_pages);
  return launch_check("k_kv8_append");
}

}  // namespace q8

using namespace q8;

extern "C" int q8op_kv8_append(const void* k, int64_t ldk, const void* v, int64_t ldv, int dtype, int64_t rows,
                               const int32_t* seq_start, const int32_t* ctx, int64_t S, const q8_kv8_pages* kv,
                               const int32_t* block_table, int max_pages, void* stream) {
  Q8_TRY(kv8_check("q8op_kv8_append", kv, seq_start, ctx, S, rows, block_table, max_pages));
  Q8_CHECK_ARG(dtype == Q8_F32 || dtype == Q8_BF16 || dtype == Q8_F16, "q8op_kv8_append: bad dtype %d", dtype);
  if (rows == 0 || S == 0) return Q8_OK;
  const int64_t width = (int64_t)kv->n_kv * kv->head_dim;
  Q8_CHECK_ARG(k && v && ldk >= width && ldv >= width, "q8op_kv8_append: k and v rows need %lld elements",
               (long long)width);
  const Kv8Rows kr{k, ldk}, vr{v, ldv};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == Q8_F32)
    return append_run<float>(kr, vr, (int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, st);
  if (dtype == Q8_BF16)
    return append_run<__nv_bfloat16>(kr, vr, (int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, st);
  return append_run<__half>(kr, vr, (int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, st);
}

extern "C" int q8op_kv8_read(const q8_kv8_pages* kv, const int32_t* seq_start, const int32_t* ctx, int64_t S,
                             const int32_t* block_table, int max_pages, float* k, float* v, int64_t rows,
                             void* stream) {
  Q8_TRY(kv8_check("q8op_kv8_read", kv, seq_start, ctx, S, rows, block_table, max_pages));
  if (rows == 0 || S == 0) return Q8_OK;
  Q8_CHECK_ARG(k && v, "q8op_kv8_read: null output");
  cudaStream_t st = (cudaStream_t)stream;
  if (kv->head_dim == 64)
    k_kv8_read<64><<<(int)rows, 256, 0, st>>>((int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, k, v);
  else
    k_kv8_read<128><<<(int)rows, 256, 0, st>>>((int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, k, v);
  return launch_check("k_kv8_read");
}
