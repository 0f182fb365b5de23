// Causal GQA attention over the 8-bit paged cache (layout: q8_kv8.cuh):
//   o = sum_j softmax_j(sk_j (q.ck_j) / sqrt(hd)) sv_j cv_j
// over the visible positions j of the row's sequence, ck, cv the codes and
// sk, sv their block's scales.
#include "q8_kernels.h"
#include "q8_kv8.cuh"

#include <math.h>

namespace q8 {

// One warp per (row, query head): a lane scores one of 32 keys at a time, the
// warp keeps a running maximum and sum, and each lane owns HD/32 output dims.
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_kv8_attn(const T* __restrict__ q, int64_t ldq, int rows,
                                                  const int32_t* __restrict__ starts, const int32_t* __restrict__ ctx,
                                                  int S, int n_heads, q8_kv8_pages kv,
                                                  const int32_t* __restrict__ table, int max_pages,
                                                  T* __restrict__ out, int64_t ldo) {
  constexpr int E = HD / 32;
  __shared__ float s_q[4][HD];
  __shared__ int s_cnt;
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int b = threadIdx.x; b < S; b += blockDim.x) before += min(max(starts[b], 0), rows) <= t;
  if (threadIdx.x == 0) s_cnt = 0;
  __syncthreads();
  if (before) atomicAdd(&s_cnt, before);
  __syncthreads();
  const int b = s_cnt - 1;
  if (b < 0) return;
  const Kv8Seq sq = kv8_seq(starts, ctx, b, rows);
  const int head = blockIdx.y * 4 + warp;
  if (t >= sq.row0 + sq.n || head >= n_heads) return;
  const int h = head / (n_heads / kv.n_kv);
  const int64_t end = sq.pos0 + (t - sq.row0) + 1;  // visible positions
  const float qs = 1.4426950408889634f / sqrtf((float)HD);
  for (int d = lane; d < HD; d += 32) s_q[warp][d] = (float)q[(int64_t)t * ldq + head * HD + d] * qs;
  __syncwarp();
  const int32_t* trow = table + (int64_t)b * max_pages;
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int64_t j0 = 0; j0 < end; j0 += 32) {
    const int64_t j = j0 + lane;
    const int pg = j < end ? kv8_page(trow, max_pages, kv.num_pages, kv.page, j) : -1;
    float s = -INFINITY, sv = 0.f;
    int64_t off = 0;
    if (pg >= 0) {
      const int64_t cell = (int64_t)pg * kv.n_kv + h;
      const int tok = (int)(j % kv.page);
      off = (cell * kv.page + tok) * HD;
      float acc = 0.f;
      for (int d = 0; d < HD; ++d) acc = fmaf(s_q[warp][d], (float)kv.k[off + d], acc);
      const int64_t si = cell * (kv.page / KV8_BLOCK) + tok / KV8_BLOCK;
      s = acc * kv.k_scale[si];
      sv = kv.v_scale[si];
    }
    const float mn = fmaxf(m, warp_max(s));
    if (mn == -INFINITY) continue;
    const float corr = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float p = s == -INFINITY ? 0.f : exp2f(s - mn);
    m = mn;
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= corr;
    const float w = p * sv;
    for (int i = 0; i < 32; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const int64_t oi = __shfl_sync(0xffffffffu, off, i);
      if (__shfl_sync(0xffffffffu, pg, i) < 0) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(wi, (float)kv.v[oi + lane * E + e], o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    out[(int64_t)t * ldo + head * HD + lane * E + e] = (T)(l > 0.f ? o[e] / l : 0.f);
}

template <typename T>
static int attn_run(const void* q, int64_t ldq, int rows, const int32_t* starts, const int32_t* ctx, int S,
                    int n_heads, const q8_kv8_pages& kv, const int32_t* table, int max_pages, void* out, int64_t ldo,
                    cudaStream_t st) {
  const dim3 grid(rows, ceil_div(n_heads, 4));
  if (kv.head_dim == 64)
    k_kv8_attn<T, 64><<<grid, 128, 0, st>>>((const T*)q, ldq, rows, starts, ctx, S, n_heads, kv, table, max_pages,
                                            (T*)out, ldo);
  else
    k_kv8_attn<T, 128><<<grid, 128, 0, st>>>((const T*)q, ldq, rows, starts, ctx, S, n_heads, kv, table, max_pages,
                                             (T*)out, ldo);
  return launch_check("k_kv8_attn");
}

}  // namespace q8

using namespace q8;

extern "C" int q8op_kv8_attention(const void* q, int64_t ldq, int dtype, int64_t rows, const int32_t* seq_start,
                                  const int32_t* ctx, int64_t S, int n_heads, const q8_kv8_pages* kv,
                                  const int32_t* block_table, int max_pages, void* out, int64_t ldo, void* stream) {
  Q8_TRY(kv8_check("q8op_kv8_attention", kv, seq_start, ctx, S, rows, block_table, max_pages));
  Q8_CHECK_ARG(dtype == Q8_F32 || dtype == Q8_BF16 || dtype == Q8_F16, "q8op_kv8_attention: bad dtype %d", dtype);
  Q8_CHECK_ARG(n_heads > 0 && n_heads % kv->n_kv == 0, "q8op_kv8_attention: %d heads over %d kv heads", n_heads,
               kv->n_kv);
  if (rows == 0 || S == 0) return Q8_OK;
  const int64_t width = (int64_t)n_heads * kv->head_dim;
  Q8_CHECK_ARG(q && out && ldq >= width && ldo >= width, "q8op_kv8_attention: q and out rows need %lld elements",
               (long long)width);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == Q8_F32)
    return attn_run<float>(q, ldq, (int)rows, seq_start, ctx, (int)S, n_heads, *kv, block_table, max_pages, out, ldo,
                           st);
  if (dtype == Q8_BF16)
    return attn_run<__nv_bfloat16>(q, ldq, (int)rows, seq_start, ctx, (int)S, n_heads, *kv, block_table, max_pages,
                                   out, ldo, st);
  return attn_run<__half>(q, ldq, (int)rows, seq_start, ctx, (int)S, n_heads, *kv, block_table, max_pages, out, ldo,
                          st);
}
