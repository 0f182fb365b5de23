// Probabilities of logits, and verification of drafted tokens against them.
//
// Probabilities follow q8op_sample's weights (sample(), src/sample.mojo:15-59,
// before its nucleus): w = exp((l - max) / temp) for the logits >= max - 16,
// else 0; p = w / sum w.  temp <= 0: the greedy choice, 1 at the first maximum.
//
// Verification (speculative sampling): the draft x behind row r is kept while
// u_r q_r(x) < p_r(x); at the first refused row a token is drawn from
// max(p - q, 0), after the last kept one from the last row's p.  A token drawn
// this way is distributed as p.  Products, differences and sums are 64-bit: a
// 128,000-entry cumulative sum in 32 bits would move the drawn token in about
// one of a hundred draws.
#include "q8_kernels.h"

#include <math.h>

namespace q8 {

__device__ __forceinline__ void vf_best(float& bv, int& bi, float ov, int oi) {
  if (ov > bv || (ov == bv && oi < bi)) {
    bv = ov;
    bi = oi;
  }
}

__global__ void __launch_bounds__(1024) k_probs(const float* __restrict__ logits, int n, int64_t ld, float temp,
                                                float* __restrict__ out, int64_t ldo) {
  __shared__ float s_v[32];
  __shared__ int s_i[32];
  __shared__ double s_d[32];
  const float* x = logits + (int64_t)blockIdx.x * ld;
  float* y = out + (int64_t)blockIdx.x * ldo;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (x[i] > -INFINITY) vf_best(bv, bi, x[i], i);
  for (int o = 16; o > 0; o >>= 1)
    vf_best(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  if (lane == 0) {
    s_v[w] = bv;
    s_i[w] = bi;
  }
  __syncthreads();
  for (int k = 0; k < 32; ++k) vf_best(bv, bi, s_v[k], s_i[k]);
  if (bi == 0x7fffffff) bi = 0;  // nothing above -inf: as q8op_argmax
  if (!(temp > 0.f) || bv == -INFINITY) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) y[i] = i == bi ? 1.f : 0.f;
    return;
  }
  const float low = bv - 16.f;
  auto weight = [&](float l) {
    if (!(l >= low)) return 0.f;
    return l == bv ? 1.f : expf((l - bv) / temp);
  };
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) sum += (double)weight(x[i]);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_d[w] = sum;
  __syncthreads();
  sum = 0.0;
  for (int k = 0; k < 32; ++k) sum += s_d[k];
  const float inv = (float)(1.0 / sum);
  for (int i = threadIdx.x; i < n; i += blockDim.x) y[i] = weight(x[i]) * inv;
}

// One CTA per sequence.
__global__ void __launch_bounds__(1024) k_verify(const float* __restrict__ p, int64_t ldp, const float* __restrict__ q,
                                                 int64_t ldq, int q_rows, const int32_t* __restrict__ ids,
                                                 const int32_t* __restrict__ starts, int rows, int S, int n,
                                                 const float* __restrict__ u, int32_t* __restrict__ taken,
                                                 int32_t* __restrict__ tokens) {
  __shared__ double s_d[1024];
  __shared__ int s_i[32];
  __shared__ int s_stop, s_filled;
  const int b = blockIdx.x, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int r0 = min(max(starts[b], 0), rows), r1 = min(max(starts[b + 1], r0), rows);
  if (r1 <= r0) {
    if (threadIdx.x == 0) taken[b] = 0;
    return;
  }
  // q has no row for a sequence's last row: row r's is r - (sequences with rows before b)
  int filled = 0;
  for (int k = threadIdx.x; k < b; k += blockDim.x)
    filled += min(max(starts[k + 1], 0), rows) > min(max(starts[k], 0), rows);
  if (threadIdx.x == 0) {
    s_stop = r1 - 1;
    s_filled = 0;
  }
  __syncthreads();
  if (filled) atomicAdd(&s_filled, filled);
  __syncthreads();
  const int q0 = -s_filled;  // r + q0: the row of q
  for (int r = r0 + threadIdx.x; r < r1 - 1; r += blockDim.x) {
    const int x = ids[r + 1];
    bool keep = false;
    if (x >= 0 && x < n && (!q || r + q0 < q_rows)) {
      const double qx = q ? (double)q[(int64_t)(r + q0) * ldq + x] : 1.0;
      keep = (double)u[r] * qx < (double)p[(int64_t)r * ldp + x];
    }
    if (!keep) atomicMin(&s_stop, r);
  }
  __syncthreads();
  const int stop = s_stop;
  const float* pr = p + (int64_t)stop * ldp;
  const float* qr = q && stop < r1 - 1 && stop + q0 < q_rows ? q + (int64_t)(stop + q0) * ldq : nullptr;
  const int gone = !q && stop < r1 - 1 ? ids[stop + 1] : -1;
  const int per = (n + blockDim.x - 1) / blockDim.x;
  const int lo = min(n, (int)threadIdx.x * per), hi = min(n, lo + per);
  bool rest = true;  // weights of the residual; false: of p itself
  auto weight = [&](int i) {
    double a = (double)pr[i];
    if (rest && qr) a -= (double)qr[i];
    if (rest && i == gone) a = 0.0;
    return a > 0.0 ? a : 0.0;
  };
  double before = 0.0, total = 0.0, mine = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    mine = 0.0;
    for (int i = lo; i < hi; ++i) mine += weight(i);
    __syncthreads();
    s_d[threadIdx.x] = mine;
    __syncthreads();
    before = total = 0.0;
    for (int k = 0; k < (int)blockDim.x; ++k) {
      if (k == (int)threadIdx.x) before = total;
      total += s_d[k];
    }
    if (total > 0.0 || !rest) break;
    rest = false;  // p == q: the refusal was a rounding's
  }
  // first index whose cumulative weight exceeds u total; if rounding leaves
  // none, the last index with a weight
  const double r = (double)u[r1 - 1] * total;
  int first = 0x7fffffff, last = -1;
  double cum = before;
  for (int i = lo; i < hi; ++i) {
    const double a = weight(i);
    if (!(a > 0.0)) continue;
    cum += a;
    last = i;
    if (first == 0x7fffffff && cum > r) first = i;
  }
  first = __reduce_min_sync(0xffffffffu, first);
  last = __reduce_max_sync(0xffffffffu, last);
  __shared__ int s_l[32];
  if (lane == 0) {
    s_i[wid] = first;
    s_l[wid] = last;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 0; k < 32; ++k) {
      first = min(first, s_i[k]);
      last = max(last, s_l[k]);
    }
    taken[b] = stop - r0;
    tokens[stop] = first != 0x7fffffff ? first : max(last, 0);
  }
  for (int i = r0 + threadIdx.x; i < r1; i += blockDim.x)
    if (i != stop) tokens[i] = i < stop ? ids[i + 1] : -1;
}

}  // namespace q8

using namespace q8;

extern "C" int q8op_probs(const float* logits, int64_t rows, int64_t n, int64_t ld, float temp, float* out,
                          int64_t ldo, void* stream) {
  Q8_CHECK_ARG(rows >= 0 && rows <= (1 << 24) && n >= 1 && n <= (1 << 28) && ld >= n && ldo >= n,
               "q8op_probs: bad shape");
  Q8_CHECK_ARG(!isnan(temp), "q8op_probs: temp must not be NaN");
  if (rows == 0) return Q8_OK;
  Q8_CHECK_ARG(logits && out, "q8op_probs: null pointer");
  k_probs<<<(int)rows, 1024, 0, (cudaStream_t)stream>>>(logits, (int)n, ld, temp, out, ldo);
  return launch_check("k_probs");
}

extern "C" int q8op_verify(const float* p, int64_t ldp, const float* q, int64_t ldq, int64_t q_rows,
                           const int32_t* ids, const int32_t* seq_start, int64_t rows, int64_t S, int64_t n,
                           const float* u, int32_t* n_accepted, int32_t* tokens, void* stream) {
  Q8_CHECK_ARG(rows >= 0 && rows <= (1 << 24) && S >= 0 && S <= (1 << 20) && n >= 1 && n <= (1 << 28) && ldp >= n &&
                   (!q || (ldq >= n && q_rows >= 0 && q_rows <= (1 << 24))),
               "q8op_verify: bad shape");
  if (S == 0) return Q8_OK;
  Q8_CHECK_ARG(seq_start && n_accepted && (rows == 0 || (p && ids && u && tokens)), "q8op_verify: null pointer");
  k_verify<<<(int)S, 1024, 0, (cudaStream_t)stream>>>(p, ldp, q, ldq, (int)q_rows, ids, seq_start, (int)rows, (int)S, (int)n, u,
                                                      n_accepted, tokens);
  return launch_check("k_verify");
}
