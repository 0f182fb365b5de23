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

#include <algorithm>
#include <cooperative_groups.h>
#include <math.h>
#include <type_traits>

namespace cg = cooperative_groups;

namespace q8 {

constexpr int VF_THREADS = 512;
constexpr int VF_WARPS = VF_THREADS / 32;
constexpr int VF_MAX_CLUSTER = 16;
constexpr int VF_Q = 10;                           // four-logit pieces that a thread of k_probs holds
constexpr int vf_slice(int threads) { return threads * 4 * VF_Q; }  // logits of a row per CTA of k_probs, at most

__device__ __forceinline__ uint32_t vf_map(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ int vf_peer(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(vf_map(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ double vf_peer(const double* p, int rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(vf_map(p, rank)) : "memory");
  return v;
}

// Sum over the warp, the same order on every lane.
__device__ __forceinline__ double vf_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void vf_send(const float* p, int rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(vf_map(p, rank)), "f"(v) : "memory");
}
__device__ __forceinline__ void vf_send(const int* p, int rank, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(vf_map(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void vf_send(const double* p, int rank, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(vf_map(p, rank)), "d"(v) : "memory");
}

// A cluster of CTAs per row, each with a slice of it in registers: logits are
// read once and probabilities written once (8 bytes a logit).  Every warp sends
// its maximum, then its sum, to all CTAs; each adds up all warps' numbers in the
// same order.  Nobody reads from a peer, so that only the sums' barrier is waited
// for at the end.
//
// (l - max) / temp log2(e) + 64 is taken as y + z, y the f32 multiply-add with
// c = ch + cl and z what it lost, so that the exponent's rounding does not grow
// with it: w = 2^y (1 + z ln 2).  The 64 keeps the weights that count, from 2^-96
// to 2^64, among the normal numbers.  Four are added in 32 bits, those sums in 64.
//
// 320 rows of 151,936: 92 us for 389 MB (4.2 TB/s, 0.64 of a copy's rate); two CTAs
// an SM take turns in loading, waiting for one another and storing.  One row of
// 128,256: 5.4 us; CTAs of 256 threads took 6.0 where CTAs of 512 took 8.1.  At 98
// us, sending by st.async took 102 and clusters that stay and load a row ahead 107;
// three CTAs an SM of 13 a row took 109, one of 1024 threads 107 at 92.
template <int THREADS, bool WIDE>  // WIDE: rows to 16 bytes; loads behind a branch each would wait for one another
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    k_probs(const float* logits, int n, int64_t ld, float temp, float ch, float cl, float* out, int64_t ldo,
            int per) {  // out may be logits
  constexpr int WARPS = THREADS / 32;
  __shared__ float s_v[VF_MAX_CLUSTER * WARPS];
  __shared__ int s_i[VF_MAX_CLUSTER * WARPS];
  __shared__ double s_d[VF_MAX_CLUSTER * WARPS];
  cluster_leave();  // that all CTAs have begun
  const cg::cluster_group cluster = cg::this_cluster();
  const int nc = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / nc;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int lo = min(n, rank * per), cnt = min(n, lo + per) - lo;
  const float* src = logits + (int64_t)row * ld + lo;
  float* dst = out + (int64_t)row * ldo + lo;
  const int at = threadIdx.x * 4;  // piece k: at + k * 4 * THREADS
  float v[VF_Q][4];
#pragma unroll
  for (int k = 0; k < VF_Q; ++k) {
    const int i = at + k * 4 * THREADS;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = -INFINITY;
    if constexpr (WIDE) {
      if (i + 4 <= cnt) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(src + i));
        v[k][0] = f.x, v[k][1] = f.y, v[k][2] = f.z, v[k][3] = f.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < cnt) v[k][e] = src[i + e];
    }
  }
  if (WIDE && (cnt & 3)) {
#pragma unroll
    for (int k = 0; k < VF_Q; ++k) {
      const int i = at + k * 4 * THREADS;
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (i + 4 > cnt && i + e < cnt) v[k][e] = src[i + e];
    }
  }
  float bv = -INFINITY;
#pragma unroll
  for (int k = 0; k < VF_Q; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) bv = fmaxf(bv, v[k][e]);  // a NaN is passed over
  bv = warp_max(bv);
  cluster_left();
  if (lane < nc) vf_send(&s_v[rank * WARPS + w], lane, bv);
  cluster_wait_all();
  for (int k = lane; k < nc * WARPS; k += 32) bv = fmaxf(bv, s_v[k]);
  bv = warp_max(bv);
  if (!(temp > 0.f) || bv == -INFINITY) {
    int bi = 0x7fffffff;
#pragma unroll
    for (int k = VF_Q - 1; k >= 0; --k)
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[k][e] == bv && bv > -INFINITY) bi = lo + at + k * 4 * THREADS + e;
    bi = __reduce_min_sync(0xffffffffu, bi);
    if (lane < nc) vf_send(&s_i[rank * WARPS + w], lane, bi);
    cluster_wait_all();
    for (int k = lane; k < nc * WARPS; k += 32) bi = min(bi, s_i[k]);
    bi = __reduce_min_sync(0xffffffffu, bi);
    if (bi == 0x7fffffff) bi = 0;  // nothing above -inf: as q8op_argmax
    for (int i = threadIdx.x; i < cnt; i += THREADS) dst[i] = lo + i == bi ? 1.f : 0.f;
    return;
  }
  double sum = 0.0;
  if (bv == INFINITY) {  // the infinite ones alone
#pragma unroll
    for (int k = 0; k < VF_Q; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = v[k][e] == bv ? 1.f : 0.f;
      sum += (double)((v[k][0] + v[k][1]) + (v[k][2] + v[k][3]));
    }
  } else {
    const float low = fmaxf(bv - 16.f, bv - 160.f / ch);  // 2^-160 is 0, and y stays finite
    const uint64_t top2 = f2_pack(-bv, -bv), ch2 = f2_pack(ch, ch), cl2 = f2_pack(cl, cl), up = f2_pack(64.f, 64.f),
                   minus = f2_pack(-1.f, -1.f), ln2 = f2_pack(0.69314718f, 0.69314718f);
#pragma unroll
    for (int k = 0; k < VF_Q; ++k) {
      uint64_t p[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float l0 = v[k][2 * e], l1 = v[k][2 * e + 1];
        const uint64_t d = f2_add(f2_pack(l0, l1), top2), y = f2_fma(d, ch2, up);
        // y - 64 is exact for y >= 32; below, weights under 2^-32 of the largest are off by up to 1.3e-6
        const uint64_t z = f2_fma(d, cl2, f2_fma(d, ch2, f2_fma(y, minus, up)));
        float p0, p1;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(f2_lo(y)));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(f2_hi(y)));
        p[e] = f2_pack(p0, p1);
        p[e] = f2_fma(f2_mul(p[e], ln2), z, p[e]);
        v[k][2 * e] = l0 >= low ? f2_lo(p[e]) : 0.f;
        v[k][2 * e + 1] = l1 >= low ? f2_hi(p[e]) : 0.f;
      }
      const uint64_t two = f2_add(f2_pack(v[k][0], v[k][1]), f2_pack(v[k][2], v[k][3]));
      sum += (double)(f2_lo(two) + f2_hi(two));
    }
  }
  sum = vf_warp_sum(sum);
  if (lane < nc) vf_send(&s_d[rank * WARPS + w], lane, sum);
  cluster_wait_all();
  sum = 0.0;
  for (int k = lane; k < nc * WARPS; k += 32) sum += s_d[k];
  sum = vf_warp_sum(sum);
  const float inv = (float)(1.0 / sum);
#pragma unroll
  for (int k = 0; k < VF_Q; ++k) {
    const int i = at + k * 4 * THREADS;
    if (WIDE && i + 4 <= cnt) {
      __stcs(reinterpret_cast<float4*>(dst + i),
             make_float4(v[k][0] * inv, v[k][1] * inv, v[k][2] * inv, v[k][3] * inv));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < cnt) dst[i + e] = v[k][e] * inv;
    }
  }
}

// A cluster of CTAs per sequence; all of them find the refused row, then each
// adds up a slice of its weights, in segments of 128 per warp, so that the
// drawn index is found in one segment: p and q rows are read once.  64 sequences,
// 151,936 columns, 78 MB: 16.1 us from the L2, 24 from memory (3.2 TB/s), a launch
// and four steps that wait for one another; one sequence 7.0 us.  Segments of 512
// took 19.2 at 18.5.
constexpr int VF_SEG = 128;

__global__ void __launch_bounds__(VF_THREADS) k_verify(const float* __restrict__ p, int64_t ldp,
                                                       const float* __restrict__ q, int64_t ldq, int q_rows,
                                                       const int32_t* __restrict__ ids,
                                                       const int32_t* __restrict__ starts, int rows, int n,
                                                       const float* __restrict__ u, int32_t* __restrict__ taken,
                                                       int32_t* __restrict__ tokens, int per) {
  extern __shared__ double s_seg[];  // the slice's segments, in order
  __shared__ double s_sum;
  __shared__ int s_stop, s_filled, s_last;
  const cg::cluster_group cluster = cg::this_cluster();
  const int nc = cluster.num_blocks(), rank = cluster.block_rank(), b = blockIdx.x / nc;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int r0 = min(max(starts[b], 0), rows), r1 = min(max(starts[b + 1], r0), rows);
  if (r1 <= r0) {
    if (rank == 0 && threadIdx.x == 0) taken[b] = 0;
    return;
  }
  const float draw = u[r1 - 1];
  // q has no row for a sequence's last row: row r's is r - (sequences with rows before b)
  int filled = 0;
  if (q)
    for (int k = threadIdx.x; k < b; k += VF_THREADS)
      filled += min(max(starts[k + 1], 0), rows) > min(max(starts[k], 0), rows);
  if (threadIdx.x == 0) {
    s_stop = r1 - 1;
    s_filled = 0;
    s_last = -1;
  }
  __syncthreads();
  filled = __reduce_add_sync(0xffffffffu, filled);
  if (lane == 0 && filled) atomicAdd(&s_filled, filled);
  __syncthreads();
  const int q0 = -s_filled;  // r + q0: the row of q
  for (int r = r0 + threadIdx.x; r < r1 - 1; r += VF_THREADS) {
    const int x = ids[r + 1];
    bool keep = false;
    if (x >= 0 && x < n && (!q || r + q0 < q_rows)) {
      const double w = q ? (double)q[(int64_t)(r + q0) * ldq + x] : 1.0, qx = w < 0.0 ? 0.0 : w;
      keep = (double)u[r] * qx < (double)p[(int64_t)r * ldp + x];  // never with a NaN
    }
    if (!keep) atomicMin(&s_stop, r);
  }
  __syncthreads();
  const int stop = s_stop;
  const float* pr = p + (int64_t)stop * ldp;
  const float* qr = q && stop < r1 - 1 && stop + q0 < q_rows ? q + (int64_t)(stop + q0) * ldq : nullptr;
  int gone = !q && stop < r1 - 1 ? ids[stop + 1] : -1;
  const int lo = min(n, rank * per), hi = min(n, lo + per);
  const int segs = (hi - lo + VF_SEG - 1) / VF_SEG;
  const bool wide = (((uintptr_t)pr | (uintptr_t)qr) & 15) == 0;  // lo is a multiple of VF_SEG
  // the lane's four weights of a segment; HOW 0: p alone, 1: p - q, both by 16 bytes and the
  // segment full, 2: any
  auto weights_of = [&](auto how, int seg, double (&v)[4]) {
    constexpr int HOW = decltype(how)::value;
    const int i = lo + seg * VF_SEG + lane * 4;
    float a[4] = {0.f, 0.f, 0.f, 0.f}, c[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (HOW < 2) {
      const float4 f = *reinterpret_cast<const float4*>(pr + i);
      a[0] = f.x, a[1] = f.y, a[2] = f.z, a[3] = f.w;
      if constexpr (HOW == 1) {
        const float4 h = *reinterpret_cast<const float4*>(qr + i);
        c[0] = h.x, c[1] = h.y, c[2] = h.z, c[3] = h.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < hi) {
          a[e] = pr[i + e];
          if (qr) c[e] = qr[i + e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double d = (double)a[e] - (c[e] < 0.f ? 0.0 : (double)c[e]);
      v[e] = d > 0.0 && i + e != gone ? d : 0.0;
    }
  };
  const int plain = wide ? (hi - lo) / VF_SEG : 0;  // segments that loads of 16 bytes can take
  double total = 0.0, before = 0.0;
  for (;;) {
    int last = -1;
    auto add_up = [&](auto how, int s) {
      double v[4];
      weights_of(how, s, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] > 0.0) last = lo + s * VF_SEG + lane * 4 + e;
      const double sum = vf_warp_sum((v[0] + v[1]) + (v[2] + v[3]));
      if (lane == 0) s_seg[s] = sum;
    };
    int s = wid;  // a branch around the loads, not one at each
    if (qr) {
#pragma unroll 4
      for (; s < plain; s += VF_WARPS) add_up(std::integral_constant<int, 1>(), s);
    } else {
#pragma unroll 4
      for (; s < plain; s += VF_WARPS) add_up(std::integral_constant<int, 0>(), s);
    }
    for (; s < segs; s += VF_WARPS) add_up(std::integral_constant<int, 2>(), s);
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0 && last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    // running sums of the segments by one warp, a stretch of them per lane
    if (wid == 0) {
      const int each = (segs + 31) / 32;
      double mine = 0.0;
      for (int k = lane * each; k < min(segs, (lane + 1) * each); ++k) s_seg[k] = mine += s_seg[k];
      double up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += y;
      }
      double base = __shfl_up_sync(0xffffffffu, up, 1);
      if (lane == 0) base = 0.0;
      for (int k = lane * each; k < min(segs, (lane + 1) * each); ++k) s_seg[k] += base;
      __syncwarp();
      if (lane == 0) s_sum = segs ? s_seg[segs - 1] : 0.0;
    }
    cluster_wait_all();
    total = before = 0.0;
    for (int k = 0; k < nc; ++k) {
      if (k == rank) before = total;
      total += vf_peer(&s_sum, k);
    }
    if (total > 0.0 || !(qr || gone >= 0)) break;
    // p <= q everywhere: the refusal was a rounding's, p itself is drawn from
    cluster_wait_all();
    qr = nullptr;
    gone = -1;
  }
  int tail = -1;  // the last index with a weight, for rank 0
  if (rank == 0 && wid == 0) tail = __reduce_max_sync(0xffffffffu, lane < nc ? vf_peer(&s_last, lane) : -1);
  __syncwarp();
  cluster_leave();
  // the first index whose cumulative weight exceeds u total lies in the CTA
  // that reaches beyond it; if rounding leaves none, the last index with a weight
  const double r = fmax((double)draw * total, 0.0);  // a draw that is none gives the first weight
  if (wid == 0) {
    const bool mine = before <= r && before + s_sum > r;
    if (mine) {
      // first segment that reaches beyond r
      int a = 0, z = segs - 1;
      while (a < z) {
        const int mid = (a + z) / 2;
        if (before + s_seg[mid] > r) z = mid;
        else a = mid + 1;
      }
      // the lanes of the running sums add in different orders, so a segment without a weight can begin beyond r by a
      // rounding: the weights that got there lie before it
      double v[4], cum;
      for (;; --a) {
        weights_of(std::integral_constant<int, 2>(), a, v);
        cum = ((v[0] + v[1]) + v[2]) + v[3];
        if (a == 0 || __any_sync(0xffffffffu, cum > 0.0)) break;
      }
      double up = cum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += y;
      }
      double base = __shfl_up_sync(0xffffffffu, up, 1);
      if (lane == 0) base = 0.0;
      base += before + (a ? s_seg[a - 1] : 0.0);
      int first = 0x7fffffff, last = -1;
      double run = 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        run += v[e];
        if (!(v[e] > 0.0)) continue;
        last = lo + a * VF_SEG + lane * 4 + e;
        if (first == 0x7fffffff && base + run > r) first = last;
      }
      first = __reduce_min_sync(0xffffffffu, first);
      last = __reduce_max_sync(0xffffffffu, last);
      if (lane == 0) tokens[stop] = first != 0x7fffffff ? first : last;
    }
    if (rank == 0 && !(r < total) && lane == 0) tokens[stop] = max(tail, 0);
  }
  if (rank == nc - 1) {
    if (threadIdx.x == 0) taken[b] = stop - r0;
    for (int i = r0 + threadIdx.x; i < r1; i += VF_THREADS)
      if (i != stop) tokens[i] = i < stop ? ids[i + 1] : -1;
  }
  cluster_left();  // nobody leaves while its sums are read
}

// CTAs per row: what `least` asks for, more while the GPU has room and a CTA keeps 2048 entries.
static int vf_cluster(int64_t rows, int64_t n, int64_t least, int64_t room) {
  int c = 1;
  while (c < VF_MAX_CLUSTER && (c < least || (rows * c * 2 <= room && n / c > 4096))) c *= 2;
  return c;
}

template <auto kern>
struct VfKernel {
  static constexpr auto value = kern;
};

template <auto kern, typename... Args>
static int vf_launch(const char* what, int64_t rows, int c, int threads, size_t smem, int most, cudaStream_t st,
                     Args... args) {
  static bool ready[64] = {false};  // of this kernel
  int dev = 0;
  Q8_CUDA(cudaGetDevice(&dev));
  if (!ready[dev & 63]) {
    Q8_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    Q8_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ready[dev & 63] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)c, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * c));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launch_status(what, cudaLaunchKernelEx(&cfg, kern, args...));
}

}  // namespace q8

using namespace q8;

constexpr int64_t VF_PROBS_MAX = (int64_t)VF_MAX_CLUSTER * vf_slice(VF_THREADS);  // 327,680
constexpr int VF_SEGS = 20000;                         // sums that a CTA of k_verify holds
constexpr int64_t VF_SLICE = (int64_t)VF_SEGS * VF_SEG;  // and the columns of them
constexpr int64_t VF_VERIFY_MAX = VF_MAX_CLUSTER * VF_SLICE;

extern "C" int q8op_probs(const float* logits, int64_t rows, int64_t n, int64_t ld, float temp, float* out,
                          int64_t ldo, void* stream) {
  Q8_CHECK_ARG(rows >= 0 && rows <= (1 << 24) && n >= 1 && n <= VF_PROBS_MAX && ld >= n && ldo >= n,
               "q8op_probs: bad shape (%lld rows of %lld, at most %lld)", (long long)rows, (long long)n,
               (long long)VF_PROBS_MAX);
  Q8_CHECK_ARG(!isnan(temp), "q8op_probs: temp must not be NaN");
  if (rows == 0) return Q8_OK;
  Q8_CHECK_ARG(logits && out, "q8op_probs: null pointer");
  // one round of small CTAs if they fit, else large ones
  const int64_t c_fine = (n + vf_slice(256) - 1) / vf_slice(256);
  const bool fine = c_fine <= VF_MAX_CLUSTER && rows * c_fine <= 4 * num_sms();
  const int slice = vf_slice(fine ? 256 : VF_THREADS);
  const int c = vf_cluster(rows, n, (n + slice - 1) / slice, 2 * num_sms());
  const int per = (int)((n + c - 1) / c + 3) & ~3;
  const double scale = std::min(1.4426950408889634 / (double)temp, 3e38);  // a subnormal temp: still no 0 x infinity
  const float ch = (float)scale, cl = (float)(scale - (double)ch);
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = (((uintptr_t)logits | (uintptr_t)out | (uintptr_t)(ld * 4) | (uintptr_t)(ldo * 4)) & 15) == 0;
  auto go = [&](auto kernel, int threads) {
    return vf_launch<decltype(kernel)::value>("k_probs", rows, c, threads, 0, 0, st, logits, (int)n, ld, temp,
                                              ch, cl, out, ldo, per);
  };
  if (fine) return wide ? go(VfKernel<k_probs<256, true>>{}, 256) : go(VfKernel<k_probs<256, false>>{}, 256);
  return wide ? go(VfKernel<k_probs<VF_THREADS, true>>{}, VF_THREADS)
              : go(VfKernel<k_probs<VF_THREADS, false>>{}, VF_THREADS);
}

extern "C" int q8op_verify(const float* p, int64_t ldp, const float* q, int64_t ldq, int64_t q_rows,
                           const int32_t* ids, const int32_t* seq_start, int64_t rows, int64_t S, int64_t n,
                           const float* u, int32_t* n_accepted, int32_t* tokens, void* stream) {
  Q8_CHECK_ARG(rows >= 0 && rows <= (1 << 24) && S >= 0 && S <= (1 << 20) && n >= 1 && n <= VF_VERIFY_MAX &&
                   ldp >= n && (!q || (ldq >= n && q_rows >= 0 && q_rows <= (1 << 24))),
               "q8op_verify: bad shape");
  if (S == 0) return Q8_OK;
  Q8_CHECK_ARG(seq_start && n_accepted && (rows == 0 || (p && ids && u && tokens)), "q8op_verify: null pointer");
  const int c = vf_cluster(S, n, (n + VF_SLICE - 1) / VF_SLICE, 2 * num_sms());
  const int per = (int)(((n + c - 1) / c + VF_SEG - 1) / VF_SEG * VF_SEG);
  return vf_launch<k_verify>("k_verify", S, c, VF_THREADS, (size_t)(per / VF_SEG) * 8, VF_SEGS * 8, (cudaStream_t)stream, p, ldp, q,
                   ldq, (int)q_rows, ids, seq_start, (int)rows, (int)n, u, n_accepted, tokens, per);
}
