// Attention over the 8-bit cache for many query rows per kv head (chunks of
// prompts), on the 5th-generation tensor cores (tcgen05 + TMEM).  The operator
// and its softmax statistics (running M of s + log2(sv), weights e sv): see
// q8_kv8_attn.cu.
//
// A CTA takes 128 rows (tokens x the heads that share a kv head) against key
// tiles of 64 positions, four scale blocks:
//   warps 4-7  load the tile's codes and write them as f16 (exact) into shared
//              memory, rows of 64 dims in the 128-byte swizzle; K is read
//              K-major, V (same layout) MN-major.
//   warp 8     one lane issues S = Q K^T (128 x 64 x hd) into TMEM and, once the
//              weights are there, O += P V (128 x hd x 64), P read from TMEM.
//   warps 0-3  a thread per row: reads its 64 scores from TMEM, keeps M and l,
//              writes P over them.  S / P have two buffers, so the next tile's
//              scores are computed meanwhile.
// p = ph + pl, two products (22 bits; the codes need one f16); f32 rows: q = qh + ql
// too.  4 x 128 x 64 x hd multiply-adds a tile, bf16 / f16 rows 3.
// M moves only when it has grown by more than 1, so that O in TMEM is scaled
// seldom.
//
// Bound.  2 x 1024 f32 rows of 32 heads on 8 of 128, 8000 and 2524 positions: 380 us
// for 159 GFLOP, 319 in f16 products (0.84 PFLOP/s, 0.50 of cuBLAS's bf16 rate, at
// which they take 192 us).  The tensor pipes are busy 40 % of the time, the issue
// slots 52 %: the chain of a tile, codes to f16 to scores to weights to product, is
// what is waited for, with one buffer each for K and V.  bf16 rows, 239 GFLOP in
// products: 383 us (356 with one f16 a weight).
//
// Two CTAs an SM (256 TMEM columns each) cover one another's waits.  Their
// number is fixed; each takes an equal stretch of all units' work and leaves
// partial results where it begins or ends inside a unit (q8_kv8_attn.cu).
// Every wait is bounded (mbar_wait).
#include "q8_kv8_attn.h"

namespace q8 {

constexpr int KT_BLOCKS = KV8_TILE, KT_KEYS = KT_BLOCKS * KV8_BLOCK;
constexpr int KT_THREADS = 288;
constexpr float KT_LIFT = KA_LIFT / 2;  // M lags by up to 1: weights are 2^15 at most
constexpr int KT_FIXED = 512;  // work of beginning and ending a unit, in positions

__device__ __forceinline__ void kt_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void kt_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void kt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One lane of a converged warp.  Products are issued under this predicate rather
// than a lane's number: their descriptors then stay in uniform registers (110
// clocks each otherwise, whatever their size; measured).
__device__ __forceinline__ bool kt_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// Shared-memory matrix descriptors, 128-byte swizzle (layout type 2, version 1),
// atoms of 8 rows x 128 bytes 1024 apart (SBO).  lbo: bytes between the 64-dim
// halves of an MN-major operand.
__device__ __forceinline__ uint64_t kt_desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// d += A B with A from shared memory, and with A from TMEM
__device__ __forceinline__ void kt_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(0));
}
__device__ __forceinline__ void kt_mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
      "r"(ta), "l"(db), "r"(idesc), "r"(acc), "r"(0));
}

__device__ __forceinline__ void kt_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void kt_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void kt_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void kt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The largest score + log2(sv) of a row's tile; left: positions of the tile that the row sees.
template <bool MASKED>
__device__ __forceinline__ float kt_top(uint32_t addr, const float4* sc, float fac, int left) {
  float top = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    float v[32];
    kt_ld32(addr + h * 32, v);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 s = sc[h * 2 + k];
      float bm = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!MASKED || k * 16 + i < left - h * 32) bm = fmaxf(bm, v[k * 16 + i]);
      if (!MASKED || bm > -INFINITY) top = fmaxf(top, fmaf(bm, fac * s.x, s.z));  // masked: no 0 x infinity
    }
  }
  return top;
}

// Scores -> weights, in place; returns their sum before sv.
template <bool MASKED>
__device__ __forceinline__ float kt_weights(uint32_t addr, const float4* sc, float fac, float ref, int left) {
  uint64_t sum = 0ull;
  const uint64_t minus = f2_pack(-1.f, -1.f);
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    float v[32];
    kt_ld32(addr + h * 32, v);
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 s = sc[h * 2 + k];
      const float f = fac * s.x, b = s.z == -INFINITY ? -INFINITY : -ref;  // a missing page: 0 s - infinity
      const uint64_t f2 = f2_pack(f, f), b2 = f2_pack(b, b), w2 = f2_pack(s.y, s.y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int q = k * 16 + 2 * i;
        const uint64_t x = f2_fma(f2_pack(v[q], v[q + 1]), f2, b2);
        float e0 = ka_exp2(f2_lo(x)), e1 = ka_exp2(f2_hi(x));
        if (MASKED) {
          if (q >= left - h * 32) e0 = 0.f;
          if (q + 1 >= left - h * 32) e1 = 0.f;
        }
        const uint64_t e = f2_pack(e0, e1), p = f2_mul(e, w2);
        sum = f2_add(sum, e);
        hi[k * 8 + i] = ka_pack(f2_lo(p), f2_hi(p));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi[k * 8 + i]));
        const uint64_t r = f2_fma(f2_pack(y.x, y.y), minus, p);
        lo[k * 8 + i] = ka_pack(f2_lo(r), f2_hi(r));
      }
    }
    kt_st16(addr + h * 32, hi);
    kt_st16(addr + h * 32 + 16, lo);
  }
  return f2_lo(sum) + f2_hi(sum);
}

// The tensor cores cut sums off where an f32 addition rounds, and O has eight
// additions a tile (four k-steps, two halves of P).  125 tiles in one go came out
// 7.9e-6 too small (relative, least squares over all outputs, scores of deviation
// 1.6).  So O goes into f32 sums in the workspace, which L2 holds, every KT_FLUSH
// tiles.  f32 rows, 8 tiles: errors of whole outputs against 8000 positions, q of
// deviation 0.5, 2 and 8, are 0.8e-6, 1.5e-6 and 0.6e-6, those of elementary f32
// operations 1.6e-6, 2.0e-6 and 1.8e-6.  Scores add the products with ql first: the
// other way round all of them were cut off at the scores' size, 2.5e-6 for q of
// deviation 2.  4 tiles: 417 us for 383 (2 x 1024 rows of 32 heads, 8000 and 2524
// positions; no flush 355, adding in L2 by red.add 481).
// 16-bit rows, 64 tiles: 8.8e-6, a fiftieth of f16's rounding, at no cost to speak of.
template <bool WIDE>
constexpr int KT_FLUSH = WIDE ? 8 : 64;

template <bool WIDE, int HD>
struct KtShape {
  static constexpr int HALVES = HD / 64;            // 64-dim planes of an operand
  static constexpr int QP = KT_ROWS * 128;          // bytes of a plane of q
  static constexpr int Q = QP * HALVES * (WIDE ? 2 : 1);
  static constexpr int KP = KT_KEYS * 128, K = KP * HALVES;
  static constexpr int SMEM = Q + 2 * K + 1024;     // + alignment
  static constexpr int REC = KT_ROWS * (HD + 2), FLUSH = KT_FLUSH<WIDE>;
};

// The units of a CTA's stretch, one after the other.  A unit (group of QT tokens,
// kv head) weighs KT_FIXED + the positions that its last token sees; units are
// ordered by (sequence, group, kv head).  Every warp walks for itself.
struct KtWalk {
  int b;
  int64_t off, left;
  // the unit
  KaUnit u;
  int t0, n;  // its tiles here
  bool begins, ends;

  static __device__ __forceinline__ int64_t sum_to(const Kv8AttnArgs& a, int64_t base, int64_t i) {
    return (int64_t)a.kv.n_kv * a.hgroups * (i * (KT_FIXED + base) + a.QT * (i * (i + 1) / 2));
  }
  static __device__ __forceinline__ int64_t weight(const Kv8AttnArgs& a, int b) {
    const Kv8Seq sq = kv8_seq(a.starts, a.ctx, b, a.rows);
    return sum_to(a, max(sq.pos0, (int64_t)0), (sq.n + a.QT - 1) / a.QT);
  }

  __device__ __forceinline__ bool next(const Kv8AttnArgs& a) {
    while (left > 0 && b < a.S) {
      const Kv8Seq sq = kv8_seq(a.starts, a.ctx, b, a.rows);
      const int64_t base = max(sq.pos0, (int64_t)0);
      const int groups = (sq.n + a.QT - 1) / a.QT;
      const int64_t w = sum_to(a, base, groups);
      while (off < w && left > 0) {
        int gi = 0;  // the last group whose sum_to is not beyond off
        for (int hi = groups; hi - gi > 1;) {
          const int mid = (gi + hi) / 2;
          if (sum_to(a, base, mid) <= off) gi = mid;
          else hi = mid;
        }
        const int64_t each = KT_FIXED + base + (int64_t)(gi + 1) * a.QT, rest = off - sum_to(a, base, gi);
        const int head = (int)(rest / each);
        const int64_t w0 = rest - head * each, take = min(left, each - w0);
        ends = w0 + take == each;
        u = ka_unit(a, sq, head, gi * a.QT);
        const int tiles = (u.nblk + KT_BLOCKS - 1) / KT_BLOCKS;
        t0 = (int)min((int64_t)tiles, max(w0 - KT_FIXED, (int64_t)0) / KT_KEYS);
        const int t1 = ends ? tiles : (int)min((int64_t)tiles, max(w0 + take - KT_FIXED, (int64_t)0) / KT_KEYS);
        begins = w0 <= KT_FIXED || t0 == 0;
        n = t1 - t0;
        off += take;
        left -= take;
        if (t1 > 0 || ends) return true;  // else the next CTA begins it
      }
      off = 0;
      ++b;
    }
    return false;
  }
};

template <bool WIDE, int HD>
__global__ void __launch_bounds__(KT_THREADS, 2) k_kv8_attn_tc(Kv8AttnArgs a) {
  using Sh = KtShape<WIDE, HD>;
  constexpr int HALVES = Sh::HALVES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sq_ = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // q | k | v
  uint8_t *sk_ = sq_ + Sh::Q, *sv_ = sk_ + Sh::K;
  __shared__ __align__(8) uint64_t qfull, kfull, kfree, vfull, pvdone[2], sfull[2], pfull[2], scfull[4];
  __shared__ uint32_t s_tmem;
  __shared__ float s_fac[KT_ROWS], s_ms[KT_ROWS];  // s_ms: M of the flushed sums, which lie as [dim / 4][row]
  __shared__ float4 s_sc[4][KT_BLOCKS];  // sk, sv KT_LIFT, its part of M (-inf: no page)
  __shared__ int64_t s_scan[KT_THREADS / 32], s_at;
  __shared__ int s_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();

  if (threadIdx.x == 0) {
    mbar_init(&qfull, 4);
    mbar_init(&kfull, 4);
    mbar_init(&kfree, 1);
    mbar_init(&vfull, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&pvdone[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&scfull[i], 1);
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&s_tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  kt_fence_before();
  __syncthreads();
  kt_fence_after();
  const uint32_t tmem = s_tmem, tmem_o = tmem + 2 * KT_KEYS;

  // where the CTA's stretch begins
  const int c = blockIdx.x, nc = gridDim.x;
  int64_t all = 0, mine = 0;
  for (int b = threadIdx.x; b < a.S; b += KT_THREADS) all += mine = KtWalk::weight(a, b);
  int64_t total;
  ka_scan(all, s_scan, &total);
  const int64_t at = total / nc * c + total % nc * c / nc, end = total / nc * (c + 1) + total % nc * (c + 1) / nc;
  if (threadIdx.x == 0) a.work_meta[2 * c] = a.work_meta[2 * c + 1] = make_int4(-1, 0, 0, 0);
  int64_t before = 0;
  for (int b0 = 0; b0 < a.S && at < end; b0 += KT_THREADS) {
    const int b = b0 + threadIdx.x;
    if (a.S > KT_THREADS) mine = b < a.S ? KtWalk::weight(a, b) : 0;
    int64_t sum;
    const int64_t to = before + ka_scan(mine, s_scan, &sum);
    if (to > at && to - mine <= at) {
      s_b = b;
      s_at = at - (to - mine);
    }
    before += sum;
    if (before > at) break;
  }
  __syncthreads();
  KtWalk w;
  w.b = at < end ? s_b : 0;
  w.off = at < end ? s_at : 0;
  w.left = end - at;

  // T counts tiles, U units with tiles: the phases of all barriers.  No role waits for
  // another but through them; q's buffer is free once the scores of a unit's
  // last tile have been read, O once the softmax warps have taken it, before
  // they announce the next unit's first weights.  A softmax warp may pass over
  // pvdone of a tile: two barriers in turn keep it from taking the one before
  // for the one that it waits for (the scores of tile t come after O of t - 2).
  uint32_t T = 0;
  if (warp < 4) {
    // ---- softmax, a thread per row
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int r = threadIdx.x;
    const int64_t room = (int64_t)a.max_pages * a.kv.page;
    const bool aligned = (((uintptr_t)a.q | (uintptr_t)(a.ldq * (WIDE ? 4 : 2))) & 15) == 0;
    const bool wide_out = (((uintptr_t)a.out | (uintptr_t)(a.ldo * (WIDE ? 4 : 2))) & 15) == 0;
    while (w.next(a)) {
      const int nrow = w.u.toks * a.GH;
      // q into shared memory: a warp its 32 rows, eight at a time, a lane HD / 32 dims of each
      constexpr int E = HD / 32;
#pragma unroll 1
      for (int i0 = 0; i0 < 32 && w.n > 0; i0 += 8) {
        float x[8][E];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = warp * 32 + i0 + i;
#pragma unroll
          for (int e = 0; e < E; ++e) x[i][e] = 0.f;
          if (row >= nrow || row % a.GH >= w.u.heads) continue;
          const int64_t at_q = (int64_t)(w.u.row0 + row / a.GH) * a.ldq + (w.u.head0 + row % a.GH) * HD + lane * E;
          if constexpr (WIDE) {
            const float* p = (const float*)a.q + at_q;
            if (E == 4 && aligned) {
              const float4 f = *reinterpret_cast<const float4*>(p);
              x[i][0] = f.x, x[i][1] = f.y, x[i][E - 2] = f.z, x[i][E - 1] = f.w;
            } else {
#pragma unroll
              for (int e = 0; e < E; ++e) x[i][e] = p[e];
            }
          } else {
            const uint16_t* p = (const uint16_t*)a.q + at_q;
            uint32_t u[E / 2];
            if (E == 4 && aligned) {
              const uint2 f = *reinterpret_cast<const uint2*>(p);
              u[0] = f.x, u[E / 2 - 1] = f.y;
            } else {
#pragma unroll
              for (int e = 0; e < E / 2; ++e) u[e] = p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
            }
#pragma unroll
            for (int e = 0; e < E / 2; ++e) {
              const float2 f = __half22float2(*reinterpret_cast<__half2*>(&u[e]));
              x[i][2 * e] = a.dtype == Q8_BF16 ? __uint_as_float(u[e] << 16) : f.x;
              x[i][2 * e + 1] = a.dtype == Q8_BF16 ? __uint_as_float(u[e] & 0xffff0000u) : f.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = warp * 32 + i0 + i;
          // the largest |q| into [2^14, 2^15): times 2^k, k from its exponent, at most 126
          unsigned top = 0u;
#pragma unroll
          for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
          top = __reduce_max_sync(0xffffffffu, top);
          const int ex = top >> 23, k = top == 0u || ex == 255 ? 0 : min(141 - ex, 126);
          const float up = __uint_as_float((unsigned)(127 + k) << 23);
          if (lane == 0)
            s_fac[row] = 1.4426950408889634f / (HD == 64 ? 8.f : 11.313708498984761f) *
                         __uint_as_float((unsigned)(127 - k) << 23);
          uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            const float y0 = x[i][2 * e] * up, y1 = x[i][2 * e + 1] * up;
            hi[e] = ka_pack(y0, y1);
            const float2 f = __half22float2(*reinterpret_cast<__half2*>(&hi[e]));
            lo[e] = ka_pack(y0 - f.x, y1 - f.y);
          }
          const int dim = lane * E;
          uint8_t* to = sq_ + (dim >> 6) * Sh::QP + row * 128 + ((((dim >> 3) & 7) ^ (row & 7)) << 4) + (dim & 7) * 2;
          if constexpr (E == 4) {
            *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[E / 2 - 1]);
            if (WIDE) *reinterpret_cast<uint2*>(to + HALVES * Sh::QP) = make_uint2(lo[0], lo[E / 2 - 1]);
          } else {
            *reinterpret_cast<uint32_t*>(to) = hi[0];
            if (WIDE) *reinterpret_cast<uint32_t*>(to + HALVES * Sh::QP) = lo[0];
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0 && w.n > 0) kt_arrive(&qfull);

      float m = -INFINITY, l = 0.f;
      const float fac = s_fac[r];
      const int lim = r < nrow ? (int)min(max(w.u.pos0 + r / a.GH + 1, (int64_t)0), room) : 0;
      const int seen = (int)min(max(w.u.pos0 + 1, (int64_t)0), room);  // by the first token: no tile before needs a mask
      for (int j = 0; j < w.n; ++j) {
        const uint32_t t = T + j, at_s = tmem + lanes + (t & 1) * KT_KEYS;
        const int p0 = (w.t0 + j) * KT_KEYS, left = lim - p0;
        const bool masked = p0 > seen - KT_KEYS;
        mbar_wait(&scfull[t & 3], (t >> 2) & 1);
        mbar_wait(&sfull[t & 1], (t >> 1) & 1);
        kt_fence_after();
        const float top = masked ? kt_top<true>(at_s, s_sc[t & 3], fac, left)
                                 : kt_top<false>(at_s, s_sc[t & 3], fac, left);
        float alpha = 1.f;
        const bool grew = top > m + 1.f || (m == -INFINITY && top > -INFINITY);
        if (grew) {
          alpha = ka_lower<false>(l, m - top);
          m = top;
        }
        if (j > 0 && j % Sh::FLUSH == 0) {  // PV of this tile begins O anew
          float4* kept = reinterpret_cast<float4*>(a.work + (int64_t)(2 * gridDim.x + blockIdx.x) * Sh::REC) + r;
          const bool add = j > Sh::FLUSH;
          const float beta = add && s_ms[r] > -INFINITY ? ka_exp2(s_ms[r] - m) : 0.f;
          s_ms[r] = m;
          mbar_wait(&pvdone[(t - 1) & 1], ((t - 1) >> 1) & 1);
          kt_fence_after();
#pragma unroll 1
          for (int h = 0; h < HD / 16; ++h, kept += 4 * KT_ROWS) {
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = add ? __ldcg(kept + i * KT_ROWS) : make_float4(0.f, 0.f, 0.f, 0.f);
            float v[16];
            kt_ld16(tmem_o + lanes + h * 16, v);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              __stcg(kept + i * KT_ROWS, make_float4(fmaf(y[i].x, beta, v[4 * i] * alpha), fmaf(y[i].y, beta, v[4 * i + 1] * alpha),
                                                     fmaf(y[i].z, beta, v[4 * i + 2] * alpha),
                                                     fmaf(y[i].w, beta, v[4 * i + 3] * alpha)));
          }
        } else if (j > 0 && __any_sync(0xffffffffu, grew)) {
          mbar_wait(&pvdone[(t - 1) & 1], ((t - 1) >> 1) & 1);  // O is up to date
          kt_fence_after();
#pragma unroll 1
          for (int h = 0; h < HD / 32; ++h) {
            float v[32];
            kt_ld32(tmem_o + lanes + h * 32, v);
            uint32_t x[2][16];
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i >> 4][i & 15] = __float_as_uint(v[i] * alpha);
            kt_st16(tmem_o + lanes + h * 32, x[0]);
            kt_st16(tmem_o + lanes + h * 32 + 16, x[1]);
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        l += masked ? kt_weights<true>(at_s, s_sc[t & 3], fac, ref, left)
                    : kt_weights<false>(at_s, s_sc[t & 3], fac, ref, left);
        kt_wait_st();
        kt_fence_before();
        __syncwarp();
        if (lane == 0) kt_arrive(&pfull[t & 1]);
      }
      T += w.n;

      // results
      const bool whole = w.begins && w.ends, live = r < nrow && r % a.GH < w.u.heads;
      float* rec = a.work + (int64_t)(2 * c + (w.begins ? 1 : 0)) * Sh::REC;
      if (w.n > 0) {
        mbar_wait(&pvdone[(T - 1) & 1], ((T - 1) >> 1) & 1);
        kt_fence_after();
      }
      const float beta = w.n > Sh::FLUSH && s_ms[r] > -INFINITY ? ka_exp2(s_ms[r] - m) : 0.f;
      const float4* kept = reinterpret_cast<const float4*>(a.work + (int64_t)(2 * nc + c) * Sh::REC) + r;
      const float scale = whole ? (l > 0.f ? 1.f / (KT_LIFT * l) : 0.f * l) : KA_LIFT / KT_LIFT;
      const int64_t o0 = (int64_t)(w.u.row0 + r / a.GH) * a.ldo + (int64_t)(w.u.head0 + r % a.GH) * HD;
#pragma unroll 1
      for (int h = 0; h < HD / 32; ++h) {
        float v[32];
        if (w.n > 0) {
          kt_ld32(tmem_o + lanes + h * 32, v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        if (w.n > Sh::FLUSH) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 y = __ldcg(kept + (h * 8 + i) * KT_ROWS);
            v[4 * i] = fmaf(y.x, beta, v[4 * i]), v[4 * i + 1] = fmaf(y.y, beta, v[4 * i + 1]);
            v[4 * i + 2] = fmaf(y.z, beta, v[4 * i + 2]), v[4 * i + 3] = fmaf(y.w, beta, v[4 * i + 3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= scale;
        if (!whole) {
          if (r < nrow) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(rec + r * HD + h * 32 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        } else if (live) {
          if (WIDE && wide_out) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>((float*)a.out + o0 + h * 32 + i) =
                  make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          } else if (!WIDE && wide_out) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t u[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) u[k] = ka_pack16(a.dtype, v[i + 2 * k], v[i + 2 * k + 1]);
              *reinterpret_cast<uint4*>((uint16_t*)a.out + o0 + h * 32 + i) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) ka_store<WIDE>(a, o0 + h * 32 + i, v[i]);
          }
        }
      }
      if (!whole) {
        rec[KT_ROWS * HD + r] = m;
        rec[KT_ROWS * HD + KT_ROWS + r] = l;
        if (threadIdx.x == 0)
          a.work_meta[2 * c + (w.begins ? 1 : 0)] =
              make_int4(w.u.row0, w.u.head0, w.u.toks | w.u.heads << 16, w.ends);
      }
      kt_fence_before();
      __syncwarp();  // s_fac is written again
    }
  } else if (warp < 8) {
    // ---- codes to f16
    constexpr int CPR = HD / 16, STEP = 128 / CPR, NI = KT_KEYS / STEP;
    const int ct = threadIdx.x - 128, qd = ct % CPR, r0 = ct / CPR, ppb = a.kv.page / KV8_BLOCK;
    while (w.next(a)) {
      const int n = w.n;
      if (n <= 0) continue;
      const int32_t* trow = a.table + (int64_t)w.u.b * a.max_pages;
      uint4 kc[NI], vc[NI];
      // lanes 0-3: the block of a tile, by page column and block within the page
      int blk = w.t0 * KT_BLOCKS + lane, col = blk / ppb, in = blk % ppb;
      const int last = min(w.u.nblk, (w.t0 + n) * KT_BLOCKS);
      auto look_up = [&]() { return lane < KT_BLOCKS && blk < last ? trow[col] : -1; };
      auto step = [&]() {
        blk += KT_BLOCKS;
        in += KT_BLOCKS;
        while (in >= ppb) in -= ppb, ++col;
      };
      auto id_of = [&](int e, int in_) {  // pool number, -1: no page
        return e >= 0 && e < a.kv.num_pages ? (e * a.kv.n_kv + w.u.h) * ppb + in_ : -1;
      };
      auto load = [&](uint4 (&cs)[NI], const int8_t* codes, int ids) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = r0 + i * STEP, id = __shfl_sync(0xffffffffu, ids, row >> 4);
          cs[i] = make_uint4(0u, 0u, 0u, 0u);
          if (id >= 0)
            cs[i] = __ldg(reinterpret_cast<const uint4*>(codes + (int64_t)id * (KV8_BLOCK * HD) + (row & 15) * HD +
                                                         qd * 16));
        }
      };
      auto put = [&](uint8_t* plane0, const uint4 (&cs)[NI]) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = r0 + i * STEP;
          const uint32_t wd[4] = {cs[i].x ^ 0x80808080u, cs[i].y ^ 0x80808080u, cs[i].z ^ 0x80808080u,
                                  cs[i].w ^ 0x80808080u};
          uint4 x[2];
          x[0] = make_uint4(ka_f16(wd[0], 0x5140), ka_f16(wd[0], 0x5342), ka_f16(wd[1], 0x5140), ka_f16(wd[1], 0x5342));
          x[1] = make_uint4(ka_f16(wd[2], 0x5140), ka_f16(wd[2], 0x5342), ka_f16(wd[3], 0x5140), ka_f16(wd[3], 0x5342));
          uint8_t* to = plane0 + (qd >> 2) * Sh::KP + row * 128;
          const int c0 = (2 * qd) & 7, first = (qd >> 2) & 1;  // the planes' lanes take turns: no bank twice
          *reinterpret_cast<uint4*>(to + (((c0 + first) ^ (row & 7)) << 4)) = first ? x[1] : x[0];
          *reinterpret_cast<uint4*>(to + (((c0 + 1 - first) ^ (row & 7)) << 4)) = first ? x[0] : x[1];
        }
      };
      // the fence holds up later loads: they are issued before it
      auto done = [&](uint64_t* bar) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) kt_arrive(bar);
      };
      float sk = 0.f, sv = 0.f;
      auto scales = [&](int id) {
        if (warp != 4) return;
        sk = id >= 0 ? a.kv.k_scale[id] : 0.f;
        sv = id >= 0 ? a.kv.v_scale[id] : 0.f;
      };
      auto scales_out = [&](uint32_t t, int id) {
        if (warp != 4) return;
        if (lane < KT_BLOCKS)
          s_sc[t & 3][lane] = make_float4(sk, sv * KT_LIFT,
                                          id >= 0 ? fmaxf(__log2f(sv), KA_LEAST) - KA_DOWN : -INFINITY, 0.f);
        __syncwarp();
        if (lane == 0) kt_arrive(&scfull[t & 3]);
      };
      // of tiles j (V), j + 1 (K) and, by its table entry, j + 2
      const int id0 = id_of(look_up(), in);
      step();
      int id1 = id_of(look_up(), in);
      step();
      int e2 = look_up(), in2 = in;
      load(kc, a.kv.k, id0);
      load(vc, a.kv.v, id0);
      scales(id0);
      mbar_wait(&kfree, (T & 1) ^ 1);  // K of the first tile
      scales_out(T, id0);
      put(sk_, kc);
      load(kc, a.kv.k, id1);
      scales(id1);
      done(&kfull);
      for (int j = 0; j < n; ++j) {  // K of tile j + 1, then V of tile j; their registers are loaded again at once
        const uint32_t t = T + j;
        const int id2 = id_of(e2, in2);
        step();
        in2 = in;
        if (j + 1 < n) {
          mbar_wait(&kfree, t & 1);
          scales_out(t + 1, id1);
          put(sk_, kc);
          e2 = look_up();
          load(kc, a.kv.k, id2);
          scales(id2);
          done(&kfull);
        }
        mbar_wait(&pvdone[(t - 1) & 1], ((t - 1) >> 1) & 1);
        put(sv_, vc);
        load(vc, a.kv.v, id1);
        done(&vfull);
        id1 = id2;
      }
      T += n;
    }
  } else {
    // ---- products: f32 sums (bit 4), f16 operands, M = 128; V is MN-major (bit 16)
    const uint32_t is = (1u << 4) | ((uint32_t)(KT_KEYS >> 3) << 17) | ((uint32_t)(KT_ROWS >> 4) << 24);
    const uint32_t io = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(KT_ROWS >> 4) << 24);
    const uint64_t dq = kt_desc(smem_u32(sq_), 16), dk = kt_desc(smem_u32(sk_), 16),
                   dv = kt_desc(smem_u32(sv_), Sh::KP);
    for (uint32_t U = 0; w.next(a);) {
      const int n = w.n;
      if (n <= 0) continue;
      mbar_wait(&qfull, U & 1);
      ++U;
      for (int j = 0; j <= n; ++j) {
        const uint32_t t = T + j;
        if (j < n) {  // scores of tile j
          mbar_wait(&kfull, t & 1);
          kt_fence_after();
          const uint32_t d = tmem + (t & 1) * KT_KEYS;
          if (kt_elect()) {
#pragma unroll
            for (int x = WIDE ? 1 : 0; x >= 0; --x)  // the small halves first: little of their sums is cut off
#pragma unroll
              for (int k = 0; k < HD / 16; ++k)  // 16 dims: 32 bytes further inside the swizzle atom
                kt_mma_ss(d, dq + (x * HALVES + (k >> 2)) * (Sh::QP >> 4) + (k & 3) * 2,
                          dk + (k >> 2) * (Sh::KP >> 4) + (k & 3) * 2, is, x != (WIDE ? 1 : 0) || k != 0);
            kt_commit(&kfree);
            kt_commit(&sfull[t & 1]);
          }
          __syncwarp();
        }
        if (j > 0) {  // outputs of the tile before
          const uint32_t p = t - 1;
          mbar_wait(&vfull, p & 1);
          mbar_wait(&pfull[p & 1], (p >> 1) & 1);
          kt_fence_after();
          if (kt_elect()) {
#pragma unroll
            for (int x = 1; x >= 0; --x)
#pragma unroll
              for (int k = 0; k < KT_KEYS / 16; ++k)  // 16 positions: two atoms further
                kt_mma_ts(tmem_o, tmem + (p & 1) * KT_KEYS + (k >> 1) * 32 + x * 16 + (k & 1) * 8, dv + k * (2048 >> 4),
                          io, x == 0 || k != 0 || (j - 1) % Sh::FLUSH != 0);
            kt_commit(&pvdone[p & 1]);
          }
          __syncwarp();
        }
      }
      T += n;
    }
  }
  kt_fence_before();
  __syncthreads();
  if (warp == 8) {
    kt_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem));
  }
}

int kv8_attn_tc_ctas() { return 2 * num_sms(); }

template <bool WIDE, int HD>
static int tc_run(const Kv8AttnArgs& a, int ctas, cudaStream_t st) {
  using Sh = KtShape<WIDE, HD>;
  static bool ready[64] = {false};
  int dev = 0;
  Q8_CUDA(cudaGetDevice(&dev));
  if (!ready[dev & 63]) {
    Q8_CUDA(cudaFuncSetAttribute(k_kv8_attn_tc<WIDE, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
    ready[dev & 63] = true;
  }
  k_kv8_attn_tc<WIDE, HD><<<ctas, KT_THREADS, Sh::SMEM, st>>>(a);
  return launch_check("k_kv8_attn_tc");
}

int kv8_attn_tc(const Kv8AttnArgs& a, int ctas, cudaStream_t st) {
  if (a.kv.head_dim == 128) return a.dtype == Q8_F32 ? tc_run<true, 128>(a, ctas, st) : tc_run<false, 128>(a, ctas, st);
  return a.dtype == Q8_F32 ? tc_run<true, 64>(a, ctas, st) : tc_run<false, 64>(a, ctas, st);
}

int kv8_attn_tc_poll_error() {
  int v = 0;
  Q8_CUDA(cudaMemcpyFromSymbol(&v, g_q8_device_error, sizeof(int)));
  if (v == 0) return Q8_OK;
  const int z = 0;
  Q8_CUDA(cudaMemcpyToSymbol(g_q8_device_error, &z, sizeof(int)));
  set_error("k_kv8_attn_tc: a barrier wait timed out (device status %d)", v);
  return v;
}

}  // namespace q8
