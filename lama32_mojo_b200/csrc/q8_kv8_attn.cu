// Causal GQA attention over the 8-bit paged cache (layout: q8_kv8.cuh):
//   o = sum_j softmax_j(sk_j (q.ck_j) / sqrt(hd)) sv_j cv_j
// over the visible positions j of the row's sequence, ck, cv the codes and
// sk, sv their block's scales.
//
// k_kv8_attn: a CTA takes a group of query rows that share a kv head (QT
// tokens of a sequence x the heads of the group) and a stretch of the
// sequence; its warps take 16-position blocks in turn, with no barrier between
// them.  A block is exactly one m16 tile of mma.sync: keys are the A operand
// (16 positions x hd), query rows the B columns, so one pass over the codes
// serves all rows of the group.
//   S^T[16 x cols] = K[16 x hd] q^T      O^T[hd x cols] += V^T[hd x 16] P^T
// f32 rows: q becomes three signed 8-bit digits, q = s (65536 a + 256 b + c)
// with s = max|q| / (127 65536) (23 bits of the row's largest element), one
// column each, and the scores are exact integer products (m16n8k32) of the
// codes as they are; P is split into two f16 halves (22 bits).  bf16 / f16 rows:
// q scaled by a power of two to the top of the f16 range, one column, the codes
// as f16 (exact); P is one f16.
// The order of a dot product's terms is free, so lane (g, t) = (lane / 4,
// lane % 4) reads its operand bytes straight from the cache rows: of K a
// quarter of rows g and g + 8, of V the g-th eighth of rows 2t, 2t + 1, 2t + 8,
// 2t + 9 (output row g of tile m is dim (hd/8) g + 2m, row g + 8 the next
// one).  No shared memory, no barrier: a block's registers are loaded again as
// soon as its products are issued, and wait there while the others work.  P^T
// becomes the B operand by movmatrix.
//
// Softmax: base 2, running maximum M of s + log2(sv) rather than of s: the
// weights that meet the codes are e sv, e = 2^(s - M), so they stay within
// (0, 1] whatever the blocks' scales are, and l = sum e is kept against the same
// M (a sv of 0 counts as 2^-100 in M).  They are lifted by 2^15 to the top of the
// f16 range, whose smallest step, 2^-24, is then 2^-39 of the row's largest one.
//
// Joining.  The warps of a CTA join through shared memory.  Few units of work
// (group x kv head): the CTAs that share a unit form a cluster and join through
// distributed shared memory, in one launch.  Many units: the blocks of all
// units, in order, are cut into equal stretches, one for each CTA that the GPU
// holds, whatever the sequences' lengths are; a stretch that begins or ends
// inside a unit leaves its partial result in the workspace, and
// k_kv8_attn_join adds those up.  No atomics, a fixed order of every sum: the
// same bits every time.
#include "q8_kv8_attn.h"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace q8 {

template <int N>
__device__ __forceinline__ void ka_load(uint32_t (&r)[N], const int8_t* p) {
  static_assert(N == 2 || N == 4 || N == 8, "8, 16 or 32 bytes");
  if constexpr (N == 8)
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
  else if constexpr (N == 4)
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "l"(p));
  else
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
}

__device__ __forceinline__ void ka_imma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ka_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t ka_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ka_remote(const float* p, int rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Sequence of slot g: slots of sequence b start at starts[b] / QT + E b.
// All threads of the CTA call it.
__device__ __forceinline__ int kv8_find(const int32_t* starts, int S, int rows, int QT, int E, int slot) {
  int n = 0;
  for (int b0 = 0; b0 < S; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    n += __syncthreads_count(b < S && min(max(starts[b], 0), rows) / QT + E * b <= slot);
  }
  return n - 1;
}

template <bool WIDE, int HD, int NT>  // WIDE: f32 rows, digits of q, halves of P
struct KaShape {
  static constexpr int RPT = WIDE ? 4 : 8;      // rows per n-tile of the outputs
  static constexpr int RMAX = NT * RPT;
  static constexpr int RT = WIDE ? 1 : 2;       // rows per n-tile whose scores a lane holds
  static constexpr int BPI = NT <= 2 ? 2 : 1;   // blocks per iteration
  static constexpr int WARPS = NT == 1 ? 12 : 8;  // that an SM holds
  static constexpr int QSMEM = NT == 1 ? 0 : NT * (HD / 16) * 32 * 8;
  static constexpr int REC = RMAX * (HD + 2);   // floats of a partial result: o, m, l
  static constexpr int smem(int warps) { return warps * REC * 4 + QSMEM + 3 * RMAX * 4; }
};

// Blocks [lo, hi) of a unit by the whole CTA.  Leaves the joined o in part
// ([RMAX][HD], lifted by KA_LIFT), m and l in s_m, s_l.
template <bool WIDE, int HD, int NT>
__device__ __forceinline__ void ka_stretch(const Kv8AttnArgs& a, const KaUnit& un, int lo, int hi, uint8_t* smem) {
  using Sh = KaShape<WIDE, HD, NT>;
  constexpr int RPT = Sh::RPT, RMAX = Sh::RMAX, RT = Sh::RT, BPI = Sh::BPI;
  constexpr int KW = HD / 16, VW = HD / 32, OT = HD / 16;  // words of a K quarter row, of a V eighth; output tiles
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  const int h = un.h, nrow = un.toks * a.GH;  // row r: token r / GH, head r % GH
  const int64_t room = (int64_t)a.max_pages * a.kv.page;
  const int32_t* trow = a.table + (int64_t)un.b * a.max_pages;
  const int ppb = a.kv.page / KV8_BLOCK;
  float* part = reinterpret_cast<float*>(smem);  // [warp][RMAX][HD]
  float* pm = part + warps * RMAX * HD;          // [warp][RMAX]
  float* pl = pm + warps * RMAX;                 // [warp][RMAX]
  uint2* qs = reinterpret_cast<uint2*>(pl + warps * RMAX);
  float* s_fac = reinterpret_cast<float*>(smem + warps * Sh::REC * 4 + Sh::QSMEM);
  float *s_m = s_fac + RMAX, *s_l = s_m + RMAX;

  // A warp's iteration takes BPI neighbouring blocks.  Lane j keeps number in
  // the pool (-1: no page) and scales of the j-th of the next 32 blocks.
  const int nit = lo + warp * BPI < hi ? (hi - lo - warp * BPI + warps * BPI - 1) / (warps * BPI) : 0;
  int ids = -1;
  float sks = 0.f, svs = 0.f;
  auto look_up = [&](int it) {
    const int i = it + lane / BPI;
    const int blk = lo + (warp + i * warps) * BPI + lane % BPI;
    ids = -1;
    sks = svs = 0.f;
    if (i < nit && blk < hi) {
      const int e = trow[blk / ppb];
      if (e >= 0 && e < a.kv.num_pages) {
        ids = (e * a.kv.n_kv + h) * ppb + blk % ppb;
        sks = a.kv.k_scale[ids];
        svs = a.kv.v_scale[ids];
      }
    }
  };
  const int8_t* kbase = a.kv.k + g * HD + t * (HD / 4);
  const int8_t* vbase = a.kv.v + 2 * t * HD + g * (HD / 8);
  uint32_t kr[BPI][2][KW], vr[BPI][4][VW];
#pragma unroll
  for (int j = 0; j < BPI; ++j) {
#pragma unroll
    for (int i = 0; i < KW; ++i) kr[j][0][i] = kr[j][1][i] = 0u;
#pragma unroll
    for (int i = 0; i < VW; ++i) vr[j][0][i] = vr[j][1][i] = vr[j][2][i] = vr[j][3][i] = 0u;
  }
  auto load_k = [&](int j, int id) {
    if (id < 0) return;
    const int8_t* p = kbase + (int64_t)id * (KV8_BLOCK * HD);
    ka_load(kr[j][0], p);
    ka_load(kr[j][1], p + 8 * HD);
  };
  auto load_v = [&](int j, int id) {
    if (id < 0) return;
    const int8_t* p = vbase + (int64_t)id * (KV8_BLOCK * HD);
    ka_load(vr[j][0], p);
    ka_load(vr[j][1], p + HD);
    ka_load(vr[j][2], p + 8 * HD);
    ka_load(vr[j][3], p + 9 * HD);
  };
  int id[BPI];
  look_up(0);
#pragma unroll
  for (int j = 0; j < BPI; ++j) {
    id[j] = __shfl_sync(0xffffffffu, ids, j);
    load_k(j, id[j]);
    load_v(j, id[j]);
  }

  // q: a lane holds its B column's words for the dims of its K quarter
  uint2 qf[NT == 1 ? KW : 1];
  const bool aligned = (((uintptr_t)a.q | (uintptr_t)(a.ldq * (WIDE ? 4 : 2))) & 15) == 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (NT > 1 && nt % warps != warp) continue;
    const int r = nt * RPT + (WIDE ? g >> 1 : g);
    float x[HD / 4];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) x[i] = 0.f;
    if (r < nrow && r % a.GH < un.heads)
      ka_row<WIDE>(x, a.q, (int64_t)(un.row0 + r / a.GH) * a.ldq + (un.head0 + r % a.GH) * HD + t * (HD / 4), a.dtype,
                   aligned);
    bool odd = false;  // NaN or infinite
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      top = fmaxf(top, fabsf(x[i]));
      odd |= !(fabsf(x[i]) < INFINITY);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    odd = __ballot_sync(0xffffffffu, odd) >> (lane & ~3) & 15u;
    float fac = 1.4426950408889634f / sqrtf((float)HD);
    if constexpr (WIDE) {
      const float pre = top < 0x1p-60f ? 0x1p90f : 1.f;  // 127 65536 / top would overflow for a subnormal top
      const float up = top > 0.f ? 8323072.f / (top * pre) : 0.f;
      fac *= top / 8323072.f;
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        uint32_t w0 = 0u, w1 = 0u;  // digit 0 or 1, and digit 2
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int X = odd ? 0 : __float2int_rn(x[4 * i + j] * pre * up);
          const int d2 = (int)(int8_t)X, X1 = (X - d2) >> 8;
          const int d1 = (int)(int8_t)X1, d0 = (X1 - d1) >> 8;
          w0 |= ((uint32_t)((g & 1) ? d1 : d0) & 255u) << (8 * j);
          w1 |= ((uint32_t)((g & 1) ? 0 : d2) & 255u) << (8 * j);
        }
        if (NT == 1) qf[i] = make_uint2(w0, w1);
        else qs[(nt * KW + i) * 32 + lane] = make_uint2(w0, w1);
      }
      if (odd) fac = __int_as_float(0x7fc00000);  // NaN scores
    } else {
      const int k = top > 0.f && top < INFINITY ? min(14 - ilogbf(top), 126) : 0;
      const float up = scalbnf(1.f, k);
      fac = scalbnf(fac, -k);
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        const uint2 w = make_uint2(ka_pack(x[4 * i] * up, x[4 * i + 1] * up),
                                   ka_pack(x[4 * i + 2] * up, x[4 * i + 3] * up));
        if (NT == 1) qf[i] = w;
        else qs[(nt * KW + i) * 32 + lane] = w;
      }
    }
    if (t == 0 && (!WIDE || (g & 1) == 0)) s_fac[r] = fac;
  }
  __syncthreads();
  float fac[NT][RT], m[NT][RT], l[NT][RT], o[OT][NT][4];
  int lim[NT][RT];  // positions that the lane's rows see
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const int r = nt * RPT + t * RT + j;
      fac[nt][j] = s_fac[r];
      lim[nt][j] = r < nrow ? (int)min(max(un.pos0 + r / a.GH + 1, (int64_t)0), room) : 0;
      m[nt][j] = -INFINITY;
      l[nt][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
  }

  int src = 0;  // lane that holds the iteration's first block
  for (int it = 0; it < nit; ++it) {
    float sk[BPI], sv[BPI];
    bool live[BPI];
#pragma unroll
    for (int j = 0; j < BPI; ++j) {
      sk[j] = __shfl_sync(0xffffffffu, sks, src + j);
      sv[j] = __shfl_sync(0xffffffffu, svs, src + j);
      live[j] = id[j] >= 0;
    }
    src += BPI;
    if (src == 32) {
      src = 0;
      look_up(it + 1);
    }
#pragma unroll
    for (int j = 0; j < BPI; ++j) id[j] = __shfl_sync(0xffffffffu, ids, src + j);

    // scores: positions g and g + 8 of each block
    float s[BPI][NT][RT][2];
#pragma unroll
    for (int j = 0; j < BPI; ++j) {
      if constexpr (WIDE) {
        int d[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[nt][0][e] = d[nt][1][e] = 0;
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
          const uint32_t f[4] = {kr[j][0][2 * i], kr[j][1][2 * i], kr[j][0][2 * i + 1], kr[j][1][2 * i + 1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 q0 = NT == 1 ? qf[2 * i] : qs[(nt * KW + 2 * i) * 32 + lane];
            const uint2 q1 = NT == 1 ? qf[2 * i + 1] : qs[(nt * KW + 2 * i + 1) * 32 + lane];
            ka_imma(d[nt][0], f, q0.x, q1.x);
            ka_imma(d[nt][1], f, q0.y, q1.y);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            s[j][nt][0][e] = fmaf((float)d[nt][0][2 * e], 65536.f, (float)(d[nt][0][2 * e + 1] * 256 + d[nt][1][2 * e]));
      } else {
        float d[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[nt][e] = 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t xu = kr[j][0][i] ^ 0x80808080u, yu = kr[j][1][i] ^ 0x80808080u;
          const uint32_t f[4] = {ka_f16(xu, 0x5140), ka_f16(yu, 0x5140), ka_f16(xu, 0x5342), ka_f16(yu, 0x5342)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 q0 = NT == 1 ? qf[i] : qs[(nt * KW + i) * 32 + lane];
            ka_mma(d[nt], f, q0.x, q0.y);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][nt][e & (RT - 1)][e >> 1] = d[nt][e];
      }
      load_k(j, id[j]);  // of the next iteration
    }

    float lsv[BPI];
    const int p0 = (lo + (warp + it * warps) * BPI) * KV8_BLOCK + g;
#pragma unroll
    for (int j = 0; j < BPI; ++j) lsv[j] = fmaxf(__log2f(sv[j]), -100.f);
    uint32_t pb[BPI][NT][2];
    bool moved = false;
    float alpha[NT][RT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < BPI; ++j) {
          const float f = fac[nt][r] * sk[j];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = s[j][nt][r][e] * f;
            s[j][nt][r][e] = live[j] && p0 + j * KV8_BLOCK + 8 * e < lim[nt][r] ? x : -INFINITY;
          }
          top = fmaxf(top, fmaxf(s[j][nt][r][0], s[j][nt][r][1]) + lsv[j]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float mn = fmaxf(m[nt][r], top);
        const float ref = mn == -INFINITY ? 0.f : mn;
        alpha[nt][r] = ka_exp2(m[nt][r] - ref);
        moved |= mn != m[nt][r];
        m[nt][r] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < BPI; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[j][nt][r][e] = ka_exp2(s[j][nt][r][e] - ref);
            sum += s[j][nt][r][e];
          }
        l[nt][r] = l[nt][r] * alpha[nt][r] + sum;
      }
#pragma unroll
      for (int j = 0; j < BPI; ++j) {
        const float w = sv[j] * KA_LIFT;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = s[j][nt][0][e] * w;
          uint32_t x;
          if (WIDE) {
            const float ph = __half2float(__float2half_rn(p));
            x = ka_pack(ph, p - ph);
          } else {
            x = ka_pack(p, s[j][nt][RT - 1][e] * w);
          }
          pb[j][nt][e] = ka_transpose(x);
        }
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][nt][e] *= alpha[nt][e & (RT - 1)];
    }
#pragma unroll
    for (int j = 0; j < BPI; ++j) {
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        // codes 4w .. 4w + 3 of the lane's dims; pairs of positions side by side
        const uint32_t e0 = __byte_perm(vr[j][0][w], vr[j][1][w], 0x5140) ^ 0x80808080u;
        const uint32_t e1 = __byte_perm(vr[j][0][w], vr[j][1][w], 0x7362) ^ 0x80808080u;
        const uint32_t d0 = __byte_perm(vr[j][2][w], vr[j][3][w], 0x5140) ^ 0x80808080u;
        const uint32_t d1 = __byte_perm(vr[j][2][w], vr[j][3][w], 0x7362) ^ 0x80808080u;
        const uint32_t fa[4] = {ka_f16(e0, 0x5140), ka_f16(e0, 0x5342), ka_f16(d0, 0x5140), ka_f16(d0, 0x5342)};
        const uint32_t fb[4] = {ka_f16(e1, 0x5140), ka_f16(e1, 0x5342), ka_f16(d1, 0x5140), ka_f16(d1, 0x5342)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          ka_mma(o[2 * w][nt], fa, pb[j][nt][0], pb[j][nt][1]);
          ka_mma(o[2 * w + 1][nt], fb, pb[j][nt][0], pb[j][nt][1]);
        }
      }
      load_v(j, id[j]);  // of the next iteration
    }
  }

#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const int r = nt * RPT + t * RT + j;
      float x = l[nt][j];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) {
        pm[warp * RMAX + r] = m[nt][j];
        pl[warp * RMAX + r] = x;
      }
      float2* row = reinterpret_cast<float2*>(part + (warp * RMAX + r) * HD + g * (HD / 8));
#pragma unroll
      for (int i = 0; i < OT; ++i)
        row[i] = WIDE ? make_float2(o[i][nt][0] + o[i][nt][1], o[i][nt][2] + o[i][nt][3])
                      : make_float2(o[i][nt][j], o[i][nt][2 + j]);
    }
  __syncthreads();
  // join the warps; the CTA's result replaces warp 0's
  if (threadIdx.x < RMAX) {
    float mx = -INFINITY, sum = 0.f;
    for (int w = 0; w < warps; ++w) mx = fmaxf(mx, pm[w * RMAX + threadIdx.x]);
    for (int w = 0; w < warps; ++w) {
      const float mw = pm[w * RMAX + threadIdx.x];
      const float x = mw == -INFINITY ? 0.f : exp2f(mw - mx);
      sum += x * pl[w * RMAX + threadIdx.x];
      pm[w * RMAX + threadIdx.x] = x;
    }
    s_m[threadIdx.x] = mx;
    s_l[threadIdx.x] = sum;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < nrow * HD; k += blockDim.x) {
    const int r = k / HD;
    float x = 0.f;
    for (int w = 0; w < warps; ++w) x += pm[w * RMAX + r] * part[w * RMAX * HD + k];
    part[k] = x;
  }
}

// Few units: a cluster of CTAs for each.
template <bool WIDE, int HD, int NT>
__global__ void __launch_bounds__(KaShape<WIDE, HD, NT>::WARPS * 32, 1) k_kv8_attn(Kv8AttnArgs a) {
  using Sh = KaShape<WIDE, HD, NT>;
  constexpr int RMAX = Sh::RMAX;
  extern __shared__ __align__(16) uint8_t smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int nsplit = cluster.num_blocks(), split = cluster.block_rank();
  const int slot = blockIdx.x / nsplit;
  const int E = a.QT > 1 ? 1 : 0;
  int b = slot;
  if (!(E == 0 && slot < a.S && a.starts[slot] <= slot && a.starts[slot + 1] > slot))
    b = kv8_find(a.starts, a.S, a.rows, a.QT, E, slot);
  if (b < 0) return;
  const Kv8Seq sq = kv8_seq(a.starts, a.ctx, b, a.rows);
  const int i0 = (slot - (sq.row0 / a.QT + E * b)) * a.QT;
  if (i0 >= sq.n) return;
  const KaUnit u = ka_unit(a, sq, blockIdx.y, i0);
  const int per = ((u.nblk + nsplit - 1) / nsplit + Sh::BPI - 1) / Sh::BPI * Sh::BPI;
  const int lo = min(u.nblk, split * per), hi = min(u.nblk, lo + per);
  ka_stretch<WIDE, HD, NT>(a, u, lo, hi, smem);
  const float* part = reinterpret_cast<float*>(smem);
  const float* s_m = reinterpret_cast<float*>(smem + (blockDim.x >> 5) * Sh::REC * 4 + Sh::QSMEM) + RMAX;
  const float* s_l = s_m + RMAX;
  const int n = u.toks * a.GH * HD;
  if (nsplit == 1) {
    for (int k = threadIdx.x; k < n; k += blockDim.x)
      ka_write<WIDE, HD>(a, u.row0, u.head0, u.heads, k, part[k], s_l[k / HD]);
    return;
  }
  cluster.sync();
  for (int k = split * blockDim.x + threadIdx.x; k < n; k += nsplit * blockDim.x) {
    const int r = k / HD;
    float mx = -INFINITY;
    for (int c = 0; c < nsplit; ++c) mx = fmaxf(mx, ka_remote(s_m + r, c));
    float x = 0.f, sum = 0.f;
    for (int c = 0; c < nsplit; ++c) {
      const float mc = ka_remote(s_m + r, c);
      const float w = mc == -INFINITY ? 0.f : exp2f(mc - mx);
      x += w * ka_remote(part + k, c);
      sum += w * ka_remote(s_l + r, c);
    }
    ka_write<WIDE, HD>(a, u.row0, u.head0, u.heads, k, x, sum);
  }
  cluster.sync();  // nobody leaves while its memory is read
}

// Many units: CTA c takes the c-th of gridDim.x equal stretches of all units'
// work, units ordered by (sequence, group, kv head).  A unit's work is its
// iterations (BPI blocks each) behind KA_FIXED more for its start and end.
constexpr int KA_FIXED = 16;

template <bool WIDE, int HD, int NT>
__global__ void __launch_bounds__(128, KaShape<WIDE, HD, NT>::WARPS / 4) k_kv8_attn_many(Kv8AttnArgs a) {
  using Sh = KaShape<WIDE, HD, NT>;
  constexpr int RMAX = Sh::RMAX, BPI = Sh::BPI;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_scan[4];
  __shared__ int64_t s_at;
  __shared__ int s_b;
  pdl_trigger();
  const int H = a.kv.n_kv * a.hgroups, c = blockIdx.x, nc = gridDim.x;
  // work of a sequence's groups, the last (longest) one's for each
  auto weight = [&](int b, int64_t* each) -> int64_t {
    const Kv8Seq sq = kv8_seq(a.starts, a.ctx, b, a.rows);
    *each = KA_FIXED + (ka_blocks(a, sq.pos0 + sq.n) + BPI - 1) / BPI;
    return (int64_t)((sq.n + a.QT - 1) / a.QT) * H * *each;
  };
  int64_t all = 0, each = 1, mine = 0;
  for (int b = threadIdx.x; b < a.S; b += blockDim.x) all += mine = weight(b, &each);
  int64_t total;
  ka_scan(all, s_scan, &total);
  // [at, end): the CTA's stretch
  const int64_t at = total / nc * c + total % nc * c / nc, end = total / nc * (c + 1) + total % nc * (c + 1) / nc;
  if (threadIdx.x == 0) a.work_meta[2 * c] = a.work_meta[2 * c + 1] = make_int4(-1, 0, 0, 0);
  if (at >= end) return;
  int64_t before = 0;
  for (int b0 = 0; b0 < a.S; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    if (a.S > blockDim.x) mine = b < a.S ? weight(b, &each) : 0;
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
  int b = s_b;
  int64_t off = s_at, left = end - at;
  while (left > 0) {
    const Kv8Seq sq = kv8_seq(a.starts, a.ctx, b, a.rows);
    const int64_t w = weight(b, &each);
    while (off < w && left > 0) {
      const int64_t k = off / each;  // unit within the sequence
      const int w0 = (int)(off - k * each), take = (int)min(left, each - w0);
      const int u0 = max(0, w0 - KA_FIXED), u1 = max(0, w0 + take - KA_FIXED);  // iterations
      const bool begins = u0 == 0, ends = w0 + take == each;
      off += take;
      left -= take;
      if (u1 == 0 && !ends) continue;  // the next CTA begins it
      const KaUnit u = ka_unit(a, sq, (int)(k % H), (int)(k / H) * a.QT);
      ka_stretch<WIDE, HD, NT>(a, u, min(u.nblk, u0 * BPI), min(u.nblk, u1 * BPI), smem);
      const float* part = reinterpret_cast<float*>(smem);
      const float* s_m = reinterpret_cast<float*>(smem + 4 * Sh::REC * 4 + Sh::QSMEM) + RMAX;
      const float* s_l = s_m + RMAX;
      const int n = u.toks * a.GH * HD;
      if (begins && ends) {
        for (int i = threadIdx.x; i < n; i += blockDim.x)
          ka_write<WIDE, HD>(a, u.row0, u.head0, u.heads, i, part[i], s_l[i / HD]);
      } else {
        // record 1: a unit that begins here, record 0: one that goes on from the CTA before
        const int rec = 2 * c + (begins ? 1 : 0);
        float* to = a.work + (int64_t)rec * Sh::REC;
        for (int i = threadIdx.x; i < n; i += blockDim.x) to[i] = part[i];
        if (threadIdx.x < RMAX) {
          to[RMAX * HD + threadIdx.x] = s_m[threadIdx.x];
          to[RMAX * HD + RMAX + threadIdx.x] = s_l[threadIdx.x];
        }
        if (threadIdx.x == 0) a.work_meta[rec] = make_int4(u.row0, u.head0, u.toks | u.heads << 16, ends);
      }
      __syncthreads();  // shared memory is used again
    }
    off = 0;
    do ++b;
    while (left > 0 && b < a.S && weight(b, &each) == 0);
    if (b >= a.S) break;
  }
}

// A unit that begins in CTA c and goes on behind it: record 1 of c, then
// records 0 of the next ones up to the one that ends it.  A warp per row.
template <bool WIDE, int HD>
__global__ void __launch_bounds__(256) k_kv8_attn_join(Kv8AttnArgs a, int RMAX) {
  constexpr int E = HD / 32;
  pdl_wait();
  const int c = blockIdx.x, nc = gridDim.x, REC = RMAX * (HD + 2), lane = threadIdx.x & 31;
  const int r = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int4 me = a.work_meta[2 * c + 1];
  const int toks = me.z & 0xffff, heads = me.z >> 16;
  if (me.x < 0 || r >= toks * a.GH || r % a.GH >= heads) return;
  int last = c + 1;  // CTAs without work (x < 0) may lie between
  while (last < nc - 1 && !a.work_meta[2 * last].w) ++last;
  float mx = -INFINITY, sum = 0.f, x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.f;
  for (int i = c; i <= last; ++i) {
    if (i != c && a.work_meta[2 * i].x < 0) continue;
    const float* rec = a.work + (int64_t)(2 * i + (i == c)) * REC;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = rec[r * HD + lane * E + e];
    const float m = rec[RMAX * HD + r], l = rec[RMAX * HD + RMAX + r];
    const float top = fmaxf(mx, m), ref = top == -INFINITY ? 0.f : top;
    const float f0 = exp2f(mx - ref), f1 = exp2f(m - ref);
    sum = sum * f0 + l * f1;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * f0 + v[e] * f1;
    mx = top;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    ka_write<WIDE, HD>(a, me.x, me.y, heads, r * HD + lane * E + e, x[e], sum);
}

template <bool WIDE, int HD>
static int join_run(const Kv8AttnArgs& a, int ctas, int RMAX, cudaStream_t st) {
  return launch_pdl("k_kv8_attn_join", k_kv8_attn_join<WIDE, HD>, dim3(ctas, ceil_div(RMAX, 8)), dim3(256), 0, st, a,
                    RMAX);
}

int kv8_attn_join(const Kv8AttnArgs& a, int ctas, int RMAX, cudaStream_t st) {
  if (a.kv.head_dim == 128)
    return a.dtype == Q8_F32 ? join_run<true, 128>(a, ctas, RMAX, st) : join_run<false, 128>(a, ctas, RMAX, st);
  return a.dtype == Q8_F32 ? join_run<true, 64>(a, ctas, RMAX, st) : join_run<false, 64>(a, ctas, RMAX, st);
}

struct KaPlan {
  bool tc;   // k_kv8_attn_tc
  int nt, GH, hgroups, QT, ctas;  // ctas: stretches of k_kv8_attn_many, 0: clusters
  int64_t slots, units;
  size_t meta, bytes;  // workspace
};

static KaPlan ka_plan(bool wide, int hd, int64_t rows, int64_t S, int n_heads, int n_kv) {
  KaPlan p{};
  const int G = n_heads / n_kv;
  const int64_t want = (rows + S - 1) / S * (int64_t)G;  // rows per kv head of an average sequence
  const int cols = wide ? 2 : 1;
  p.nt = want * cols <= 8 ? 1 : want * cols <= 16 ? 2 : 4;
  p.tc = want >= 64 && G <= KT_ROWS;
  const int rmax = p.tc ? KT_ROWS : 8 * p.nt / cols;
  p.GH = std::min(G, rmax);
  p.hgroups = ceil_div(G, p.GH);
  p.QT = rows <= S ? 1 : rmax / p.GH;
  p.slots = p.QT > 1 ? rows / p.QT + S : rows;
  p.units = p.slots * n_kv * p.hgroups;
  // One n-tile: a unit is cheap to begin and its partial results are small.
  if (p.tc || (p.nt == 1 && p.units > num_sms())) {
    p.ctas = p.tc ? kv8_attn_tc_ctas() : 3 * num_sms();
    p.meta = (size_t)p.ctas * 2 * rmax * (hd + 2) * 4;
    p.bytes = p.meta + (size_t)p.ctas * 2 * sizeof(int4);
  }
  return p;
}

template <bool WIDE, int HD, int NT>
static int attn_run(Kv8AttnArgs& a, const KaPlan& p, cudaStream_t st) {
  using Sh = KaShape<WIDE, HD, NT>;
  auto few = k_kv8_attn<WIDE, HD, NT>;
  static bool ready[64] = {false};
  int dev = 0;
  Q8_CUDA(cudaGetDevice(&dev));
  if (!ready[dev & 63]) {
    Q8_CUDA(cudaFuncSetAttribute(few, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::smem(Sh::WARPS)));
    Q8_CUDA(cudaFuncSetAttribute(few, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ready[dev & 63] = true;
  }
  if constexpr (NT == 1) {
    if (p.ctas) {
      k_kv8_attn_many<WIDE, HD, NT><<<p.ctas, 128, Sh::smem(4), st>>>(a);
      Q8_TRY(launch_check("k_kv8_attn_many"));
      return kv8_attn_join(a, p.ctas, Sh::RMAX, st);
    }
  }
  // a cluster's CTAs: an SM each, but an iteration for every warp at the longest context
  const int64_t most = ((int64_t)a.max_pages * a.kv.page / KV8_BLOCK + Sh::BPI * Sh::WARPS - 1) / (Sh::BPI * Sh::WARPS);
  int nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({16, most, num_sms() / p.units}));
  Q8_CHECK_ARG(p.slots * nsplit < ((int64_t)1 << 31) && (int64_t)a.kv.n_kv * a.hgroups <= 65535,
               "q8op_kv8_attention: too many rows or heads");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)nsplit, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.slots * nsplit), a.kv.n_kv * a.hgroups);
  cfg.blockDim = dim3(Sh::WARPS * 32);
  cfg.dynamicSmemBytes = Sh::smem(Sh::WARPS);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  Q8_CUDA(cudaLaunchKernelEx(&cfg, few, a));
  return Q8_OK;
}

template <bool WIDE, int HD>
static int attn_pick(Kv8AttnArgs& a, const KaPlan& p, cudaStream_t st) {
  if (p.nt == 1) return attn_run<WIDE, HD, 1>(a, p, st);
  if (p.nt == 2) return attn_run<WIDE, HD, 2>(a, p, st);
  return attn_run<WIDE, HD, 4>(a, p, st);
}

}  // namespace q8

using namespace q8;

extern "C" size_t q8op_kv8_attention_workspace(int dtype, int64_t rows, int64_t S, int n_heads, int n_kv,
                                               int head_dim) {
  if (rows <= 0 || S <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || head_dim <= 0) return 0;
  return ka_plan(dtype == Q8_F32, head_dim, rows, S, n_heads, n_kv).bytes;
}

extern "C" int q8op_kv8_attention(const void* q, int64_t ldq, int dtype, int64_t rows, const int32_t* seq_start,
                                  const int32_t* ctx, int64_t S, int n_heads, const q8_kv8_pages* kv,
                                  const int32_t* block_table, int max_pages, void* out, int64_t ldo, void* work,
                                  size_t work_bytes, void* stream) {
  Q8_TRY(kv8_check("q8op_kv8_attention", kv, seq_start, ctx, S, rows, block_table, max_pages));
  Q8_CHECK_ARG(dtype == Q8_F32 || dtype == Q8_BF16 || dtype == Q8_F16, "q8op_kv8_attention: bad dtype %d", dtype);
  Q8_CHECK_ARG(n_heads > 0 && n_heads % kv->n_kv == 0 && n_heads / kv->n_kv <= 65535,
               "q8op_kv8_attention: %d heads over %d kv heads", n_heads, kv->n_kv);
  if (rows == 0 || S == 0) return Q8_OK;
  const int64_t width = (int64_t)n_heads * kv->head_dim;
  Q8_CHECK_ARG(q && out && ldq >= width && ldo >= width, "q8op_kv8_attention: q and out rows need %lld elements",
               (long long)width);
  const KaPlan p = ka_plan(dtype == Q8_F32, kv->head_dim, rows, S, n_heads, kv->n_kv);
  Q8_CHECK_ARG(p.bytes == 0 || (work && work_bytes >= p.bytes && ((uintptr_t)work & 15) == 0),
               "q8op_kv8_attention: workspace of %zu bytes (16-byte aligned), %zu needed", work ? work_bytes : (size_t)0,
               p.bytes);
  Kv8AttnArgs a{q,   ldq,   dtype,       (int)rows, seq_start, ctx,  (int)S, n_heads,   *kv, block_table, max_pages,
                out, ldo,   p.QT,        p.GH,      p.hgroups, (float*)work, (int4*)((char*)work + p.meta)};
  cudaStream_t st = (cudaStream_t)stream;
  if (p.tc) {
    Q8_TRY(kv8_attn_tc(a, p.ctas, st));
    return kv8_attn_join(a, p.ctas, KT_ROWS, st);
  }
  if (kv->head_dim == 128) return dtype == Q8_F32 ? attn_pick<true, 128>(a, p, st) : attn_pick<false, 128>(a, p, st);
  return dtype == Q8_F32 ? attn_pick<true, 64>(a, p, st) : attn_pick<false, 64>(a, p, st);
}
