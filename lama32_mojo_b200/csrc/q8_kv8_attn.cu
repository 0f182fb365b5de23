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
// codes as they are; the two f16 halves of P (22 bits) are two more columns.
// bf16 / f16 rows: q scaled by a power of two to the top of the f16 range, one
// column, the codes as f16 (exact); the halves of P are two products.  One f16
// alone would move an f16 result by as much again as its own rounding.
// The order of a dot product's terms is free, so lane (g, t) = (lane / 4,
// lane % 4) reads its operand bytes straight from the cache rows: of K a
// quarter of rows g and g + 8, of V the g-th eighth of rows 2t, 2t + 1, 2t + 8,
// 2t + 9 (output row g of tile m is dim (hd/8) g + 2m, row g + 8 the next
// one).  No shared memory, no barrier: a block's registers are loaded again as
// soon as its products are issued, and wait there while the others work.  P^T
// becomes the B operand by movmatrix.
//
// Softmax: base 2, running maximum M of s + log2(sv) rather than of s: the
// weights that meet the codes are e sv, e = 2^(s - M), so they stay within one
// range whatever the blocks' scales are, and l = sum e is kept against the same
// M.  The largest is 2^15, at the top of the f16 range, whose smallest step,
// 2^-24, is then 2^-39 of it.  How M is shifted for that: KA_DOWN.
//
// Joining.  The warps of a CTA join through shared memory.  Few units of work
// (group x kv head): the CTAs that share a unit form a cluster and join through
// distributed shared memory, in one launch.  Many units: the blocks of all
// units, in order, are cut into equal stretches, one for each CTA that the GPU
// holds, whatever the sequences' lengths are; a stretch that begins or ends
// inside a unit leaves its partial result in the workspace, and
// k_kv8_attn_join adds those up.  No atomics, a fixed order of every sum: the
// same bits every time.
//
// Bound.  64 f32 rows, one each for sequences up to 8192 positions, 32 heads on 8
// of 128: 94 us for 557 MB, 5.9 TB/s or 0.90 of a copy's rate; 39 % of the issue
// slots, so the cache's rows are what it waits for.  80 bf16 rows of 16 sequences,
// 24 heads: 37 us for 76 MB: launch, search and join take half (33 with one f16 a weight).  One row and 523
// positions, heads of 64: 5.9 us, a launch and a chain of dependent loads (6.8
// before the warps shared the work on the query rows: 3000 of 8500 clocks).
#include "q8_kv8_attn.h"

#include <algorithm>
#include <type_traits>
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

constexpr int ka_bpi(int nt) { return nt == 1 ? 2 : 1; }
constexpr int ka_warps(int nt) { return nt <= 2 ? 12 : 8; }

template <bool WIDE, int HD, int NT>  // WIDE: f32 rows, digits of q, halves of P
struct KaShape {
  static constexpr int RPT = WIDE ? 4 : 8;      // rows per n-tile of the outputs
  static constexpr int RMAX = NT * RPT;
  static constexpr int RT = WIDE ? 1 : 2;       // rows per n-tile whose scores a lane holds
  static constexpr int BPI = ka_bpi(NT);        // blocks per iteration
  static constexpr int WARPS = ka_warps(NT);     // that an SM holds
  static constexpr int QSMEM = NT * (HD / 16) * 32 * 8;
  static constexpr int REC = RMAX * (HD + 2);   // floats of a partial result: o, m, l
  static constexpr int smem(int warps) { return warps * REC * 4 + QSMEM + 3 * RMAX * 4; }
};

// Blocks [lo, hi) of a unit by the whole CTA.  At the end a warp takes a row r at
// a time: sink(r, x, m, l), x the lane's HD / 32 dims of the sum lifted by KA_LIFT.
template <bool WIDE, int HD, int NT, int warps, typename Sink>
__device__ __forceinline__ void ka_stretch(const Kv8AttnArgs& a, const KaUnit& un, int lo, int hi, uint8_t* smem,
                                           Sink sink) {
  using Sh = KaShape<WIDE, HD, NT>;
  constexpr int RPT = Sh::RPT, RMAX = Sh::RMAX, RT = Sh::RT, BPI = Sh::BPI;
  constexpr int KW = HD / 16, VW = HD / 32, OT = HD / 16;  // words of a K quarter row, of a V eighth; output tiles
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int h = un.h, nrow = un.toks * a.GH;  // row r: token r / GH, head r % GH
  const unsigned per_gh = (65535u + a.GH) / a.GH;
  auto tok_of = [&](int r) { return (int)(r * per_gh >> 16); };  // exact: both are at most 128
  const int64_t room = (int64_t)a.max_pages * a.kv.page;
  const int32_t* trow = a.table + (int64_t)un.b * a.max_pages;
  const int ppb = a.kv.page / KV8_BLOCK;
  float* part = reinterpret_cast<float*>(smem);  // [warp][RMAX][HD]
  float* pm = part + warps * RMAX * HD;          // [warp][RMAX]
  float* pl = pm + warps * RMAX;                 // [warp][RMAX]
  uint2* qs = reinterpret_cast<uint2*>(pl + warps * RMAX);
  float* s_fac = reinterpret_cast<float*>(smem + warps * Sh::REC * 4 + Sh::QSMEM);

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
  // q: four dims a lane, a warp 128 / HD rows at a time.  Loaded before anything
  // waits for the table.
  constexpr int LPR = HD / 4, RPP = 32 / LPR, RPW = (RMAX + warps * RPP - 1) / (warps * RPP);
  float x[RPW][4];
  auto load_q = [&](auto by16) {
#pragma unroll
    for (int k = 0; k < RPW; ++k) {
      const int r = (k * warps + warp) * RPP + lane / LPR;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[k][i] = 0.f;
      const int tok = tok_of(r), head = r - tok * a.GH;
      if (r < nrow && head < un.heads)
        ka_four<WIDE, decltype(by16)::value>(
            x[k], a.q, (int64_t)(un.row0 + tok) * a.ldq + (un.head0 + head) * HD + lane % LPR * 4, a.dtype);
    }
  };
  if ((((uintptr_t)a.q | (uintptr_t)(a.ldq * (WIDE ? 4 : 2))) & 15) == 0) load_q(std::true_type());
  else load_q(std::false_type());
  int id[BPI];
  look_up(0);
#pragma unroll
  for (int j = 0; j < BPI; ++j) {
    id[j] = __shfl_sync(0xffffffffu, ids, j);
    load_k(j, id[j]);
    load_v(j, id[j]);
  }

  // the B columns' words, by lane: of lane (g, t) and word i, column g's codes of
  // the dims t HD / 4 + 4 i .. + 3
#pragma unroll
  for (int k = 0; k < RPW; ++k) {
    const int r = (k * warps + warp) * RPP + lane / LPR, w = lane % LPR;
    unsigned bits = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) bits = max(bits, __float_as_uint(x[k][i]) & 0x7fffffffu);
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
    if (r >= RMAX) continue;
    const bool odd = bits >= 0x7f800000u;  // NaN or infinite
    uint2* to = qs + (r / RPT * KW + w % KW) * 32 + w / KW;
    float fac = 1.4426950408889634f / sqrtf((float)HD);
    if constexpr (WIDE) {
      const float top = __uint_as_float(bits);
      const float pre = top < 0x1p-60f ? 0x1p90f : 1.f;  // 127 65536 / top would overflow for a subnormal top
      const float up = top > 0.f ? 8323072.f / (top * pre) : 0.f;
      fac *= top / 8323072.f;
      uint32_t d0 = 0u, d1 = 0u, d2 = 0u;  // digits
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int X = odd ? 0 : __float2int_rn(x[k][j] * pre * up);
        const int c2 = (int)(int8_t)X, X1 = (X - c2) >> 8;
        const int c1 = (int)(int8_t)X1, c0 = (X1 - c1) >> 8;
        d0 |= ((uint32_t)c0 & 255u) << (8 * j);
        d1 |= ((uint32_t)c1 & 255u) << (8 * j);
        d2 |= ((uint32_t)c2 & 255u) << (8 * j);
      }
      to[r % RPT * 8] = make_uint2(d0, d2);  // columns 2 r and 2 r + 1
      to[r % RPT * 8 + 4] = make_uint2(d1, 0u);
      if (odd) fac = __int_as_float(0x7fc00000);  // NaN scores
    } else {
      // the largest element into [2^14, 2^15)
      const int sh = bits == 0u || odd ? 0 : min(141 - (int)(bits >> 23), 126);
      const float up = __uint_as_float((unsigned)(127 + sh) << 23);
      fac *= __uint_as_float((unsigned)(127 - sh) << 23);
      to[r % RPT * 4] = make_uint2(ka_pack(x[k][0] * up, x[k][1] * up), ka_pack(x[k][2] * up, x[k][3] * up));
    }
    if (w == 0) s_fac[r] = fac;
  }
  __syncthreads();
  uint2 qf[NT == 1 ? KW : 1];
  if (NT == 1) {
#pragma unroll
    for (int i = 0; i < KW; ++i) qf[i] = qs[i * 32 + lane];
  }
  float fac[NT][RT], m[NT][RT], l[NT][RT], o[OT][NT][4];
  int lim[NT][RT];  // positions that the lane's rows see
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const int r = nt * RPT + t * RT + j;
      fac[nt][j] = s_fac[r];
      lim[nt][j] = r < nrow ? (int)min(max(un.pos0 + tok_of(r) + 1, (int64_t)0), room) : 0;
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
    for (int j = 0; j < BPI; ++j) lsv[j] = fmaxf(__log2f(sv[j]), KA_LEAST) - KA_DOWN;
    uint32_t pb[BPI][NT][2], pr[BPI][WIDE ? 1 : NT][2];  // pr: what the f16 of pb leave of the weights
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
        alpha[nt][r] = ka_lower<false>(l[nt][r], m[nt][r] - ref);
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
        l[nt][r] += sum;
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
            const float p1 = s[j][nt][RT - 1][e] * w;
            x = ka_pack(p, p1);
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&x));
            pr[j][WIDE ? 0 : nt][e] = ka_transpose(ka_pack(p - h.x, p1 - h.y));
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
          if constexpr (!WIDE) {
            ka_mma(o[2 * w][nt], fa, pr[j][nt][0], pr[j][nt][1]);
            ka_mma(o[2 * w + 1][nt], fb, pr[j][nt][0], pr[j][nt][1]);
          }
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
  // join the warps: lane w knows warp w's m and l
  constexpr int D = HD / 32;
  for (int r = warp; r < nrow; r += warps) {
    const float mw = lane < warps ? pm[lane * RMAX + r] : -INFINITY, mx = warp_max(mw);
    float lw = lane < warps ? pl[lane * RMAX + r] : 0.f;
    const float f = ka_lower<true>(lw, mw - (mx == -INFINITY ? 0.f : mx));
    const float sum = warp_sum(lw);
    float x[D];
#pragma unroll
    for (int e = 0; e < D; ++e) x[e] = 0.f;
    const float* p = part + r * HD + lane * D;
#pragma unroll 4
    for (int w = 0; w < warps; ++w, p += RMAX * HD) {
      const float fw = __shfl_sync(0xffffffffu, f, w);
      float y[D];
      if constexpr (D == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        y[0] = v.x, y[1] = v.y, y[D - 2] = v.z, y[D - 1] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        y[0] = v.x, y[1] = v.y;
      }
#pragma unroll
      for (int e = 0; e < D; ++e) x[e] += fw * y[e];
    }
    sink(r, x, mx, sum);
  }
}

// The lane's dims of row r of a unit, from its lifted sums x and the sum of the weights.
template <bool WIDE, int HD>
__device__ __forceinline__ void ka_out(const Kv8AttnArgs& a, int row0, int head0, int heads, int r,
                                       const float (&x)[HD / 32], float sum) {
  constexpr int D = HD / 32;
  const int tok = r / a.GH, h = r - tok * a.GH;
  if (h >= heads) return;
  const int64_t i = (int64_t)(row0 + tok) * a.ldo + (head0 + h) * HD + (threadIdx.x & 31) * D;
  const float inv = 1.f / (KA_LIFT * sum);
  float y[D];
#pragma unroll
  for (int e = 0; e < D; ++e) y[e] = sum > 0.f ? x[e] * inv : 0.f * (x[e] + sum);  // no position: 0; NaN stays
  const bool aligned = (((uintptr_t)a.out | (uintptr_t)(a.ldo * (WIDE ? 4 : 2))) & (D * (WIDE ? 4 : 2) - 1)) == 0;
  if (!aligned) {
#pragma unroll
    for (int e = 0; e < D; ++e) ka_store<WIDE>(a, i + e, y[e]);
  } else if constexpr (WIDE) {
    float* to = (float*)a.out + i;
    if constexpr (D == 4) *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
    else *reinterpret_cast<float2*>(to) = make_float2(y[0], y[1]);
  } else {
    uint32_t u[D / 2];
#pragma unroll
    for (int k = 0; k < D / 2; ++k) u[k] = ka_pack16(a.dtype, y[2 * k], y[2 * k + 1]);
    uint16_t* to = (uint16_t*)a.out + i;
    if constexpr (D == 4) *reinterpret_cast<uint2*>(to) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(to) = u[0];
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
  if (nsplit == 1) {
    ka_stretch<WIDE, HD, NT, Sh::WARPS>(a, u, lo, hi, smem, [&](int r, const float (&x)[HD / 32], float, float l) {
      ka_out<WIDE, HD>(a, u.row0, u.head0, u.heads, r, x, l);
    });
    return;
  }
  // the CTA's result takes warp 0's place
  float* part = reinterpret_cast<float*>(smem);
  float *s_m = reinterpret_cast<float*>(smem + (blockDim.x >> 5) * Sh::REC * 4 + Sh::QSMEM) + RMAX, *s_l = s_m + RMAX;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  ka_stretch<WIDE, HD, NT, Sh::WARPS>(a, u, lo, hi, smem, [&](int r, const float (&x)[HD / 32], float m, float l) {
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) part[r * HD + lane * (HD / 32) + e] = x[e];
    if (lane == 0) {
      s_m[r] = m;
      s_l[r] = l;
    }
  });
  cluster_wait_all();
  // 32 elements to a warp, the clusters' warps in turn; lane c knows CTA c's m and l
  const int n = u.toks * a.GH * HD, step = (blockDim.x >> 5) * nsplit * 32;
  int k0 = (warp * nsplit + split) * 32;
  if (k0 >= n) cluster_leave();
  for (; k0 < n; k0 += step) {
    const int r = k0 / HD;
    const float m = lane < nsplit ? ka_remote(s_m + r, lane) : -INFINITY;
    float l = lane < nsplit ? ka_remote(s_l + r, lane) : 0.f;
    const float mx = warp_max(m), f = ka_lower<true>(l, m - (mx == -INFINITY ? 0.f : mx));
    const float sum = warp_sum(l);
    float x = 0.f;
    for (int c = 0; c < nsplit; ++c) x += __shfl_sync(0xffffffffu, f, c) * ka_remote(part + k0 + lane, c);
    if (k0 + step >= n) cluster_leave();
    ka_write<WIDE, HD>(a, u.row0, u.head0, u.heads, k0 + lane, x, sum);
  }
  cluster_left();  // nobody leaves while its memory is read
}

// Many units: CTA c takes the c-th of gridDim.x equal stretches of all units'
// work, units ordered by (sequence, group, kv head).  A unit's work is its
// iterations (BPI blocks each) behind some more for its start and end (7 us,
// an iteration of a CTA's four warps taking 0.45 us with one n-tile and two
// blocks, 0.3 us with two n-tiles and one).
constexpr int ka_fixed(int nt) { return nt == 1 ? 14 : 28; }

template <bool WIDE, int HD, int NT>
__global__ void __launch_bounds__(128, KaShape<WIDE, HD, NT>::WARPS / 4) k_kv8_attn_many(Kv8AttnArgs a) {
  using Sh = KaShape<WIDE, HD, NT>;
  constexpr int RMAX = Sh::RMAX, BPI = Sh::BPI, KA_FIXED = ka_fixed(NT);
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
      const int lo = min(u.nblk, u0 * BPI), hi = min(u.nblk, u1 * BPI);
      // record 1: a unit that begins here, record 0: one that goes on from the CTA before
      const bool whole = begins && ends;
      const int rec = 2 * c + (begins ? 1 : 0), lane = threadIdx.x & 31;
      float* to = a.work + (int64_t)rec * Sh::REC;
      ka_stretch<WIDE, HD, NT, 4>(a, u, lo, hi, smem, [&](int r, const float (&x)[HD / 32], float m, float l) {
        if (whole) {
          ka_out<WIDE, HD>(a, u.row0, u.head0, u.heads, r, x, l);
          return;
        }
        if constexpr (HD == 128)
          *reinterpret_cast<float4*>(to + r * HD + lane * 4) = make_float4(x[0], x[1], x[HD / 32 - 2], x[HD / 32 - 1]);
        else
          *reinterpret_cast<float2*>(to + r * HD + lane * 2) = make_float2(x[0], x[1]);
        if (lane == 0) {
          to[RMAX * HD + r] = m;
          to[RMAX * HD + RMAX + r] = l;
        }
      });
      if (!whole && threadIdx.x == 0)
        a.work_meta[rec] = make_int4(u.row0, u.head0, u.toks | u.heads << 16, ends);
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
    const float m = rec[RMAX * HD + r];
    float l = rec[RMAX * HD + RMAX + r];
    const float top = fmaxf(mx, m), ref = top == -INFINITY ? 0.f : top;
    const float f0 = ka_lower<true>(sum, mx - ref), f1 = ka_lower<true>(l, m - ref);
    sum += l;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * f0 + v[e] * f1;
    mx = top;
  }
  ka_out<WIDE, HD>(a, me.x, me.y, heads, r, x, sum);
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

// Clusters of c CTAs, each with an SM to itself, that the device holds at once.
static int ka_clusters(int c) {
  static int held[64][9];  // 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int& n = held[dev & 63][c];
  if (n == 0) {
    auto kern = k_kv8_attn<true, 128, 1>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)c, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c);
    cfg.blockDim = dim3(KaShape<true, 128, 1>::WARPS * 32);
    cfg.dynamicSmemBytes = KaShape<true, 128, 1>::smem(KaShape<true, 128, 1>::WARPS);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess) {
      cudaGetLastError();
      got = 0;
    }
    n = got > 0 ? got : -1;
  }
  return n > 0 ? n : 0;
}

// How a call is cut up.  Every sequence is taken to have rows / S rows and the
// table's width of positions.  The three forms cost, fitted to 531 shapes of 1 to
// 64 sequences, 600 to 20,000 positions, 1 to 24 rows a sequence (us, head size
// 128; 64 in brackets):
//   clusters  5 + 3 a wave + 1.25 (0.75) an iteration of a warp; 9 for 5 with 4
//             n-tiles, whose results take longer to join
//   many      14 (16 with 4 n-tiles) + 0.94 (0.56) an iteration: even stretches,
//             a second launch
//   tcgen05   24 + 1.4 (1.2) a tile of a CTA for f32 rows, 1.0 (0.85) for 16-bit
//             ones: pays when 128 rows share a reading
// The form chosen so was within 1 % of the best one on average, 27 % at worst, with
// tables as wide as the longest sequence.  Wider ones mislead it: 8 sequences of 512
// positions take 7.9 us, 12.3 with 2048 columns of 64; 5 rows each 13.6 and 26.0.
// (16-bit rows: fitted when a weight was one f16, which made all forms 5 to 12 %
// faster.)
// f32 rows, 32 heads on 8 of 128, us for the three: 8 sequences of 4000 positions,
// 1 row, 16.0, 21.7, 39.4; 16 of 8000, 39.4, 31.7, 90.1; 16 of 4500, 24 rows, 212,
// 187, 88.
struct KaPlan {
  bool tc;     // k_kv8_attn_tc
  int nt, GH, hgroups, QT;
  int ctas;    // stretches of k_kv8_attn_many or k_kv8_attn_tc, 0: clusters
  int nsplit;  // CTAs of a cluster
  int64_t slots;
  size_t meta, bytes;  // workspace
};

static KaPlan ka_plan(bool wide, int hd, int64_t rows, int64_t S, int n_heads, int n_kv, int64_t positions) {
  KaPlan p{};
  const int G = n_heads / n_kv, sms = num_sms();
  const int64_t avg = (rows + S - 1) / S, want = avg * G;  // rows per kv head of an average sequence
  const int64_t blocks = (positions + KV8_BLOCK - 1) / KV8_BLOCK;
  const int cols = wide ? 2 : 1;
  p.nt = want * cols <= 8 ? 1 : want * cols <= 16 ? 2 : 4;
  // groups of a sequence on all kv heads: `rmax` rows each
  auto cut = [&](int rmax) {
    p.GH = std::min(G, rmax);
    p.hgroups = ceil_div(G, p.GH);
    p.QT = rows <= S ? 1 : rmax / p.GH;
    return (avg + p.QT - 1) / p.QT * n_kv * p.hgroups;
  };
  int rmax = 8 * p.nt / cols;
  const int64_t reg = S * cut(rmax), tc = S * cut(KT_ROWS);
  const int per_it = ka_bpi(p.nt) * ka_warps(p.nt);
  const int64_t most = (blocks + per_it - 1) / per_it;
  p.nsplit = 1;
  for (int c = 8; c > 1 && p.nsplit == 1; --c)
    if (c <= most && reg <= ka_clusters(c)) p.nsplit = c;
  const int64_t waves = (reg * p.nsplit + sms - 1) / sms, its = (most + p.nsplit - 1) / p.nsplit;
  // at most 8 CTAs to a unit: their results are joined one after the other
  const int many_ctas = (int)std::min<int64_t>(ka_warps(p.nt) / 4 * sms, reg * 8);
  const int tc_ctas = (int)std::min<int64_t>(kv8_attn_tc_ctas(), tc * 8);
  const double turn = hd == 128 ? 1.25 : 0.75;
  const double t_cluster = (p.nt < 4 ? 5 : 9) + waves * (3 + turn * its);
  const double t_many =
      (p.nt < 4 ? 14 : 16) + 0.75 * turn * reg * blocks / (ka_bpi(p.nt) * 4.0 * many_ctas);
  const double t_tc = 24 + (hd == 128 ? 1.0 : 0.85) * (wide ? 1.4 : 1.0) * tc * ((blocks + KV8_TILE - 1) / KV8_TILE) / tc_ctas;
  p.tc = p.nt == 4 && G <= KT_ROWS && t_tc < std::min(t_cluster, t_many);
  if (p.tc || t_many < t_cluster) p.ctas = p.tc ? tc_ctas : many_ctas;
  if (p.tc) rmax = KT_ROWS;
  cut(rmax);
  p.slots = p.QT > 1 ? rows / p.QT + S : rows;  // room for the groups, about half of it used where QT > 1
  if (p.ctas) {
    p.meta = (size_t)p.ctas * (p.tc ? 3 : 2) * rmax * (hd + 2) * 4;  // tc: and a place for flushed sums
    p.bytes = p.meta + (size_t)p.ctas * 2 * sizeof(int4);
  }
  return p;
}

template <bool WIDE, int HD, int NT>
static int attn_run(const Kv8AttnArgs& a, const KaPlan& p, cudaStream_t st) {
  using Sh = KaShape<WIDE, HD, NT>;
  auto few = k_kv8_attn<WIDE, HD, NT>;
  auto many = k_kv8_attn_many<WIDE, HD, NT>;
  static bool ready[64] = {false};
  int dev = 0;
  Q8_CUDA(cudaGetDevice(&dev));
  if (!ready[dev & 63]) {
    Q8_CUDA(cudaFuncSetAttribute(few, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::smem(Sh::WARPS)));
    Q8_CUDA(cudaFuncSetAttribute(many, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::smem(4)));
    ready[dev & 63] = true;
  }
  if (p.ctas) {
    many<<<p.ctas, 128, Sh::smem(4), st>>>(a);
    Q8_TRY(launch_check("k_kv8_attn_many"));
    return kv8_attn_join(a, p.ctas, Sh::RMAX, st);
  }
  Q8_CHECK_ARG(p.slots * p.nsplit < ((int64_t)1 << 31) && (int64_t)a.kv.n_kv * a.hgroups <= 65535,
               "q8op_kv8_attention: too many rows or heads");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)p.nsplit, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.slots * p.nsplit), a.kv.n_kv * a.hgroups);
  cfg.blockDim = dim3(Sh::WARPS * 32);
  cfg.dynamicSmemBytes = Sh::smem(Sh::WARPS);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launch_status("k_kv8_attn", cudaLaunchKernelEx(&cfg, few, a));
}

template <bool WIDE, int HD>
static int attn_pick(const Kv8AttnArgs& a, const KaPlan& p, cudaStream_t st) {
  if (p.nt == 1) return attn_run<WIDE, HD, 1>(a, p, st);
  if (p.nt == 2) return attn_run<WIDE, HD, 2>(a, p, st);
  return attn_run<WIDE, HD, 4>(a, p, st);
}

}  // namespace q8

using namespace q8;

extern "C" size_t q8op_kv8_attention_workspace(int dtype, int64_t rows, int64_t S, int n_heads, int n_kv, int head_dim,
                                               int64_t positions) {
  if (rows <= 0 || S <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || head_dim <= 0 || positions < 0) return 0;
  return ka_plan(dtype == Q8_F32, head_dim, rows, S, n_heads, n_kv, positions).bytes;
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
  const KaPlan p = ka_plan(dtype == Q8_F32, kv->head_dim, rows, S, n_heads, kv->n_kv, (int64_t)max_pages * kv->page);
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
