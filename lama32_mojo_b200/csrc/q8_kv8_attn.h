// Shared by the attention kernels of the 8-bit cache: q8_kv8_attn.cu (entry
// point, few rows per kv head: decode steps and drafts) and q8_kv8_attn_tc.cu
// (many rows: chunks of prompts).
#pragma once
#include "q8_kernels.h"
#include "q8_kv8.cuh"

#include <math.h>

namespace q8 {

// M of a block: s + log2(sv) less KA_DOWN, a sv below 2^KA_LEAST counting as that, so that e = 2^(s - M) is
// between 2^(24 - 121) for the largest sv and 2^(24 + 72) for the least one: l = sum e of 2^31 positions
// stays finite, and what e can lose below f32's smallest normal number is 2^-29 of the row's largest weight.
constexpr float KA_DOWN = 24.f, KA_LEAST = -72.f;
constexpr float KA_LIFT = 0x1p-9f;  // weights are e sv KA_LIFT: the largest is 2^15

struct Kv8AttnArgs {
  const void* q;
  int64_t ldq;
  int dtype, rows;
  const int32_t* starts;
  const int32_t* ctx;
  int S, n_heads;
  q8_kv8_pages kv;
  const int32_t* table;
  int max_pages;
  void* out;
  int64_t ldo;
  int QT, GH, hgroups;  // tokens per group, heads per group, head groups per kv head
  float* work;          // two partial results for every CTA, then k_kv8_attn_tc's flushed sums
  int4* work_meta;      // and what they are
};

// four biased codes (c + 128) -> f16 pairs (bytes 0, 1) and (bytes 2, 3): 0x64uu is 1024 + u
__device__ __forceinline__ uint32_t ka_f16(uint32_t u, uint32_t sel) {
  uint32_t x;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(x) : "r"(u), "r"(0x64646464u), "r"(sel));
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&x), __half2half2(__ushort_as_half((unsigned short)0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t ka_pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// two floats as two bf16 or f16
__device__ __forceinline__ uint32_t ka_pack16(int dtype, float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return dtype == Q8_BF16 ? *reinterpret_cast<const uint32_t*>(&b) : ka_pack(lo, hi);
}

__device__ __forceinline__ float ka_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// l 2^d and 2^d, d <= 0 the step of a running maximum.  Between blocks of the least and the largest scales d lies
// below f32's exponents (-193 and the scores' difference), but l, 2^96 against 2^-97, does not.
template <bool EXACT>
__device__ __forceinline__ float ka_lower(float& l, float d) {
  const bool far = d < -100.f;
  const float e = far ? d + 96.f : d;
  const float f = EXACT ? exp2f(e) : ka_exp2(e);
  l *= f;
  if (far) l *= 0x1p-96f;
  return far ? 0.f : f;
}

// four consecutive elements from element i0 on as floats
template <bool WIDE, bool ALIGNED>
__device__ __forceinline__ void ka_four(float (&v)[4], const void* base, int64_t i0, int dtype) {
  if constexpr (WIDE) {
    const float* p = (const float*)base + i0;
    if constexpr (ALIGNED) {
      const float4 u = *reinterpret_cast<const float4*>(p);
      v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = p[i];
    }
  } else {
    const uint16_t* p = (const uint16_t*)base + i0;
    uint32_t w[2];
    if constexpr (ALIGNED) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w[i]));
      v[2 * i] = dtype == Q8_BF16 ? __uint_as_float(w[i] << 16) : f.x;
      v[2 * i + 1] = dtype == Q8_BF16 ? __uint_as_float(w[i] & 0xffff0000u) : f.y;
    }
  }
}

template <bool WIDE>
__device__ __forceinline__ void ka_store(const Kv8AttnArgs& a, int64_t i, float x) {
  if (WIDE) ((float*)a.out)[i] = x;
  else if (a.dtype == Q8_BF16) ((__nv_bfloat16*)a.out)[i] = __float2bfloat16_rn(x);
  else ((__half*)a.out)[i] = __float2half_rn(x);
}

// A group of rows on one kv head.
struct KaUnit {
  int b, row0, toks;  // sequence, first row, tokens
  int h, head0, heads;
  int64_t pos0;       // position of the first token
  int nblk;           // blocks that the last token sees
};

__device__ __forceinline__ int ka_blocks(const Kv8AttnArgs& a, int64_t end) {
  const int64_t room = (int64_t)a.max_pages * a.kv.page;
  return (int)((min(max(end, (int64_t)0), room) + KV8_BLOCK - 1) / KV8_BLOCK);
}

// j: kv head x head group; i0: first row of the group within the sequence
__device__ __forceinline__ KaUnit ka_unit(const Kv8AttnArgs& a, const Kv8Seq& sq, int j, int i0) {
  KaUnit u;
  const int G = a.n_heads / a.kv.n_kv, hg = j % a.hgroups;
  u.b = sq.b;
  u.row0 = sq.row0 + i0;
  u.toks = min(a.QT, sq.n - i0);
  u.h = j / a.hgroups;
  u.head0 = u.h * G + hg * a.GH;
  u.heads = min(a.GH, G - hg * a.GH);
  u.pos0 = sq.pos0 + i0;
  u.nblk = ka_blocks(a, u.pos0 + u.toks);
  return u;
}

// Element k of a unit's rows, from its lifted sum x and the sum of the weights.
template <bool WIDE, int HD>
__device__ __forceinline__ void ka_write(const Kv8AttnArgs& a, int row0, int head0, int heads, int k, float x,
                                         float sum) {
  const int r = k / HD;
  if (r % a.GH >= heads) return;
  ka_store<WIDE>(a, (int64_t)(row0 + r / a.GH) * a.ldo + (head0 + r % a.GH) * HD + k % HD,
                 sum > 0.f ? x * (1.f / KA_LIFT) / sum : 0.f * (x + sum));  // no position: 0; NaN stays
}

// Inclusive sum over the CTA's threads; *total: all of them.  s: a word per warp.
__device__ __forceinline__ int64_t ka_scan(int64_t v, int64_t* s, int64_t* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // s may still be read
  if (lane == 31) s[w] = v;
  __syncthreads();
  int64_t sum = 0;
  for (int k = 0; k < nw; ++k) {
    if (k == w) v += sum;
    sum += s[k];
  }
  *total = sum;
  return v;
}

// Adds the partial results of units that several CTAs of a launch share
// (records of RMAX rows: o [RMAX][HD], m [RMAX], l [RMAX]).
int kv8_attn_join(const Kv8AttnArgs& a, int ctas, int RMAX, cudaStream_t st);
// Many rows per kv head (tcgen05): 128 rows to a group.
constexpr int KT_ROWS = 128;
constexpr int KV8_TILE = 4;  // blocks of a key tile
int kv8_attn_tc_ctas();
int kv8_attn_tc(const Kv8AttnArgs& a, int ctas, cudaStream_t st);

}  // namespace q8
