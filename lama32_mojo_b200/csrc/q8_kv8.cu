// 8-bit paged KV cache: append and read back.  Layout and packing of a call's
// rows: q8_kv8.cuh.  The f32 cache's append is k_rope_kv (q8_ops.cu).
#include "q8_kernels.h"
#include "q8_kv8.cuh"

#include <math.h>
#include <type_traits>

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
  Q8_CHECK_ARG((int64_t)max_pages * kv->page <= INT32_MAX, "%s: the table has more than 2^31 - 1 positions", what);
  return Q8_OK;
}

// round(x / s), ties to even, within +-127: the quotient of the real numbers,
// not of their f32 rounding.  The estimate r is off by one at most, next to a
// tie; x - r s is exact there: a multiple of the smaller ulp of x and s and at
// most about s / 2.  s > 0; an infinite x gives +-127.
__device__ __forceinline__ int kv8_code(float x, float s) {
  float r = rintf(__fdiv_rn(x, s));
  const float d = fmaf(-r, s, x), two = fabsf(d) * 2.f;
  if (two >= s && (two > s || ((int)r & 1))) r += d > 0.f ? 1.f : -1.f;
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// round(c s0 / s1), ties to even, for a code that stays while its block's scale
// grows; ratio = s0 / s1 rounded.  c ratio is off by less than 127 2^-23, so
// only next to a tie the exact products (64 bits hold them) have to decide.
__device__ __forceinline__ int kv8_rescale(int c, float ratio, float s0, float s1) {
  const float y = (float)c * ratio;
  int r = __float2int_rn(y);
  if (fabsf(fabsf(y - (float)r) - 0.5f) < 0x1p-14f) {
    const double d = (double)c * (double)s0 - (double)r * (double)s1, two = 2.0 * fabs(d);
    if (two > (double)s1 || (two == (double)s1 && (r & 1))) r += d > 0.0 ? 1 : -1;
  }
  return r;
}

// k or v rows of one call
struct Kv8Rows {
  const void* x;
  int64_t ld;
};

__device__ __forceinline__ float kv8_f32(float x) { return x; }
__device__ __forceinline__ float kv8_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float kv8_f32(__half x) { return __half2float(x); }

// elements 2i and 2i + 1 of a 16-byte piece
template <typename T>
__device__ __forceinline__ uint64_t kv8_pair(const uint32_t (&u)[4], int i) {
  if constexpr (sizeof(T) == 4) {
    return (uint64_t)u[2 * i + 1] << 32 | u[2 * i];
  } else if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    return f2_pack(f.x, f.y);
  } else {
    return (uint64_t)(u[i] & 0xffff0000u) << 32 | u[i] << 16;
  }
}

// the larger of top and |w|, by pairs for 16-bit elements; NaN is the largest
template <typename T>
__device__ __forceinline__ unsigned kv8_max(unsigned top, unsigned w) {
  if constexpr (sizeof(T) == 4) {
    return max(top, w & 0x7fffffffu);
  } else {
    typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
    w &= 0x7fff7fffu;
    const T2 m = __hmax2_nan(*reinterpret_cast<T2*>(&top), *reinterpret_cast<T2*>(&w));
    return *reinterpret_cast<const unsigned*>(&m);
  }
}

// One warp per (block of 16 positions, kv head, k or v).  A lane takes 16 bytes
// of a row, the warp as many rows as fit; the rows are read twice, for the
// scale and for the codes (the second time from the caches), which takes half
// the registers of keeping them and leaves room for twice the warps.  Slots
// number the touched blocks: sequence b's start at starts[b]/16 + 2b, which
// leaves room for the n/16 + 2 blocks that n rows can touch.  Bytes: the rows
// once, a quarter or half of that in codes.  12,562 bf16 rows of 8 kv heads of
// 128, 77 MB: 17.4 us with the rows in the L2, 28.7 (under ncu) with nothing there,
// bound by some 20 instructions an element and by the chain from sequence to page
// to rows (no row is loaded before the table has answered, though it could be).
//
// Codes, two at a time in packed f32 operations: m = fma(x, 1/s, 1.5 2^23) rounds to the whole number nearest to the
// estimated quotient and holds it in its low byte; r = m - 1.5 2^23.  The
// estimate is 2 ulps off at most, so r is right, or by one off next to a tie;
// d = x - r s, which is exact, tells: r moves towards x where |d| > s / 2, or
// where it is s / 2 and r odd (m's last bit).  Blocks with numbers that are not
// finite, or scales far outside the usual ones, go the long way (kv8_code).
template <typename T, int HD, bool ALIGNED>  // rows to 16 bytes; known when compiled: a branch at each load costs 4 us
__global__ void __launch_bounds__(128, 10) k_kv8_append(Kv8Rows kr, Kv8Rows vr, int rows,
                                                        const int32_t* __restrict__ starts,
                                                        const int32_t* __restrict__ ctx, int S, q8_kv8_pages kv,
                                                        const int32_t* __restrict__ table, int max_pages) {
  constexpr int E = 16 / sizeof(T), LPR = HD / E, RPI = 32 / LPR;
  const int slot = blockIdx.x, lane = threadIdx.x & 31;
  const int unit = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit >= 2 * kv.n_kv) return;
  const int b = kv8_find_warp(starts, S, rows, KV8_BLOCK, 2, slot);
  if (b < 0) return;
  const Kv8Seq sq = kv8_seq(starts, ctx, b, rows);
  if (sq.n <= 0) return;
  const int64_t first = max(sq.pos0, (int64_t)0);
  const int64_t blk = first / KV8_BLOCK + (slot - (sq.row0 / KV8_BLOCK + 2 * b));
  const int64_t lo = max(blk * KV8_BLOCK, first);
  const int64_t hi = min((blk + 1) * KV8_BLOCK, sq.pos0 + sq.n);
  if (lo >= hi) return;
  const int in = (int)(lo % KV8_BLOCK), cnt = (int)(hi - lo);
  const int row = sq.row0 + (int)(lo - sq.pos0);
  const int h = unit >> 1, tk = lane / LPR, el = (lane % LPR) * E;
  const bool isv = unit & 1;
  const Kv8Rows src = isv ? vr : kr;
  const T* x = (const T*)src.x + (int64_t)row * src.ld + h * HD + el;
  union Piece {
    uint4 w;
    uint32_t u[4];
    T e[E];
    __device__ Piece() {}
  };
  auto load = [&](Piece& v, int t) {
    if constexpr (ALIGNED) {
      v.w = *reinterpret_cast<const uint4*>(x + (int64_t)t * src.ld);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v.e[e] = x[(int64_t)t * src.ld + e];
    }
  };
  const int pg = kv8_page(table + (int64_t)b * max_pages, max_pages, kv.num_pages, kv.page, lo);
  if (pg < 0) return;
  const int64_t cell = (int64_t)pg * kv.n_kv + h;
  const int tok0 = (int)((uint32_t)(blk * KV8_BLOCK) % (uint32_t)kv.page);
  int8_t* codes = (isv ? kv.v : kv.k) + (cell * kv.page + tok0) * HD + el;
  float* scale = (isv ? kv.v_scale : kv.k_scale) + cell * (kv.page / KV8_BLOCK) + tok0 / KV8_BLOCK;
  const float old = in > 0 ? *scale : 0.f;
  // the largest |x| by its bits, which order as the numbers do; non-finite ones lie above
  unsigned top = 0u;
#pragma unroll 4
  for (int t = tk; t < cnt; t += RPI) {
    Piece v;
    load(v, t);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      top = kv8_max<T>(top, v.u[e]);
  }
  if (sizeof(T) == 2) {
    const unsigned short bits = (unsigned short)max(top & 0xffffu, top >> 16);
    top = __float_as_uint(kv8_f32(*reinterpret_cast<const T*>(&bits)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const bool finite = top < 0x7f800000u;
  if (!finite) {  // NaN counts as 0, and infinities do not enter the scale
    top = 0u;
#pragma unroll 1
    for (int t = tk; t < cnt; t += RPI)
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const unsigned a = __float_as_uint(kv8_f32(x[(int64_t)t * src.ld + e])) & 0x7fffffffu;
        if (a < 0x7f800000u) top = max(top, a);
      }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  const float s = fmaxf(old, __fdiv_rn(__uint_as_float(top), 127.f));
  union Codes {
    int8_t c[E];
    typename std::conditional<E == 8, uint2, uint32_t>::type w;
  };
  using Word = decltype(Codes::w);
  if (s != old && in > 0) {
    const float ratio = __fdiv_rn(old, s);
#pragma unroll 4
    for (int t = tk; t < in; t += RPI) {
      Codes k;
      k.w = *reinterpret_cast<const Word*>(codes + t * HD);
#pragma unroll
      for (int e = 0; e < E; ++e) k.c[e] = (int8_t)kv8_rescale(k.c[e], ratio, old, s);
      *reinterpret_cast<Word*>(codes + t * HD) = k.w;
    }
  }
  if (lane == 0) *scale = s;
  const bool plain = finite && s > 0x1p-100f && s < 0x1p100f;
  if (!plain) {
#pragma unroll 1
    for (int t = tk; t < cnt; t += RPI)
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const float a = kv8_f32(x[(int64_t)t * src.ld + e]);
        int c = 0;
        if (a == a) c = s > 0.f ? kv8_code(a, s) : fabsf(a) == INFINITY ? (a < 0.f ? -127 : 127) : 0;
        codes[(in + t) * HD + e] = (int8_t)c;
      }
    return;
  }
  const float inv = 1.f / s, half = s * 0.5f;
  const uint64_t inv2 = f2_pack(inv, inv), s2 = f2_pack(s, s), magic = f2_pack(12582912.f, 12582912.f),
                 minus = f2_pack(-1.f, -1.f);
#pragma unroll 2
  for (int t = tk; t < cnt; t += RPI) {
    Piece v;
    load(v, t);
    uint64_t m[E / 2], d[E / 2];
    bool near = false;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const uint64_t a = kv8_pair<T>(v.u, e);
      m[e] = f2_fma(a, inv2, magic);
      d[e] = f2_fma(f2_fma(m[e], minus, magic), s2, a);
      near |= fabsf(f2_lo(d[e])) >= half || fabsf(f2_hi(d[e])) >= half;
    }
    if (near) {  // next to a tie
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        float mi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float di = i ? f2_hi(d[e]) : f2_lo(d[e]);
          mi[i] = i ? f2_hi(m[e]) : f2_lo(m[e]);
          if (fabsf(di) > half || (fabsf(di) == half && (__float_as_int(mi[i]) & 1))) mi[i] += copysignf(1.f, di);
        }
        m[e] = f2_pack(mi[0], mi[1]);
      }
    }
    uint32_t w[E / 4];
#pragma unroll
    for (int e = 0; e < E / 4; ++e)
      w[e] = __byte_perm(__byte_perm((uint32_t)m[2 * e], (uint32_t)(m[2 * e] >> 32), 0x0040),
                         __byte_perm((uint32_t)m[2 * e + 1], (uint32_t)(m[2 * e + 1] >> 32), 0x0040), 0x5410);
    if constexpr (E == 8) *reinterpret_cast<uint2*>(codes + (in + t) * HD) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(codes + (in + t) * HD) = w[0];
  }
}

// One warp per row of the call; rows without a page read as zeros.  12,599 rows
// of 8 kv heads of 128: 21.3 us for 129 MB (6.1 TB/s, 0.92 of a copy's rate); 27.6
// without streaming stores, four fifths of the bytes being written.
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_read(int rows, const int32_t* __restrict__ starts,
                                                  const int32_t* __restrict__ ctx, int S, q8_kv8_pages kv,
                                                  const int32_t* __restrict__ table, int max_pages,
                                                  float* __restrict__ ko, float* __restrict__ vo) {
  const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= rows) return;
  const int b = kv8_find_warp(starts, S, rows, 1, 0, t);
  if (b < 0) return;
  const Kv8Seq sq = kv8_seq(starts, ctx, b, rows);
  if (t >= sq.row0 + sq.n) return;  // behind the last sequence
  const int64_t p = sq.pos0 + (t - sq.row0);
  const int pg = kv8_page(table + (int64_t)b * max_pages, max_pages, kv.num_pages, kv.page, p);
  const int tok = pg < 0 ? 0 : (int)((uint32_t)p % (uint32_t)kv.page);
  const int64_t cell = (int64_t)max(pg, 0) * kv.n_kv, step = (int64_t)kv.page * HD;
  const int64_t code0 = cell * step + (int64_t)tok * HD, scale0 = cell * (kv.page / KV8_BLOCK) + tok / KV8_BLOCK;
  const int64_t o0 = (int64_t)t * kv.n_kv * HD;
#pragma unroll 4
  for (int i = lane * 4; i < kv.n_kv * HD; i += 128) {
    const int h = i / HD, d = i % HD;
    float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
    if (pg >= 0) {
      const int64_t at = code0 + h * step + d;
      const char4 ck = *reinterpret_cast<const char4*>(kv.k + at), cv = *reinterpret_cast<const char4*>(kv.v + at);
      const int64_t si = scale0 + (int64_t)h * (kv.page / KV8_BLOCK);
      const float sk = kv.k_scale[si], sv = kv.v_scale[si];
      k = make_float4(ck.x * sk, ck.y * sk, ck.z * sk, ck.w * sk);
      v = make_float4(cv.x * sv, cv.y * sv, cv.z * sv, cv.w * sv);
    }
    __stcs(reinterpret_cast<float4*>(ko + o0 + i), k);
    __stcs(reinterpret_cast<float4*>(vo + o0 + i), v);
  }
}

template <typename T, int HD>
static int append_run(const Kv8Rows& k, const Kv8Rows& v, int rows, const int32_t* starts, const int32_t* ctx, int S,
                      const q8_kv8_pages& kv, const int32_t* table, int max_pages, cudaStream_t st) {
  const dim3 grid(rows / KV8_BLOCK + 2 * S, ceil_div(2 * kv.n_kv, 4));
  const bool aligned = (((uintptr_t)k.x | (uintptr_t)v.x | (k.ld * sizeof(T)) | (v.ld * sizeof(T))) & 15) == 0;
  auto kern = aligned ? k_kv8_append<T, HD, true> : k_kv8_append<T, HD, false>;
  kern<<<grid, 128, 0, st>>>(k, v, rows, starts, ctx, S, kv, table, max_pages);
  return launch_check("k_kv8_append");
}

template <typename T>
static int append_run(const Kv8Rows& k, const Kv8Rows& v, int rows, const int32_t* starts, const int32_t* ctx, int S,
                      const q8_kv8_pages& kv, const int32_t* table, int max_pages, cudaStream_t st) {
  return kv.head_dim == 64 ? append_run<T, 64>(k, v, rows, starts, ctx, S, kv, table, max_pages, st)
                           : append_run<T, 128>(k, v, rows, starts, ctx, S, kv, table, max_pages, st);
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
  Q8_CHECK_ARG(k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, "q8op_kv8_read: null or unaligned output");
  cudaStream_t st = (cudaStream_t)stream;
  if (kv->head_dim == 64)
    k_kv8_read<64><<<ceil_div(rows, 8), 256, 0, st>>>((int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, k, v);
  else
    k_kv8_read<128><<<ceil_div(rows, 8), 256, 0, st>>>((int)rows, seq_start, ctx, (int)S, *kv, block_table, max_pages, k, v);
  return launch_check("k_kv8_read");
}
