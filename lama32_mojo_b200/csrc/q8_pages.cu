// Page tables of a paged KV cache on the device: truncating and freeing,
// forking with shared pages, reserving (allocation and copy-on-write),
// compacting the pool, and the page copies that the last two ask for.
//
// State: table [S, max_pages] int32 (negative: no page), ctx [S] int32
// lengths, refs [num_pages] int32, the table entries that hold a page; 0 is
// free.  There is no list of free pages: a page is taken by scanning refs, the
// lowest number first, so equal states give equal results.  Sums into refs are
// integer atomics; their order does not matter.
//
// Bound: chains of loads and barriers, not bytes.  64 sequences, 17 columns, 389
// pages, everything in the caches: truncate 1.8, fork 4.9, reserve 3.7, compact
// 4.5 us (3.6, 7.0, 10.9 and, of 3000 pages, 8.3 with nothing there).  Truncate has
// a CTA for each sequence (2048 columns: 3.5 us); the others are one CTA each and
// grow:  fork with the table's columns, a strip of 4 to 32 after the other whatever
// the lengths are (2048 columns: 112 us; 1024 sequences 1.3 ms);  reserve and compact
// with the pool, 1024 counts in a round of three barriers, compact three times (16,384
// pages: 12.6 and 25 us, 262,144: 149 and 375);  reserve also compares every
// sequence that writes into a shared page with all sequences.
#include "q8_kernels.h"

#include <algorithm>

namespace q8 {

constexpr int PG_MAX_SEQS = 8192;

struct PageState {
  int32_t* table;
  int S, max_pages;
  int32_t* ctx;
  int32_t* refs;
  int num_pages, page;
};

__device__ __forceinline__ bool pg_valid(const PageState& p, int e) { return e >= 0 && e < p.num_pages; }

// Exclusive prefix sum of one int per thread of a 1024-thread block; total in *sum.
__device__ __forceinline__ int pg_scan(int v, int* s_warp, int* sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s_warp may still be read from an earlier call
  if (lane == 31) s_warp[w] = x;
  __syncthreads();
  if (w == 0) {
    int y = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    s_warp[lane] = y;
  }
  __syncthreads();
  *sum = s_warp[31];
  return x - v + (w ? s_warp[w - 1] : 0);
}

// ------------------------------------------------------------------ truncate
__global__ void __launch_bounds__(256) k_pg_truncate(PageState p, const int32_t* __restrict__ new_len) {
  const int s = blockIdx.x;
  const int len = new_len[s];
  if (len < 0) return;
  const int cut = min(len, max(p.ctx[s], 0));
  __syncthreads();
  if (threadIdx.x == 0) p.ctx[s] = cut;
  int32_t* row = p.table + (int64_t)s * p.max_pages;
  for (int j = cut / p.page + (cut % p.page != 0) + threadIdx.x; j < p.max_pages; j += blockDim.x) {
    const int e = row[j];
    if (e < 0) continue;
    if (pg_valid(p, e)) atomicSub(p.refs + e, 1);
    row[j] = -1;
  }
}

// ------------------------------------------------------------------ fork
// One CTA.  Columns of the table do not touch one another, so a strip of
// columns is read for every pair before it is written for any: sources that
// are destinations of other pairs are taken as they were before the call.
__global__ void __launch_bounds__(1024) k_pg_fork(PageState p, const int32_t* __restrict__ src,
                                                  const int32_t* __restrict__ dst, int n, int strip) {
  extern __shared__ int sm[];
  int* owner = sm;          // [S] the last pair that writes a sequence, -1: none
  int* lens = sm + p.S;     // [n] length of the pair's source
  int* ent = lens + n;      // [n][strip]
  for (int s = threadIdx.x; s < p.S; s += blockDim.x) owner[s] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int a = src[i], b = dst[i];
    if (a < 0 || a >= p.S || b < 0 || b >= p.S) continue;
    lens[i] = max(p.ctx[a], 0);
    atomicMax(owner + b, i);
  }
  __syncthreads();
  for (int c0 = 0; c0 < p.max_pages; c0 += strip) {
    for (int k = threadIdx.x; k < n * strip; k += blockDim.x) {
      const int i = k / strip, c = c0 + k % strip;
      const int b = dst[i];
      if (b < 0 || b >= p.S || owner[b] != i || c >= p.max_pages) continue;
      const int e = p.table[(int64_t)src[i] * p.max_pages + c];
      ent[k] = (int64_t)c * p.page < lens[i] && pg_valid(p, e) ? e : -1;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < n * strip; k += blockDim.x) {
      const int i = k / strip, c = c0 + k % strip;
      const int b = dst[i];
      if (b < 0 || b >= p.S || owner[b] != i || c >= p.max_pages) continue;
      int32_t* at = p.table + (int64_t)b * p.max_pages + c;
      const int old = *at, now = ent[k];
      if (pg_valid(p, old)) atomicSub(p.refs + old, 1);
      if (now >= 0) atomicAdd(p.refs + now, 1);
      *at = now;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int b = dst[i];
    if (b >= 0 && b < p.S && owner[b] == i) p.ctx[b] = lens[i];
  }
}

// ------------------------------------------------------------------ reserve
// One CTA.  Requests are ordered by (sequence, position); request k takes the
// k-th free page.  Nothing changes unless every request can be met.
__global__ void __launch_bounds__(1024) k_pg_reserve(PageState p, const int32_t* __restrict__ n_new,
                                                     int32_t* __restrict__ src, int32_t* __restrict__ dst,
                                                     int32_t* __restrict__ status, int32_t* __restrict__ work) {
  extern __shared__ int sm[];
  int* edge = sm;         // [S] shared page that the first new token falls into, -1: none
  int* cnt = sm + p.S;    // [S] pages wanted; then the number of the first
  __shared__ int s_warp[32];
  __shared__ int s_over;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (threadIdx.x == 0) s_over = 0;
  __syncthreads();
  // a warp per sequence: missing entries among the columns it will write
  for (int s = w; s < p.S; s += nw) {
    const int n = n_new[s], len = max(p.ctx[s], 0);
    const int32_t* row = p.table + (int64_t)s * p.max_pages;
    int c = 0, e0 = -1;
    if (n > 0) {
      const int64_t a = len / p.page, z = ((int64_t)len + n - 1) / p.page;
      if (z >= p.max_pages) {
        if (lane == 0) s_over = 1;
      } else {
        for (int64_t j = a + lane; j <= z; j += 32) c += row[j] < 0;
        c = __reduce_add_sync(0xffffffffu, c);
        if (len % p.page) {
          const int e = row[a];
          if (pg_valid(p, e) && p.refs[e] > 1) e0 = e;
        }
      }
    }
    if (lane == 0) {
      edge[s] = e0;
      cnt[s] = c;
    }
  }
  __syncthreads();
  // the first of a page's sharers keeps it when all of them write
  for (int s = threadIdx.x; s < p.S; s += blockDim.x) {
    const int e = edge[s];
    if (e < 0) continue;
    int all = 0, lower = 0;
    for (int t = 0; t < p.S; ++t) {
      const bool same = edge[t] == e;
      all += same;
      lower += same && t < s;
    }
    if (!(all == p.refs[e] && lower == 0)) cnt[s] |= 1 << 30;  // copies: one page more
  }
  __syncthreads();
  int total = 0;
  for (int s0 = 0; s0 < p.S; s0 += blockDim.x) {
    const int s = s0 + threadIdx.x;
    const int raw = s < p.S ? cnt[s] : 0;
    const bool cow = raw >> 30 & 1;
    int sum;
    const int at = total + pg_scan((raw & ~(1 << 30)) + cow, s_warp, &sum);
    if (s < p.S) {
      cnt[s] = at;
      if (!cow) edge[s] = -1;
    }
    total += sum;
  }
  int free_pages = 0;
  for (int e0 = 0; e0 < p.num_pages; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const bool f = e < p.num_pages && p.refs[e] <= 0;
    int sum;
    const int at = free_pages + pg_scan(f, s_warp, &sum);
    if (f && at < total) work[at] = e;
    free_pages += sum;
  }
  __syncthreads();
  const bool ok = !s_over && total <= free_pages;
  if (threadIdx.x == 0) {
    status[0] = ok ? Q8_OK : Q8_ERR_KV_FULL;
    status[1] = total;
    status[2] = ok ? free_pages - total : free_pages;
  }
  for (int s = w; s < p.S; s += nw) {
    const int n = n_new[s], e0 = edge[s];
    int got = -1;
    if (ok && n > 0) {
      const int len = max(p.ctx[s], 0);
      int32_t* row = p.table + (int64_t)s * p.max_pages;
      const int64_t a = len / p.page, z = ((int64_t)len + n - 1) / p.page;
      int at = cnt[s];
      if (e0 >= 0) {
        got = work[at];
        if (lane == 0) {
          atomicSub(p.refs + e0, 1);
          p.refs[got] = 1;
          row[a] = got;
        }
        ++at;
      }
      for (int64_t j0 = a + (e0 >= 0); j0 <= z; j0 += 32) {
        const int64_t j = j0 + lane;
        const bool miss = j <= z && row[j] < 0;
        const unsigned m = __ballot_sync(0xffffffffu, miss);
        if (miss) {
          const int e = work[at + __popc(m & ((1u << lane) - 1u))];
          row[j] = e;
          p.refs[e] = 1;
        }
        at += __popc(m);
      }
      __syncwarp();
      if (lane == 0) p.ctx[s] = len + n;
    }
    if (lane == 0) {
      src[s] = got < 0 ? -1 : e0;
      dst[s] = got;
    }
  }
}

// ------------------------------------------------------------------ compact
// One CTA: pages in use keep their order where they move to: the k-th used
// page above the number of used pages goes to the k-th free one below it.
__global__ void __launch_bounds__(1024) k_pg_compact(PageState p, int32_t* __restrict__ src, int32_t* __restrict__ dst,
                                                     int32_t* __restrict__ work) {
  __shared__ int s_warp[32];
  int used = 0;
  for (int e0 = 0; e0 < p.num_pages; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int sum;
    pg_scan(e < p.num_pages && p.refs[e] > 0, s_warp, &sum);
    used += sum;
  }
  int nsrc = 0, ndst = 0;
  for (int e0 = 0; e0 < p.num_pages; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const bool u = e < p.num_pages && p.refs[e] > 0;
    const bool from = u && e >= used, to = e < p.num_pages && !u && e < used;
    int a, b;
    const int ia = nsrc + pg_scan(from, s_warp, &a), ib = ndst + pg_scan(to, s_warp, &b);
    if (from) src[ia] = e;
    if (to) dst[ib] = e;
    if (e < p.num_pages) work[e] = e;
    nsrc += a;
    ndst += b;
  }
  for (int k = nsrc + threadIdx.x; k < p.num_pages / 2; k += blockDim.x) src[k] = dst[k] = -1;
  __syncthreads();
  for (int k = threadIdx.x; k < nsrc; k += blockDim.x) {
    const int a = src[k], b = dst[k];
    p.refs[b] = p.refs[a];
    p.refs[a] = 0;
    work[a] = b;
  }
}

// table entries -> new numbers; an entry whose page nobody counted stays
__global__ void k_pg_remap(PageState p, const int32_t* __restrict__ work) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)p.S * p.max_pages) return;
  const int e = p.table[i];
  if (pg_valid(p, e)) p.table[i] = work[e];
}

// ------------------------------------------------------------------ copies
constexpr int PG_MAX_POOLS = 64;
constexpr int PG_WINDOW = 1 << 18;  // page numbers per pass of the bitmaps

struct PoolList {
  uint8_t* base[PG_MAX_POOLS];
  int64_t bytes[PG_MAX_POOLS];
  int n;
};

// A pair is left out when its destination is a source of the call, or the
// destination of another pair: what such copies leave would depend on their
// order.  Every CTA marks the call's page numbers in bitmaps (sources,
// destinations, destinations seen twice), lists the pairs that remain, and
// takes its share of their 16 KB pieces: 64 bytes of a piece per thread, all
// loaded before the first is stored.  0.77 GB: 123 us, 6.3 TB/s or 0.96 of a
// copy's rate; 50 MB: 10 us.
constexpr int PG_COPY_THREADS = 256;
constexpr int PG_PIECE = PG_COPY_THREADS * 64;
constexpr int PG_LIST = 2048;  // pairs per pass

__global__ void __launch_bounds__(PG_COPY_THREADS) k_pg_copy(PoolList pools, int num_pages,
                                                             const int32_t* __restrict__ src,
                                                             const int32_t* __restrict__ dst, int n) {
  extern __shared__ unsigned bits[];
  __shared__ int2 s_list[PG_LIST];
  __shared__ int s_at[PG_MAX_POOLS + 1];  // first piece of each pool within a page
  __shared__ int s_warp[PG_COPY_THREADS / 32];
  const int words = (min(num_pages, PG_WINDOW) + 31) / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned *is_src = bits, *is_dst = bits + words, *twice = bits + 2 * words;
  if (threadIdx.x == 0) {
    int at = 0;
    for (int k = 0; k < pools.n; ++k) {
      s_at[k] = at;
      at += (int)((pools.bytes[k] + PG_PIECE - 1) / PG_PIECE);
    }
    s_at[pools.n] = at;
  }
  for (int w0 = 0; w0 < num_pages; w0 += PG_WINDOW) {
    __syncthreads();
    for (int i = threadIdx.x; i < 3 * words; i += PG_COPY_THREADS) bits[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PG_COPY_THREADS) {
      const int a = src[i], b = dst[i];
      if (a < 0 || a >= num_pages || b < 0 || b >= num_pages) continue;
      const int ra = a - w0, rb = b - w0;
      if (ra >= 0 && ra < PG_WINDOW) atomicOr(is_src + (ra >> 5), 1u << (ra & 31));
      if (rb >= 0 && rb < PG_WINDOW) {
        const unsigned bit = 1u << (rb & 31);
        if (atomicOr(is_dst + (rb >> 5), bit) & bit) atomicOr(twice + (rb >> 5), bit);
      }
    }
    __syncthreads();
    for (int p0 = 0; p0 < n; p0 += PG_LIST) {
      int listed = 0;
      for (int i0 = p0; i0 < min(n, p0 + PG_LIST); i0 += PG_COPY_THREADS) {
        const int i = i0 + threadIdx.x;
        int a = -1, b = -1;
        if (i < n) a = src[i], b = dst[i];
        const int rb = b - w0;
        bool ok = a >= 0 && a < num_pages && b >= 0 && b < num_pages && rb >= 0 && rb < PG_WINDOW;
        if (ok) ok = !((is_src[rb >> 5] | twice[rb >> 5]) >> (rb & 31) & 1);
        const unsigned m = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) s_warp[warp] = __popc(m);
        __syncthreads();
        int at = listed;
        for (int k = 0; k < PG_COPY_THREADS / 32; ++k) {
          if (k < warp) at += s_warp[k];
          listed += s_warp[k];
        }
        if (ok) s_list[at + __popc(m & ((1u << lane) - 1u))] = make_int2(a, b);
        __syncthreads();
      }
      const int per = s_at[pools.n];
      for (int64_t u = blockIdx.x; u < (int64_t)listed * per; u += gridDim.x) {
        const int2 pair = s_list[u / per];
        const int c = (int)(u % per);
        int k = 0;
        while (c >= s_at[k + 1]) ++k;
        const int64_t bytes = pools.bytes[k], o = (int64_t)(c - s_at[k]) * PG_PIECE;
        const uint8_t* from = pools.base[k] + pair.x * bytes + o;
        uint8_t* to = pools.base[k] + pair.y * bytes + o;
        const int len = (int)min((int64_t)PG_PIECE, bytes - o);
        if ((((uintptr_t)pools.base[k] | bytes) & 15) == 0) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = (i * PG_COPY_THREADS + threadIdx.x) * 16;
            if (at < len) v[i] = __ldcs(reinterpret_cast<const uint4*>(from + at));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = (i * PG_COPY_THREADS + threadIdx.x) * 16;
            if (at < len) __stcs(reinterpret_cast<uint4*>(to + at), v[i]);
          }
        } else {
          for (int i = threadIdx.x; i < len; i += PG_COPY_THREADS) to[i] = from[i];
        }
      }
      __syncthreads();  // the list is used again
    }
  }
}

static int pg_check(const char* what, const void* table, int64_t S, int max_pages, const void* refs,
                    int64_t num_pages, int page) {
  Q8_CHECK_ARG((table || S == 0) && refs, "%s: null pointer", what);  // an empty tensor's address is null
  Q8_CHECK_ARG(S >= 0 && S <= PG_MAX_SEQS && max_pages > 0 && max_pages <= (1 << 24),
               "%s: bad table (%lld sequences, at most %d; %d columns)", what, (long long)S, PG_MAX_SEQS, max_pages);
  Q8_CHECK_ARG(num_pages > 0 && num_pages <= (1 << 30) && page > 0 && page <= (1 << 20),
               "%s: bad pool (%lld pages of %d tokens)", what, (long long)num_pages, page);
  Q8_CHECK_ARG(S * max_pages <= INT32_MAX && (int64_t)max_pages * page <= INT32_MAX,
               "%s: the table has more than 2^31 - 1 entries or positions", what);
  return Q8_OK;
}

// Opt-in above 48 KB (the kernels' static arrays included): always the kernel's own largest size, so that two threads
// that call at once ask for the same.
template <typename K>
static int pg_smem(K kern, size_t bytes, int most) {
  if (bytes > 24 * 1024) Q8_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  return Q8_OK;
}

}  // namespace q8

using namespace q8;

extern "C" int q8op_kv_truncate(int32_t* block_table, int64_t S, int max_pages, int32_t* ctx, int32_t* refs,
                                int64_t num_pages, int page, const int32_t* new_len, void* stream) {
  Q8_TRY(pg_check("q8op_kv_truncate", block_table, S, max_pages, refs, num_pages, page));
  if (S == 0) return Q8_OK;
  Q8_CHECK_ARG(ctx && new_len, "q8op_kv_truncate: null pointer");
  const PageState p{block_table, (int)S, max_pages, ctx, refs, (int)num_pages, page};
  k_pg_truncate<<<(int)S, 256, 0, (cudaStream_t)stream>>>(p, new_len);
  return launch_check("k_pg_truncate");
}

extern "C" int q8op_kv_fork(int32_t* block_table, int64_t S, int max_pages, int32_t* ctx, int32_t* refs,
                            int64_t num_pages, int page, const int32_t* src, const int32_t* dst, int64_t n,
                            void* stream) {
  Q8_TRY(pg_check("q8op_kv_fork", block_table, S, max_pages, refs, num_pages, page));
  Q8_CHECK_ARG(n >= 0 && n <= PG_MAX_SEQS, "q8op_kv_fork: %lld pairs, at most %d", (long long)n, PG_MAX_SEQS);
  if (S == 0 || n == 0) return Q8_OK;
  Q8_CHECK_ARG(ctx && src && dst, "q8op_kv_fork: null pointer");
  const PageState p{block_table, (int)S, max_pages, ctx, refs, (int)num_pages, page};
  const int strip = (int)std::min<int64_t>(32, 32768 / n);
  const size_t smem = (size_t)(S + n + n * strip) * 4;
  Q8_TRY(pg_smem(k_pg_fork, smem, (2 * PG_MAX_SEQS + 32768) * 4));
  k_pg_fork<<<1, 1024, smem, (cudaStream_t)stream>>>(p, src, dst, (int)n, strip);
  return launch_check("k_pg_fork");
}

extern "C" int q8op_kv_reserve(int32_t* block_table, int64_t S, int max_pages, int32_t* ctx, int32_t* refs,
                               int64_t num_pages, int page, const int32_t* n_new, int32_t* src, int32_t* dst,
                               int32_t* status, int32_t* work, void* stream) {
  Q8_TRY(pg_check("q8op_kv_reserve", block_table, S, max_pages, refs, num_pages, page));
  Q8_CHECK_ARG((S == 0 || (ctx && n_new && src && dst)) && status && work, "q8op_kv_reserve: null pointer");
  const PageState p{block_table, (int)S, max_pages, ctx, refs, (int)num_pages, page};
  const size_t smem = (size_t)S * 8;
  Q8_TRY(pg_smem(k_pg_reserve, smem, PG_MAX_SEQS * 8));
  k_pg_reserve<<<1, 1024, smem, (cudaStream_t)stream>>>(p, n_new, src, dst, status, work);
  return launch_check("k_pg_reserve");
}

extern "C" int q8op_kv_compact(int32_t* block_table, int64_t S, int max_pages, int32_t* refs, int64_t num_pages,
                               int32_t* src, int32_t* dst, int32_t* work, void* stream) {
  Q8_TRY(pg_check("q8op_kv_compact", block_table, S, max_pages, refs, num_pages, 1));
  Q8_CHECK_ARG((num_pages < 2 || (src && dst)) && work, "q8op_kv_compact: null pointer");
  const PageState p{block_table, (int)S, max_pages, nullptr, refs, (int)num_pages, 1};
  cudaStream_t st = (cudaStream_t)stream;
  k_pg_compact<<<1, 1024, 0, st>>>(p, src, dst, work);
  Q8_TRY(launch_check("k_pg_compact"));
  if (S == 0) return Q8_OK;
  k_pg_remap<<<ceil_div(S * max_pages, 256), 256, 0, st>>>(p, work);
  return launch_check("k_pg_remap");
}

extern "C" int q8op_kv_copy_pages(void* const* pools, const int64_t* page_bytes, int n_pools, int64_t num_pages,
                                  const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  Q8_CHECK_ARG(n_pools >= 0 && n_pools <= PG_MAX_POOLS, "q8op_kv_copy_pages: %d pools, at most %d", n_pools,
               PG_MAX_POOLS);
  Q8_CHECK_ARG(n >= 0 && n <= (1 << 30) && num_pages > 0 && num_pages <= (1 << 30),
               "q8op_kv_copy_pages: bad shape (%lld pairs, %lld pages)", (long long)n, (long long)num_pages);
  if (n == 0 || n_pools == 0) return Q8_OK;
  Q8_CHECK_ARG(pools && page_bytes && src && dst, "q8op_kv_copy_pages: null pointer");
  PoolList l{};
  l.n = n_pools;
  int64_t pieces = 0;
  for (int i = 0; i < n_pools; ++i) {
    Q8_CHECK_ARG(pools[i] && page_bytes[i] > 0, "q8op_kv_copy_pages: pool %d is null or empty", i);
    l.base[i] = (uint8_t*)pools[i];
    l.bytes[i] = page_bytes[i];
    pieces += (page_bytes[i] + PG_PIECE - 1) / PG_PIECE;
  }
  Q8_CHECK_ARG(pieces < ((int64_t)1 << 30), "q8op_kv_copy_pages: pages of more than 16 TB");
  const size_t smem = (size_t)((std::min<int64_t>(num_pages, PG_WINDOW) + 31) / 32) * 12;
  Q8_TRY(pg_smem(k_pg_copy, smem, PG_WINDOW / 32 * 12));
  const int grid = (int)std::min<int64_t>(n * pieces, 6 * num_sms());
  k_pg_copy<<<grid, PG_COPY_THREADS, smem, (cudaStream_t)stream>>>(l, (int)num_pages, src, dst, (int)n);
  return launch_check("k_pg_copy");
}
