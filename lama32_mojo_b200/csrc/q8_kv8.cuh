// What the kernels of the 8-bit paged KV cache share (q8_kv8.cu, q8_kv8_attn.cu).
//
// Pages of one layer: codes [num_pages, n_kv, page, hd] int8 and one f32 scale
// for every 16 tokens of a kv head, [num_pages, n_kv, page/16]; a value is
// code * scale.  A call's rows are packed: rows starts[b] .. starts[b+1]-1
// belong to sequence b and are its last positions, ctx[b]-n .. ctx[b]-1.
// Everything that comes from device memory (starts, ctx, table) is bounded
// before it is used as an index: a table entry outside [0, num_pages) or a
// position past the table is a page that is not there.
#pragma once
#include "q8_common.cuh"

namespace q8 {

constexpr int KV8_BLOCK = Q8_KV8_BLOCK;

// The rows of one sequence in a call.
struct Kv8Seq {
  int b;        // sequence, -1: none
  int row0;     // its first row
  int n;        // its rows
  int64_t pos0; // position of row0 (negative: rows before the sequence's start)
};

__device__ __forceinline__ Kv8Seq kv8_seq(const int32_t* starts, const int32_t* ctx, int b, int rows) {
  Kv8Seq s;
  s.b = b;
  s.row0 = min(max(starts[b], 0), rows);
  s.n = min(max(starts[b + 1], s.row0), rows) - s.row0;
  s.pos0 = (int64_t)ctx[b] - s.n;
  return s;
}

// Page of position p, or -1.
__device__ __forceinline__ int kv8_page(const int32_t* table_row, int max_pages, int64_t num_pages, int page,
                                        int64_t p) {
  if (p < 0) return -1;
  const uint32_t j = (uint32_t)p / (uint32_t)page;  // a position is below ctx, an int32
  if (j >= (uint32_t)max_pages) return -1;
  const int e = table_row[j];
  return e >= 0 && e < num_pages ? e : -1;
}

// Sequence of slot g, slots of sequence b starting at starts[b] / per + more b,
// by one warp; -1: before the first.
__device__ __forceinline__ int kv8_find_warp(const int32_t* starts, int S, int rows, int per, int more, int slot) {
  int n = 0;
  for (int b = threadIdx.x & 31; b < S; b += 32) n += min(max(starts[b], 0), rows) / per + more * b <= slot;
  return __reduce_add_sync(0xffffffffu, n) - 1;
}

int kv8_check(const char* what, const q8_kv8_pages* kv, const int32_t* seq_start, const int32_t* ctx, int64_t S,
              int64_t rows, const int32_t* block_table, int max_pages);

}  // namespace q8
