// Work lists of attention over sequences that are packed back to back: what the attention kernels walk instead of
// (batch, tile) coordinates.  Written by mb_packed_plan (packed_plan.cu) from offsets in device memory, read by the packed
// forms of the attention kernels.
#pragma once

#include <stdint.h>

struct __align__(16) PackedItem {
  int q_row, sq;      // first row and length of the sequence's queries
  int k_row, sk;      // and of its keys
  int first;          // forward: first query of a pair of 128-row tiles; backward: first key of a 128-row block
  int pad[3];
};

// A plan in memory: four lists one behind the other, each a header of 16 bytes (the number of items first) and its items;
// [forward, backward] x [whole sequences visible, causal].  The items of a list are ordered by cost, dearest first.
__host__ __device__ inline long packed_forward_items(long total_q, long n) { return total_q / 256 + n + 1; }
__host__ __device__ inline long packed_backward_items(long total_k, long n) { return total_k / 128 + n + 1; }
__host__ __device__ inline long packed_list_bytes(long items) { return 16 + items * static_cast<long>(sizeof(PackedItem)); }
__host__ __device__ inline long packed_list_offset(long total_q, long total_k, long n, int backward, int causal) {
  const long f = packed_list_bytes(packed_forward_items(total_q, n)), b = packed_list_bytes(packed_backward_items(total_k, n));
  return backward ? 2 * f + causal * b : causal * f;
}
