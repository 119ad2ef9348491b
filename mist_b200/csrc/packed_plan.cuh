// Work lists of attention over sequences that are packed back to back: what the attention kernels walk instead of
// (batch, tile) coordinates.  Written by mb_packed_plan (packed_plan.cu) from offsets in device memory, read by the packed
// forms of the attention kernels.
#pragma once

#include "sm100.cuh"

struct __align__(16) PackedItem {
  int q_row, sq;      // first row and length of the sequence's queries
  int k_row, sk;      // and of its keys
  int first;          // forward: first query of a pair of 128-row tiles; backward: first key of a 128-row block
  int pad[3];
};

// A plan in memory: four lists one behind the other, each a header and its items; [forward, backward] x [whole sequences
// visible, causal].  The items of a list are ordered by cost (blocks of 128 rows that they walk), dearest first.
struct PackedHeader {
  int count, cost, dearest, pad;      // items, what they cost together, what the dearest costs
};
__host__ __device__ inline long packed_forward_items(long total_q, long n) { return total_q / 256 + n + 1; }
__host__ __device__ inline long packed_backward_items(long total_k, long n) { return total_k / 128 + n + 1; }
__host__ __device__ inline long packed_list_bytes(long items) {
  return static_cast<long>(sizeof(PackedHeader)) + items * static_cast<long>(sizeof(PackedItem));
}
__host__ __device__ inline long packed_list_offset(long total_q, long total_k, long n, int backward, int causal) {
  const long f = packed_list_bytes(packed_forward_items(total_q, n)), b = packed_list_bytes(packed_backward_items(total_k, n));
  return backward ? 2 * f + causal * b : causal * f;
}
// Behind the lists: every query row's place in its sequence (int64), then, a byte per row, whether at most one block of keys
// is visible from the row's tile (bit 0: whole sequences visible, bit 1: causal).
__host__ __device__ inline long packed_positions_offset(long total_q, long total_k, long n) {
  return packed_list_offset(total_q, total_k, n, 1, 1) + packed_list_bytes(packed_backward_items(total_k, n));
}
__host__ __device__ inline long packed_single_offset(long total_q, long total_k, long n) {
  return packed_positions_offset(total_q, total_k, n) + 8 * total_q;
}
// Blocks of 128 keys that a tile of 128 queries from q0 on sees, in a sequence of sq queries and sk keys.
__host__ __device__ inline int packed_key_blocks(int q0, int sq, int sk, bool causal) {
  int keys = sk;
  if (causal) {
    const int seen = q0 + 128 + sk - sq;
    keys = seen < keys ? seen : keys;
  }
  return keys > 0 ? (keys + 127) / 128 : 0;
}

// Work items are dealt as they are asked for: a tile of a long sequence takes tens of times as long as one of a short
// sequence, and dealing them in turn left a third of the chip idle at the end (16384 tokens in 14 documents, 32 heads of 128
// over 8: backward 1262 us, forward 481 in the worst order of groups).  The thread that loads claims the next item when it
// has issued the last load of this one, and hands it to the other warps through a ring in shared memory.  Claiming earlier
// would tie items to CTAs that are still busy.

// Heads that are walked together: those whose tensors share L2, but so many that the dearest item, with which the last group
// begins, is no longer than the group's share of a CTA (16384 tokens in 14 documents, 8 units of 4 heads: backward 897 us in
// groups of 1, 845 of 2, 788 of 4, 858 of 8).
__device__ __forceinline__ int heads_together(const PackedHeader* h, int in_l2, int heads) {
  const long cost = h->cost > 0 ? h->cost : 1;
  const long need = (static_cast<long>(h->dearest) * gridDim.x + cost - 1) / cost;
  return static_cast<int>(need > heads ? heads : (need > in_l2 ? need : in_l2));
}

struct ItemRing {
  static constexpr int kSlots = 4;
  static constexpr int kBytes = kSlots * 32 + 2 * kSlots * 8;
  int4* slot;            // {q_row, sq, k_row, sk}, {first, head, valid, -}
  uint64_t* full;
  uint64_t* empty;
  __device__ __forceinline__ explicit ItemRing(uint8_t* at)
      : slot(reinterpret_cast<int4*>(at)), full(reinterpret_cast<uint64_t*>(at + kSlots * 32)), empty(full + kSlots) {}
  __device__ __forceinline__ void init(int consumer_warps) const {
    for (int i = 0; i < kSlots; ++i) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], consumer_warps);
    }
  }
  // Claims item r of this CTA (the first one is the CTA's index) out of items x heads and publishes it; by one thread.
  // false: the wait gave up, or there is no item; a and b are the item.  `group` heads are walked together.
  __device__ __forceinline__ bool claim(int r, int* counter, const PackedItem* items, int count, int heads, int group, int4& a,
                                        int4& b, bool& ok) const {
    const int total = count * heads;
    int t = blockIdx.x;
    if (r > 0) t = counter ? static_cast<int>(gridDim.x) + atomicAdd(counter, 1) : total;
    a = b = make_int4(0, 0, 0, 0);
    if (t < total) {
      const int per_group = group * count;
      const int g = t / per_group, rest = t - g * per_group;
      const int gsize = min(group, heads - g * group);
      const int at = rest / gsize;
      a = *reinterpret_cast<const int4*>(&items[at]);
      b = make_int4(items[at].first, g * group + rest % gsize, 1, 0);
    }
    const int s = r % kSlots;
    if (r >= kSlots && !sm100::mbar_wait(&empty[s], (r / kSlots - 1) & 1)) {
      ok = false;
      return false;
    }
    slot[2 * s] = a;
    slot[2 * s + 1] = b;
    sm100::mbar_arrive(&full[s]);
    return b.z != 0;
  }
  // Item r, by a whole warp (or by the one lane of it that works); false where there is none or the wait gives up.
  template <bool WARP>
  __device__ __forceinline__ bool take(int r, int4& a, int4& b) const {
    const int s = r % kSlots;
    if (!sm100::mbar_wait(&full[s], (r / kSlots) & 1)) return false;
    a = slot[2 * s];
    b = slot[2 * s + 1];
    if (WARP) sm100::mbar_arrive_warp(&empty[s]);
    else sm100::mbar_arrive(&empty[s]);
    return b.z != 0;
  }
};
