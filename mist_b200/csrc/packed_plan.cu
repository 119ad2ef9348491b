// Builds the work lists of attention over packed sequences (packed_plan.cuh) on the device, so that the offsets never
// have to be read back to the host.  A step builds them once and every layer's attention walks them.
#include "common.cuh"
#include "packed_plan.cuh"
#include <string.h>

namespace {

constexpr int kThreads = 1024;
constexpr int kCosts = 8192;       // blocks of 128 a tile walks; dearer ones count as the dearest

// Blocks 0 - 3: one list each.  Counting sort by cost: a warp per sequence, a lane per item.  The offsets are clamped to the tensors,
// so no content of theirs makes an attention kernel leave them.  Rows behind the last sequence get items without keys (or
// queries), whose outputs are zeros.  Items of one cost come in no fixed order; no result depends on it but the order in
// which dQ is summed.
__global__ void __launch_bounds__(kThreads)
packed_plan_kernel(const int* cu_q, const int* cu_k, int n, int total_q, int total_k, uint8_t* plan, int* ends) {
  if (ends && blockIdx.x == gridDim.x - 1) {      // where the offsets end, or -1 for impossible ones
    const int* cu[2] = {cu_q, cu_k};
    const int total[2] = {total_q, total_k};
    for (int u = 0; u < 2; ++u) {
      bool bad = cu[u][0] != 0 || cu[u][n] > total[u];
      for (int i = threadIdx.x; i < n; i += kThreads) bad |= cu[u][i + 1] < cu[u][i];
      bad = __syncthreads_or(bad);
      if (threadIdx.x == 0) ends[u] = bad ? -1 : cu[u][n];
    }
    if (threadIdx.x == 0) __threadfence_system();
    return;
  }
  __shared__ int count[kCosts];
  __shared__ int part[32], all_costs, dearest;
  auto clamped = [](int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); };
  if (blockIdx.x >= 4) {      // a row's place in its sequence: the last offset that is not above it
    const int row = (blockIdx.x - 4) * kThreads + threadIdx.x;
    if (row >= total_q) return;
    int lo = 0, hi = n;       // the first offset counts as 0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu_q[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    const int q0 = lo ? cu_q[lo] : 0, at = row - q0;
    reinterpret_cast<int64_t*>(plan + packed_positions_offset(total_q, total_k, n))[row] = at;
    // the numbers of the sequence as the lists have them
    const int k0 = lo ? clamped(cu_k[lo], 0, total_k) : 0;
    const int sq = (lo < n ? clamped(cu_q[lo + 1], q0, total_q) : total_q) - q0;
    const int sk = lo < n ? clamped(cu_k[lo + 1], k0, total_k) - k0 : 0;
    plan[packed_single_offset(total_q, total_k, n) + row] =
        (packed_key_blocks(at & ~127, sq, sk, false) <= 1 ? 1 : 0) | (packed_key_blocks(at & ~127, sq, sk, true) <= 1 ? 2 : 0);
    return;
  }
  const int backward = blockIdx.x >> 1, causal = blockIdx.x & 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* list = plan + packed_list_offset(total_q, total_k, n, backward, causal);
  PackedHeader* header = reinterpret_cast<PackedHeader*>(list);
  PackedItem* items = reinterpret_cast<PackedItem*>(header + 1);
  const int cap = static_cast<int>(backward ? packed_backward_items(total_k, n) : packed_forward_items(total_q, n));
  for (int i = tid; i < kCosts; i += kThreads) count[i] = 0;
  if (tid == 0) all_costs = dearest = 0;
  __syncthreads();
  auto walk = [&](auto&& f) {
    for (int b = warp; b <= n; b += kThreads / 32) {
      PackedItem it;
      const int q0 = b ? clamped(cu_q[b], 0, total_q) : 0, k0 = b ? clamped(cu_k[b], 0, total_k) : 0;
      const int q1 = b < n ? clamped(cu_q[b + 1], q0, total_q) : total_q;
      const int k1 = b < n ? clamped(cu_k[b + 1], k0, total_k) : total_k;
      it.q_row = q0;
      it.sq = (b == n && backward) ? 0 : q1 - q0;
      it.k_row = k0;
      it.sk = (b == n && !backward) ? 0 : k1 - k0;
      it.pad[0] = it.pad[1] = it.pad[2] = 0;
      const int step = backward ? 128 : 256, len = backward ? it.sk : it.sq;
      for (int first = lane * step; first < len; first += 32 * step) {
        it.first = first;
        const int off = it.sk - it.sq;        // query i sees keys up to i + off
        int cost;
        if (backward) {
          const int from = causal ? max(0, first - off) / 128 : 0;
          cost = max(0, (it.sq + 127) / 128 - from);
        } else {
          const int last = causal ? min(it.sk, min(it.sq, first + 256) + off) : it.sk;
          cost = max(0, last + 127) / 128;
        }
        f(it, kCosts - 1 - min(cost, kCosts - 1));
      }
    }
  };
  walk([&](const PackedItem&, int c) {
    atomicAdd(&count[c], 1);
    atomicMax(&dearest, kCosts - 1 - c);
  });
  __syncthreads();
  // exclusive sum over the costs
  constexpr int per = kCosts / kThreads;
  int mine[per], sum = 0;
#pragma unroll
  for (int i = 0; i < per; ++i) {
    mine[i] = sum;
    sum += count[tid * per + i];
  }
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) part[warp] = upto;
  __syncthreads();
  int before = upto - sum;
  for (int w = 0; w < warp; ++w) before += part[w];
#pragma unroll
  for (int i = 0; i < per; ++i) count[tid * per + i] = before + mine[i];
  int costs = 0;
#pragma unroll
  for (int i = 0; i < per; ++i) costs += ((i + 1 < per ? mine[i + 1] : sum) - mine[i]) * (kCosts - 1 - (tid * per + i));
  if (costs) atomicAdd(&all_costs, costs);
  __syncthreads();
  if (tid == kThreads - 1) {
    header->count = min(before + sum, cap);
    header->cost = all_costs;
    header->dearest = dearest;
    header->pad = 0;
  }
  walk([&](const PackedItem& it, int c) {
    const int at = atomicAdd(&count[c], 1);
    if (at < cap) items[at] = it;
  });
}

// Offsets that the host knows, as many as the arguments of a launch take.
constexpr int kOffsets = 992;
struct Offsets {
  int at[kOffsets];
};
__global__ void __launch_bounds__(256)
packed_offsets_kernel(const __grid_constant__ Offsets offsets, int n, int* out) {
  for (int i = threadIdx.x; i < n; i += 256) out[i] = offsets.at[i];
}

// Reports sequences of more than `most` rows, as the plan has them.
__global__ void __launch_bounds__(256)
packed_limit_kernel(const int* cu, int n, int total, int most, int* status) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= n) return;
  const int first = b ? max(0, min(cu[b], total)) : 0, end = min(cu[b + 1], total);
  if (end - first > most) atomicCAS(status, 0, MB_ERR_POSITION);
}

}  // namespace

MB_API int* mb_status_device_ptr();

// Bytes of a plan for n sequences in tensors of total_q and total_k rows.
MB_API long mb_packed_plan_bytes(int n, int total_q, int total_k) {
  if (n < 0 || total_q < 0 || total_k < 0) return 0;
  return packed_single_offset(total_q, total_k, n) + total_q;
}
// Where in a plan every query row's place in its sequence stands: total_q numbers of 64 bits.
MB_API long mb_packed_plan_positions(int n, int total_q, int total_k) { return packed_positions_offset(total_q, total_k, n); }

// cu_q, cu_k: n + 1 offsets each, in device memory; host_q, host_k: null, or the offsets in host memory, which are then
// written there first.  The plan (16-byte aligned) serves causal and full attention, forward and backward, with any number of
// heads.  ends: null, or two numbers in pinned host memory that get the last offsets, or -1 where they are impossible.
MB_API int mb_packed_plan(int* cu_q, int* cu_k, const int* host_q, const int* host_k, int n, int total_q, int total_k, void* plan,
                          int* ends, cudaStream_t stream) {
  if (n < 0 || total_q < 0 || total_k < 0 || (reinterpret_cast<uintptr_t>(plan) & 15)) return -1;
  const int* from[2] = {host_q, host_k};
  int* to[2] = {cu_q, cu_k};
  for (int u = 0; u < 2; ++u) {
    for (int first = 0; from[u] && first <= n; first += kOffsets) {
      Offsets part;
      const int count = n + 1 - first < kOffsets ? n + 1 - first : kOffsets;
      memcpy(part.at, from[u] + first, sizeof(int) * count);
      packed_offsets_kernel<<<1, 256, 0, stream>>>(part, count, to[u] + first);
    }
  }
  packed_plan_kernel<<<4 + (total_q + kThreads - 1) / kThreads + (ends ? 1 : 0), kThreads, 0, stream>>>(
      cu_q, cu_k, n, total_q, total_k, static_cast<uint8_t*>(plan), ends);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// cu: n + 1 offsets in device memory.  A sequence of more than `most` of the `total` rows sets the status word.
MB_API int mb_packed_limit(const int* cu, int n, int total, int most, cudaStream_t stream) {
  int* status = mb_status_device_ptr();
  if (n < 0 || total < 0 || most < 0 || !status) return -1;
  if (n == 0) return 0;
  packed_limit_kernel<<<(n + 255) / 256, 256, 0, stream>>>(cu, n, total, most, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}
