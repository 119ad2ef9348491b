// Embedding lookup and its gradient by sorted tokens.
//
//   out[t]  = scale * wte[ids[t] - v0]  (zero for an id outside [v0, v0 + rows))  +  wpe[position of t]
//   dwte[v] = scale * sum of dout[t] over the tokens t with id v0 + v          (wpe alike, without the scale)
//
// The gradient is a sum over the tokens of each row.  Tokens are sorted by row first (a stable radix sort, so the
// tokens of a row keep their order), then every row of the table is summed in fp32 by the threads that write it: each
// row of dout is read once, each row of the table is written once in its own type, and the sums have one order, so
// results repeat bit for bit.  The traffic that stays is that of the definition; it is bound by memory.
// Measured: 16384 tokens of 2560, tables of 50304 and 2048 rows: lookup 35 us, sort 16, sums 67 (390 MB, 5.8 TB/s); 8192
// tokens of 4096, 32000 rows: 19, 11, 51.  (A scatter with atomics into fp32 tables and a cast of those took 1300 us.)
//
// Reference counterpart: the embedding modules of mist/modules/embedding.py:207-281 (gradient by torch's scatter-add).
#include "common.cuh"
#include <cooperative_groups.h>
#include <string.h>

MB_API int* mb_status_device_ptr();

namespace cg = cooperative_groups;

namespace {

// ------------------------------------------------------------------------------------------------ lookup
// N words of two values each, in one access of 16 or 32 bytes.
template <int N>
__device__ __forceinline__ void load_words(uint32_t* w, const uint32_t* p) {
  if (N == 8) {
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[N - 4]), "=r"(w[N - 3]), "=r"(w[N - 2]), "=r"(w[N - 1])
                 : "l"(p));
  } else {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  }
}
template <int N>
__device__ __forceinline__ void store_words(uint32_t* p, const uint32_t* w) {
  if (N == 8) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[N - 4]), "r"(w[N - 3]), "r"(w[N - 2]), "r"(w[N - 1]) : "memory");
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// One warp per token and slice of its row, `per_warp` vectors of 2 N values, 64 bytes of each table in flight per lane.  (In
// accesses of 32 bytes 16384 x 2560 with positions take 34.8 us and 8192 x 4096 19.4, of 16 bytes 39.4 and 24.7; more CTAs per
// SM with less in flight 36 - 50.)
template <int N>
__global__ void __launch_bounds__(256, 4)
embed_fwd_kernel(const int64_t* __restrict__ ids, const int64_t* __restrict__ pos, const uint32_t* __restrict__ wte,
                 const uint32_t* __restrict__ wpe, uint32_t* __restrict__ out, int tokens, int seq, int h, int64_t v0, int rows,
                 int positions, float scale, int per_warp, bool strict, int* status) {
  constexpr int kRounds = 16 / N;
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const int from = blockIdx.y * per_warp, to = min(h / (2 * N), from + per_warp);
  const int64_t row = ids[t] - v0;
  const bool in = row >= 0 && row < rows;
  int64_t p = -1;
  if (wpe) {
    p = pos ? pos[t] : t % seq;
    if (strict && p < 0) p += positions;
    if (p < 0 || p >= positions) {
      if (strict && status && lane == 0 && blockIdx.y == 0) atomicCAS(status, 0, MB_ERR_POSITION);
      p = -1;
    }
  }
  const int64_t words = h >> 1;
  const uint32_t* we = wte + (in ? row : 0) * words;
  const uint32_t* pe = wpe + (p >= 0 ? p : 0) * words;
  uint32_t* dst = out + t * words;
  for (int c0 = from + lane; c0 < to; c0 += 32 * kRounds) {
    uint32_t a[kRounds][N], b[kRounds][N];
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
      memset(a[u], 0, sizeof(a[u]));
      if (in && c0 + 32 * u < to) load_words<N>(a[u], we + static_cast<int64_t>(c0 + 32 * u) * N);
      if (p >= 0 && c0 + 32 * u < to) load_words<N>(b[u], pe + static_cast<int64_t>(c0 + 32 * u) * N);
    }
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
      const int c = c0 + 32 * u;
      if (c >= to) break;
      uint32_t o[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float x = __uint_as_float(a[u][k] << 16), y = __uint_as_float(a[u][k] & 0xffff0000u);
        if (p >= 0) {
          const float gx = __uint_as_float(b[u][k] << 16), gy = __uint_as_float(b[u][k] & 0xffff0000u);
          x = in ? fmaf(x, scale, gx) : gx;
          y = in ? fmaf(y, scale, gy) : gy;
        } else {
          x = in ? x * scale : 0.f;
          y = in ? y * scale : 0.f;
        }
        const __nv_bfloat162 both = __floats2bfloat162_rn(x, y);
        o[k] = *reinterpret_cast<const uint32_t*>(&both);
      }
      store_words<N>(dst + static_cast<int64_t>(c) * N, o);
    }
  }
}

// -------------------------------------------------------------------------------------------------- sort
// Work area of one table's sort, 16-byte aligned arrays in a row: two buffers each of keys and tokens [tokens], counters
// and partial sums of the rows whose tokens lie in several tiles.
constexpr int kTile = 32;        // sorted tokens that a warp sums
constexpr int kChunk = 256;      // columns of them

struct Area {
  uint32_t* key[2];
  int* tok[2];
  int* arrived;      // [tile][first, last row of it][column chunk]
  float* part;       // [tile][first, last row of it][h]
};

struct Sort {
  const int64_t* ids;
  int64_t v0;
  int rows;          // keys are 0 ... rows - 1, and rows for tokens that belong to no row
  int passes;
  bool from_end;     // negative rows count from the end
  Area area;
};

constexpr int kSortThreads = 1024;
constexpr int kSortCluster = 8;

// The sorts take 8 bits of the key a pass.  A warp owns a stretch of consecutive tokens; ballots over the bits rank equal
// digits inside 32 of them (__match_any_sync takes 270 cycles of a scheduler), a histogram per warp counts those before.
// Latency is all that they cost: 8 us a pass of 16384 tokens, most of it the exchange between the CTAs and the scatter.
struct SortSpace {
  int hist[32][256];
  int totals[256], base[256], warp_part[8], quarter[4][256];
};

// The digits of a pass have been counted, hist[warp][digit]; what stands there becomes the number of equal digits of this CTA
// in the warps before, and base[digit] the place of the digit's first token of this CTA.  All(tid, own) adds up the CTAs:
// {tokens of the digit in the CTAs before, in all}.
template <typename All>
__device__ __forceinline__ void sort_offsets(SortSpace& z, All&& all_of) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __syncthreads();
  // exclusive sum of a digit over the warps, a quarter of them per thread
  int* column = &z.hist[8 * (tid >> 8)][tid & 255];
  int sum = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const int n = column[256 * w];
    column[256 * w] = sum;
    sum += n;
  }
  z.quarter[tid >> 8][tid & 255] = sum;
  __syncthreads();
  const int2 counts = all_of(tid);
  // exclusive sum over the digits
  int upto = counts.y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += n;
  }
  if (tid < 256 && lane == 31) z.warp_part[warp] = upto;
  __syncthreads();
  if (tid < 256) {
    int start = upto - counts.y + counts.x;
    for (int w = 0; w < warp; ++w) start += z.warp_part[w];
    z.base[tid] = start;
  }
  __syncthreads();
}
__device__ __forceinline__ unsigned digit_of(uint32_t key, int shift, bool live) { return live ? (key >> shift) & 255u : 256u; }
// Counts 32 tokens of the warp and returns the rank of the lane's among the warp's tokens of its digit.
__device__ __forceinline__ int sort_count(SortSpace& z, unsigned digit) {
  unsigned same = __ballot_sync(0xffffffffu, digit < 256);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const bool one = (digit >> b) & 1;
    const unsigned ones = __ballot_sync(0xffffffffu, one);
    same &= one ? ones : ~ones;
  }
  const int before = __popc(same & ((1u << (threadIdx.x & 31)) - 1u));
  int* count = &z.hist[threadIdx.x >> 5][digit & 255];
  int rank = 0;
  if (digit < 256) rank = *count + before;
  __syncwarp();
  if (digit < 256 && before == 0) *count += __popc(same);
  __syncwarp();
  return rank;
}
// The place of a token of that rank, after sort_offsets.
__device__ __forceinline__ int sort_place(const SortSpace& z, unsigned digit, int rank) {
  const int warp = threadIdx.x >> 5;
  int at = z.base[digit] + z.hist[warp][digit] + rank;
  for (int q = 0; q < (warp >> 3); ++q) at += z.quarter[q][digit];
  return at;
}
__device__ __forceinline__ uint32_t row_of(const Sort& s, int i) {
  int64_t r = s.ids[i] - s.v0;
  if (s.from_end && r < 0) r += s.rows;
  return (r >= 0 && r < s.rows) ? static_cast<uint32_t>(r) : static_cast<uint32_t>(s.rows);
}

// Up to kBlockSort tokens: one CTA per table, everything in its shared memory between the passes.  (Of 16384 tokens a CTA
// takes 51 us, a cluster 19.)
constexpr int kHeld = 2;         // tokens of a lane
constexpr int kBlockSort = kSortThreads * kHeld;
constexpr int kBlockSortBytes = sizeof(SortSpace) + 8 * kBlockSort;
__global__ void __launch_bounds__(kSortThreads)
embed_sort_block_kernel(const __grid_constant__ Sort s0, const __grid_constant__ Sort s1, int tokens, int counters) {
  extern __shared__ __align__(16) uint8_t sort_smem[];
  SortSpace& z = *reinterpret_cast<SortSpace*>(sort_smem);
  uint2* pairs = reinterpret_cast<uint2*>(sort_smem + sizeof(SortSpace));
  const Sort& s = blockIdx.x ? s1 : s0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int per_warp = ((tokens + 31) / 32 + 31) & ~31, begin = warp * per_warp, end = min(begin + per_warp, tokens);
  mb::let_next_kernel_start();      // the row sums wait for this kernel's end, but not for their launch
  for (int i = tid; i < counters; i += kSortThreads) s.area.arrived[i] = 0;
  uint32_t key[kHeld], tok[kHeld];      // tok: the token, and above it, once it is known, its rank
  static_assert(kBlockSort <= 1 << 16 && kBlockSort / 32 <= 1 << 16, "token and rank share 32 bits");
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int i = begin + 32 * u + lane;
    tok[u] = i;
    key[u] = i < end ? row_of(s, i) : 0u;
  }
  for (int pass = 0; pass < s.passes; ++pass) {
    const int shift = 8 * pass;
    for (int d = lane; d < 256; d += 32) z.hist[warp][d] = 0;
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (begin + 32 * u < end) tok[u] |= sort_count(z, digit_of(key[u], shift, begin + 32 * u + lane < end)) << 16;
    sort_offsets(z, [&](int t) {
      return make_int2(0, t < 256 ? z.quarter[0][t] + z.quarter[1][t] + z.quarter[2][t] + z.quarter[3][t] : 0);
    });
    const bool last = pass + 1 == s.passes;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      if (begin + 32 * u + lane < end) {
        const int at = sort_place(z, digit_of(key[u], shift, true), tok[u] >> 16);
        if (last) {
          s.area.key[pass & 1][at] = key[u];
          s.area.tok[pass & 1][at] = tok[u] & 0xffffu;
        } else {
          pairs[at] = make_uint2(key[u], tok[u] & 0xffffu);
        }
      }
    }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int i = begin + 32 * u + lane;
      if (i < end) {
        const uint2 p = pairs[i];
        key[u] = p.x;
        tok[u] = p.y;
      }
    }
  }
}

// More tokens: one cluster per table.  The CTAs exchange their digit counts through distributed shared memory.  HELD: a lane's
// tokens fit its registers.
constexpr int kClusterHeld = 4;
template <bool HELD>
__global__ void __launch_bounds__(kSortThreads)
embed_sort_cluster_kernel(const __grid_constant__ Sort s0, const __grid_constant__ Sort s1, int tokens, int counters) {
  __shared__ SortSpace z;
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int ctas = kSortCluster;
  const int rank = cluster.block_rank();
  const Sort& s = (blockIdx.x / ctas) ? s1 : s0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int warps = ctas * 32;
  const int per_warp = ((tokens + warps - 1) / warps + 31) & ~31;
  const long first = static_cast<long>(rank * 32 + warp) * per_warp;
  const int begin = static_cast<int>(first < tokens ? first : tokens);
  const int end = static_cast<int>(first + per_warp < tokens ? first + per_warp : tokens);
  mb::let_next_kernel_start();
  for (int i = rank * kSortThreads + tid; i < counters; i += ctas * kSortThreads) s.area.arrived[i] = 0;
  for (int pass = 0; pass < s.passes; ++pass) {
    const int shift = 8 * pass;
    const uint32_t* src_key = s.area.key[(pass + 1) & 1];
    const int* src_tok = s.area.tok[(pass + 1) & 1];
    auto key_at = [&](int i) -> uint32_t { return i >= end ? 0u : (pass > 0 ? __ldcg(src_key + i) : row_of(s, i)); };
    uint32_t key[kClusterHeld];
    int tok[kClusterHeld], rank_of[kClusterHeld];
    if (HELD) {
#pragma unroll
      for (int u = 0; u < kClusterHeld; ++u) {
        const int i = begin + 32 * u + lane;
        key[u] = key_at(i);
        tok[u] = pass > 0 && i < end ? __ldcg(src_tok + i) : i;
      }
    }
    for (int d = lane; d < 256; d += 32) z.hist[warp][d] = 0;
    __syncwarp();
    if (HELD) {
#pragma unroll
      for (int u = 0; u < kClusterHeld; ++u)
        if (begin + 32 * u < end) rank_of[u] = sort_count(z, digit_of(key[u], shift, begin + 32 * u + lane < end));
    } else {
      for (int i = begin + lane; i - lane < end; i += 32) sort_count(z, digit_of(key_at(i), shift, i < end));
    }
    sort_offsets(z, [&](int t) {
      if (t < 256) z.totals[t] = z.quarter[0][t] + z.quarter[1][t] + z.quarter[2][t] + z.quarter[3][t];
      cluster.sync();
      int2 n = make_int2(0, 0);
      if (t < 256) {
        int x[ctas];
#pragma unroll
        for (int c = 0; c < ctas; ++c) x[c] = cluster.map_shared_rank(z.totals, c)[t];
#pragma unroll
        for (int c = 0; c < ctas; ++c) {
          if (c < rank) n.x += x[c];
          n.y += x[c];
        }
      }
      return n;
    });
    if (HELD) {
#pragma unroll
      for (int u = 0; u < kClusterHeld; ++u) {
        if (begin + 32 * u + lane < end) {
          const int at = sort_place(z, digit_of(key[u], shift, true), rank_of[u]);
          s.area.key[pass & 1][at] = key[u];
          s.area.tok[pass & 1][at] = tok[u];
        }
      }
    } else {
      // counted once more, now from the offsets on: sort_count's rank is then the place inside the CTA's share
      for (int i = begin + lane; i - lane < end; i += 32) {
        const uint32_t key = key_at(i);
        const unsigned digit = digit_of(key, shift, i < end);
        const int rank = sort_count(z, digit);
        if (i < end) {
          int at = z.base[digit] + rank;
          for (int q = 0; q < (warp >> 3); ++q) at += z.quarter[q][digit];
          s.area.key[pass & 1][at] = key;
          s.area.tok[pass & 1][at] = pass > 0 ? __ldcg(src_tok + i) : i;
        }
      }
    }
    cluster.sync();      // the next pass reads what other CTAs wrote; nobody reads totals any more
  }
}

// ---------------------------------------------------------------------------------------------- row sums
struct Table {
  const uint32_t* key;   // sorted rows; null: row r has the tokens r, r + stride, ... (`tokens` of them in all)
  const int* tok;
  int* arrived;
  float* part;
  void* out;             // [rows][h]
  int rows, stride;
  float scale;
};

// First i of [0, n) with key[i] >= x, by a warp: 32 probes a step.
__device__ __forceinline__ int warp_lower_bound(const uint32_t* key, int n, uint32_t x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int step = (hi - lo + 31) >> 5;
    const long at = lo + static_cast<long>(lane) * step;
    const bool less = at < hi && key[at] < x;
    const int c = __popc(__ballot_sync(0xffffffffu, less));
    if (c == 0) break;
    const long next = lo + static_cast<long>(c) * step;
    lo += (c - 1) * step + 1;
    hi = next < hi ? static_cast<int>(next) : hi;
  }
  return lo;
}

__device__ __forceinline__ void add8(float* acc, const mb::bf16x8& v) {
  float f[8];
  mb::unpack8(v, f);
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] += f[k];
}

// How a table is written; a template parameter, because all four in every place cost registers and a third of the time.
enum Mode : int { kBf16 = 0, kBf16Add = 1, kF32 = 2, kF32Add = 3 };

// out[0..8) (+)= scale * acc, rounded once
template <int MODE>
__device__ __forceinline__ void write8(const Table& t, long at, const float* acc) {
  float f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = acc[k] * t.scale;
  if (MODE >= kF32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(t.out) + at);
    if (MODE == kF32Add) {
      const float4 x = dst[0], y = dst[1];
      f[0] += x.x; f[1] += x.y; f[2] += x.z; f[3] += x.w;
      f[4] += y.x; f[5] += y.y; f[6] += y.z; f[7] += y.w;
    }
    dst[0] = make_float4(f[0], f[1], f[2], f[3]);
    dst[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    mb::bf16x8* dst = reinterpret_cast<mb::bf16x8*>(static_cast<__nv_bfloat16*>(t.out) + at);
    if (MODE == kBf16Add) add8(f, *dst);
    *dst = mb::pack8(f);
  }
}

constexpr int kSumThreads = 256;
constexpr int kZeroRows = 16;

// A part of a row that lies in several tiles has been written: the warp that counts the last one adds all in order.
// [a, b): the row's sorted tokens.
template <int MODE>
__device__ __noinline__ void count_part(const Table& t, int h, int chunk, int chunks, uint32_t row, int a, int b) {
  const int lane = threadIdx.x & 31, c = chunk * 32 + lane;
  const int tile0 = a / kTile, parts = (b - 1) / kTile - tile0 + 1;
  const int slot0 = 2 * tile0 + (a % kTile != 0);      // in the row's first tile; in the others the row is the first
  __threadfence();
  __syncwarp();
  int last = 0;
  if (lane == 0) last = atomicAdd(&t.arrived[slot0 * chunks + chunk], 1) == parts - 1;
  if (!__shfl_sync(0xffffffffu, last, 0)) return;
  __threadfence();
  if (c >= (h >> 3)) return;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int q = 0; q < parts; ++q) {
    const float4* src = reinterpret_cast<const float4*>(t.part + static_cast<long>(q ? 2 * (tile0 + q) : slot0) * h + 8 * c);
    const float4 x = __ldcg(src), y = __ldcg(src + 1);
    sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
    sum[4] += y.x; sum[5] += y.y; sum[6] += y.z; sum[7] += y.w;
  }
  write8<MODE>(t, static_cast<long>(row) * h + 8 * c, sum);
}

// One warp: the columns of a chunk, of the rows whose tokens are in a tile of kTile sorted ones.  However the ids are
// distributed, a warp has the same work.  A row that lies in several tiles leaves a part in each.
template <int MODE>
__device__ __forceinline__ void sum_tile(const Table& t, const __nv_bfloat16* dout, int tokens, int h, int tile, int chunk,
                                         int chunks) {
  const int lane = threadIdx.x & 31, vpr = h >> 3, c = chunk * 32 + lane;
  const bool live = c < vpr;
  const int p0 = tile * kTile, all = min(kTile, tokens - p0);
  const uint32_t key = lane < all ? t.key[p0 + lane] : 0xffffffffu;
  const int tok = lane < all ? t.tok[p0 + lane] : 0;
  const int n = __popc(__ballot_sync(0xffffffffu, key < static_cast<uint32_t>(t.rows)));      // tokens of no row come last
  if (n == 0) return;
  const uint32_t before = p0 > 0 ? t.key[p0 - 1] : 0xffffffffu;
  const uint32_t after = n == all && p0 + n < tokens ? t.key[p0 + n] : 0xffffffffu;
  uint32_t left = __shfl_up_sync(0xffffffffu, key, 1);
  if (lane == 0) left = before;
  // bit j: token j is the first of its row
  const unsigned starts = __ballot_sync(0xffffffffu, lane < n && key != left);
  const bool begun = !(starts & 1u), goes_on = after == __shfl_sync(0xffffffffu, key, n - 1);
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.f;
  auto store_part = [&](int slot) {
    if (!live) return;
    float4* dst = reinterpret_cast<float4*>(t.part + (2l * tile + slot) * h + 8 * c);
    dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  };
  int from = 0, first_end = n;                     // first token of the row in hand; end of the tile's first row
  for (int j = 0; j < n; j += 8) {
    mb::bf16x8 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long at = __shfl_sync(0xffffffffu, tok, (j + u) & 31);
      if (live && j + u < n) v[u] = *reinterpret_cast<const mb::bf16x8*>(dout + at * h + 8 * c);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (j + u < n) {
        if (j + u > 0 && ((starts >> (j + u)) & 1u)) {
          const long row = __shfl_sync(0xffffffffu, key, from);
          if (from == 0) first_end = j + u;
          if (from == 0 && begun) store_part(0);
          else if (live) write8<MODE>(t, row * h + 8 * c, acc);
          from = j + u;
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = 0.f;
        }
        add8(acc, v[u]);
      }
    }
  }
  const uint32_t row = __shfl_sync(0xffffffffu, key, from), row0 = __shfl_sync(0xffffffffu, key, 0);
  if (goes_on || (from == 0 && begun)) store_part(from != 0);
  else if (live) write8<MODE>(t, static_cast<long>(row) * h + 8 * c, acc);
  if (begun) {
    const int a = warp_lower_bound(t.key, tokens, row0);
    const int b = first_end == n && goes_on ? warp_lower_bound(t.key, tokens, row0 + 1) : p0 + first_end;
    count_part<MODE>(t, h, chunk, chunks, row0, a, b);
  }
  if (goes_on && (from != 0 || !begun))
    count_part<MODE>(t, h, chunk, chunks, row, p0 + from, warp_lower_bound(t.key, tokens, row + 1));
}

// Rows that get no token, where the table is stored.
template <int MODE>
__device__ __forceinline__ void zero_rows(const Table& t, int tokens, int h, int block) {
  __shared__ uint8_t used[kZeroRows];
  __shared__ int range[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = block * kZeroRows, nrows = min(kZeroRows, t.rows - r0);
  if (threadIdx.x < kZeroRows) used[threadIdx.x] = 0;
  if (warp < 2) {
    const int at = warp_lower_bound(t.key, tokens, static_cast<uint32_t>(warp ? r0 + nrows : r0));
    if (lane == 0) range[warp] = at;
  }
  __syncthreads();
  for (int i = range[0] + threadIdx.x; i < range[1]; i += kSumThreads) used[t.key[i] - r0] = 1;
  __syncthreads();
  const int bytes = h * (MODE >= kF32 ? 4 : 2);
  uint8_t* out = static_cast<uint8_t*>(t.out) + static_cast<long>(r0) * bytes;
  const bool wide = ((reinterpret_cast<uintptr_t>(t.out) | bytes) & 31) == 0;      // whole sectors
  for (int r = warp; r < nrows; r += kSumThreads / 32) {
    if (used[r]) continue;
    uint8_t* row = out + static_cast<long>(r) * bytes;
    if (wide) {
      for (int at = 32 * lane; at < bytes; at += 1024)
        asm volatile("st.global.v8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};\n" ::"l"(row + at), "r"(0) : "memory");
    } else {
      for (int at = 16 * lane; at < bytes; at += 512) *reinterpret_cast<uint4*>(row + at) = make_uint4(0, 0, 0, 0);
    }
  }
}

// A row of positions by place: token r of every sample.  One warp: a row's columns of a chunk.
__device__ __forceinline__ void sum_stride(const Table& t, const __nv_bfloat16* dout, int tokens, int h, int row, int chunk) {
  const int c = chunk * 32 + (threadIdx.x & 31);
  if (c >= (h >> 3)) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (row < t.stride) {
#pragma unroll 4
    for (long j = row; j < tokens; j += t.stride) add8(acc, *reinterpret_cast<const mb::bf16x8*>(dout + j * h + 8 * c));
  }
  write8<kBf16>(t, static_cast<long>(row) * h + 8 * c, acc);
}

// What the blocks do: items of sum_tile (or rows of sum_stride), one per warp, of table 0 and of table 1, then rows without a
// token of table 0 and of table 1.  The sums wait for memory, the zeros fill its queues behind them.
struct Blocks {
  int sums0, sums1, zeros0;      // numbers of blocks; the rest are the zeros of table 1
};
template <int MODE>
__global__ void __launch_bounds__(kSumThreads, 4)
embed_sum_kernel(const __grid_constant__ Table t0, const __grid_constant__ Table t1, const __nv_bfloat16* dout, int tokens,
                 int h, int chunks, const Blocks blocks) {
  mb::wait_for_previous_kernel();
  int b = blockIdx.x;
  if (b < blocks.sums0 + blocks.sums1) {
    const bool second = b >= blocks.sums0;
    if (second) b -= blocks.sums0;
    const long item = static_cast<long>(b) * (kSumThreads / 32) + (threadIdx.x >> 5);
    const int at = static_cast<int>(item / chunks), chunk = static_cast<int>(item - static_cast<long>(at) * chunks);
    const bool inside = static_cast<long>(at) * kTile < tokens;
    if (!second) {      // (a reference to one of the two would put both in local memory)
      if (inside) sum_tile<MODE>(t0, dout, tokens, h, at, chunk, chunks);
    } else if (t1.key) {
      if (inside) sum_tile<kBf16>(t1, dout, tokens, h, at, chunk, chunks);
    } else if (at < t1.rows) {
      sum_stride(t1, dout, tokens, h, at, chunk);
    }
    return;
  }
  b -= blocks.sums0 + blocks.sums1;
  if (b < blocks.zeros0) zero_rows<MODE & ~1>(t0, tokens, h, b);
  else zero_rows<kBf16>(t1, tokens, h, b - blocks.zeros0);
}

size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }
int tiles_of(int tokens) { return static_cast<int>((tokens + static_cast<long>(kTile) - 1) / kTile); }
int chunks_of(int h) { return (h + kChunk - 1) / kChunk; }

size_t area_bytes(int tokens, int h) {
  return 4 * up16(4ul * tokens) + up16(8ul * tiles_of(tokens) * chunks_of(h)) + up16(8ul * tiles_of(tokens) * h);
}
Area make_area(uint8_t* at, int tokens, int h) {
  Area a;
  const size_t n = up16(4ul * tokens);
  for (int i = 0; i < 2; ++i) {
    a.key[i] = reinterpret_cast<uint32_t*>(at + 2 * i * n);
    a.tok[i] = reinterpret_cast<int*>(at + (2 * i + 1) * n);
  }
  a.arrived = reinterpret_cast<int*>(at + 4 * n);
  a.part = reinterpret_cast<float*>(at + 4 * n + up16(8ul * tiles_of(tokens) * chunks_of(h)));
  return a;
}
Sort make_sort(const int64_t* ids, int64_t v0, int rows, uint8_t* at, int tokens, int h) {
  Sort s;
  s.ids = ids;
  s.v0 = v0;
  s.rows = rows;
  s.from_end = false;
  s.passes = 1;
  while (s.passes < 4 && (static_cast<uint32_t>(rows) >> (8 * s.passes))) ++s.passes;
  s.area = make_area(at, tokens, h);
  return s;
}
Table make_table(const Sort& s, void* out, float scale) {
  Table t;
  t.key = s.area.key[(s.passes + 1) & 1];
  t.tok = s.area.tok[(s.passes + 1) & 1];
  t.arrived = s.area.arrived;
  t.part = s.area.part;
  t.out = out;
  t.rows = s.rows;
  t.stride = 0;
  t.scale = scale;
  return t;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// out [tokens][h] = scale * wte[ids - v0] + wpe[pos]; wpe may be null; pos null: position t % seq.  Ids outside the rows of
// wte and positions outside those of wpe add nothing; strict: negative positions count from the end of wpe, and ones outside
// it are reported as well.  h a multiple of 8, tables and out on 16 bytes.
MB_API int mb_embed_fwd(const int64_t* ids, const int64_t* pos, const void* wte, const void* wpe, void* out, int tokens,
                        int seq, int h, int64_t v0, int rows, int positions, int strict, float scale, cudaStream_t stream) {
  if (tokens < 0 || h <= 0 || h % 8 || rows < 0 || (wpe && !pos && seq <= 0)) return -1;
  if (!aligned16(wte) || !aligned16(wpe) || !aligned16(out)) return -1;
  if (tokens == 0) return 0;
  // rows of whole 32-byte sectors in accesses of as many bytes
  const bool wide = h % 16 == 0 && ((reinterpret_cast<uintptr_t>(wte) | reinterpret_cast<uintptr_t>(wpe) |
                                     reinterpret_cast<uintptr_t>(out)) & 31) == 0;
  const int vectors = h / (wide ? 16 : 8);
  // whole rows once they fill the chip (48 warps on each of 148 SMs); before that a row is cut into slices of 1024 values
  const int per_warp = tokens >= 7104 ? vectors : (wide ? 64 : 128);
  (wide ? embed_fwd_kernel<8> : embed_fwd_kernel<4>)<<<dim3((tokens + 7) / 8, (vectors + per_warp - 1) / per_warp), 256, 0,
                                                      stream>>>(
      ids, pos, static_cast<const uint32_t*>(wte), static_cast<const uint32_t*>(wpe), static_cast<uint32_t*>(out), tokens, seq, h,
      v0, rows, positions, scale, per_warp, strict != 0, strict ? mb_status_device_ptr() : nullptr);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// Bytes of workspace of mb_embed_bwd.
MB_API size_t mb_embed_bwd_workspace(int tokens, int h, int with_positions) {
  return area_bytes(tokens, h) * (with_positions ? 2 : 1);
}

// dout [tokens][h] -> dwte [rows][h] (fp32 or bf16, stored or added to) and, where dwpe is not null, dwpe [positions][h]
// (bf16, stored).  pos null: position t % seq.  Every row of a stored table is written; rows that get no token are left
// alone where it is added to.  strict: as in the lookup.  The workspace is for this call alone, on 16 bytes.  dwte may be null.
MB_API int mb_embed_bwd(const int64_t* ids, const int64_t* pos, const void* dout, void* dwte, void* dwpe, int tokens, int seq,
                        int h, int64_t v0, int rows, int positions, int strict, float scale, int dwte_fp32, int accumulate,
                        void* workspace, cudaStream_t stream) {
  if (tokens < 0 || h <= 0 || h % 8 || rows < 0 || positions < 0 || (dwpe && !pos && seq <= 0)) return -1;
  if (!aligned16(dout) || !aligned16(dwte) || !aligned16(dwpe) || !aligned16(workspace)) return -1;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  const bool sort0 = dwte && rows > 0, sort1 = dwpe && pos && positions > 0;
  Sort s[2];
  memset(s, 0, sizeof(s));
  int nsort = 0;
  Table t[2];
  memset(t, 0, sizeof(t));
  if (sort0) {
    s[nsort] = make_sort(ids, v0, rows, at, tokens, h);
    t[0] = make_table(s[nsort++], dwte, scale);
  }
  if (sort1) {
    s[nsort] = make_sort(pos, 0, positions, at + nsort * area_bytes(tokens, h), tokens, h);
    s[nsort].from_end = strict != 0;
    t[1] = make_table(s[nsort++], dwpe, 1.f);
  } else if (dwpe) {
    t[1].out = dwpe;
    t[1].rows = positions;
    t[1].stride = seq;
    t[1].scale = 1.f;
  }
  const int chunks = chunks_of(h), tiles = tiles_of(tokens);
  if (nsort && tokens > 0) {
    const long counters64 = 2l * tiles * chunks;
    if (counters64 > 0x7fffffffl) return -1;
    const int counters = static_cast<int>(counters64);
    if (tokens <= kBlockSort) {
      int dev = 0;
      static bool configured[64] = {};
      if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
      if (!configured[dev]) {
        if (cudaFuncSetAttribute(embed_sort_block_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBlockSortBytes) !=
            cudaSuccess)
          return -3;
        configured[dev] = true;
      }
      embed_sort_block_kernel<<<nsort, kSortThreads, kBlockSortBytes, stream>>>(s[0], s[1], tokens, counters);
      if (cudaGetLastError() != cudaSuccess) return -4;
    } else {
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof(cfg));
      cfg.gridDim = dim3(kSortCluster * nsort);
      cfg.blockDim = dim3(kSortThreads);
      cfg.stream = stream;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = kSortCluster;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      const bool held = tokens <= kSortCluster * kSortThreads * kClusterHeld;
      if (cudaLaunchKernelEx(&cfg, held ? embed_sort_cluster_kernel<true> : embed_sort_cluster_kernel<false>, s[0], s[1], tokens,
                             counters) != cudaSuccess)
        return -4;
    }
  }
  auto groups = [](long n, int per) { return (n + per - 1) / per; };
  const long sums0 = sort0 ? groups(static_cast<long>(tiles) * chunks, kSumThreads / 32) : 0;
  const long sums1 = sort1 ? groups(static_cast<long>(tiles) * chunks, kSumThreads / 32)
                           : (dwpe ? groups(static_cast<long>(positions) * chunks, kSumThreads / 32) : 0);
  const long zeros0 = sort0 && !accumulate ? groups(rows, kZeroRows) : 0, zeros1 = sort1 ? groups(positions, kZeroRows) : 0;
  const long blocks = sums0 + sums1 + zeros0 + zeros1;
  if (blocks == 0) return 0;
  if (blocks > 0x7fffffffl) return -1;
  Blocks of;
  of.sums0 = static_cast<int>(sums0);
  of.sums1 = static_cast<int>(sums1);
  of.zeros0 = static_cast<int>(zeros0);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kSumThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = nsort && tokens > 0 ? 1 : 0;
  const auto kernel = dwte_fp32 ? (accumulate ? embed_sum_kernel<kF32Add> : embed_sum_kernel<kF32>)
                                : (accumulate ? embed_sum_kernel<kBf16Add> : embed_sum_kernel<kBf16>);
  if (cudaLaunchKernelEx(&cfg, kernel, t[0], t[1], static_cast<const __nv_bfloat16*>(dout), tokens, h, chunks, of) !=
      cudaSuccess)
    return -4;
  return 0;
}
