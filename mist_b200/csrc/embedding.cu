// Embedding lookup and its gradient by sorted tokens.
//
//   out[t]  = scale * wte[ids[t] - v0]  (zero for an id outside [v0, v0 + rows))  +  wpe[position of t]
//   dwte[v] = scale * sum of dout[t] over the tokens t with id v0 + v          (wpe alike, without the scale)
//
// The gradient is a sum over the tokens of each row.  Tokens are sorted by row first (a stable radix sort, so the
// tokens of a row keep their order), then every row of the table is summed in fp32 by the threads that write it: each
// row of dout is read once, each row of the table is written once in its own type, and the sums have one order, so
// results repeat bit for bit.  The traffic that stays is that of the definition; it is bound by memory.
//
// Reference counterpart: the embedding modules of mist/modules/embedding.py:207-281 (gradient by torch's scatter-add).
#include "common.cuh"
#include <cooperative_groups.h>
#include <string.h>

namespace cg = cooperative_groups;

namespace {

// ------------------------------------------------------------------------------------------------ lookup
// One warp per token and slice of its row, `per_warp` vectors of 8 values, four rounds of loads in flight per lane.
__global__ void __launch_bounds__(256, 6)
embed_fwd_kernel(const int64_t* __restrict__ ids, const int64_t* __restrict__ pos, const __nv_bfloat16* __restrict__ wte,
                 const __nv_bfloat16* __restrict__ wpe, __nv_bfloat16* __restrict__ out, int tokens, int seq, int h, int64_t v0,
                 int rows, int positions, float scale, int per_warp) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const int vpr = h >> 3, from = blockIdx.y * per_warp, to = min(vpr, from + per_warp);
  const int64_t row = ids[t] - v0;
  const bool in = row >= 0 && row < rows;
  int64_t p = -1;
  if (wpe) {
    p = pos ? pos[t] : t % seq;
    if (p >= positions) p = -1;
  }
  const mb::bf16x8* we = reinterpret_cast<const mb::bf16x8*>(wte + (in ? row : 0) * h);
  const mb::bf16x8* pe = reinterpret_cast<const mb::bf16x8*>(wpe + (p >= 0 ? p : 0) * h);
  mb::bf16x8* dst = reinterpret_cast<mb::bf16x8*>(out + static_cast<int64_t>(t) * h);
  for (int c0 = from + lane; c0 < to; c0 += 128) {
    mb::bf16x8 a[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      memset(&a[u], 0, sizeof(a[u]));
      if (in && c0 + 32 * u < to) a[u] = we[c0 + 32 * u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 32 * u;
      if (c >= to) break;
      float f[8];
      mb::unpack8(a[u], f);
      if (p >= 0) {
        float g[8];
        mb::unpack8(pe[c], g);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = in ? fmaf(f[k], scale, g[k]) : g[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = in ? f[k] * scale : 0.f;
      }
      dst[c] = mb::pack8(f);
    }
  }
}

// -------------------------------------------------------------------------------------------------- sort
// Work area of one table's sort, 16-byte aligned arrays in a row: two buffers each of keys and tokens [tokens], counters
// of the long rows, partial sums of the long rows.
constexpr int kTile = 64;        // sorted tokens that are summed together where a row has more than that ("long" rows)
constexpr int kCols = 512;       // columns of such a sum that one CTA takes

struct Area {
  uint32_t* key[2];
  int* tok[2];
  int* arrived;      // [tile][first, last long row of it][column slice]
  float* part;       // [tile][first, last long row of it][h]
};

struct Sort {
  const int64_t* ids;
  int64_t v0;
  int rows;          // keys are 0 ... rows - 1, and rows for tokens that belong to no row
  int passes;
  Area area;
};

constexpr int kSortThreads = 1024;
constexpr int kSortCluster = 8;
constexpr int kHeld = 4;         // tokens that a lane keeps in registers over a pass

// One cluster (or, for few tokens, one CTA) sorts one table's tokens, 8 bits of the key a pass.  A warp owns a stretch
// of consecutive tokens; __match_any_sync ranks equal digits inside 32 of them, a histogram per warp counts those before.
// The CTAs exchange their digit counts through distributed shared memory.  Latency is what it costs: about 2 us a pass
//.
template <bool HELD>
__global__ void __launch_bounds__(kSortThreads)
embed_sort_kernel(const __grid_constant__ Sort s0, const __grid_constant__ Sort s1, int tokens, int counters) {
  __shared__ int hist[32][256];
  __shared__ int totals[256], base[256], warp_part[8], quarter[4][256];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const Sort& s = (blockIdx.x / ctas) ? s1 : s0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const unsigned below = (1u << lane) - 1u;
  const int warps = ctas * 32;
  const int per_warp = ((tokens + warps - 1) / warps + 31) & ~31;
  const long first = static_cast<long>(rank * 32 + warp) * per_warp;
  const int begin = static_cast<int>(first < tokens ? first : tokens);
  const int end = static_cast<int>(first + per_warp < tokens ? first + per_warp : tokens);

  mb::let_next_kernel_start();      // the row sums wait for this kernel's end, but not for their launch
  for (int i = rank * kSortThreads + tid; i < counters; i += ctas * kSortThreads) s.area.arrived[i] = 0;

  for (int pass = 0; pass < s.passes; ++pass) {
    const int shift = 8 * pass;
    const uint32_t* src_key = s.area.key[(pass + 1) & 1];
    const int* src_tok = s.area.tok[(pass + 1) & 1];
    uint32_t* dst_key = s.area.key[pass & 1];
    int* dst_tok = s.area.tok[pass & 1];
    auto key_at = [&](int i) -> uint32_t {
      if (pass > 0) return __ldcg(src_key + i);
      const int64_t r = s.ids[i] - s.v0;
      return (r >= 0 && r < s.rows) ? static_cast<uint32_t>(r) : static_cast<uint32_t>(s.rows);
    };
    uint32_t key[kHeld];
    int tok[kHeld];
    if (HELD) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        const int i = begin + 32 * u + lane;
        if (i < end) {
          key[u] = key_at(i);
          tok[u] = pass > 0 ? __ldcg(src_tok + i) : i;
        }
      }
    }
#pragma unroll
    for (int d = lane; d < 256; d += 32) hist[warp][d] = 0;
    __syncwarp();
    auto count = [&](int i, uint32_t k) {
      const unsigned digit = i < end ? (k >> shift) & 255u : 256u;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      if (digit < 256 && (same & below) == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
    };
    if (HELD) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (begin + 32 * u < end) count(begin + 32 * u + lane, key[u]);
    } else {
      for (int i = begin + lane; i - lane < end; i += 32) count(i, i < end ? key_at(i) : 0u);
    }
    __syncthreads();
    // exclusive sum of a digit over the warps, a quarter of them per thread
    int* column = &hist[8 * (tid >> 8)][tid & 255];
    int sum = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int n = column[256 * w];
      column[256 * w] = sum;
      sum += n;
    }
    quarter[tid >> 8][tid & 255] = sum;
    __syncthreads();
    if (tid < 256) totals[tid] = quarter[0][tid] + quarter[1][tid] + quarter[2][tid] + quarter[3][tid];
    cluster.sync();
    int before = 0, all = 0;
    if (tid < 256) {
      for (int c = 0; c < ctas; ++c) {
        const int n = cluster.map_shared_rank(totals, c)[tid];
        if (c < rank) before += n;
        all += n;
      }
    }
    // exclusive sum of `all` over the digits
    int upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    if (tid < 256 && lane == 31) warp_part[warp] = upto;
    __syncthreads();
    if (tid < 256) {
      int start = upto - all;
      for (int w = 0; w < warp; ++w) start += warp_part[w];
      base[tid] = start + before;
    }
    __syncthreads();
    auto place = [&](int i, uint32_t k, int t) {
      const unsigned digit = i < end ? (k >> shift) & 255u : 256u;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      if (digit < 256) {
        int at = base[digit] + hist[warp][digit] + __popc(same & below);
        for (int q = 0; q < (warp >> 3); ++q) at += quarter[q][digit];
        dst_key[at] = k;
        dst_tok[at] = t;
      }
      __syncwarp();
      if (digit < 256 && (same & below) == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
    };
    if (HELD) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (begin + 32 * u < end) place(begin + 32 * u + lane, key[u], tok[u]);
    } else {
      for (int i = begin + lane; i - lane < end; i += 32)
        place(i, i < end ? key_at(i) : 0u, (pass > 0 && i < end) ? __ldcg(src_tok + i) : i);
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
  int fp32, accumulate;
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

// out[0..8) (+)= scale * acc, rounded once
__device__ __forceinline__ void write8(const Table& t, long at, const float* acc) {
  float f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = acc[k] * t.scale;
  if (t.fp32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(t.out) + at);
    if (t.accumulate) {
      const float4 x = dst[0], y = dst[1];
      f[0] += x.x; f[1] += x.y; f[2] += x.z; f[3] += x.w;
      f[4] += y.x; f[5] += y.y; f[6] += y.z; f[7] += y.w;
    }
    dst[0] = make_float4(f[0], f[1], f[2], f[3]);
    dst[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    mb::bf16x8* dst = reinterpret_cast<mb::bf16x8*>(static_cast<__nv_bfloat16*>(t.out) + at);
    if (t.accumulate) add8(f, *dst);
    *dst = mb::pack8(f);
  }
}

constexpr int kRows = 8;         // table rows of a CTA
constexpr int kSumThreads = 256;

// Rows of up to kTile tokens (and rows without any): one thread per 8 columns of a row.
__device__ __forceinline__ void sum_rows(const Table& t, const __nv_bfloat16* dout, int tokens, int h, int block) {
  __shared__ int start[kRows + 1];
  const int warp = threadIdx.x >> 5;
  const int r0 = block * kRows, nrows = min(kRows, t.rows - r0), vpr = h >> 3;
  if (t.key) {
    if (warp < 2) {
      const int at = warp_lower_bound(t.key, tokens, static_cast<uint32_t>(warp ? r0 + nrows : r0));
      if ((threadIdx.x & 31) == 0) start[warp ? nrows : 0] = at;
    }
    __syncthreads();
    if (threadIdx.x > 0 && threadIdx.x < nrows) {
      int lo = start[0], hi = start[nrows];
      const uint32_t x = r0 + threadIdx.x;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t.key[mid] < x) lo = mid + 1;
        else hi = mid;
      }
      start[threadIdx.x] = lo;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < nrows * vpr; i += kSumThreads) {
    const int r = i / vpr, c = (i - r * vpr) * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t.key) {
      const int a = start[r], b = start[r + 1];
      if (b - a > kTile || (a == b && t.accumulate)) continue;      // summed by sum_long; nothing to add
      for (int j = a; j < b; j += 4) {
        mb::bf16x8 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u < b) v[u] = *reinterpret_cast<const mb::bf16x8*>(dout + static_cast<long>(t.tok[j + u]) * h + c);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u < b) add8(acc, v[u]);
      }
    } else {
      if (r0 + r >= t.stride && t.accumulate) continue;
      if (r0 + r < t.stride)
        for (long j = r0 + r; j < tokens; j += t.stride) add8(acc, *reinterpret_cast<const mb::bf16x8*>(dout + j * h + c));
    }
    write8(t, static_cast<long>(r0 + r) * h + c, acc);
  }
}

// Rows of more than kTile tokens: a CTA adds the tokens that such a row has among kTile sorted ones; a tile touches two
// of these rows at most, the row of its first token and that of its last.  The CTA that counts the last part of a row adds
// the parts in order.
__device__ void sum_long(const Table& t, const __nv_bfloat16* dout, int tokens, int h, int tile, int slice, int slices) {
  __shared__ int seg[2];
  __shared__ float red[3][kCols];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, tid = threadIdx.x;
  const int p0 = tile * kTile, p1 = min(p0 + kTile, tokens) - 1;
  const int group = tid >> 6, c = slice * kCols + (tid & 63) * 8;      // 4 groups of tokens x 64 vectors
  for (int w = 0; w < 2; ++w) {
    const uint32_t k = t.key[w ? p1 : p0];
    if (k >= static_cast<uint32_t>(t.rows) || (w && k == t.key[p0])) continue;
    // more than kTile equal keys in a row reach kTile - (tokens of this tile) further on one side
    const int left = w ? p0 : max(0, p0 - kTile), right = min(tokens - 1, p1 + kTile);
    __syncthreads();
    if (warp < 2) {
      const int at = warp_lower_bound(t.key + left, right + 1 - left, k + warp) + left;
      if ((tid & 31) == 0) seg[warp] = at;
    }
    __syncthreads();
    if (seg[1] - seg[0] <= kTile) continue;
    __syncthreads();
    if (warp < 2) {
      const int at = warp_lower_bound(t.key, tokens, k + warp);
      if ((tid & 31) == 0) seg[warp] = at;
    }
    __syncthreads();
    const int a = seg[0], b = seg[1];
    const int from = max(a, p0), to = min(b, p1 + 1), n = to - from;
    const int j0 = from + n * group / 4, j1 = from + n * (group + 1) / 4;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < h) {
      for (int j = j0; j < j1; j += 4) {
        mb::bf16x8 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u < j1) v[u] = *reinterpret_cast<const mb::bf16x8*>(dout + static_cast<long>(t.tok[j + u]) * h + c);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u < j1) add8(acc, v[u]);
      }
      if (group > 0)
#pragma unroll
        for (int u = 0; u < 8; ++u) red[group - 1][(tid & 63) * 8 + u] = acc[u];
    }
    __syncthreads();
    if (group == 0 && c < h) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int x = (tid & 63) * 8 + u;
        acc[u] += red[0][x] + (red[1][x] + red[2][x]);
      }
      float4* dst = reinterpret_cast<float4*>(t.part + (2l * tile + w) * h + c);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
    __threadfence();
    __syncthreads();
    const int tile0 = a / kTile, parts = (b - 1) / kTile - tile0 + 1;
    const int slot0 = 2 * tile0 + (a % kTile != 0);      // of the row's first tile; later tiles begin inside the row
    if (tid == 0) last = atomicAdd(&t.arrived[slot0 * slices + slice], 1) == parts - 1;
    __syncthreads();
    if (!last) continue;
    __threadfence();
    if (group == 0 && c < h) {
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int q = 0; q < parts; q += 4) {
        float4 x[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (q + u >= parts) break;
          const float4* src = reinterpret_cast<const float4*>(t.part + static_cast<long>(q + u ? 2 * (tile0 + q + u) : slot0) * h + c);
          x[u][0] = __ldcg(src);
          x[u][1] = __ldcg(src + 1);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (q + u >= parts) break;
          sum[0] += x[u][0].x; sum[1] += x[u][0].y; sum[2] += x[u][0].z; sum[3] += x[u][0].w;
          sum[4] += x[u][1].x; sum[5] += x[u][1].y; sum[6] += x[u][1].z; sum[7] += x[u][1].w;
        }
      }
      write8(t, static_cast<long>(k) * h + c, sum);
    }
  }
}

// blocks: [long rows of table 0][of table 1][rows of table 0][of table 1]
__global__ void __launch_bounds__(kSumThreads, 6)
embed_sum_kernel(const __grid_constant__ Table t0, const __grid_constant__ Table t1, const __nv_bfloat16* dout, int tokens, int h, int long0, int long1,
                 int rows0, int slices) {
  mb::wait_for_previous_kernel();
  int b = blockIdx.x;
  if (b < long0 + long1) {
    const bool second = b >= long0;
    if (second) b -= long0;
    sum_long(second ? t1 : t0, dout, tokens, h, b / slices, b % slices, slices);
    return;
  }
  b -= long0 + long1;
  if (b < rows0) sum_rows(t0, dout, tokens, h, b);
  else sum_rows(t1, dout, tokens, h, b - rows0);
}

size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }
int tiles_of(int tokens) { return tokens > kTile ? (tokens + kTile - 1) / kTile : 0; }
int slices_of(int h) { return (h + kCols - 1) / kCols; }

size_t area_bytes(int tokens, int h) {
  return 4 * up16(4ul * tokens) + up16(8ul * tiles_of(tokens) * slices_of(h)) + up16(8ul * tiles_of(tokens) * h);
}
Area make_area(uint8_t* at, int tokens, int h) {
  Area a;
  const size_t n = up16(4ul * tokens);
  for (int i = 0; i < 2; ++i) {
    a.key[i] = reinterpret_cast<uint32_t*>(at + 2 * i * n);
    a.tok[i] = reinterpret_cast<int*>(at + (2 * i + 1) * n);
  }
  a.arrived = reinterpret_cast<int*>(at + 4 * n);
  a.part = reinterpret_cast<float*>(at + 4 * n + up16(8ul * tiles_of(tokens) * slices_of(h)));
  return a;
}
Sort make_sort(const int64_t* ids, int64_t v0, int rows, uint8_t* at, int tokens, int h) {
  Sort s;
  s.ids = ids;
  s.v0 = v0;
  s.rows = rows;
  s.passes = 1;
  while (s.passes < 4 && (static_cast<uint32_t>(rows) >> (8 * s.passes))) ++s.passes;
  s.area = make_area(at, tokens, h);
  return s;
}
Table make_table(const Sort& s, void* out, int fp32, int accumulate, float scale) {
  Table t;
  t.key = s.area.key[(s.passes + 1) & 1];
  t.tok = s.area.tok[(s.passes + 1) & 1];
  t.arrived = s.area.arrived;
  t.part = s.area.part;
  t.out = out;
  t.rows = s.rows;
  t.stride = 0;
  t.fp32 = fp32;
  t.accumulate = accumulate;
  t.scale = scale;
  return t;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// out [tokens][h] = scale * wte[ids - v0] + wpe[pos]; wpe may be null; pos null: position t % seq.  Ids outside the rows of
// wte and positions outside those of wpe add nothing.  h a multiple of 8, tables and out on 16 bytes.
MB_API int mb_embed_fwd(const int64_t* ids, const int64_t* pos, const void* wte, const void* wpe, void* out, int tokens,
                        int seq, int h, int64_t v0, int rows, int positions, float scale, cudaStream_t stream) {
  if (tokens < 0 || h <= 0 || h % 8 || rows < 0 || (wpe && !pos && seq <= 0)) return -1;
  if (!aligned16(wte) || !aligned16(wpe) || !aligned16(out)) return -1;
  if (tokens == 0) return 0;
  // whole rows once they fill the chip (48 warps on each of 148 SMs); before that a row is cut into slices of 128 vectors
  const int per_warp = tokens >= 7104 ? h / 8 : 128;
  embed_fwd_kernel<<<dim3((tokens + 7) / 8, (h / 8 + per_warp - 1) / per_warp), 256, 0, stream>>>(
      ids, pos, static_cast<const __nv_bfloat16*>(wte), static_cast<const __nv_bfloat16*>(wpe),
      static_cast<__nv_bfloat16*>(out), tokens, seq, h, v0, rows, positions, scale, per_warp);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

// Bytes of workspace of mb_embed_bwd.
MB_API size_t mb_embed_bwd_workspace(int tokens, int h, int with_positions) {
  return area_bytes(tokens, h) * (with_positions ? 2 : 1);
}

// dout [tokens][h] -> dwte [rows][h] (fp32 or bf16, stored or added to) and, where dwpe is not null, dwpe [positions][h]
// (bf16, stored).  pos null: position t % seq.  Every row of a stored table is written; rows that get no token are left
// alone where it is added to.  The workspace is for this call alone, on 16 bytes.  dwte may be null.
MB_API int mb_embed_bwd(const int64_t* ids, const int64_t* pos, const void* dout, void* dwte, void* dwpe, int tokens, int seq,
                        int h, int64_t v0, int rows, int positions, float scale, int dwte_fp32, int accumulate,
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
    t[0] = make_table(s[nsort++], dwte, dwte_fp32, accumulate, scale);
  }
  if (sort1) {
    s[nsort] = make_sort(pos, 0, positions, at + nsort * area_bytes(tokens, h), tokens, h);
    t[1] = make_table(s[nsort++], dwpe, 0, 0, 1.f);
  } else if (dwpe) {
    t[1].out = dwpe;
    t[1].rows = positions;
    t[1].stride = seq;
    t[1].scale = 1.f;
  }
  const int slices = slices_of(h), tiles = tiles_of(tokens);
  if (nsort && tokens > 0) {
    // one CTA up to 2048 tokens: a cluster's exchange costs more than the shorter stretches of its warps save
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    const int ctas = tokens <= 2048 ? 1 : kSortCluster;
    cfg.gridDim = dim3(ctas * nsort);
    cfg.blockDim = dim3(kSortThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool held = tokens <= ctas * kSortThreads * kHeld;
    if (cudaLaunchKernelEx(&cfg, held ? embed_sort_kernel<true> : embed_sort_kernel<false>, s[0], s[1], tokens, 2 * tiles * slices) != cudaSuccess) return -4;
  }
  const long rows0 = sort0 ? (rows + kRows - 1) / kRows : 0, rows1 = dwpe ? (positions + kRows - 1) / kRows : 0;
  const long long0 = sort0 ? static_cast<long>(tiles) * slices : 0, long1 = sort1 ? static_cast<long>(tiles) * slices : 0;
  const long blocks = rows0 + rows1 + long0 + long1;
  if (blocks == 0) return 0;
  if (blocks > 0x7fffffffl) return -1;
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
  if (cudaLaunchKernelEx(&cfg, embed_sum_kernel, t[0], t[1], static_cast<const __nv_bfloat16*>(dout), tokens, h,
                         static_cast<int>(long0), static_cast<int>(long1), static_cast<int>(rows0), slices) != cudaSuccess)
    return -4;
  return 0;
}
