// bf16 GEMM on CTA pairs: two CTAs on neighbouring SMs compute one 256 x 256 output tile with
// `tcgen05.mma.cta_group::2`.  Each CTA stages 128 rows of A and 128 rows of B per k-block
// (32 KB instead of the 48 KB a lone CTA needs for a 128 x 256 tile), so the shared-memory
// read traffic per MMA drops by a third and six stages fit.  The leader CTA issues the MMAs;
// each CTA keeps its 128 x 256 half of the accumulator in its own TMEM and runs its own
// epilogue (TMEM -> registers -> swizzled staging tile -> TMA store / reduce-add).
//
//   C[M,N] (op)= A[M,K] * B[N,K]^T, operands K-major or MN-major as in the single-CTA kernel.
//
// Same role split per CTA (192 threads): warp 0 TMA producer, warp 1 MMA issuer (leader CTA
// only), warps 2..5 epilogue; two accumulator stages in TMEM.  Loads are per-CTA TMA copies
// (never multicast) whose completion bytes are counted on the leader's barrier.
//
// Reference counterpart: the cuBLAS(Lt) calls of csrc/fused_dense_lib/fused_dense_cuda.cu:19-167.
#include "sm100_pair.cuh"
#include <string.h>
#include <stdio.h>

using namespace sm100;

namespace {

constexpr int BM = 128;       // rows per CTA (256 per pair)
constexpr int BN = 256;       // columns per pair; each CTA stages BN / 2 rows of B
constexpr int BNH = BN / 2;
constexpr int BK = 64;
// Six pipeline stages; the kernels whose epilogue reads a second operand (gelu' or residual) give one
// stage up for two staging tiles that TMA fills with that operand ahead of the epilogue.
constexpr int kStagesPlain = 6;
constexpr int kStagesAux = 5;
constexpr int kThreads = 192;

enum EpiFlags : int {
  EPI_BIAS = 1, EPI_GELU = 2, EPI_SAVE_PRE = 4, EPI_ACCUM = 8, EPI_DGELU = 16, EPI_OUT_FP32 = 32, EPI_RESIDUAL = 64
};

struct PairParams {
  int M, N, K;
  const __nv_bfloat16* bias;
  const __nv_bfloat16* aux;   // DGELU: pre-activation, RESIDUAL: tensor to add; [M][N] bf16 with row stride ldc
  int ldc;
  int flags;
  float alpha;
  int* status;
  // The tiles of the last, partly filled wave (tail_tiles of them) are cut along K into `splits` parts each, so that the
  // pairs without a tile take a share.  Every part goes to `part` in fp32; the CTA that counts the last part of its half
  // tile in `arrived` adds them in K order and runs the epilogue.  tail_tiles = 0: nothing is split.
  int tail_tiles, splits;
  float* part;      // [tail tile][split][CTA of the pair][column / 4][row][4]
  int* arrived;     // [tail tile][CTA of the pair], zero at the start
};

template <bool AUX>
struct Layout {
  static constexpr int kStages = AUX ? kStagesAux : kStagesPlain;
  static constexpr int kABytes = BM * BK * 2;
  static constexpr int kBBytes = BNH * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStagingBytes = BM * 128;
  static constexpr int kStagingOffset = kStages * kStageBytes;
  static constexpr int kAuxOffset = kStagingOffset + 2 * kStagingBytes;          // two tiles, AUX only
  static constexpr int kBarOffset = kAuxOffset + (AUX ? 2 * kStagingBytes : 0);
  // full[S], empty[S], tmem_full[2], tmem_empty[2], aux_full[2], tmem base word
  static constexpr int kTotal = kBarOffset + (2 * kStages + 6) * 8 + 16;
};

__device__ __forceinline__ void report(int* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// What a kernel's epilogue does beside the common part.  The split form is a kernel of its own: its second source of the
// products cost the others 4 - 9 % where the epilogue is the bound (13760 x 6664 x 128: 81.7 us against 87.4).
enum Kind : int { kPlain = 0, kAux = 1, kSplit = 2, kXentStats = 3, kXentGrad = 4, kXentKeep = 5 };

// Vocabulary projection with cross entropy: C, the logits, is not stored (kXentKeep: 16 bits of each).  The statistics' epilogue
// hides behind the products (4096 x 2048, vocabulary 50304 with bias: 496 us, 1.70 PFLOP/s, tensor pipe 97 % busy), the
// gradient's almost (25344 columns of the same: 259 us, 1.64 PFLOP/s, 88 %).  Long runs of both passes are bound by the power
// cap: 8192 x 2560 x 50304 6.4 ms for 8 T H V operations, 5.4 where kXentKeep spares the backward pass the logits (its own 1440
// us against 1290: 824 MB more to write, one stage less).  A struct of its own, because a parameter more changes the code of
// the other kinds (registers of the split one 238 -> 164).
struct XentParams : PairParams {
  const int64_t* labels;      // [M]; the label's column is labels[m] - v0
  int64_t v0, ignore;
  int segments;               // parts of K whose sums are added in registers
  float2* stats;              // kXentStats: [column tile][M] {maximum * log2(e), sum of 2^(x * log2(e) - that)}; kXentKeep: of
                              // every 128 columns
  float* target;              // kXentStats, kXentKeep: [M], written where the label's column is among these
  const float *lse, *gloss;   // kXentGrad: [M]
  float* col_sums;            // kXentGrad: [32 rows][N], column sums of what is stored, or null
};
template <int KIND> struct ParamsOf { using type = PairParams; };
template <> struct ParamsOf<kXentStats> { using type = XentParams; };
template <> struct ParamsOf<kXentGrad> { using type = XentParams; };
template <> struct ParamsOf<kXentKeep> { using type = XentParams; };

// What kXentKeep stores of a logit: how far it is below the greatest of its row's 128 columns, in 16 bits of 2^-10 octaves.
// The probability it stands for is right to 2^-11 octaves, 3.4e-4 of itself, a sixth of the rounding of the gradient to bf16,
// whatever its size (fp16 would lose the small ones, bf16 has a coarser step); 64 octaves below count as 0.
constexpr float kKeptStep = 1024.f;
constexpr uint32_t kKeptZero = 65535u;
// Two logits; `top` is the greatest in the same units.  2^23 is added instead of a conversion, which the unit of the
// exponentials would do; a NaN becomes 0 here and is one again by its row's sum.
__device__ __forceinline__ uint32_t kept_code2(float a, float b, float top) {
  constexpr float kScale = -1.4426950408889634f * kKeptStep, kMost = static_cast<float>(kKeptZero);
  const uint32_t x = __float_as_uint(fminf(fmaxf(fmaf(a, kScale, top), 0.f), kMost) + 8388608.f);
  const uint32_t y = __float_as_uint(fminf(fmaxf(fmaf(b, kScale, top), 0.f), kMost) + 8388608.f);
  return __byte_perm(x, y, 0x5410);
}
// The way back: 2^13 + code * 2^-10 has the code in its low half.
__device__ __forceinline__ float kept_below(uint32_t pair, int which) {
  static_assert(kKeptStep == 1024.f, "the step is 2^-10");
  return __uint_as_float(__byte_perm(pair, 0x46000000u, which ? 0x7632 : 0x7610)) - 8192.f;
}

// The bias of N columns, what the sums of their logits start from.
template <int N>
__device__ __forceinline__ void xent_start(const XentParams& p, float* v, int col0) {
  if (!(p.flags & EPI_BIAS)) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
  } else if (col0 + N <= p.N && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 8) mb::unpack8(*reinterpret_cast<const mb::bf16x8*>(p.bias + col0 + i), v + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __bfloat162float(p.bias[min(col0 + i, p.N - 1)]);
  }
}

// Statistics of the logits of one row over half a tile.  The maximum is kept in units of log2(e),
// so that an exponential is one FFMA and one ex2: 128 of them per thread, 2048 cycles of the special-function units per
// tile, against 8 cycles per unit of K of the products.
__device__ __forceinline__ float2 xent_row_stats(const XentParams& p, float* v, int col0, int lab, float& target) {
  constexpr float kLog2e = 1.4426950408889634f;
  if (col0 + 128 > p.N) {
#pragma unroll
    for (int i = 0; i < 128; ++i) v[i] = col0 + i < p.N ? v[i] : -INFINITY;
  }
  if (lab >= 0) {
#pragma unroll
    for (int i = 0; i < 128; ++i) target = lab == i ? v[i] : target;
  }
  float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
  const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kLog2e;
  const float m_use = m == -INFINITY ? 0.f : m;       // nothing but -inf: the exponentials are 0
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 128; ++i) s[i & 3] += mb::fast_exp2(fmaf(v[i], kLog2e, -m_use));
  return make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
}

// Threads of a kind's CTA: the epilogues of cross entropy have two warps for each 32 rows.
__host__ __device__ constexpr bool is_xent(int kind) { return kind >= kXentStats; }
__host__ __device__ constexpr int threads_of(int kind) { return is_xent(kind) ? 320 : kThreads; }
__host__ __device__ constexpr int staged_tiles(int kind) { return kind == kAux || kind == kXentGrad || kind == kXentKeep ? 4 : 2; }

template <bool A_MN, bool B_MN, int KIND>
__global__ void __launch_bounds__(threads_of(KIND), 1)
gemm_pair_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                 const __grid_constant__ CUtensorMap tma_c, const __grid_constant__ CUtensorMap tma_aux,
                 const typename ParamsOf<KIND>::type p) {
  constexpr bool AUX = KIND == kAux, SPLIT = KIND == kSplit, XENT = is_xent(KIND), KEEP = KIND == kXentKeep, STATS = KIND == kXentStats || KEEP;
  using L = Layout<staged_tiles(KIND) == 4>;
  constexpr int STAGES = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // Both CTAs of the pair must use the same offsets: the dynamic segment starts at the same
  // shared-memory address in every CTA of a launch, so the same rounding applies.
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* aux_full = tempty_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux_full + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader_cta = (rank == 0);
  const int pair = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;

  const int num_m = (p.M + 2 * BM - 1) / (2 * BM);
  const int num_n = (p.N + BN - 1) / BN;
  const int num_kb = (p.K + BK - 1) / BK;
  const int full_tiles = num_m * num_n - (SPLIT ? p.tail_tiles : 0);
  int num_items = full_tiles + (SPLIT ? p.tail_tiles * p.splits : 0);
  if constexpr (XENT)       // a pair's tiles, each as many items in a row as K has segments
    num_items = pair + num_pairs * p.segments * ((full_tiles - pair + num_pairs - 1) / num_pairs);
  // 256-row tiles per raster group: neighbours share B panels in L2.  The vocabulary's weight passes through memory once per
  // group, and the power that takes is missing to the products: 8192 tokens of 2560, vocabulary 50304, both passes 6790 us in
  // groups of 4, 6675 of 8, 6565 of 16.
  constexpr int GM = XENT ? 16 : 4;

  auto tile_coords = [&](int t, int& m0, int& n0) {
    int per_group = GM * num_n;
    int g = t / per_group;
    int first_m = g * GM;
    int gsz = min(num_m - first_m, GM);
    int r = t - g * per_group;
    m0 = (first_m + r % gsz) * (2 * BM) + static_cast<int>(rank) * BM;   // this CTA's rows
    n0 = (r / gsz) * BN;
  };

  // Item w of the list: tile t, K blocks [kb0, kb1); split is -1 for a whole tile.
  auto item_at = [&](int w, int& t, int& kb0, int& kb1, int& split) {
    t = w;
    kb0 = 0;
    kb1 = num_kb;
    split = -1;
    if constexpr (XENT) {
      const int q = (w - pair) / num_pairs, seg = q % p.segments;
      t = pair + q / p.segments * num_pairs;
      kb0 = seg * num_kb / p.segments;
      kb1 = (seg + 1) * num_kb / p.segments;
    }
    if (SPLIT && w >= full_tiles) {
      const int u = w - full_tiles;
      split = u / p.tail_tiles;
      t = full_tiles + u - split * p.tail_tiles;
      kb0 = split * num_kb / p.splits;
      kb1 = (split + 1) * num_kb / p.splits;
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);    // leader's: its own arrive.expect_tx covering both CTAs' bytes
      mbar_init(&empty_bar[s], 1);   // one MMA commit, broadcast to both CTAs
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);   // one MMA commit, broadcast to both CTAs
      mbar_init(&tempty_bar[a], XENT ? 16 : 8);  // leader's: the epilogue warps of both CTAs, 4 (8) each
      mbar_init(&aux_full[a], 1);    // second epilogue operand staged by TMA (AUX kernels)
    }
    fence_barrier_init();
    prefetch_tmap(&tma_a);
    prefetch_tmap(&tma_b);
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer's barriers exist before anything is signalled on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      uint32_t it = 0;
      uint32_t armed[STAGES];
      for (int s = 0; s < STAGES; ++s) armed[s] = 0;
      bool ok = true;
      for (int w = pair; w < num_items && ok; w += num_pairs) {
        int t, kb0, kb1, split, m0, n0;
        item_at(w, t, kb0, kb1, split);
        tile_coords(t, m0, n0);
        const int nb0 = n0 + static_cast<int>(rank) * BNH;   // this CTA's rows of B
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          int s = it % STAGES;
          uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(&empty_bar[s], ph ^ 1)) {
            report(p.status, MB_ERR_TIMEOUT_EMPTY);
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * L::kStageBytes;
          uint8_t* sb = sa + L::kABytes;
          if (leader_cta) {
            mbar_expect_tx(&full_bar[s], 2 * L::kStageBytes);
            armed[s]++;
          }
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[s]), 0);
          if (!A_MN) {
            tma_load_2d_pair(sa, &tma_a, bar, kb * BK, m0);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d_pair(sa + j * (BK * 128), &tma_a, bar, m0 + 64 * j, kb * BK);
          }
          if (!B_MN) {
            tma_load_2d_pair(sb, &tma_b, bar, kb * BK, nb0);
          } else {
#pragma unroll
            for (int j = 0; j < BNH / 64; ++j)
              tma_load_2d_pair(sb + j * (BK * 128), &tma_b, bar, nb0 + 64 * j, kb * BK);
          }
        }
      }
      if (!ok && leader_cta) {
        for (int s = 0; s < STAGES; ++s)
          if (armed[s]) mbar_wait(&full_bar[s], (armed[s] - 1) & 1, 50);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------- MMA issuer (leader CTA only)
    if (leader_cta) {
      constexpr uint32_t idesc = make_idesc_bf16(2 * BM, BN, A_MN ? 1 : 0, B_MN ? 1 : 0);
      uint32_t it = 0, tcount = 0;
      bool ok = true;
      for (int w = pair; w < num_items && ok; w += num_pairs, ++tcount) {
        int t, kb0, kb1, split;
        item_at(w, t, kb0, kb1, split);
        int acc = tcount & 1;
        uint32_t acc_ph = (tcount >> 1) & 1;
        if (!mbar_wait(&tempty_bar[acc], acc_ph ^ 1)) {
          report(p.status, MB_ERR_TIMEOUT_TMEM);
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          int s = it % STAGES;
          uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(&full_bar[s], ph)) {
            report(p.status, MB_ERR_TIMEOUT_FULL);
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            uint32_t sa = smem_u32(smem + s * L::kStageBytes);
            uint32_t sb = sa + L::kABytes;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              uint64_t ad = A_MN ? make_smem_desc_sw128(sa + k * 2048, BK * 128, 1024)
                                 : make_smem_desc_sw128(sa + k * 32, 16, 1024);
              uint64_t bd = B_MN ? make_smem_desc_sw128(sb + k * 2048, BK * 128, 1024)
                                 : make_smem_desc_sw128(sb + k * 32, 16, 1024);
              mma_f16_ss_pair(d_tmem, ad, bd, idesc, ((kb - kb0) | k) != 0 ? 1u : 0u);
            }
            mma_commit_pair(&empty_bar[s]);   // frees the stage in both CTAs
          }
          __syncwarp();
        }
        if (ok && elect_one()) mma_commit_pair(&tfull_bar[acc]);
        __syncwarp();
      }
    }
  } else if constexpr (XENT) {
    // --------------------------------------------- cross entropy of the logits (both CTAs)
    // Two warps for 32 rows, 128 columns each.  A tensor-core sum truncates, which makes logits of a long K too small by
    // some 2^-24 of themselves per 16 products (hidden size 4096: a loss 1.5e-6 off); so for the statistics K is cut into
    // segments of 1024 at most, whose sums are added here.  The accumulator goes back before the exponentials.
    const int q = warp & 3, half = (warp - 2) >> 2, r = q * 32 + lane;
    const bool leader = (warp & 3) == 2 && lane == 0;                        // of this half's 128 threads
    float2* meet = reinterpret_cast<float2*>(smem + L::kStagingOffset);      // [parity of the tile][row]
    uint32_t count = 0, stored = 0;
    int parity = 0;
    bool ok = true;
    auto wait_sum = [&](uint32_t n) -> bool {
      if (mbar_wait(&tfull_bar[n & 1], (n >> 1) & 1)) return true;
      report(p.status, MB_ERR_TIMEOUT_TMEM);
      return false;
    };
    auto add32 = [&](float* v, uint32_t n, int c) {      // columns c ... of this half
      uint32_t rr[32];
      tmem_ld32(tmem_base + (n & 1) * BN + half * 128 + c + (static_cast<uint32_t>(q * 32) << 16), rr);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(rr[i]);
    };
    auto give_back = [&](uint32_t n) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty_bar[n & 1]), 0));
    };
    auto label_at = [&](bool live, int row, int col, int width) -> int {      // the label's place among these, or -1
      if (!live) return -1;
      const int64_t at = p.labels[row] - p.v0 - col;
      return at >= 0 && at < min(width, p.N - col) ? static_cast<int>(at) : -1;
    };
    for (int t = pair; t < full_tiles && ok; t += num_pairs, parity ^= 1) {
      int m0, n0;
      tile_coords(t, m0, n0);
      const int row = m0 + r, col0 = n0 + half * 128;
      const bool live = row < p.M;
      if constexpr (STATS) {
        float v[128];
        xent_start<128>(p, v, col0);
#pragma unroll 1
        for (int seg = 0; seg < p.segments && ok; ++seg, ++count) {
          ok = wait_sum(count);
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 128; c += 32) add32(v + c, count, c);
          give_back(count);
        }
        if (!ok || m0 >= p.M) continue;
        const int lab = label_at(live, row, col0, 128);
        float target = 0.f;
        float2 mine = xent_row_stats(p, v, col0, lab, target);
        if (lab >= 0) p.target[row] = target;
        if constexpr (KEEP) {
          if (live) p.stats[(2 * static_cast<size_t>(n0 / BN) + half) * p.M + row] = mine;
          const float top = mine.x == -INFINITY ? 0.f : mine.x * kKeptStep;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (col0 + 64 * u >= p.N) break;
            uint8_t* stg = smem + L::kStagingOffset + (2 * half + (stored & 1)) * L::kStagingBytes;
            if (leader) tma_wait_read<1>();
            asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              uint32_t c[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) c[i] = kept_code2(v[64 * u + 8 * g + 2 * i], v[64 * u + 8 * g + 2 * i + 1], top);
              *reinterpret_cast<uint4*>(stg + r * 128 + ((g ^ (r & 7)) << 4)) = make_uint4(c[0], c[1], c[2], c[3]);
            }
            fence_async_smem();
            asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
            if (leader) {
              tma_store_2d(&tma_c, stg, col0 + 64 * u, m0);
              tma_commit();
            }
            ++stored;
          }
          continue;
        }
        if (half) meet[parity * BM + r] = mine;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
        if (!half) {
          const float2 other = meet[parity * BM + r];
          const float m = fmaxf(mine.x, other.x), use = m == -INFINITY ? 0.f : m;
          mine = make_float2(m, mine.y * mb::fast_exp2(mine.x - use) + other.y * mb::fast_exp2(other.x - use));
          if (live) p.stats[static_cast<size_t>(n0 / BN) * p.M + row] = mine;
        }
      } else {
        // (softmax - [label]) * gradient of the loss, 0 in an ignored row; 64 columns at a time through staging
        const bool skipped = !live || p.labels[row] == p.ignore;
        const float lse2 = live ? p.lse[row] * 1.4426950408889634f : 0.f, gloss = live ? p.gloss[row] : 0.f;
        ok = wait_sum(count);
        tc_fence_after();
#pragma unroll 1
        for (int u = 0; u < 2 && ok; ++u) {
          const int ucol0 = col0 + 64 * u;
          float v[64];
          xent_start<64>(p, v, ucol0);
          add32(v, count, 64 * u);
          add32(v + 32, count, 64 * u + 32);
          if (u == 1) give_back(count);
          if (m0 >= p.M || ucol0 >= p.N) continue;
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = mb::fast_exp2(fmaf(v[i], 1.4426950408889634f, -lse2));
          const int lab = label_at(live, row, ucol0, 64);
          if (lab >= 0) {
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = i == lab ? v[i] - 1.f : v[i];
          }
          uint8_t* stg = smem + L::kStagingOffset + (2 * half + (stored & 1)) * L::kStagingBytes;
          if (leader) tma_wait_read<1>();
          asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = skipped ? 0.f : v[8 * g + i] * gloss;
            *reinterpret_cast<mb::bf16x8*>(stg + r * 128 + ((g ^ (r & 7)) << 4)) = mb::pack8(f);
          }
          if (p.col_sums && m0 + q * 32 < p.M) {
            // column sums of what is stored (the bias' gradient): a lane adds two columns of its warp's 32 rows
            __syncwarp();
            float s0 = 0.f, s1 = 0.f;
#pragma unroll 8
            for (int i = 0; i < 32; ++i) {
              const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(
                  stg + (q * 32 + i) * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4));
              s0 += x.x;
              s1 += x.y;
            }
            float* dst = p.col_sums + static_cast<size_t>((m0 >> 5) + q) * p.N + ucol0 + 2 * lane;
            if (ucol0 + 2 * lane < p.N) dst[0] = s0;
            if (ucol0 + 2 * lane + 1 < p.N) dst[1] = s1;
          }
          fence_async_smem();
          asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
          if (leader) {
            tma_store_2d(&tma_c, stg, ucol0, m0);
            tma_commit();
          }
          ++stored;
        }
        ++count;
      }
    }
    if (leader) tma_wait_all<0>();
  } else {
    // ----------------------------------------------------------- epilogue (both CTAs)
    const int q = warp & 3;
    const int r = q * 32 + lane;
    const bool leader = (threadIdx.x == 64);
    const bool out_fp32 = (p.flags & EPI_OUT_FP32) != 0;
    const int cols_per_unit = out_fp32 ? 32 : 64;
    const int units = BN / cols_per_unit;
    const int npass = (p.flags & EPI_SAVE_PRE) ? 2 : 1;
    uint32_t tcount = 0, epi_units = 0, aux_units = 0;
    bool ok = true;
    for (int w = pair; w < num_items && ok; w += num_pairs, ++tcount) {
      int t, kb0, kb1, split, m0, n0;
      item_at(w, t, kb0, kb1, split);
      tile_coords(t, m0, n0);
      int acc = tcount & 1;
      uint32_t acc_ph = (tcount >> 1) & 1;
      if (AUX && leader && m0 < p.M) {
        // the first two operand tiles of this output tile travel while the main loop still runs
        const int live = min(units, (p.N - n0 + cols_per_unit - 1) / cols_per_unit);
        for (int u = 0; u < 2 && u < live; ++u) {
          const uint32_t au = aux_units + u;
          mbar_expect_tx(&aux_full[au & 1], L::kStagingBytes);
          tma_load_2d(smem + L::kAuxOffset + (au & 1) * L::kStagingBytes, &tma_aux, &aux_full[au & 1],
                      n0 + u * cols_per_unit, m0);
        }
      }
      if (!mbar_wait(&tfull_bar[acc], acc_ph)) {
        report(p.status, MB_ERR_TIMEOUT_TMEM);
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
      auto release_accumulator = [&]() {     // tell the leader's MMA warp (one arrival per warp)
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty_bar[acc]), 0));
      };
      const float4* parts = nullptr;         // the tile's parts in K order, where it was split
      if (SPLIT && split >= 0) {
        constexpr int kPart4 = BM * BN / 4;  // float4s of a CTA's half of a part
        const int tail = t - full_tiles;
        float4* all = reinterpret_cast<float4*>(p.part) + static_cast<size_t>(tail) * p.splits * 2 * kPart4 + rank * kPart4 + r;
        float4* mine = all + static_cast<size_t>(split) * 2 * kPart4;
        for (int c = 0; c < BN; c += 32) {
          uint32_t rr[32];
          tmem_ld32(taddr + c, rr);
          tmem_ld_wait();
#pragma unroll
          for (int g = 0; g < 8; ++g)
            mine[(c / 4 + g) * BM] = make_float4(__uint_as_float(rr[4 * g]), __uint_as_float(rr[4 * g + 1]),
                                                 __uint_as_float(rr[4 * g + 2]), __uint_as_float(rr[4 * g + 3]));
        }
        release_accumulator();
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (leader) tmem_slot[1] = (atomicAdd(&p.arrived[2 * tail + rank], 1) == p.splits - 1);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (!tmem_slot[1]) continue;
        __threadfence();
        parts = all;
      }
      const bool rows_live = m0 < p.M;   // the second CTA of a pair can hang over the bottom edge
      int units_live = 0;
      if (rows_live) units_live = min(units, (p.N - n0 + cols_per_unit - 1) / cols_per_unit);
      for (int u = 0; u < units && rows_live; ++u) {
        const int ucol0 = n0 + u * cols_per_unit;
        if (ucol0 >= p.N) break;
        if (AUX) {
          const uint32_t au = aux_units + u;
          if (!mbar_wait(&aux_full[au & 1], (au >> 1) & 1)) {
            report(p.status, MB_ERR_TIMEOUT_FULL);
            ok = false;
            break;
          }
        }
        for (int pass = 0; pass < npass; ++pass) {
          uint8_t* stg = smem + L::kStagingOffset + (epi_units & 1) * L::kStagingBytes;
          if (leader) tma_wait_read<1>();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          const int halves = out_fp32 ? 1 : 2;
          for (int hh = 0; hh < halves; ++hh) {
            float v[32];
            const int col0 = ucol0 + hh * 32;
            if (SPLIT && parts) {
              const float4* at = parts + (u * cols_per_unit + hh * 32) / 4 * BM;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
              for (int sp = 0; sp < p.splits; ++sp, at += 2 * (BM * BN / 4)) {
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                  const float4 x = __ldcg(at + g * BM);
                  v[4 * g] += x.x; v[4 * g + 1] += x.y; v[4 * g + 2] += x.z; v[4 * g + 3] += x.w;
                }
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= p.alpha;
            } else {
              uint32_t rr[32];
              tmem_ld32(taddr + u * cols_per_unit + hh * 32, rr);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(rr[i]) * p.alpha;
            }
            if (p.flags & EPI_BIAS) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += __bfloat162float(p.bias[min(col0 + i, p.N - 1)]);
            }
            if (AUX) {
              // second operand from the tile TMA staged for this unit (same swizzle as the output tile)
              const uint8_t* at = smem + L::kAuxOffset + ((aux_units + u) & 1) * L::kStagingBytes;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float f[8];
                mb::unpack8(*reinterpret_cast<const mb::bf16x8*>(at + r * 128 + (((hh * 4 + j) ^ (r & 7)) << 4)), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  if (p.flags & EPI_DGELU) v[8 * j + i] *= mb::gelu_tanh_grad(f[i]);
                  else v[8 * j + i] += f[i];
                }
              }
            }
            if ((p.flags & EPI_GELU) && (pass == npass - 1)) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = mb::gelu_tanh(v[i]);
            }
            if (out_fp32) {
#pragma unroll
              for (int g = 0; g < 8; ++g)
                *reinterpret_cast<float4*>(stg + r * 128 + ((g ^ (r & 7)) << 4)) =
                    make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                *reinterpret_cast<mb::bf16x8*>(stg + r * 128 + (((hh * 4 + g) ^ (r & 7)) << 4)) = mb::pack8(v + 8 * g);
            }
          }
          fence_async_smem();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (AUX && leader && u + 2 < units_live) {
            // every thread has read this unit's operand tile: refill the buffer for the unit after next
            const uint32_t au = aux_units + u + 2;
            mbar_expect_tx(&aux_full[au & 1], L::kStagingBytes);
            tma_load_2d(smem + L::kAuxOffset + (au & 1) * L::kStagingBytes, &tma_aux, &aux_full[au & 1],
                        n0 + (u + 2) * cols_per_unit, m0);
          }
          if (leader) {
            const CUtensorMap* dst = (npass == 2 && pass == 0) ? &tma_aux : &tma_c;
            if ((p.flags & EPI_ACCUM) && out_fp32) {
              asm volatile(
                  "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];\n" ::
                      "l"(reinterpret_cast<uint64_t>(dst)),
                  "r"(smem_u32(stg)), "r"(ucol0), "r"(m0)
                  : "memory");
            } else {
              tma_store_2d(dst, stg, ucol0, m0);
            }
            tma_commit();
          }
          ++epi_units;
        }
      }
      aux_units += units_live;
      if (!SPLIT || split < 0) release_accumulator();
    }
    if (leader) tma_wait_all<0>();
  }

  // Neither CTA may leave while the other can still read its shared memory, signal its
  // barriers or use the paired TMEM allocation.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * BN);
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}
bool make_map(CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols,
              uint32_t box_rows, bool fp32, bool promote) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld * (fp32 ? 4u : 2u)};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return encode_with_context([&] {
    return fn(m, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, promote ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

int g_sms = 0;

struct Split {
  int tail_tiles, splits;
};
// How the last wave is cut.  Splitting saves the K blocks that a part leaves to others; against that stand the parts
// written to memory and read back by one CTA in the end, and an epilogue that no longer overlaps anything: about 20 K blocks
// and 12 more for each part, measured over 76 - 688 tiles, tails of 2 - 70 tiles, 8 - 256 K blocks and 2 - 8 parts.  Parts
// that need a wave of their own never paid.  So it is the long sums with a nearly empty last wave that are split, above
// all weight gradients, whose K is the number of tokens: of 256 K blocks 76 tiles (tail 2) 171 -> 134 us, 300 tiles (tail 4)
// 491 -> 445; of 128 K blocks 76 tiles 90 -> 79 us, 256 tiles (tail 34) 208 -> 204.  Of 64 K blocks no tail gained (86 tiles,
// tail 12: 47 -> 50 us), nor did a tail of 38 tiles of 128 (90 -> 96 us in three parts).
Split choose_split(int M, int N, int K, int flags, int max_ctas) {
  Split none = {0, 1};
  const int pairs = max_ctas / 2, num_kb = (K + BK - 1) / BK;
  const long tiles = static_cast<long>((M + 2 * BM - 1) / (2 * BM)) * ((N + BN - 1) / BN);
  if (pairs < 1 || tiles < pairs || (flags & (EPI_DGELU | EPI_RESIDUAL))) return none;
  const int tail = static_cast<int>(tiles % pairs);
  int best = 12, splits = 1;
  for (int s = 2; s <= 8 && tail > 0 && s * tail <= pairs && num_kb / s >= 8; ++s) {
    const int gain = num_kb - (num_kb + s - 1) / s - 20 - 12 * s - tail * s / 10;
    if (gain > best) {
      best = gain;
      splits = s;
    }
  }
  if (splits == 1) return none;
  return {tail, splits};
}
int clamp_ctas(int max_ctas) {
  if (!g_sms) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&g_sms, cudaDevAttrMultiProcessorCount, dev);
  }
  return (max_ctas <= 0 || max_ctas > g_sms) ? g_sms : max_ctas;
}
size_t arrived_bytes(const Split& s) { return (static_cast<size_t>(s.tail_tiles) * 2 * 4 + 255) / 256 * 256; }

template <bool A_MN, bool B_MN, int KIND>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const CUtensorMap& tx,
           const typename ParamsOf<KIND>::type& p, int max_ctas, cudaStream_t stream) {
  constexpr int smem = Layout<staged_tiles(KIND) == 4>::kTotal + 1024;
  static bool configured[64] = {};      // of each device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  auto kern = gemm_pair_kernel<A_MN, B_MN, KIND>;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -3;
    configured[dev] = true;
  }
  int tiles = ((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + BN - 1) / BN);
  int pairs = max_ctas / 2;
  if (pairs > tiles) pairs = tiles;
  if (pairs < 1) return -1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  cfg.blockDim = dim3(threads_of(KIND), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, tx, p) == cudaSuccess ? 0 : -4;
}

template <int KIND>
int dispatch(bool a_mn, bool b_mn, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
             const CUtensorMap& tx, const PairParams& p, int max_ctas, cudaStream_t stream) {
  if (!a_mn && !b_mn) return launch<false, false, KIND>(ta, tb, tc, tx, p, max_ctas, stream);
  if (!a_mn && b_mn) return launch<false, true, KIND>(ta, tb, tc, tx, p, max_ctas, stream);
  if (a_mn && !b_mn) return launch<true, false, KIND>(ta, tb, tc, tx, p, max_ctas, stream);
  return launch<true, true, KIND>(ta, tb, tc, tx, p, max_ctas, stream);
}

}  // namespace

MB_API int* mb_status_device_ptr();

// Same contract as mb_gemm_bf16 for the epilogues the TMA-store path covers (bias, GELU with
// optional pre-activation copy, bf16 or fp32 output, fp32 accumulation, and for bf16 output
// multiplication by gelu'(aux) or addition of aux).  Returns 1 without
// launching when the arguments need the single-CTA kernel (other epilogue flags, unaligned C,
// fewer than two 256 x 256 tiles); the caller then uses mb_gemm_bf16.
static char g_pair_err[256] = "";
// Arguments of the last mb_gemm_pair_bf16 call that got as far as building its tensor maps.
MB_API const char* mb_gemm_pair_last_error(void) { return g_pair_err; }

// Bytes of workspace with which mb_gemm_pair_bf16 would split the tiles of its last wave; 0: nothing to split.
MB_API size_t mb_gemm_pair_workspace(int M, int N, int K, int flags, int max_ctas) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Split s = choose_split(M, N, K, flags, clamp_ctas(max_ctas));
  if (!s.tail_tiles) return 0;
  return arrived_bytes(s) + static_cast<size_t>(s.tail_tiles) * s.splits * 2 * BM * BN * sizeof(float);
}

// mb_gemm_pair_bf16 (below) with a workspace of as many bytes as mb_gemm_pair_workspace says, aligned to 16 and for this
// call alone; null: no tile is split.
MB_API int mb_gemm_pair_split_bf16(const void* A, const void* B, void* C, int M, int N, int K, int lda, int ldb,
                                   int ldc, int a_mn_major, int b_mn_major, int flags, const void* bias, void* aux,
                                   float alpha, int max_ctas, void* workspace, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if ((lda & 7) || (ldb & 7) || (reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(B) & 15))
    return -1;
  const bool out_fp32 = (flags & EPI_OUT_FP32) != 0;
  const int esz = out_fp32 ? 4 : 2;
  const int ok_flags = EPI_BIAS | EPI_GELU | EPI_SAVE_PRE | EPI_OUT_FP32 | (out_fp32 ? EPI_ACCUM : 0) |
                       (out_fp32 ? 0 : (EPI_DGELU | EPI_RESIDUAL));
  if ((flags & ~ok_flags) || (reinterpret_cast<uintptr_t>(C) & 15) || ((static_cast<long>(ldc) * esz) % 16) ||
      ((flags & EPI_GELU) && out_fp32))
    return 1;
  if ((flags & EPI_SAVE_PRE) && (!aux || (reinterpret_cast<uintptr_t>(aux) & 15) || !(flags & EPI_GELU))) return 1;
  if (flags & (EPI_DGELU | EPI_RESIDUAL)) {
    // one second operand only, read with 16-byte loads at row stride ldc
    if (!aux || (reinterpret_cast<uintptr_t>(aux) & 15) || (ldc & 7) || (flags & (EPI_GELU | EPI_SAVE_PRE)) ||
        ((flags & EPI_DGELU) && (flags & EPI_RESIDUAL)))
      return 1;
  }
  max_ctas = clamp_ctas(max_ctas);
  const long tiles = static_cast<long>((M + 2 * BM - 1) / (2 * BM)) * ((N + BN - 1) / BN);
  if (tiles < max_ctas / 2) return 1;     // cannot fill the machine with 256 x 256 tiles
  CUtensorMap ta, tb, tc, tx;
  memset(&tx, 0, sizeof(tx));
  // a tensor map that cannot be encoded: -21 (A), -22 (B), -23 (C), -24 (second epilogue operand); the arguments
  // of the refused call can be read back with mb_gemm_pair_last_error
  snprintf(g_pair_err, sizeof(g_pair_err), "A=%p B=%p C=%p aux=%p M=%d N=%d K=%d lda=%d ldb=%d ldc=%d a_mn=%d b_mn=%d flags=%d",
           A, B, C, aux, M, N, K, lda, ldb, ldc, a_mn_major, b_mn_major, flags);
  if (!(a_mn_major ? make_map(&ta, A, K, M, lda, 64, BK, false, true) : make_map(&ta, A, M, K, lda, 64, BM, false, true)))
    return -21;
  if (!(b_mn_major ? make_map(&tb, B, K, N, ldb, 64, BK, false, true) : make_map(&tb, B, N, K, ldb, 64, BNH, false, true)))
    return -22;
  if (!make_map(&tc, C, M, N, ldc, out_fp32 ? 32 : 64, BM, out_fp32, false)) return -23;
  const bool has_aux = (flags & (EPI_DGELU | EPI_RESIDUAL)) != 0;
  if (((flags & EPI_SAVE_PRE) || has_aux) && !make_map(&tx, aux, M, N, ldc, 64, BM, false, false)) return -24;
  PairParams p;
  p.M = M; p.N = N; p.K = K;
  p.bias = reinterpret_cast<const __nv_bfloat16*>(bias);
  p.aux = reinterpret_cast<const __nv_bfloat16*>(aux);
  p.ldc = ldc;
  p.flags = flags;
  p.alpha = alpha;
  p.status = mb_status_device_ptr();
  Split split = {0, 1};
  if (workspace && !(reinterpret_cast<uintptr_t>(workspace) & 15)) split = choose_split(M, N, K, flags, max_ctas);
  p.tail_tiles = split.tail_tiles;
  p.splits = split.splits;
  p.arrived = reinterpret_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + arrived_bytes(split));
  if (split.tail_tiles && cudaMemsetAsync(workspace, 0, arrived_bytes(split), stream) != cudaSuccess) return -4;
  if (has_aux) return dispatch<kAux>(a_mn_major != 0, b_mn_major != 0, ta, tb, tc, tx, p, max_ctas, stream);
  if (split.tail_tiles) return dispatch<kSplit>(a_mn_major != 0, b_mn_major != 0, ta, tb, tc, tx, p, max_ctas, stream);
  return dispatch<kPlain>(a_mn_major != 0, b_mn_major != 0, ta, tb, tc, tx, p, max_ctas, stream);
}

namespace {

// One thread adds a sixteenth of a row's tiles; a block takes 32 rows.
__global__ void __launch_bounds__(512)
xent_combine_kernel(const float2* __restrict__ stats, const float* __restrict__ target, const int64_t* __restrict__ labels,
                    float* __restrict__ loss, float* __restrict__ lse, float* __restrict__ out_stats, int rows, int tiles,
                    int cols, int64_t v0, int64_t ignore) {
  __shared__ float2 part[16][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float2 x) {
    const float n = fmaxf(m, x.x), use = n == -INFINITY ? 0.f : n;
    s = s * exp2f(m - use) + x.y * exp2f(x.x - use);
    m = n;
  };
  if (row < rows) {
    for (int t = w; t < tiles; t += 128) {
      float2 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        x[u] = t + 16 * u < tiles ? stats[static_cast<size_t>(t + 16 * u) * rows + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) add(x[u]);
    }
  }
  part[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w || row >= rows) return;
  for (int k = 1; k < 16; ++k) add(part[k][lane]);
  const int64_t lab = labels[row], at = lab - v0;
  const float hit = (at >= 0 && at < cols) ? target[row] : 0.f;
  constexpr double kLn2 = 0.6931471805599453;
  if (out_stats) {
    out_stats[3l * row] = static_cast<float>(m * kLn2);
    out_stats[3l * row + 1] = s;
    out_stats[3l * row + 2] = hit;
  } else {
    const float l = static_cast<float>((static_cast<double>(m) + log2f(s)) * kLn2);
    lse[row] = l;
    loss[row] = lab == ignore ? 0.f : l - hit;
  }
}

// Sum over the groups of 32 rows, in a fixed order; a block takes 32 columns.
__global__ void __launch_bounds__(256)
xent_bias_grad_kernel(const float* __restrict__ sums, void* __restrict__ out, int groups, int cols, int fp32) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int g = w; g < groups; g += 8) a += sums[static_cast<size_t>(g) * cols + c];
  }
  part[w][lane] = a;
  __syncthreads();
  if (w || c >= cols) return;
  for (int k = 1; k < 8; ++k) a += part[k][lane];
  if (fp32) static_cast<float*>(out)[c] = a;
  else static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16(a);
}

// Gradient of a piece of the logits from what kXentKeep stored: 32 rows x 512 columns per block, 8 columns of 8 rows per thread.
// The label's column is computed from the logit itself, so that a row whose label is all but certain keeps its small gradient.
// Bound by memory: 8192 x 12800 72 us, 5.8 TB/s (146 with conversions between integers and floats, which share the unit of the
// exponentials, and every check per element).
template <bool SUMS>
__global__ void __launch_bounds__(256)
xent_kept_grad_kernel(const uint16_t* __restrict__ kept, int ldk, const float2* __restrict__ stats, const float* __restrict__ target,
                      const int64_t* __restrict__ labels, const float* __restrict__ lse, const float* __restrict__ gloss,
                      __nv_bfloat16* __restrict__ out, int ldd, float* __restrict__ col_sums, int rows, int c0, int cols,
                      int64_t v0, int64_t ignore) {
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ float top[4][32], grad[32], hit[32], part[3][SUMS ? 512 : 1];
  __shared__ int at[32];
  __shared__ bool skip[32];
  const int tid = threadIdx.x, r0 = blockIdx.y * 32, col = blockIdx.x * 512 + 8 * (tid & 63), line = tid >> 6;
  uint4 c[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int row = r0 + 4 * k + line;
    if (col < cols && row < rows) c[k] = *reinterpret_cast<const uint4*>(kept + static_cast<size_t>(row) * ldk + c0 + col);
  }
  if (tid < 32) {
    const int row = r0 + tid;
    const bool none = row >= rows || labels[row] == ignore;
    const int64_t a = none ? -1 : labels[row] - v0 - c0;
    const bool here = a >= 0 && a < cols;
    skip[tid] = none;
    grad[tid] = none ? 0.f : gloss[row];
    hit[tid] = here ? mb::fast_exp2(kLog2e * target[row] - kLog2e * lse[row]) - 1.f : 0.f;
    at[tid] = here ? static_cast<int>(a) : -8;
  } else if (tid >= 64 && tid < 192) {
    const int q = (tid - 64) >> 5, row = r0 + (tid & 31), first = blockIdx.x * 512 + 128 * q;
    if (row < rows && first < cols)
      top[q][tid & 31] = stats[static_cast<size_t>((c0 + first) / 128) * rows + row].x - kLog2e * lse[row];
  }
  __syncthreads();
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < cols) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int in = 4 * k + line, row = r0 + in;
      if (row >= rows) break;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (!skip[in]) {
        const float t = top[(tid & 63) >> 4][in], g = grad[in];
        const uint32_t w[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
        uint32_t zeros = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) zeros |= (~w[i] - 0x00010001u) & w[i] & 0x80008000u;      // halves that are all ones
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = g * mb::fast_exp2(t - kept_below(w[i >> 1], i & 1));
        const int label = at[in] - col;
        if (zeros || static_cast<unsigned>(label) < 8u || col + 8 > cols) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (((w[i >> 1] >> (16 * (i & 1))) & 0xffffu) == kKeptZero) f[i] = 0.f;
            if (i == label) f[i] = g * hit[in];
            if (col + i >= cols) f[i] = 0.f;
          }
        }
      }
      *reinterpret_cast<mb::bf16x8*>(out + static_cast<size_t>(row) * ldd + col) = mb::pack8(f);
      if (SUMS) {      // before the rounding
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += f[i];
      }
    }
  }
  if (!SUMS) return;
  if (line) {
#pragma unroll
    for (int i = 0; i < 8; ++i) part[line - 1][8 * (tid & 63) + i] = sum[i];
  }
  __syncthreads();
  if (line || col >= cols) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (col + i < cols)
      col_sums[static_cast<size_t>(blockIdx.y) * cols + col + i] =
          (sum[i] + part[0][8 * tid + i]) + (part[1][8 * tid + i] + part[2][8 * tid + i]);
  }
}

// Both operands K-major, the vocabulary on the B side; no rule on the number of tiles: there is one kernel for all sizes.
// out: the gradient of the logits (kXentGrad), what is kept of them (kXentKeep), or nothing.
int xent_gemm(const void* x, const void* w, void* dlogits, int ldd, XentParams& p, int ldx, int ldw, int max_ctas,
              cudaStream_t stream, bool keep = false) {
  CUtensorMap ta, tb, tc, tx;
  memset(&tc, 0, sizeof(tc));
  memset(&tx, 0, sizeof(tx));
  if (!make_map(&ta, x, p.M, p.K, ldx, 64, BM, false, true)) return -21;
  if (!make_map(&tb, w, p.N, p.K, ldw, 64, BNH, false, true)) return -22;
  if (dlogits && !make_map(&tc, dlogits, p.M, p.N, ldd, 64, BM, false, false)) return -23;
  p.alpha = 1.f;
  p.status = mb_status_device_ptr();
  p.splits = 1;
  max_ctas = clamp_ctas(max_ctas);
  if (max_ctas < 2) max_ctas = 2;      // a pair
  if (keep) return launch<false, false, kXentKeep>(ta, tb, tc, tx, p, max_ctas, stream);
  return dlogits ? launch<false, false, kXentGrad>(ta, tb, tc, tx, p, max_ctas, stream)
                 : launch<false, false, kXentStats>(ta, tb, tc, tx, p, max_ctas, stream);
}

bool xent_args_ok(const void* x, const void* w, int M, int V, int K, int ldx, int ldw) {
  return M >= 0 && V > 0 && K > 0 && !((K | ldx | ldw) & 7) && ldx >= K && ldw >= K &&
         !((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15);
}

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// Work area of the backward pass: gradient of a piece's logits, its column sums, dx in fp32 (several pieces), and what
// the products split (the largest of them; calls follow one another on the stream).
struct XentArea {
  size_t dlogits, col_sums, dx32, gemm, total;
};
XentArea xent_area(int M, int V, int K, int piece, bool want_x, bool want_w, bool want_b, int dw_flags, int max_ctas) {
  XentArea a;
  const size_t wide = (static_cast<size_t>(piece) + 7) / 8 * 8;
  const bool many = piece < V;
  a.dlogits = up256(2 * wide * M);
  a.col_sums = want_b ? up256(4ul * piece * ((M + 31) / 32)) : 0;
  a.dx32 = want_x && many ? up256(4ul * M * K) : 0;
  a.gemm = 0;
  auto need = [&](int m, int n, int k, int flags) {
    const size_t b = mb_gemm_pair_workspace(m, n, k, flags, max_ctas);
    if (b > a.gemm) a.gemm = b;
  };
  for (int n : {piece, V % piece ? V % piece : piece}) {
    if (want_x) need(M, K, n, many ? EPI_OUT_FP32 : 0);
    if (want_w) need(n, K, M, dw_flags);
  }
  a.total = a.dlogits + a.col_sums + a.dx32 + up256(a.gemm);
  return a;
}

}  // namespace

MB_API int mb_gemm_bf16(const void* A, const void* B, void* C, int M, int N, int K, int lda, int ldb, int ldc, int a_mn_major,
                        int b_mn_major, int flags, const void* bias, void* aux, float alpha, int tile_n, int max_ctas,
                        cudaStream_t stream);
MB_API int mb_cast_f32_to_bf16(const float* in, void* out, size_t n, float scale, cudaStream_t s);

// Tiles of the vocabulary that mb_xent_linear_fwd keeps statistics of.
MB_API int mb_xent_linear_tiles(int V) { return (V + BN - 1) / BN; }

// Cross entropy of logits = x [M,K] * w [V,K]^T + bias, which are not stored.  stats: [tiles][M][2] fp32 and target: [M]
// fp32, workspaces of this call.  out_stats null: loss [M] (0 where the label is `ignore`) and lse [M], natural logarithms;
// a label outside [v0, v0 + V) has the logit 0.  out_stats [M][3]: {maximum, sum of exponentials relative to it, label's
// logit (0 outside)} instead, which a group of vocabulary slices combines.  K and the leading dimensions multiples of 8.
// Where kept is given, 16 bits of every logit are stored there, [M][ldk] (ldk >= V, a multiple of 8), for the backward pass, which
// then needs stats, [2 * tiles][M][2] in this case, and target as well.
MB_API int mb_xent_linear_fwd(const void* x, const void* w, const void* bias, const int64_t* labels, float* stats,
                              float* target, float* loss, float* lse, float* out_stats, void* kept, int ldk, int M, int V, int K,
                              int ldx, int ldw, int64_t v0, int64_t ignore, int max_ctas, cudaStream_t stream) {
  if (!xent_args_ok(x, w, M, V, K, ldx, ldw)) return -1;
  if (kept && (ldk < V || ldk % 8 || (reinterpret_cast<uintptr_t>(kept) & 15))) return -1;
  if (M == 0) return 0;
  XentParams p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = V; p.K = K;
  p.bias = reinterpret_cast<const __nv_bfloat16*>(bias);
  p.flags = bias ? EPI_BIAS : 0;
  p.labels = labels;
  p.v0 = v0;
  p.segments = (K + 1023) / 1024;
  p.stats = reinterpret_cast<float2*>(stats);
  p.target = target;
  const int rc = xent_gemm(x, w, kept, ldk, p, ldx, ldw, max_ctas, stream, kept != nullptr);
  if (rc != 0) return rc;
  xent_combine_kernel<<<(M + 31) / 32, 512, 0, stream>>>(p.stats, target, labels, loss, lse, out_stats, M,
                                                         mb_xent_linear_tiles(V) * (kept ? 2 : 1), V, v0, ignore);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}
// Bytes of workspace of mb_xent_linear_bwd, which holds the gradient of `piece` columns of logits at a time.
MB_API size_t mb_xent_linear_bwd_workspace(int M, int V, int K, int piece, int want_x, int want_w, int want_b, int dw_fp32,
                                           int accumulate, int max_ctas) {
  if (M <= 0 || V <= 0 || K <= 0 || piece <= 0) return 0;
  return xent_area(M, V, K, piece < V ? piece : V, want_x, want_w, want_b,
                   (dw_fp32 ? EPI_OUT_FP32 : 0) | (accumulate ? EPI_ACCUM : 0), clamp_ctas(max_ctas)).total;
}

// Gradients of the loss, gloss [M] being what it is differentiated by: with d[t,v] = (exp(logit - lse) - [label]) * gloss
// (rows whose label is `ignore`: 0), computed again piece by piece and rounded to bf16, dx [M][K] = d w (bf16), dw [V][K]
// (+)= d^T x (bf16 or fp32, row stride lddw), dbias [V] = column sums of d (bf16 or fp32).  dx, dw and dbias may be null.
// piece: a multiple of 256, or V.  kept, stats and target: what the forward pass kept, or null to compute the logits again.
MB_API int mb_xent_linear_bwd(const void* x, const void* w, const void* bias, const int64_t* labels, const float* lse,
                              const float* gloss, void* dx, void* dw, void* dbias, const void* kept, int ldk, const float* stats,
                              const float* target, int M, int V, int K, int ldx, int ldw, int lddw, int dw_fp32, int accumulate,
                              int dbias_fp32, int64_t v0, int64_t ignore, int piece, int max_ctas, void* workspace,
                              cudaStream_t stream) {
  if (!xent_args_ok(x, w, M, V, K, ldx, ldw) || M == 0 || piece <= 0) return -1;
  if (kept && (ldk < V || ldk % 8 || (reinterpret_cast<uintptr_t>(kept) & 15) || (M + 31) / 32 > 65535)) return -1;
  if (piece >= V) piece = V;
  else if (piece % 256) return -1;
  if ((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(workspace)) & 15) return -1;
  const int dw_flags = (dw_fp32 ? EPI_OUT_FP32 : 0) | (accumulate ? EPI_ACCUM : 0);
  const XentArea area = xent_area(M, V, K, piece, dx, dw, dbias, dw_flags, clamp_ctas(max_ctas));
  uint8_t* at = static_cast<uint8_t*>(workspace);
  void* dl = at;
  float* sums = dbias ? reinterpret_cast<float*>(at + area.dlogits) : nullptr;
  float* dx32 = reinterpret_cast<float*>(at + area.dlogits + area.col_sums);
  void* gemm_area = area.gemm ? at + area.dlogits + area.col_sums + area.dx32 : nullptr;
  auto gemm = [&](const void* a, const void* b, void* c, int m, int n, int k, int lda, int ldb, int ldc, int a_mn, int flags) {
    const int rc = max_ctas == 1 ? 1      // no pair
                                 : mb_gemm_pair_split_bf16(a, b, c, m, n, k, lda, ldb, ldc, a_mn, 1, flags, nullptr, nullptr,
                                                           1.f, max_ctas, gemm_area, stream);
    return rc != 1 ? rc : mb_gemm_bf16(a, b, c, m, n, k, lda, ldb, ldc, a_mn, 1, flags, nullptr, nullptr, 1.f, 0, max_ctas,
                                       stream);
  };
  for (int c0 = 0; c0 < V; c0 += piece) {
    const int n = V - c0 < piece ? V - c0 : piece, ldd = (n + 7) / 8 * 8;
    const __nv_bfloat16* wp = static_cast<const __nv_bfloat16*>(w) + static_cast<size_t>(c0) * ldw;
    XentParams p;
    memset(&p, 0, sizeof(p));
    p.M = M; p.N = n; p.K = K;
    p.bias = bias ? static_cast<const __nv_bfloat16*>(bias) + c0 : nullptr;
    p.flags = bias ? EPI_BIAS : 0;
    p.labels = labels;
    p.v0 = v0 + c0;
    p.ignore = ignore;
    p.lse = lse;
    p.gloss = gloss;
    p.segments = 1;
    p.col_sums = sums;
    int rc = 0;
    if (kept) {
      (sums ? xent_kept_grad_kernel<true> : xent_kept_grad_kernel<false>)<<<dim3((n + 511) / 512, (M + 31) / 32), 256, 0, stream>>>(
          static_cast<const uint16_t*>(kept), ldk, reinterpret_cast<const float2*>(stats), target, labels, lse, gloss,
          static_cast<__nv_bfloat16*>(dl), ldd, sums, M, c0, n, v0, ignore);
      if (cudaGetLastError() != cudaSuccess) rc = -4;
    } else {
      rc = xent_gemm(x, wp, dl, ldd, p, ldx, ldw, max_ctas, stream);
    }
    if (rc == 0 && dbias) {
      void* dst = static_cast<uint8_t*>(dbias) + static_cast<size_t>(c0) * (dbias_fp32 ? 4 : 2);
      xent_bias_grad_kernel<<<(n + 31) / 32, 256, 0, stream>>>(sums, dst, (M + 31) / 32, n, dbias_fp32);
      if (cudaGetLastError() != cudaSuccess) rc = -4;
    }
    if (rc == 0 && dx)
      rc = piece == V ? gemm(dl, wp, dx, M, K, n, ldd, ldw, K, 0, 0)
                      : gemm(dl, wp, dx32, M, K, n, ldd, ldw, K, 0, EPI_OUT_FP32 | (c0 ? EPI_ACCUM : 0));
    if (rc == 0 && dw)
      rc = gemm(dl, x, static_cast<uint8_t*>(dw) + static_cast<size_t>(c0) * lddw * (dw_fp32 ? 4 : 2), n, K, M, ldd, ldx, lddw,
                1, dw_flags);
    if (rc != 0) return rc;
  }
  return dx && piece < V ? mb_cast_f32_to_bf16(dx32, dx, static_cast<size_t>(M) * K, 1.f, stream) : 0;
}

MB_API int mb_gemm_pair_bf16(const void* A, const void* B, void* C, int M, int N, int K, int lda, int ldb, int ldc,
                             int a_mn_major, int b_mn_major, int flags, const void* bias, void* aux, float alpha,
                             int max_ctas, cudaStream_t stream) {
  return mb_gemm_pair_split_bf16(A, B, C, M, N, K, lda, ldb, ldc, a_mn_major, b_mn_major, flags, bias, aux, alpha,
                                 max_ctas, nullptr, stream);
}
