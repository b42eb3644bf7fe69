// Gated feed-forward block for sm_100a, forward and backward:
//   H = act(G) * U with G = X Wg^T, U = X Wu^T      (X [M,K], Wg, Wu [F,K])
//   dU = dH * act(G), dG = dH * U * act'(G)
//   dX = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X
// in bf16 with fp32 accumulation in TMEM.  One persistent, warp-specialised
// kernel (roles, ring, bounded waits and teardown as in gemm_sm100.cuh) with
// three kinds of tile, which differ in what feeds the two operands of an MMA
// and in what is done with the accumulator:
//   gated  A = X, B = Wg and Wu; a tile's accumulator holds a block of G next
//          to the same block of U, and the epilogue combines them, so neither
//          goes to memory unless the caller keeps it.
//   dX     one sum over the 2F products: first dG (A) with Wg (B), then dU
//          with Wu, so dX is written once.  Wg is [F,K] and F is summed over,
//          so B is read "MN-major": a TMA box is 64 columns (of the output) x
//          64 rows (of the sum).
//   dW     dWg's tile rows, then dWu's.  The sum runs over the M rows, so
//          dG/dU and X are both read MN-major.
// MN-major operands cost nothing over K-major ones: the same bytes per stage
// in the same 128-byte swizzle, two 8 KB boxes instead of one of 16 KB.  No
// transposed copy of anything is made.
//
// dX and dW run in one launch: dX's tiles are few and long (a sum over 2F),
// dW's many and short, so the clusters that get no dX tile, or one less, take
// dW tiles meanwhile (ffn_unit), where two launches would leave most SMs idle
// behind dX's last wave.
//
// Bound by the tensor cores where M is large: their pipe is active for 83% of
// the cycles forward (2048 x 14336 x 4096, 256-wide tiles) and 90% backward.
// Measured, 8192 x 14336 x 4096: forward with G and U kept 1.27 ms = 1.52
// PFLOP/s, gradients 2.55 ms = 1.51 PFLOP/s for a few calls after a pause; 1.49
// and 2.99 ms = 1.29 PFLOP/s in a loop of seconds, under the power cap.  Library
// products of the same operations, without the element-wise work: 1.24 and 2.49,
// 1.44 and 2.91 ms.  Smaller sizes lose to whole tiles and waves and to the first
// fetches and last epilogue, which nothing overlaps: 777 x 5120 x 2048 (a quarter
// of the tiles' rows are padding) takes 40 us, twice its operations' time.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>

#include "gemm_sm100.cuh"

namespace b200gemm {

enum FfnKind { kGated = 0, kGrads = 1 };

struct FfnOut {
  uint16_t* ptr;   // bf16 bits
  long long ld;    // row pitch in elements
};

// One set of equal tiles.
struct FfnSet {
  int M, N;          // rows and columns of one output matrix (gated: N = F)
  int num_kb;        // K blocks of a tile
  int tiles_m;       // tile rows (dW: of one of the two matrices)
  int tiles_n;       // tile columns
  int tiles;         // tiles in all (dW: of both matrices; dX: of every K range)
};

struct FfnParams {
  FfnSet first;      // gated, or dX
  FfnSet second;     // dW
  int seg_kb;        // dX: K blocks of the first product (num_kb = 2 seg_kb)
  // dX split over its sum, where it has too few tiles for the clusters: range
  // s of `split` covers K blocks [s slice_kb, ..) and writes fp32 partial sums
  // to partials[s][M][N] (dX_sum_kernel adds them); split = 1: none of that.
  int split, slice_kb;
  float* partials;
  int ahead;         // dW tiles that a cluster without a last dX tile takes meanwhile
  int band;          // tile rows per band of the tile order
  int act;           // kAct*
  int save;          // gated: G and U are written too
  FfnOut out[3];     // gated: H, G, U; gradients: dX, dWg, dWu
  unsigned int* status;
  unsigned long long timeout_ns;
};

// Tensor maps of a launch.
struct FfnMaps {
  CUtensorMap a0, a1;   // gated: X; dX: dG, dU (K-major)
  CUtensorMap b0, b1;   // gated: Wg, Wu (K-major); dX: Wg, Wu (MN-major)
  CUtensorMap w0, w1;   // dW: dG, dU (MN-major)
  CUtensorMap x;        // dW: X (MN-major)
  CUtensorMap c[3];     // the outputs
};

// NB = 2: 256 x 512 accumulators, a single one: two N = 256 MMAs per K step
//         share the A stage.  kGated: G's 256 columns, then U's (256
//         columns of H per tile); otherwise 512 columns of the output.
// NB = 1: 256 x 256 accumulators, two of them, so a tile's epilogue
//         overlaps the next tile's MMAs.  kGated: the N = 256 MMA takes its
//         first 128 B rows from the even CTA and the others from the odd one,
//         so the even CTA loads rows of Wg and the odd one the same rows of
//         Wu (128 columns of H per tile).  MN = 192 (gated only) and 128 are
//         the same with narrower MMAs, for sizes that 256 cuts into a mostly
//         idle last wave, or into fewer tiles than there are clusters.
template <int KIND, int NB, int STAGES, int MN = 256>
struct FfnCfg {
  static_assert(MN == 256 || (NB == 1 && (MN == 128 || (MN == 192 && KIND == kGated))), "MMA width");
  static constexpr int kKind = KIND;
  static constexpr int kNB = NB;
  static constexpr int kStages = STAGES;
  static constexpr int kMmaN = MN;
  static constexpr int kTileN = KIND == kGated ? MN / 2 * NB : MN * NB;  // output columns per tile
  static constexpr int kAccBufs = NB == 1 ? 2 : 1;
  static constexpr int kEpiWarps = 4 * NB;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kWarpCols = kTileN / NB;              // output columns one epilogue warp writes
  static constexpr int kWarpChunks = kWarpCols / kCBoxCols;
  static constexpr int kCBufs = NB == 2 ? 4 : 2;
  static constexpr int kBRows = MN / 2;                      // one CTA's half of one MMA's B rows
  static constexpr int kBlockBytesB = kBRows * kBlockK * 2;
  static constexpr int kStageBytesB = NB * kBlockBytesB;
  static constexpr uint32_t kTxBytes = 2 * (kStageBytesA + kStageBytesB);
  static constexpr int kA = 0;
  static constexpr int kB = kA + STAGES * kStageBytesA;
  static constexpr int kC = kB + STAGES * kStageBytesB;
  static constexpr int kFull = kC + kEpiWarps * kCBufs * kCStageBytes;
  static constexpr int kEmpty = kFull + 8 * STAGES;
  static constexpr int kTFull = kEmpty + 8 * STAGES;
  static constexpr int kTEmpty = kTFull + 8 * kAccBufs;
  static constexpr int kDrain = kTEmpty + 8 * kAccBufs;
  static constexpr int kTmemSlot = kDrain + 8;
  static constexpr int kAbort = kTmemSlot + 4;
  static constexpr int kEnd = kAbort + 4;
  static constexpr int kSmemBytes = kEnd + 1024;
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB per-CTA shared memory limit");
  static_assert(kSmemBytes > 116 * 1024, "one CTA per SM: two that want TMEM could wait for one another's");
};

// Matrix descriptor of an MN-major operand in the 128-byte swizzle: 64
// consecutive MN elements form a 128-byte row, 8 rows (of K) a 1024-byte
// atom; the next 8 K rows follow 1024 B on (stride offset) and the next 64
// MN elements one 64 x 64 box = 8192 B on (leading offset).  A K step of 16
// is two atoms, 2048 B.
constexpr uint64_t kSmemDescHiMn = (uint64_t(1024 >> 4) << 32) | (uint64_t(8192 >> 4) << 16) |
                                   (uint64_t(1) << 46) | (uint64_t(2) << 61);
template <bool MN>
__device__ __forceinline__ uint64_t ffn_desc(uint32_t addr) {
  return (MN ? kSmemDescHiMn : kSmemDescHi) | uint64_t((addr & 0x3FFFFu) >> 4);
}
// Descriptor units (16 B) from one K step of 16 to the next.
template <bool MN>
constexpr uint64_t kDescStep = MN ? 128 : 2;

// Instruction descriptor: kind::f16, D f32, A and B bf16, M = 256 (pair),
// N = MN; bits 15 and 16 say that A or B is MN-major.
template <int MN, bool A_MN, bool B_MN>
constexpr uint32_t kFfnIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u) |
                               (static_cast<uint32_t>(MN >> 3) << 17) | ((256u >> 4) << 24);

// Tile t of a set in the band order: bands of `band` tile rows, each swept
// column by column, so the band's A rows and one column of B stay in L2
// meanwhile.
__device__ __forceinline__ void ffn_tile(int band, int tiles_m, int tiles_n, int t, int& tm, int& tn) {
  const int per_band = band * tiles_n;
  const int b = t / per_band, r = t - b * per_band;
  const int rows = min(band, tiles_m - b * band);
  tn = r / rows;
  tm = b * band + (r - tn * rows);
}

// The i-th unit of cluster c of g: a tile of the first set (round robin), then
// of the second.  Where the first set's tiles do not divide evenly, the
// clusters that have one less take `ahead` tiles of the second set meanwhile,
// and the rest go round all clusters.  False past the last unit.
struct FfnUnit {
  bool second;   // of the second set: dW
  bool up;       // dW: a tile of dWu
  int slice;     // dX: its K range
  int tm, tn;
};
template <int KIND>
__device__ __forceinline__ bool ffn_unit(const FfnParams& p, int c, int g, int i, FfnUnit& u) {
  const int q = p.first.tiles / g, r = p.first.tiles - q * g;
  const int mine = q + (c < r ? 1 : 0);
  u.second = u.up = false;
  u.slice = 0;
  if (i < mine) {
    int t = i * g + c;
    if (KIND == kGrads && p.split > 1) {  // a range's tiles follow one another
      const int cells = p.first.tiles_m * p.first.tiles_n;
      u.slice = t / cells;
      t -= u.slice * cells;
    }
    ffn_tile(p.band, p.first.tiles_m, p.first.tiles_n, t, u.tm, u.tn);
    return true;
  }
  if constexpr (KIND == kGated) return false;
  const int k = i - mine, light = g - r;  // (r = 0: no cluster has more than another)
  const int ahead = r > 0 ? p.ahead : 0;
  int t;
  if (c >= r && k < ahead) t = k * light + (c - r);
  else t = ahead * light + (c >= r ? (k - ahead) * g + (c - r) : k * g + light + c);
  if (t >= p.second.tiles) return false;
  ffn_tile(p.band, 2 * p.second.tiles_m, p.second.tiles_n, t, u.tm, u.tn);
  u.second = true;
  u.up = u.tm >= p.second.tiles_m;
  if (u.up) u.tm -= p.second.tiles_m;
  return true;
}

// The normal distribution's integral Phi(x), and e = e^(-x^2/2).  By its tail,
// 1 - Phi(|x|) = e t P(t) with t = 1 / (1 + 0.33 |x|), so that it keeps its
// relative accuracy for x < 0 (as 1 + erf it would have lost all digits at
// x = -5.6, where x Phi(x) is -6e-8).  P: our own fit of degree 7 for the least
// maximal relative error over all x >= 0, 2^-19.6 with fp32's roundings.  The
// gated block 8192 x 14336 x 4096 (G and U kept) with erff, erfcf and this:
// 1.48, 1.59 and 1.46 ms; its gradients 2.96, 3.09 and 2.91 ms.
__device__ __forceinline__ float normal_cdf(float x, float& e) {
  const float t = ptx::rcp_approx(fmaf(0.33f, fabsf(x), 1.0f));
  float p = fmaf(0.033285525f, t, -0.10566421f);
  p = fmaf(p, t, 0.06743017f);
  p = fmaf(p, t, 0.033429552f);
  p = fmaf(p, t, 0.09100458f);
  p = fmaf(p, t, 0.11721682f);
  p = fmaf(p, t, 0.13164698f);
  p = fmaf(p, t, 0.13165107f);
  e = __expf(-0.5f * x * x);
  const float tail = p * t * e;
  return x < 0.0f ? tail : 1.0f - tail;
}

// act(x) for bf16 results: e^x and the reciprocal are the fast forms.  __expf(a)
// is off by up to 2 + 1.173 |a| steps of 2^-23 and what a's own roundings make
// of it, the reciprocal by one step: relative errors below 2^-16 for |a| up to
// 20 and below 2^-14 as far as e^a is finite, where bf16 rounds by 2^-8.  The
// tanh form of GELU goes through the logistic function, 0.5 (1 + tanh z) = 1 /
// (1 + e^-2z), which keeps its relative accuracy where tanh is near -1.  A NaN
// stays one under each of them.
template <int ACT>
__device__ __forceinline__ float ffn_act(float x) {
  if constexpr (ACT == kActRelu) return ptx::max_nan(x, 0.0f);
  if constexpr (ACT == kActGelu) {
    float e;
    return x * normal_cdf(x, e);
  }
  if constexpr (ACT == kActGeluTanh)
    return x * ptx::rcp_approx(1.0f + __expf(-1.5957691216057308f * fmaf(0.044715f * x, x * x, x)));
  if constexpr (ACT == kActSilu) return x * ptx::rcp_approx(1.0f + __expf(-x));
  return x;
}

// act(x) and its derivative:
//   silu       s = 1 / (1 + e^-x):     s (1 + x (1 - s))
//   gelu       Phi(x) + x phi(x)
//   gelu_tanh  s = 1 / (1 + e^-2z):    s + x s (1 - s) 2 z'
// x^2 is capped in 2 z' (it multiplies an exact zero there).
template <int ACT>
__device__ __forceinline__ void ffn_act_grad(float x, float& a, float& da) {
  if constexpr (ACT == kActRelu) {
    a = ptx::max_nan(x, 0.0f);
    da = x > 0.0f ? 1.0f : (x <= 0.0f ? 0.0f : x);
  } else if constexpr (ACT == kActGelu) {
    float e;
    const float phi = normal_cdf(x, e);
    a = x * phi;
    da = fmaf(x * 0.39894228040143268f, e, phi);
  } else if constexpr (ACT == kActGeluTanh) {
    const float x2 = x * x;
    const float s = ptx::rcp_approx(1.0f + __expf(-1.5957691216057308f * fmaf(0.044715f * x, x2, x)));
    a = x * s;
    da = fmaf(a * (1.0f - s), 1.5957691216057308f * fmaf(0.134145f, fminf(x2, 1e30f), 1.0f), s);
  } else if constexpr (ACT == kActSilu) {
    const float s = ptx::rcp_approx(1.0f + __expf(-x));
    a = x * s;
    da = fmaf(a, 1.0f - s, s);
  } else {
    a = x;
    da = 1.0f;
  }
}

// h = act(g) * u on one lane's 32 columns, rounded to bf16 pairs.  The
// activation is switched outside the straight loop.
template <int ACT>
__device__ __forceinline__ void ffn_combine32(const uint32_t (&g)[32], const uint32_t (&u)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float lo = ffn_act<ACT>(__uint_as_float(g[2 * i])) * __uint_as_float(u[2 * i]);
    const float hi = ffn_act<ACT>(__uint_as_float(g[2 * i + 1])) * __uint_as_float(u[2 * i + 1]);
    w[i] = ptx::pack_bf16x2(__float_as_uint(lo), __float_as_uint(hi));
  }
}
__device__ __forceinline__ void ffn_combine(int act, const uint32_t (&g)[32], const uint32_t (&u)[32],
                                            uint32_t (&w)[16]) {
  switch (act) {
    case kActRelu: ffn_combine32<kActRelu>(g, u, w); break;
    case kActGelu: ffn_combine32<kActGelu>(g, u, w); break;
    case kActGeluTanh: ffn_combine32<kActGeluTanh>(g, u, w); break;
    case kActSilu: ffn_combine32<kActSilu>(g, u, w); break;
    default: ffn_combine32<kActNone>(g, u, w); break;
  }
}

// One 32 x 32 chunk of a bf16 output (lane = row, w = 16 packed pairs): a
// swizzled staging buffer and a TMA store, or predicated element stores for
// the chunk that ends inside a 16-byte group (TMA clips in 16-byte units).
template <int BUFS>
__device__ __forceinline__ void ffn_store_chunk(const uint32_t (&w)[16], int col, int row, uint32_t lane,
                                                uint32_t cstage0, uint32_t& cbuf, const CUtensorMap& map,
                                                const FfnOut& o, int M, int N) {
  if (row >= M || col >= N) return;  // warp-uniform
  if ((N % 8) != 0 && col + kCBoxCols > N) {
    const int r = row + static_cast<int>(lane);
    if (r < M) {
      uint16_t* dst = o.ptr + static_cast<long long>(r) * o.ld + col;
      const int ncols = N - col;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (2 * i < ncols) dst[2 * i] = static_cast<uint16_t>(w[i] & 0xFFFFu);
        if (2 * i + 1 < ncols) dst[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
      }
    }
    return;
  }
  const uint32_t buf = cstage0 + cbuf * kCStageBytes;
  if (lane == 0) ptx::bulk_wait_group_read<BUFS - 1>();  // the store that last read this buffer is done
  __syncwarp();
  stage_chunk_row(buf, lane, w);
  ptx::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    ptx::tma_store_2d(&map, buf, col, row);
    ptx::bulk_commit_group();
  }
  if (++cbuf == BUFS) cbuf = 0;
}

// K blocks [first, end) of a unit.
template <int KIND>
__device__ __forceinline__ void ffn_range(const FfnParams& p, const FfnUnit& u, int& first, int& end) {
  first = 0;
  end = u.second ? p.second.num_kb : p.first.num_kb;
  if (KIND == kGrads && !u.second && p.split > 1) {
    first = u.slice * p.slice_kb;
    end = min(end, first + p.slice_kb);
  }
}

// The K blocks of one tile through the MMA: false when a wait ran out.
template <class Cfg, bool A_MN, bool B_MN>
__device__ __forceinline__ bool ffn_mma_tile(uint32_t sA, uint32_t sB, uint32_t full0, uint32_t own_empty0,
                                             uint32_t peer_empty0, uint32_t d_tmem, int num_kb, uint32_t& stage,
                                             uint32_t& phase, const ptx::Watchdog& wd, unsigned int unit) {
  for (int kb = 0; kb < num_kb; ++kb) {
    if (!ptx::mbar_wait(full0 + 8 * stage, phase, wd, kSiteMmaFull, unit)) return false;
    ptx::tc_fence_after();
    const uint64_t a_desc = ffn_desc<A_MN>(sA + stage * kStageBytesA);
    const uint64_t b_desc = ffn_desc<B_MN>(sB + stage * Cfg::kStageBytesB);
#pragma unroll
    for (int k = 0; k < kBlockK / kMmaK; ++k) {
#pragma unroll
      for (int h = 0; h < Cfg::kNB; ++h) {
        ptx::mma_bf16_cg2(d_tmem + h * 256u, a_desc + k * kDescStep<A_MN>,
                          b_desc + (h * Cfg::kBlockBytesB >> 4) + k * kDescStep<B_MN>, kFfnIdesc<Cfg::kMmaN, A_MN, B_MN>,
                          (kb > 0 || k > 0) ? 1u : 0u);
      }
    }
    ptx::mma_commit_cg2(own_empty0 + 8 * stage);
    ptx::mma_commit_cg2(peer_empty0 + 8 * stage);
    if (++stage == Cfg::kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  return true;
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1) __cluster_dims__(2, 1, 1)
    ffn_gemm_sm100(const __grid_constant__ FfnMaps maps, const FfnParams p) {
  constexpr int STAGES = Cfg::kStages;
  constexpr int NB = Cfg::kNB;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t rank = ptx::cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = static_cast<int>(ptx::cluster_id_x());
  const int nclusters = static_cast<int>(ptx::num_clusters_x());

  const uint32_t sA = base + Cfg::kA, sB = base + Cfg::kB, sC = base + Cfg::kC;
  const uint32_t full0 = base + Cfg::kFull, empty0 = base + Cfg::kEmpty;
  const uint32_t tfull0 = base + Cfg::kTFull, tempty0 = base + Cfg::kTEmpty;
  const uint32_t drain = base + Cfg::kDrain, tmem_slot = base + Cfg::kTmemSlot;

  ptx::Watchdog wd;
  wd.abort_flag = base + Cfg::kAbort;
  wd.peer_abort_flag = ptx::mapa(wd.abort_flag, rank ^ 1u);
  wd.status = p.status;
  wd.timeout_ns = p.timeout_ns;

  if (threadIdx.x == 0) {
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(wd.abort_flag) : "memory");
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full0 + 8 * s, 1);   // leader's expect_tx arrival (+ bytes of both CTAs)
      ptx::mbar_init(empty0 + 8 * s, 1);  // one MMA commit
    }
    for (int a = 0; a < Cfg::kAccBufs; ++a) {
      ptx::mbar_init(tfull0 + 8 * a, 1);                     // one MMA commit
      ptx::mbar_init(tempty0 + 8 * a, 2 * Cfg::kEpiWarps);   // every epilogue warp of the pair
    }
    ptx::mbar_init(drain, 1);
    ptx::fence_mbar_init_cluster();
    ptx::prefetch_tensormap(&maps.a0);
    ptx::prefetch_tensormap(&maps.b0);
    ptx::prefetch_tensormap(&maps.c[0]);
  }
  if (warp == 1) {
    ptx::tmem_alloc_cg2(tmem_slot, kTmemCols);
    ptx::tmem_relinquish_cg2();
  }
  ptx::tc_fence_before();
  ptx::cluster_sync_all();
  ptx::tc_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
  // The gradients are launched to overlap the kernel that makes dG and dU:
  // the set-up above runs during its tail, and nothing global is touched
  // before it is complete.
  ptx::griddep_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint64_t policy = ptx::policy_evict_last();
      const uint32_t full_leader0 = ptx::mapa(full0, 0);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      FfnUnit u;
      for (int i = 0; ok && ffn_unit<Cfg::kKind>(p, cluster, nclusters, i, u); ++i) {
        const int row_a = u.tm * kTileM + static_cast<int>(rank) * 128;
        const int row_b = u.tn * Cfg::kTileN + ((Cfg::kKind == kGated && NB == 1) ? 0 : static_cast<int>(rank) * Cfg::kBRows);
        int kb_first, kb_end;
        ffn_range<Cfg::kKind>(p, u, kb_first, kb_end);
        for (int kb = kb_first; kb < kb_end; ++kb) {
          if (!ptx::mbar_wait(empty0 + 8 * stage, phase ^ 1u, wd, kSiteProducer, static_cast<unsigned>(i))) {
            ok = false;
            break;
          }
          if (leader) ptx::mbar_arrive_expect_tx(full0 + 8 * stage, Cfg::kTxBytes);
          const uint32_t fb = full_leader0 + 8 * stage;
          const uint32_t da = sA + stage * kStageBytesA, db = sB + stage * Cfg::kStageBytesB;
          if constexpr (Cfg::kKind == kGated) {
            ptx::tma_load_2d_cg2(da, &maps.a0, fb, kb * kBlockK, row_a, policy);
#pragma unroll
            for (int h = 0; h < NB; ++h) {
              const bool up = NB == 2 ? h == 1 : rank == 1;
              ptx::tma_load_2d_cg2(db + h * Cfg::kBlockBytesB, up ? &maps.b1 : &maps.b0, fb, kb * kBlockK, row_b,
                                   policy);
            }
          } else {
            const bool seg1 = !u.second && kb >= p.seg_kb;
            const int k = (seg1 ? kb - p.seg_kb : kb) * kBlockK;
            if (u.second) {
              const CUtensorMap* ma = u.up ? &maps.w1 : &maps.w0;
              ptx::tma_load_2d_cg2(da, ma, fb, row_a, k, policy);
              ptx::tma_load_2d_cg2(da + 8192, ma, fb, row_a + 64, k, policy);
            } else {
              ptx::tma_load_2d_cg2(da, seg1 ? &maps.a1 : &maps.a0, fb, k, row_a, policy);
            }
            const CUtensorMap* mb = u.second ? &maps.x : (seg1 ? &maps.b1 : &maps.b0);
#pragma unroll
            for (int h = 0; h < NB; ++h) {
              const uint32_t d = db + h * Cfg::kBlockBytesB;
#pragma unroll
              for (int c = 0; c < Cfg::kBRows / 64; ++c)
                ptx::tma_load_2d_cg2(d + c * 8192, mb, fb, row_b + h * 256 + c * 64, k, policy);
            }
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    if (leader && lane == 0) {
      const uint32_t own_empty0 = ptx::mapa(empty0, 0), peer_empty0 = ptx::mapa(empty0, 1);
      const uint32_t own_tfull0 = ptx::mapa(tfull0, 0), peer_tfull0 = ptx::mapa(tfull0, 1);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      FfnUnit u;
      for (int i = 0; ffn_unit<Cfg::kKind>(p, cluster, nclusters, i, u); ++i) {
        const unsigned int unit = static_cast<unsigned int>(i);
        if (!ptx::mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1u, wd, kSiteMmaTmemEmpty, unit)) break;
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256u;
        bool ok;
        int kb_first, kb_end;
        ffn_range<Cfg::kKind>(p, u, kb_first, kb_end);
        const int num_kb = kb_end - kb_first;
        if constexpr (Cfg::kKind == kGated) {
          ok = ffn_mma_tile<Cfg, false, false>(sA, sB, full0, own_empty0, peer_empty0, d_tmem, num_kb, stage, phase,
                                               wd, unit);
        } else if (u.second) {
          ok = ffn_mma_tile<Cfg, true, true>(sA, sB, full0, own_empty0, peer_empty0, d_tmem, num_kb, stage, phase, wd,
                                             unit);
        } else {
          ok = ffn_mma_tile<Cfg, false, true>(sA, sB, full0, own_empty0, peer_empty0, d_tmem, num_kb, stage, phase, wd,
                                              unit);
        }
        if (!ok) break;
        ptx::mma_commit_cg2(own_tfull0 + 8 * acc);
        ptx::mma_commit_cg2(peer_tfull0 + 8 * acc);
        if (++acc == Cfg::kAccBufs) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      // Every MMA this thread issued must be complete before TMEM is freed
      // and before the peer CTA (whose shared memory the MMAs read) exits.
      ptx::mma_commit_cg2(ptx::mapa(drain, 0));
      ptx::Watchdog dwd = wd;
      dwd.timeout_ns = 100000000ull;
      ptx::mbar_wait_drain(drain, 0, dwd, kSiteDrain);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const uint32_t e = warp - 2u;
    const uint32_t quarter = warp & 3u;   // TMEM lanes this warp may access
    const uint32_t nblk = e >> 2;         // which kWarpCols output columns of the tile
    const uint32_t cstage0 = sC + e * Cfg::kCBufs * kCStageBytes;
    const uint32_t tempty_leader0 = ptx::mapa(tempty0, 0);
    uint32_t acc = 0, acc_phase = 0, cbuf = 0;
    FfnUnit u;
    for (int i = 0; ffn_unit<Cfg::kKind>(p, cluster, nclusters, i, u); ++i) {
      const int row = u.tm * kTileM + static_cast<int>(rank) * 128 + static_cast<int>(quarter) * 32;
      const int col0 = u.tn * Cfg::kTileN + static_cast<int>(nblk) * Cfg::kWarpCols;
      const bool full_ok = ptx::mbar_wait(tfull0 + 8 * acc, acc_phase, wd, kSiteEpilogue, static_cast<unsigned>(i));
      if (!__all_sync(0xFFFFFFFFu, full_ok)) break;
      ptx::tc_fence_after();
      const uint32_t t_row = tmem_base + ((quarter * 32u) << 16) + acc * 256u + nblk * Cfg::kWarpCols;
      auto release = [&]() {  // this warp's TMEM reads are done
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(tempty_leader0 + 8 * acc);
      };
      if constexpr (Cfg::kKind == kGated) {
        const int M = p.first.M, N = p.first.N;
        constexpr uint32_t kUp = Cfg::kMmaN / 2 * NB;  // U's columns follow G's
#pragma unroll 1
        for (int c = 0; c < Cfg::kWarpChunks; ++c) {
          uint32_t g[32], v[32], w[16];
          ptx::tmem_ld_32x32b_x32(t_row + c * kCBoxCols, g);
          ptx::tmem_ld_32x32b_x32(t_row + kUp + c * kCBoxCols, v);
          ptx::tmem_wait_ld();
          ptx::reg_fence32(g);
          ptx::reg_fence32(v);
          if (c == Cfg::kWarpChunks - 1) release();
          const int col = col0 + c * kCBoxCols;
          ffn_combine(p.act, g, v, w);
          ffn_store_chunk<Cfg::kCBufs>(w, col, row, lane, cstage0, cbuf, maps.c[0], p.out[0], M, N);
          if (p.save) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = ptx::pack_bf16x2(g[2 * j], g[2 * j + 1]);
            ffn_store_chunk<Cfg::kCBufs>(w, col, row, lane, cstage0, cbuf, maps.c[1], p.out[1], M, N);
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = ptx::pack_bf16x2(v[2 * j], v[2 * j + 1]);
            ffn_store_chunk<Cfg::kCBufs>(w, col, row, lane, cstage0, cbuf, maps.c[2], p.out[2], M, N);
          }
        }
      } else {
        const int which = u.second ? (u.up ? 2 : 1) : 0;
        const int M = u.second ? p.second.M : p.first.M, N = p.first.N;  // (N is K for all three)
        const CUtensorMap* map = &maps.c[which];
        constexpr int kHeld = Cfg::kWarpChunks - Cfg::kCBufs;
        if (!u.second && p.split > 1) {
          // fp32 partial sums of this K range, straight from the registers (a
          // lane's row, 16 bytes at a time; N % 8 == 0).
          const int r = row + static_cast<int>(lane);
          float* dst = p.partials + (static_cast<long long>(u.slice) * M + r) * N;
#pragma unroll 1
          for (int c = 0; c < Cfg::kWarpChunks; ++c) {
            uint32_t v[32];
            ptx::tmem_ld_32x32b_x32(t_row + c * kCBoxCols, v);
            ptx::tmem_wait_ld();
            ptx::reg_fence32(v);
            if (c == Cfg::kWarpChunks - 1) release();
            const int col = col0 + c * kCBoxCols;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              if (r < M && col + j < N) ptx::st_global_v4(dst + col + j, v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        } else if (NB == 2 && row < M && col0 + Cfg::kWarpCols <= N) {
          // The single accumulator holds the next tile's MMAs up until it is
          // read: half of a warp's chunks go into its staging buffers and half
          // into registers, then it is released, then the stores are issued.
          if (lane == 0) ptx::bulk_wait_group_read<0>();
          __syncwarp();
          uint32_t held[kHeld > 0 ? kHeld : 1][16];
#pragma unroll
          for (int c = 0; c < Cfg::kWarpChunks; c += 2) {
            uint32_t v0[32], v1[32];
            ptx::tmem_ld_32x32b_x32(t_row + c * kCBoxCols, v0);
            ptx::tmem_ld_32x32b_x32(t_row + (c + 1) * kCBoxCols, v1);
            ptx::tmem_wait_ld();
            ptx::reg_fence32(v0);
            ptx::reg_fence32(v1);
            if (c < Cfg::kCBufs) {
              stage_chunk_row_f32(cstage0 + c * kCStageBytes, lane, v0);
              stage_chunk_row_f32(cstage0 + (c + 1) * kCStageBytes, lane, v1);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                held[c - Cfg::kCBufs][j] = ptx::pack_bf16x2(v0[2 * j], v0[2 * j + 1]);
                held[c + 1 - Cfg::kCBufs][j] = ptx::pack_bf16x2(v1[2 * j], v1[2 * j + 1]);
              }
            }
          }
          release();
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
#pragma unroll
            for (int c = 0; c < Cfg::kCBufs; ++c) {
              ptx::tma_store_2d(map, cstage0 + c * kCStageBytes, col0 + c * kCBoxCols, row);
              ptx::bulk_commit_group();
            }
          }
          cbuf = 0;
#pragma unroll
          for (int c = 0; c < kHeld; ++c)
            ffn_store_chunk<Cfg::kCBufs>(held[c], col0 + (Cfg::kCBufs + c) * kCBoxCols, row, lane, cstage0, cbuf, *map,
                                         p.out[which], M, N);
        } else {
#pragma unroll 1
          for (int c = 0; c < Cfg::kWarpChunks; ++c) {
            uint32_t v[32], w[16];
            ptx::tmem_ld_32x32b_x32(t_row + c * kCBoxCols, v);
            ptx::tmem_wait_ld();
            ptx::reg_fence32(v);
            if (c == Cfg::kWarpChunks - 1) release();
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = ptx::pack_bf16x2(v[2 * j], v[2 * j + 1]);
            ffn_store_chunk<Cfg::kCBufs>(w, col0 + c * kCBoxCols, row, lane, cstage0, cbuf, *map, p.out[which], M, N);
          }
        }
      }
      if (++acc == Cfg::kAccBufs) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (lane == 0) ptx::bulk_wait_group_read<0>();  // staging reusable; the stores land before the kernel completes
    __syncwarp();
  }

  // --------------------------------------------------------------- teardown
  if (threadIdx.x == 0 && ptx::aborted(wd)) ptx::sleep_ns_bounded(200000ull);
  ptx::tc_fence_before();
  ptx::cluster_sync_all();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc_cg2(tmem_base, kTmemCols);
}

// dG and dU from dH, G and U, element by element: 6 bytes read and 4 written
// per element, so DRAM-bound (2048 x 14336: 43 us, in which 241 MB reach DRAM,
// 5.7 TB/s; 52 MB of the results are still in L2, where the products read them);
// a thread takes 8 columns (16 bytes of each).
// They are rounded to bf16 once, to be operands of the tensor cores.  Rows of
// the results are ldo elements (F rounded up to 8) and their padding columns
// are set to 0: the products below sum over them.
struct GatedGradParams {
  int M, F;
  const uint16_t *dh, *g, *u;
  long long lddh, ldgu;
  uint16_t *dg, *du;
  long long ldo;
};

template <int ACT>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GatedGradParams p) {
  ptx::griddep_launch_dependents();  // the products' kernel may set itself up; it waits for this one's end
  const int col = static_cast<int>(blockIdx.x * 256u + threadIdx.x) * 8;
  if (col >= p.F) return;
  for (long long r = blockIdx.y; r < p.M; r += gridDim.y) {
    uint32_t h[4], g[4], u[4], dg[4], du[4];
    load_bf16x8(p.dh + r * p.lddh, col, p.F, h);
    load_bf16x8(p.g + r * p.ldgu, col, p.F, g);
    load_bf16x8(p.u + r * p.ldgu, col, p.F, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a0, a1, d0, d1;
      ffn_act_grad<ACT>(bf16_lo(g[i]), a0, d0);
      ffn_act_grad<ACT>(bf16_hi(g[i]), a1, d1);
      const float h0 = bf16_lo(h[i]), h1 = bf16_hi(h[i]);
      du[i] = ptx::pack_bf16x2(__float_as_uint(h0 * a0), __float_as_uint(h1 * a1));
      dg[i] = ptx::pack_bf16x2(__float_as_uint(h0 * bf16_lo(u[i]) * d0), __float_as_uint(h1 * bf16_hi(u[i]) * d1));
    }
    // (columns past F were read as 0, so their products are 0 too)
    ptx::st_global_v4(p.dg + r * p.ldo + col, dg[0], dg[1], dg[2], dg[3]);
    ptx::st_global_v4(p.du + r * p.ldo + col, du[0], du[1], du[2], du[3]);
  }
}

// dX from its K ranges' partial sums, added in range order and rounded once;
// a thread takes 8 columns.  500 x 1000 from 4 ranges: 7 us by itself, mostly
// its launch and first loads; it starts when the products have ended.
__global__ void __launch_bounds__(256) dx_sum_kernel(const float* partials, int split, int M, int N, uint16_t* dx,
                                                     long long ld) {
  const int groups = N / 8;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long r = i / groups;
  if (r >= M) return;
  const int col = static_cast<int>(i - r * groups) * 8;
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
  for (int s = 0; s < split; ++s) {
    const auto* src = reinterpret_cast<const float4*>(partials + (s * static_cast<long long>(M) + r) * N + col);
    const float4 x = src[0], y = src[1];
    a.x += x.x;
    a.y += x.y;
    a.z += x.z;
    a.w += x.w;
    b.x += y.x;
    b.y += y.y;
    b.z += y.z;
    b.w += y.w;
  }
  auto pack = [](float lo, float hi) { return ptx::pack_bf16x2(__float_as_uint(lo), __float_as_uint(hi)); };
  ptx::st_global_v4(dx + r * ld + col, pack(a.x, a.y), pack(a.z, a.w), pack(b.x, b.y), pack(b.z, b.w));
}

}  // namespace b200gemm
