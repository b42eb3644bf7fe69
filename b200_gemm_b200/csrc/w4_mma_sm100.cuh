// Products with 4-bit weights (see w4_sm100.cuh for the format) for more than
// 16 rows of activations (run_w4 says when for fewer), on the 5th-generation
// tensor cores:
//   Y = X W^T,   H = act(X Wg^T) * (X Wu^T)
// 32 rows of X per CTA, or 64 from 33 on (blocks of 64 rows beyond that).
//
// With mma.sync every 8 rows of X cost as many instructions again as the
// weights' expansion; here they cost the issuing threads nothing.  128 rows of
// W are the M side of tcgen05.mma, the rows of X its N side.  A is read from
// TMEM: a thread of the expansion warps takes the codes of one row of W,
// expands them to bf16 and stores them to its TMEM lane (128 k's are 64
// columns), so that shared memory carries the codes and X alone.  With A in
// shared memory, whose writes and reads share one pipe, 192 rows of 128 k's
// took 1700 cycles; now 1000, where the codes alone take 530 to arrive.  The
// sum of a group (of 128 k's at most) is left in TMEM, from where the epilogue
// warps, whose lanes are rows of W, multiply it by the group's scale in fp32
// and add it to the row's sums in registers.  No weight is rounded.
//
// What bounds it is not taken apart.  Of 28672 x 8192, 32 rows, the tensor pipe
// is active 21% of the time, the issue slots 58%, DRAM 31%.  By w4_mma_plan's fit
// a step of 128 x 32 x 16 takes some 60 cycles with all that goes with it, a
// quarter of the rate of wide MMAs; what sets that pace (A from TMEM, sums that
// wait for one another, the hand-overs between warps) was not timed alone.
// 28416 x 4096, groups of 128, 32 rows: 26 us (mma.sync: 37), 58 MB of
// weights at 2.3 TB/s; 8192 x 8192: 18 us (25); gated 14336 x 4096: 24 us (53).
// 64 rows in one CTA take 32, 21 and 29 us (in two CTAs of 32: 51, 27 and 45):
// the MMAs take little more, the epilogue twice as long.  Its 64 sums a thread
// do not fit the 96 registers that all warps share: 48 to 108 bytes are spilled
// with two blocks of rows, but for the gated block in groups of 128 and more.
//
// Warps: 0 .. 4H-1   epilogue: block w / 4 of 128 rows, TMEM lanes 32 (w % 4) ..
//        16 or 8     expansion, two groups of eight for the steps in turn, or
//                    one: TMEM lanes 32 (w % 4) .., one half of a step's k's
//        2 or 3      TMA producer; MMA issue, the first also TMEM allocation
// H = 2 blocks of rows per CTA: Wg's and Wu's, or 256 rows of W; H = 1: 128
// rows of W.  Rows are divided evenly over the SMs and K over the CTAs of a
// cluster as in w4_nt_sm100; rows past a CTA's share are not expanded (what
// their lanes of TMEM hold gives sums that nobody reads).
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>

#include "gated_decode_sm100.cuh"
#include "gemm_sm100.cuh"
#include "w4_sm100.cuh"

namespace b200gemm {

// SG: groups per 128 k's (1 for groups of 128 and 256).
template <bool GATED, int H, int SG, int TOK>
struct W4MmaCfg {
  static_assert(TOK == 32 || TOK == 64, "rows of X");
  static_assert(H == 1 || H == 2, "blocks of 128 rows");
  static_assert(!GATED || H == 2, "Wg and Wu");
  static_assert(SG == 1 || SG == 2 || SG == 4, "groups of 128 or more, 64, 32");
  static constexpr bool kGatedOut = GATED;
  static constexpr int kH = H;
  static constexpr int kSG = SG;
  static constexpr int kTok = TOK;
  static constexpr int kStageK = 256;                  // k's of a stage of the ring
  static constexpr int kStepK = 128;                   // k's expanded and multiplied at a time: half a stage
  static constexpr int kEpiWarps = 4 * H;
  // Two groups of expansion warps take the steps in turn.  In groups of 32 the
  // epilogue is what lasts, and one group leaves it the registers to fetch its
  // next sums ahead (gated 14331 x 4096, 32 rows: 35.7 -> 31.8 us).
  static constexpr int kExpGroups = SG == 4 || TOK == 64 ? 1 : 2;
  static constexpr int kExpWarps = 8;                  // of each group
  // Two sets of accumulators, for the even and the odd steps, each of two
  // groups at most (one with 64 rows of X) and filled again for the others.
  static constexpr int kSetsPerStep = TOK == 64 ? SG : (SG == 4 ? 2 : 1);
  // Warps that issue MMAs.  One block's eight MMAs of a step take less than a
  // warp's waits and commits around them, and sets that are filled again wait more often: there
  // two warps take the steps in turn (4096 x 14336, 32 rows: 17.2 -> 15.8
  // us).  With two blocks one warp is better, as the earlier step's MMAs all
  // come first (28416 x 4096: 27.2 -> 25.8 us).
  static constexpr int kMmaWarps = H == 1 || kSetsPerStep > 1 ? 2 : 1;
  static constexpr int kThreads = 32 * (kEpiWarps + kExpGroups * kExpWarps + 1 + kMmaWarps);
  static constexpr int kCodes = 128 * 128;             // one block's codes of a stage: 128 bytes a row
  static constexpr int kStageX = 4 * kTok * 128;       // four boxes of 64 k's
  static constexpr int kStageBytes = H * kCodes + kStageX;
  static constexpr int kBlockA = kStepK / 2;           // TMEM columns of one block's operand
  static constexpr int kBufA = H * kBlockA;
  static constexpr int kBufs = H == 1 ? 4 : 2;         // operand buffers
  static constexpr int kSetGroups = SG / kSetsPerStep;
  static constexpr int kTmemSet = H * kSetGroups * kTok;
  static constexpr int kTmemAcc = kBufs * kBufA;       // the accumulators' first column
  static constexpr int kTmemUsed = kTmemAcc + 2 * kTmemSet;
  static constexpr int kTmemCols = 512;
  static_assert(kTmemUsed <= kTmemCols && kTmemUsed > 256, "TMEM columns");
  static constexpr int kBars = 256;
  static constexpr int kRing = 192 * 1024 / kStageBytes;
  static constexpr int kRingAt = 0;                    // X's boxes first in a stage: 1024-byte aligned
  static constexpr int kBarsAt = kRingAt + kRing * kStageBytes;
  static constexpr int kSmemBytes = 1024 + kBarsAt + kBars;
  static_assert((2 * kRing + 2 * kBufs + 4 + 1) * 8 + 8 <= kBars, "barriers");
  // All of an SM's TMEM for a CTA is safe as long as no other CTA that wants
  // some fits next to it: clusters of two kernels could otherwise each hold
  // what the other's last CTA waits for.
  static_assert(kSmemBytes > 190 * 1024 && kSmemBytes <= 232448, "one CTA per SM");
  // The rows' sums [kTok][kPitch], in the ring once the MMAs are done.
  static constexpr int kPitch = H * 128;
  static_assert(kTok * kPitch * 4 <= kRing * kStageBytes, "sums alias the ring");
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((static_cast<uint32_t>(kTok) >> 3) << 17) |
                                     ((128u >> 4) << 24);
};

// Eight codes (k in order, the lowest in the lowest four bits) to four bf16
// pairs of (q - 8) / 64, as in w4_sm100.cuh but adjacent k's to a pair.  The
// codes at even k are masked out in place, and those at odd k, 16 q; a byte
// permutation puts adjacent bytes into 16-bit halves.  Six bit operations and
// four multiply-adds.
struct W4PairConst {
  uint32_t even, odd, scale, offset;
};
__device__ __forceinline__ W4PairConst w4_pair_const() {
  W4PairConst c;
  asm volatile("mov.u32 %0, 0x0F0F0F0F;\n\tmov.u32 %1, 0xF0F0F0F0;\n\tmov.u32 %2, 0x7D007F00;\n\tmov.u32 %3, 0xBE00BE00;"
               : "=r"(c.even), "=r"(c.odd), "=r"(c.scale), "=r"(c.offset));
  return c;
}
__device__ __forceinline__ void w4_expand_pairs(uint32_t w, const W4PairConst& c, uint32_t* v) {
  const uint32_t e = w & c.even, o = w & c.odd;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // bytes: e_i, its sign (0), o_i, the sign of e_i
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(e), "r"(o), "r"(0x8480u + i * 0x1111u));
    v[i] = fma_bf16x2(d, c.scale, c.offset);
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1)
    w4_mma_sm100(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                 const __grid_constant__ CUtensorMap map_x, const W4NtParams p) {
  constexpr int H = Cfg::kH, SG = Cfg::kSG, RING = Cfg::kRing, BUFS = Cfg::kBufs, TOK = Cfg::kTok;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + Cfg::kBarsAt;
  const uint32_t full0 = bars, empty0 = full0 + 8 * RING;               // ring: codes and X
  const uint32_t afull0 = empty0 + 8 * RING, aempty0 = afull0 + 8 * BUFS;  // expanded operands
  const uint32_t tfull0 = aempty0 + 8 * BUFS, tempty0 = tfull0 + 16;       // accumulators
  const uint32_t drain = tempty0 + 16, tmem_slot = drain + 8;
  // (the shuffle tells the compiler that a warp has one value)
  const uint32_t warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
  constexpr uint32_t kProducer = Cfg::kEpiWarps + Cfg::kExpGroups * Cfg::kExpWarps, kMma = kProducer + 1;
  const int split = static_cast<int>(gridDim.x);   // CTAs of this cluster: K ranges
  const int rank = static_cast<int>(blockIdx.x);
  const int n0 = static_cast<int>(blockIdx.y) * p.rows;
  const int m0 = static_cast<int>(blockIdx.z) * TOK;
  const int s_begin = rank * p.stages_per_cta;
  const int count = max(0, min(p.num_stages, s_begin + p.stages_per_cta) - s_begin);
  const int cols = min(p.rows, p.N - n0);          // output columns of this CTA

  ptx::Watchdog wd;
  wd.abort_flag = tmem_slot + 4;
  wd.peer_abort_flag = ptx::mapa(wd.abort_flag, split > 1 ? static_cast<uint32_t>(rank ^ 1) : 0u);
  wd.status = p.status;
  wd.timeout_ns = p.timeout_ns;

  if (warp == kProducer && lane == 0) {
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(wd.abort_flag) : "memory");
    for (int s = 0; s < RING; ++s) {
      ptx::mbar_init(full0 + 8 * s, 1);
      ptx::mbar_init(empty0 + 8 * s, Cfg::kExpGroups * Cfg::kExpWarps + 2);  // the codes are expanded, the MMAs have read X
    }
    for (int b = 0; b < BUFS; ++b) {
      ptx::mbar_init(afull0 + 8 * b, Cfg::kExpWarps);
      ptx::mbar_init(aempty0 + 8 * b, 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(tfull0 + 8 * b, 1);
      ptx::mbar_init(tempty0 + 8 * b, Cfg::kEpiWarps);
    }
    ptx::mbar_init(drain, Cfg::kMmaWarps);
    ptx::fence_mbar_init_cluster();
    ptx::fence_proxy_async_smem();
  }
  if (warp == kMma) {
    ptx::tmem_alloc_cg1(tmem_slot, Cfg::kTmemCols);
    ptx::tmem_relinquish_cg1();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
  tmem_base = __shfl_sync(0xFFFFFFFFu, tmem_base, 0);

  float acc[TOK];  // epilogue warps: sums of this lane's row of W
#pragma unroll
  for (int t = 0; t < TOK; ++t) acc[t] = 0.0f;

  if (warp == kProducer) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint64_t policy_w = ptx::policy_evict_first();  // read once (per block of rows of X)
      const uint64_t policy_x = ptx::policy_evict_last();   // read by every CTA
      auto load_w = [&](int it, int s) {
        const uint32_t bar = full0 + 8 * s, dst = base + Cfg::kRingAt + s * Cfg::kStageBytes + Cfg::kStageX;
        ptx::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
        const int x = (s_begin + it) * 128;  // bytes: two codes each
        ptx::tma_load_2d(dst, &map_w0, bar, x, n0, policy_w);
        if (H == 2) ptx::tma_load_2d(dst + Cfg::kCodes, &map_w1, bar, x, Cfg::kGatedOut ? n0 : n0 + 128, policy_w);
      };
      auto load_x = [&](int it, int s) {
        const uint32_t dst = base + Cfg::kRingAt + s * Cfg::kStageBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ptx::tma_load_2d(dst + i * (TOK * 128), &map_x, full0 + 8 * s, (s_begin + it) * Cfg::kStageK + 64 * i, m0, policy_x);
      };
      const int pre = min(RING, count);
      if (p.pdl == kPdlWeightsEarly) {
        for (int it = 0; it < pre; ++it) load_w(it, it);
        ptx::griddep_wait();
        for (int it = 0; it < pre; ++it) load_x(it, it);
      } else {
        ptx::griddep_wait();
        for (int it = 0; it < pre; ++it) {
          load_w(it, it);
          load_x(it, it);
        }
      }
      int stage = 0;
      uint32_t phase = 1;  // after a whole ring
      for (int it = pre; it < count; ++it) {
        if (!ptx::mbar_wait_cta(empty0 + 8 * stage, phase ^ 1u, wd, kSiteProducer, blockIdx.y)) break;
        load_w(it, stage);
        load_x(it, stage);
        if (++stage == RING) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp >= kMma) {
    // ----------------------------------------------------------------- MMA
    // The whole warp runs the loop and elects a lane around the MMAs, which
    // keeps their operands in uniform registers: issued from a branch of one
    // lane, every MMA took some 60 cycles to issue, four times its work.
    const bool leader = ptx::elect_one();
    bool go = true;
    for (int it = static_cast<int>(warp - kMma); it < 2 * count && go; it += Cfg::kMmaWarps) {
      const int stage = (it >> 1) % RING, buf = it % BUFS, odd = it & 1;
      const uint32_t phase = static_cast<uint32_t>((it >> 1) / RING) & 1u, bphase = static_cast<uint32_t>(it / BUFS) & 1u;
      go = ptx::mbar_wait_cta(full0 + 8 * stage, phase, wd, kSiteMmaFull, blockIdx.y) &&
           ptx::mbar_wait_cta(afull0 + 8 * buf, bphase, wd, kSiteMmaFull, blockIdx.y);
      if (!__all_sync(0xFFFFFFFFu, go)) break;
      const uint32_t xs = base + Cfg::kRingAt + stage * Cfg::kStageBytes + odd * (2 * TOK * 128);
      constexpr int SETS = Cfg::kSetsPerStep, STEPS = 8 / SETS;  // steps of 16 k's per set
#pragma unroll
      for (int j = 0; j < SETS; ++j) {
        const uint32_t sphase = static_cast<uint32_t>((it >> 1) * SETS + j) & 1u;  // fillings of this set before
        go = ptx::mbar_wait_cta(tempty0 + 8 * odd, sphase ^ 1u, wd, kSiteMmaTmemEmpty, blockIdx.y);
        go = __all_sync(0xFFFFFFFFu, go);
        if (!go) break;
        ptx::tc_fence_after();
        if (leader) {
          // One group's MMAs wait for one another: the blocks' and the groups' in turn.
          const uint32_t a = tmem_base + buf * Cfg::kBufA;
          const uint32_t d = tmem_base + Cfg::kTmemAcc + odd * Cfg::kTmemSet;
          constexpr int GROUPS = Cfg::kSetGroups, PER = STEPS / GROUPS;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
              const int kk = j * STEPS + g * PER + i;
              const uint64_t b_desc = smem_desc(xs + (kk >> 2) * (TOK * 128)) + 2 * (kk & 3);
#pragma unroll
              for (int h = 0; h < H; ++h)
                ptx::mma_bf16_cg1_ta(d + (h * GROUPS + g) * TOK, a + h * Cfg::kBlockA + kk * 8, b_desc, Cfg::kIdesc,
                                     i > 0 ? 1u : 0u);
            }
          }
          ptx::mma_commit_cg1(tfull0 + 8 * odd);
          if (j == SETS - 1) {
            ptx::mma_commit_cg1(aempty0 + 8 * buf);
            ptx::mma_commit_cg1(empty0 + 8 * stage);
          }
        }
        __syncwarp();
      }
    }
    // Every MMA issued here must be complete before TMEM is freed.
    if (leader) {
      ptx::mma_commit_cg1(drain);
      ptx::Watchdog dwd = wd;
      dwd.timeout_ns = 100000000ull;
      ptx::mbar_wait_drain(drain, 0, dwd, kSiteDrain);
    }
    __syncwarp();
  } else if (warp >= Cfg::kEpiWarps) {
    // ----------------------------------------------------------- expansion
    // Of two groups of warps each takes one half of every stage.  A lane's row
    // of codes is eight 16-byte chunks, stored by the TMA at chunk c ^ (row % 8):
    // eight rows' chunks are then in different banks.
    const uint32_t quarter = warp & 3u, half = ((warp - Cfg::kEpiWarps) >> 2) & 1u;
    const uint32_t group = (warp - Cfg::kEpiWarps) / Cfg::kExpWarps;
    const uint32_t row = quarter * 32u + lane;
    const W4PairConst c = w4_pair_const();
    // Rows of each block that this CTA needs: whole quarters are left out.
    const int rows0 = Cfg::kGatedOut ? cols : min(cols, 128), rows1 = Cfg::kGatedOut ? cols : max(cols - 128, 0);
    const bool need[2] = {static_cast<int>(quarter * 32u) < rows0, H == 2 && static_cast<int>(quarter * 32u) < rows1};
    const uint32_t chunk0 = row * 128u + (((2u * half) ^ (row & 7u)) << 4);
    for (int it = static_cast<int>(group); it < 2 * count; it += Cfg::kExpGroups) {
      const int stage = (it >> 1) % RING, buf = it % BUFS;
      const uint32_t phase = static_cast<uint32_t>((it >> 1) / RING) & 1u, bphase = static_cast<uint32_t>(it / BUFS) & 1u;
      const bool got = ptx::mbar_wait_cta(full0 + 8 * stage, phase, wd, kSiteEpilogue, blockIdx.y) &&
                       ptx::mbar_wait_cta(aempty0 + 8 * buf, bphase ^ 1u, wd, kSiteEpilogue, blockIdx.y);
      if (!__all_sync(0xFFFFFFFFu, got)) break;
      ptx::tc_fence_after();
      const uint32_t codes = base + Cfg::kRingAt + stage * Cfg::kStageBytes + Cfg::kStageX + (chunk0 ^ ((it & 1u) << 6));
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if (!need[h]) continue;
        uint32_t q[8], v[32];
        ptx::ld_shared_v4(codes + h * Cfg::kCodes, q[0], q[1], q[2], q[3]);
        ptx::ld_shared_v4((codes + h * Cfg::kCodes) ^ 16u, q[4], q[5], q[6], q[7]);
#pragma unroll
        for (int i = 0; i < 8; ++i) w4_expand_pairs(q[i], c, v + 4 * i);
        ptx::tmem_st_32x32b_x32(tmem_base + ((quarter * 32u) << 16) + buf * Cfg::kBufA + h * Cfg::kBlockA + half * 32u, v);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive_cta(afull0 + 8 * buf);
        if (Cfg::kExpGroups == 2 || (it & 1)) ptx::mbar_arrive_cta(empty0 + 8 * stage);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const uint32_t h = warp >> 2, quarter = warp & 3u;
    const int n = n0 + (Cfg::kGatedOut ? 0 : static_cast<int>(h) * 128) + static_cast<int>(quarter * 32u + lane);
    const uint16_t* scales = ((Cfg::kGatedOut && h == 1) ? p.scales1 : p.scales0) + min(n, p.N - 1);
    // Scales are loaded two steps ahead, from lines brought into L2 some
    // sixteen steps ahead, four steps' at a time.  Past K the last group's
    // stands in (X is 0 there, and a NaN among the last makes the row NaN anyway).
    uint32_t sc_even[SG] = {}, sc_odd[SG] = {};
    const int shift = p.group_shift;
    const int last = (min(p.K, (s_begin + count) * Cfg::kStageK) - 1) >> shift;
    const int to_end = min(n + ((lane & 1u) ? 31 : 0) - static_cast<int>(lane), p.N - 1) - min(n, p.N - 1);
    const uint32_t pitch = static_cast<uint32_t>(p.N);
    auto scale_at = [&](int it, int sg) {  // of group sg of step `it`
      const int k = s_begin * Cfg::kStageK + it * Cfg::kStepK + sg * (Cfg::kStepK / SG);
      return scales + static_cast<uint64_t>(static_cast<uint32_t>(min(k >> shift, last))) * pitch;
    };
    auto load_scales = [&](int it, uint32_t (&d)[SG]) {
#pragma unroll
      for (int sg = 0; sg < SG; ++sg) d[sg] = __ldg(scale_at(it, sg));
    };
    auto prefetch_scales = [&](int it) {  // steps it .. it + 3
      // two lanes a group: the first and the last of the warp's rows
      if (lane < 8 * SG) {
        const int g = static_cast<int>(lane) / 2;
        ptx::prefetch_l2(scale_at(it + g / SG, g % SG) + to_end);
      }
    };
    if (p.pdl != kPdlWeightsEarly) ptx::griddep_wait();
    if (count > 0) {
      load_scales(0, sc_even);
      load_scales(1, sc_odd);
    }
    for (int it = 2; it < min(2 * count, 16); it += 4) prefetch_scales(it);
    const uint32_t t_row = tmem_base + ((quarter * 32u) << 16) + Cfg::kTmemAcc + h * Cfg::kSetGroups * TOK;
    uint32_t sphase = 0;
    // One filling of a set; after a step's last one its registers of scales
    // take those of the step after next (without a copy between, which would
    // wait for the load).
    auto add_set = [&](int it, int j, uint32_t (&sc)[SG]) {
      const uint32_t set = static_cast<uint32_t>(it) & 1u;
      const bool got = ptx::mbar_wait_cta(tfull0 + 8 * set, sphase, wd, kSiteEpilogue, blockIdx.y);
      if (!__all_sync(0xFFFFFFFFu, got)) return false;
      ptx::tc_fence_after();
      // Chunks of 16 columns; with a register set to spare the next one is on
      // its way while this one is added.
      constexpr int CHUNKS = Cfg::kSetGroups * TOK / 16, AHEAD = SG == 4 && TOK == 32 ? 2 : 1;
      uint32_t v[AHEAD][16];
      ptx::tmem_ld_32x32b_x16(t_row + set * Cfg::kTmemSet, v[0]);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        ptx::tmem_wait_ld();
        ptx::reg_fence16(v[c % AHEAD]);
        if (AHEAD == 2 && c + 1 < CHUNKS) ptx::tmem_ld_32x32b_x16(t_row + set * Cfg::kTmemSet + 16 * (c + 1), v[(c + 1) % AHEAD]);
        if (c + 1 == CHUNKS) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cta(tempty0 + 8 * set);
        }
        // An infinite scale counts as NaN, as it makes one of a code of 8.
        const uint32_t bits = sc[j * Cfg::kSetGroups + c * 16 / TOK];
        const float s = __uint_as_float(((bits & 0x7FFFu) == 0x7F80u ? 0x7FC0u : bits) << 16);
#pragma unroll
        for (int t = 0; t < 16; ++t)
          acc[c * 16 % TOK + t] = fmaf(s, __uint_as_float(v[c % AHEAD][t]), acc[c * 16 % TOK + t]);
        if (AHEAD == 1 && c + 1 < CHUNKS) ptx::tmem_ld_32x32b_x16(t_row + set * Cfg::kTmemSet + 16 * (c + 1), v[0]);
      }
      if (j == Cfg::kSetsPerStep - 1) load_scales(it + 2, sc);
      return true;
    };
    bool go = true;
    for (int it = 0; it < 2 * count && go; it += 2) {
      if (it % 4 == 0) prefetch_scales(it + 18);
#pragma unroll
      for (int j = 0; j < Cfg::kSetsPerStep; ++j) {
        go = go && add_set(it, j, sc_even) && add_set(it + 1, j, sc_odd);
        sphase ^= 1u;
      }
    }
    __syncwarp();
  }
  ptx::griddep_launch_dependents();

  // ------------------------------------------------------ the rows' sums
  __syncthreads();  // every MMA is done: the ring is free
  auto* sums = reinterpret_cast<float*>(smem_raw + (base - ptx::smem_u32(smem_raw)) + Cfg::kRingAt);
  if (warp < Cfg::kEpiWarps) {
#pragma unroll
    for (int t = 0; t < TOK; ++t) sums[t * Cfg::kPitch + warp * 32 + lane] = 64.0f * acc[t];
  }
  if (split > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (!ptx::aborted(wd)) {
    const int toks = min(TOK, p.M - m0);
    const uint32_t sums_at = base + Cfg::kRingAt;
    // 128 threads to a row of the result; a cluster's CTAs share the rows.
    constexpr int kRows = Cfg::kThreads / 128;
    const int row0 = static_cast<int>(threadIdx.x) / 128 + kRows * rank, row_step = kRows * split;
    auto put = [&](int tok, int c, float v, float up) {
      if constexpr (Cfg::kGatedOut) v = gated_value(p.act, v, up);
      const long long off = static_cast<long long>(m0 + tok) * p.ldo + n0 + c;
      if (p.out_type == kOutF32) static_cast<float*>(p.out)[off] = v;
      else static_cast<__nv_bfloat16*>(p.out)[off] = __float2bfloat16_rn(v);
    };
    auto total = [&](uint32_t at) {  // over the CTAs of the cluster, in their order
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        v[c] = c < split ? ld_cluster_f32(ptx::mapa(sums_at + at * 4u, static_cast<uint32_t>(c))) : 0.0f;
#pragma unroll
      for (int c = 1; c < 8; ++c) v[0] += v[c];
      return v[0];
    };
    for (int c = static_cast<int>(threadIdx.x) & 127; threadIdx.x < kRows * 128 && c < cols; c += 128) {
      if (split == 1) {
#pragma unroll 4
        for (int tok = row0; tok < toks; tok += kRows)
          put(tok, c, sums[tok * Cfg::kPitch + c], Cfg::kGatedOut ? sums[tok * Cfg::kPitch + 128 + c] : 0.0f);
      } else {
        for (int tok = row0; tok < toks; tok += row_step) {
          const uint32_t at = static_cast<uint32_t>(tok * Cfg::kPitch + c);
          put(tok, c, total(at), Cfg::kGatedOut ? total(at + 128u) : 0.0f);
        }
      }
    }
  }
  if (threadIdx.x == 0 && ptx::aborted(wd)) ptx::sleep_ns_bounded(200000ull);
  __syncwarp();
  ptx::tc_fence_before();
  if (split > 1) ptx::cluster_sync_all();  // no CTA leaves while another reads its sums
  else __syncthreads();
  ptx::tc_fence_after();
  if (warp == kMma) ptx::tmem_dealloc_cg1(tmem_base, Cfg::kTmemCols);
}

}  // namespace b200gemm
