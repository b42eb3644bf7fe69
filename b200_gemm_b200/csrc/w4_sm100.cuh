// Products of a few rows of activations with 4-bit weights for sm_100a, and the
// conversions between them and bf16:
//   Y = X W^T,   H = act(X Wg^T) * (X Wu^T)
//   W[n,k] = s[k / group, n] * (q[n,k] - 8), q in 0..15, two to a byte (even k
//   in the low four bits), s bf16
// X [M,K] bf16, at most 16 rows (more: w4_mma_sm100.cuh).
//
// Rows of W are the M side of mma.sync m16n8k16, rows of X its N side, fp32
// sums.  mma.sync, not tcgen05: the codes are expanded in registers, which
// mma.sync reads directly, and a tcgen05.mma takes the same time for 8 rows of
// X as for 32.  Both measured (us, this kernel and that one): at 8 rows 8192 x
// 8192 in groups of 128 12.9 and 16.7, of 32 14.1 and 23, 4096 x 14336 12.2 and
// 16.6; at 16 rows 16.1 and 17.4, 17.3 and 23.5, 15.0 and 16.6.  One row of
// 28672 x 8192 takes 28 us, 121 MB of codes and scales at 4.3 TB/s, with 62% of
// the issue slots and 50% of the logic pipe in use: what bounds the kernel,
// next to HBM, is the number of instructions issued per weight, so everything
// else is arranged around them:
//   * Four bits masked out in place, b = q or 16 q in a 16-bit half, are
//     b 2^-133 as bf16 (the lowest bit of the exponent counts on like one of
//     the mantissa), so a multiply-add by 2^127 or 2^123 and -1/8 makes them
//     (q - 8) / 64, exactly: five bit operations and four multiply-adds for
//     eight weights.  The last 6 bits come back with the row's finished sums.
//     (128 + q, or-ed together, costs seven bit operations and no multiply-add
//     but a sum that starts from -136 sum(x): 3 to 8% slower.)
//   * The sum of a group (of half of one, ..) is multiplied by its scale in
//     fp32 and added to the row's.
//   * One CTA of 16 warps per SM takes a range of rows of W (gated: the same
//     rows of Wg and Wu) that divides N evenly over the SMs, whatever N is,
//     and streams it through a ring of 128-byte-swizzled TMA boxes, 512 k's a
//     stage.  Warp (half, c) takes half of the rows (gated: Wg's or Wu's) and
//     k's 64 c .. of every stage, so it reads its part of X once per stage and
//     uses it for all its rows.
// The sum over k may run in any order as long as both operands use the same
// one, so a lane takes 8 consecutive k's of a row with a single load instead
// of the fragment's scattered ones.  The 8 warps' sums of a row are added in
// shared memory and, where N is too narrow to give every SM enough rows,
// those of the K ranges of a cluster of up to 8 CTAs through distributed
// shared memory, always in the same order.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>

#include "ffn_sm100.cuh"
#include "gemm_sm100.cuh"
#include "gated_decode_sm100.cuh"

namespace b200gemm {

struct W4NtParams {
  int M, N, K;             // gated: N = F
  int rows;                // rows of W (gated: of each of Wg and Wu) a CTA finishes
  int num_stages;          // ceil(K / 512)
  int stages_per_cta;      // of each CTA of a cluster
  int act;                 // gated: kAct*
  int out_type;            // kOutBf16 or kOutF32
  int group_shift;         // log2 of the group (4-bit weights)
  const uint16_t* scales0; // [K / group][N]: W, or Wg
  const uint16_t* scales1; // Wu
  void* out;
  long long ldo;           // elements
  unsigned int* status;
  unsigned long long timeout_ns;
  int pdl;
};

// MT: 16-row tiles of W per warp (and half); NT: tiles of 8 rows of X; G32:
// groups of 32 (a warp's 64 k's of a stage are two groups, not part of one).
template <bool GATED, bool G32, int MT, int NT>
struct W4NtCfg {
  static constexpr bool kGatedOut = GATED;
  static constexpr bool kG32 = G32;
  static constexpr int kMT = MT;
  static constexpr int kNT = NT;
  static constexpr int kTok = 8 * NT;
  static constexpr int kHalf = 16 * MT;                // weight rows of one half of the warps
  static constexpr int kWarps = 16;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStageK = 512;
  static constexpr int kBoxW = 2 * kHalf * 128;        // 256 k's of every weight row
  static constexpr int kStageW = 2 * kBoxW;
  // X is not swizzled: a box may then be 256 k's wide (two copies a stage, not
  // eight), and each warp reads its part of it only once.
  static constexpr int kBoxX = kTok * 512;             // 256 k's of every row of X
  static constexpr int kStageX = 2 * kBoxX;
  static constexpr int kStageBytes = kStageW + kStageX;
  // Sums, in the ring once it is drained: [8 warps][kTok][kPitch], then the
  // CTA's own [kTok][kPitch] (a pitch of 8 mod 32: a lane group's 4 tokens x 8
  // rows fall into 32 different banks).
  static constexpr int kPitch = (2 * kHalf + 31) / 32 * 32 + 8;
  static constexpr int kPart = 8 * kTok * kPitch * 4;
  static constexpr int kSums = kPart + kTok * kPitch * 4;
  static constexpr int kBars = 256;
  static constexpr int kMaxRing = 8;
  static constexpr int kRingFit = (232448 - 1024 - kBars) / kStageBytes;
  static constexpr int kRing = kRingFit > kMaxRing ? kMaxRing : kRingFit;
  static_assert(kRing >= 3, "pipeline too shallow");
  static_assert(2 * 8 * kMaxRing + 8 <= kBars, "barriers");
  static constexpr int kRingBytes = kRing * kStageBytes > kSums ? kRing * kStageBytes : kSums;
  static constexpr int kSmemBytes = 1024 + kBars + kRingBytes;
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB per-CTA shared memory limit");
};

// The same onto another accumulator, c.
__device__ __forceinline__ void mma_m16n8k16_onto(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1,
                                                  uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Eight codes of a word -> four bf16 pairs of (q - 8) / 64: pair j holds codes
// j and j + 4.  (Constants come from registers: opaque to the compiler, which
// otherwise keeps them as immediates.)
struct W4Const {
  uint32_t mask, mask16, scale, scale16, offset;
};
__device__ __forceinline__ W4Const w4_const() {
  W4Const c;
  asm volatile("mov.u32 %0, 0x000F000F;\n\tmov.u32 %1, 0x00F000F0;" : "=r"(c.mask), "=r"(c.mask16));
  asm volatile("mov.u32 %0, 0x7F007F00;\n\tmov.u32 %1, 0x7D007D00;\n\tmov.u32 %2, 0xBE00BE00;"
               : "=r"(c.scale), "=r"(c.scale16), "=r"(c.offset));
  return c;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ void w4_expand(uint32_t w, const W4Const& k, uint32_t (&v)[4]) {
  v[0] = fma_bf16x2(w & k.mask, k.scale, k.offset);
  v[1] = fma_bf16x2(w & k.mask16, k.scale16, k.offset);
  v[2] = fma_bf16x2((w >> 8) & k.mask, k.scale, k.offset);
  v[3] = fma_bf16x2((w >> 8) & k.mask16, k.scale16, k.offset);
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1)
    w4_nt_sm100(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                 const __grid_constant__ CUtensorMap map_x, const W4NtParams p) {
  constexpr int NT = Cfg::kNT, MT = Cfg::kMT, RING = Cfg::kRing;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t ring = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = ring + Cfg::kRingBytes;
  const uint32_t full0 = bars, empty0 = bars + 8 * RING;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const int split = static_cast<int>(gridDim.x);   // CTAs of this cluster: K ranges
  const int rank = static_cast<int>(blockIdx.x);
  const int n0 = static_cast<int>(blockIdx.y) * p.rows;
  const int s_begin = rank * p.stages_per_cta;
  const int count = max(0, min(p.num_stages, s_begin + p.stages_per_cta) - s_begin);

  ptx::Watchdog wd;
  wd.abort_flag = bars + 16 * RING;
  wd.peer_abort_flag = ptx::mapa(wd.abort_flag, split > 1 ? static_cast<uint32_t>(rank ^ 1) : 0u);
  wd.status = p.status;
  wd.timeout_ns = p.timeout_ns;

  const uint64_t policy_w = ptx::policy_evict_first();  // read once
  const uint64_t policy_x = ptx::policy_evict_last();   // read by every CTA
  auto load_w = [&](int it, int s) {
    const uint32_t bar = full0 + 8 * s, dst = ring + s * Cfg::kStageBytes;
    ptx::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int x = (s_begin + it) * 256 + b * 128;  // bytes: two codes each
      ptx::tma_load_2d(dst + b * Cfg::kBoxW, &map_w0, bar, x, n0, policy_w);
      if (Cfg::kGatedOut) ptx::tma_load_2d(dst + b * Cfg::kBoxW + Cfg::kHalf * 128, &map_w1, bar, x, n0, policy_w);
    }
  };
  auto load_x = [&](int it, int s) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
      ptx::tma_load_2d(ring + s * Cfg::kStageBytes + Cfg::kStageW + b * Cfg::kBoxX, &map_x, full0 + 8 * s,
                       (s_begin + it) * Cfg::kStageK + b * 256, 0, policy_x);
  };

  const uint32_t half = warp >> 3, part = warp & 7u;  // rows, and k's 64 part .. of every stage
  // Scales of this warp's rows for its k's of the next stage (one or two
  // groups), loaded one stage ahead: lane l holds rows l, l + 32, ..  The
  // first ones are asked for before the ring's copies, which would keep them
  // waiting for microseconds.
  constexpr int kHold = (Cfg::kHalf + 31) / 32, kSets = Cfg::kG32 ? 2 : 1;
  uint32_t next_sc[kSets][kHold] = {};
  const int row0 = n0 + (Cfg::kGatedOut ? 0 : static_cast<int>(half) * Cfg::kHalf) + static_cast<int>(lane);
  const uint16_t* scales = ((Cfg::kGatedOut && half == 1) ? p.scales1 : p.scales0) + row0;
  int k_next = s_begin * Cfg::kStageK + static_cast<int>(part) * 64;
  const int k_end = min(p.K, (s_begin + count) * Cfg::kStageK);  // past it: scale 0 (past K X is 0)
  auto load_scales = [&]() {
#pragma unroll
    for (int e = 0; e < kSets; ++e) {
      const bool in_k = k_next + 32 * e < k_end;
      const uint16_t* src = scales + static_cast<long long>((k_next + 32 * e) >> p.group_shift) * p.N;
#pragma unroll
      for (int r = 0; r < kHold; ++r) next_sc[e][r] = in_k && row0 + 32 * r < p.N ? __ldg(src + 32 * r) : 0;
    }
    k_next += Cfg::kStageK;
  };
  if (p.pdl != kPdlWeightsEarly) ptx::griddep_wait();
  load_scales();
  if (threadIdx.x == 0) {
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(wd.abort_flag) : "memory");
    for (int s = 0; s < RING; ++s) {
      ptx::mbar_init(full0 + 8 * s, 1);
      ptx::mbar_init(empty0 + 8 * s, Cfg::kWarps);
    }
    ptx::fence_mbar_init_cluster();
    ptx::fence_proxy_async_smem();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int pre = min(RING, count);
    if (p.pdl == kPdlWeightsEarly) {
      for (int it = 0; it < pre; ++it) load_w(it, it);
      ptx::griddep_wait();
      for (int it = 0; it < pre; ++it) load_x(it, it);
    } else {
      for (int it = 0; it < pre; ++it) {  // stage by stage: a stage's X is not kept behind the next one's W
        load_w(it, it);
        load_x(it, it);
      }
    }
  }
  __syncwarp();

  // Fragment row (or column) g of 8 stands for row tok(g), as in the bf16 kernel
  // for few rows.  The 8 rows of a 4-byte load of codes have their chunks at the
  // 8 places of the 128-byte swizzle, so a warp's lanes hit all banks.
  const uint32_t g = lane >> 2, t = lane & 3u;
  const uint32_t tokg = (g >> 1) | ((g & 1u) << 2);
  const W4Const w4c = w4_const();

  // acc[i][j]: weight rows 16 i .. of this half, tokens 8 j ..
  float acc[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
  // Shared addresses: stages, boxes and groups of 8 rows are 1024-byte
  // aligned and a row is 128 bytes, so a chunk's place is an exclusive-or.
  const uint32_t off_w = (part >> 2) * Cfg::kBoxW + half * (Cfg::kHalf * 128u) + tokg * 128u +
                         (((2u * (part & 3u)) ^ tokg) << 4) + t * 4u;
  const uint32_t off_x = Cfg::kStageW + (part >> 2) * Cfg::kBoxX + tokg * 512u + (part & 3u) * 128u + t * 16u;
  int stage = 0;
  uint32_t phase = 0;
  // The warps take turns at refilling the stage before the one at hand, part of
  // the way into it, when the others have mostly left that one (after the first
  // quarter; at the end of it, 1 to 4% slower).
  auto refill = [&](int j) {
    if (lane == 0 && j >= 0 && j + RING < count && (j & 15) == static_cast<int>(warp)) {
      const int s = stage == 0 ? RING - 1 : stage - 1;
      const uint32_t ph = stage == 0 ? phase ^ 1u : phase;
      if (ptx::mbar_wait_cta(empty0 + 8 * s, ph, wd, kSiteProducer, blockIdx.y)) {
        load_w(j + RING, s);
        load_x(j + RING, s);
      }
    }
    __syncwarp();
  };
  for (int it = 0; it < count; ++it) {
    float sc[kSets][kHold];
#pragma unroll
    for (int e = 0; e < kSets; ++e)
#pragma unroll
      for (int r = 0; r < kHold; ++r) {
        // An infinite scale counts as NaN, whatever its group's codes are: of
        // a code of 8 it makes one, and the group's sum does not tell.
        const uint32_t s = next_sc[e][r];
        sc[e][r] = __uint_as_float((s & 0x7F80u) == 0x7F80u ? 0x7FC00000u : s << 16);
      }
    load_scales();
    const bool got = ptx::mbar_wait_cta(full0 + 8 * stage, phase, wd, kSiteEpilogue, blockIdx.y);
    if (!__all_sync(0xFFFFFFFFu, got)) break;
    if ((s_begin + it) * Cfg::kStageK + static_cast<int>(part) * 64 < p.K) {
      const uint32_t aw = ring + stage * Cfg::kStageBytes + off_w;
      const uint32_t ax = ring + stage * Cfg::kStageBytes + off_x;
      // X's 8 k's of this lane in chunk e of 32, as pairs (k_j, k_j+4) like the
      // weights'.
      auto load_x = [&](int e, uint32_t (&x)[NT][4]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t x0, x1, x2, x3;
          ptx::ld_shared_v4(ax + 64u * e + j * 4096u, x0, x1, x2, x3);
          x[j][0] = __byte_perm(x0, x2, 0x5410);
          x[j][1] = __byte_perm(x0, x2, 0x7632);
          x[j][2] = __byte_perm(x1, x3, 0x5410);
          x[j][3] = __byte_perm(x1, x3, 0x7632);
        }
      };
      // acc += scale * sum for row tile i.
      auto add_scaled = [&](int i, int set, const float (&sum)[NT][4]) {
        const float v = sc[set][i >> 1];
        const float s0 = __shfl_sync(0xFFFFFFFFu, v, (i & 1) * 16 + tokg);
        const float s1 = __shfl_sync(0xFFFFFFFFu, v, (i & 1) * 16 + 8 + tokg);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[i][j][0] = fmaf(s0, sum[j][0], acc[i][j][0]);
          acc[i][j][1] = fmaf(s0, sum[j][1], acc[i][j][1]);
          acc[i][j][2] = fmaf(s1, sum[j][2], acc[i][j][2]);
          acc[i][j][3] = fmaf(s1, sum[j][3], acc[i][j][3]);
        }
      };
      uint32_t x[2][NT][4];
      const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 2; ++e) load_x(e, x[e]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (i == MT / 4) refill(it - 1);
        float sum[NT][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t lo[4], hi[4];
          w4_expand(ld_shared_u32((aw ^ (16u * e)) + i * 2048u), w4c, lo);
          w4_expand(ld_shared_u32((aw ^ (16u * e)) + i * 2048u + 1024u), w4c, hi);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (e < kSets) mma_m16n8k16_onto(sum[j], zero, lo[0], hi[0], lo[1], hi[1], x[e][j][0], x[e][j][1]);
            else mma_m16n8k16(sum[j], lo[0], hi[0], lo[1], hi[1], x[e][j][0], x[e][j][1]);
            mma_m16n8k16(sum[j], lo[2], hi[2], lo[3], hi[3], x[e][j][2], x[e][j][3]);
          }
          if (e == 1 || Cfg::kG32) add_scaled(i, e % kSets, sum);
        }
      }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive_cta(empty0 + 8 * stage);
    if (++stage == RING) {
      stage = 0;
      phase ^= 1u;
    }
  }
  ptx::griddep_launch_dependents();
  // --------------------------------------------- the CTA's sum over its K range
  __syncthreads();  // the ring is drained
  constexpr uint32_t kSlab = Cfg::kTok * Cfg::kPitch;  // floats of one warp's sums
  auto* sums = reinterpret_cast<float*>(smem_raw + (ring - ptx::smem_u32(smem_raw)));
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // column 2t + b of the fragment is token tok(2t + b) = t + 4b
        const uint32_t tok = j * 8u + t + 4u * (c & 1), row = half * Cfg::kHalf + i * 16u + 8u * (c >> 1) + tokg;
        sums[part * kSlab + tok * Cfg::kPitch + row] = 64.0f * acc[i][j][c];
      }
  __syncthreads();
  const int toks = min(Cfg::kTok, p.M);
  const int cols = min(p.rows, p.N - n0);  // output columns of this CTA
  auto warp_sum = [&](uint32_t at) {
    float v = sums[at];
#pragma unroll
    for (int c = 1; c < 8; ++c) v += sums[c * kSlab + at];
    return v;
  };
  if (split > 1) {
    for (int tok = static_cast<int>(warp); tok < toks; tok += Cfg::kWarps)
      for (int r = static_cast<int>(lane); r < 2 * Cfg::kHalf; r += 32)
        sums[Cfg::kPart / 4 + tok * Cfg::kPitch + r] = warp_sum(tok * Cfg::kPitch + r);
    ptx::cluster_sync_all();
  }

  // --------- the sum over the warps or over the cluster, whose CTAs share it out
  if (!ptx::aborted(wd)) {
    auto total = [&](uint32_t at) {
      if (split == 1) return warp_sum(at);
      const uint32_t a = ring + Cfg::kPart + at * 4u;
      float v = ld_cluster_f32(ptx::mapa(a, 0));
      for (int c = 1; c < split; ++c) v += ld_cluster_f32(ptx::mapa(a, static_cast<uint32_t>(c)));
      return v;
    };
    for (int i = static_cast<int>(threadIdx.x) + Cfg::kThreads * rank; i < toks * cols; i += Cfg::kThreads * split) {
      const int tok = i / cols, c = i - tok * cols;
      float v = total(tok * Cfg::kPitch + c);
      if constexpr (Cfg::kGatedOut) {
        v = gated_value(p.act, v, total(tok * Cfg::kPitch + Cfg::kHalf + c));
      }
      const long long off = static_cast<long long>(tok) * p.ldo + n0 + c;
      if (p.out_type == kOutF32) static_cast<float*>(p.out)[off] = v;
      else static_cast<__nv_bfloat16*>(p.out)[off] = __float2bfloat16_rn(v);
    }
  }
  if (threadIdx.x == 0 && ptx::aborted(wd)) ptx::sleep_ns_bounded(200000ull);
  __syncwarp();
  if (split > 1) ptx::cluster_sync_all();  // no CTA leaves while another reads its sums
}

// ------------------------------------------------- 4-bit weights and bf16
// Per group of one row: s = bf16(max|w| / 7), q = clamp(rint(w / s), -8, 7) + 8
// (8 where s is 0 or NaN, so a group with a NaN or infinity comes back as
// NaN).  DRAM-bound once the arithmetic is a handful of instructions per
// weight.  A block takes 32 rows x 256 k's: a warp reads 256 k's of a row, 16
// bytes a lane, four rows in flight; a group's lanes find its maximum by
// shuffles on the magnitude bits (which order NaN above all), and the block's
// scales are written row-contiguously through shared memory.  14336 x 4096 in
// groups of 128: 28 us, 148 MB at 5.3 TB/s, with 74% of the issue slots in use;
// back 24.5 us (most of it from and to L2 when just written).
struct W4Params {
  int N, K, group_shift;
  uint16_t* w;           // [N, K], row pitch ldw
  long long ldw;
  uint8_t* codes;        // [N, K / 2]
  uint16_t* scales;      // [K / group, N]
};

// Codes of 8 weights (4 words of bf16 pairs) for scale s.  The quotient of
// two bf16 numbers is either a tie k + 1/2 exactly or at least 2^-10 off one
// (2w - (2k + 1)s is a multiple of the smaller operand's last place), while
// w * (1 / s) is within 2^-20 of it below 8.  So one fused multiply-add onto
// 1.5 * 2^11, where fp32 has a spacing of 2^-12, gives the quotient on a grid
// that holds the ties and moves nothing across one, and a second addition
// onto 1.5 * 2^23 + 8 rounds it to the integer (ties to even) and leaves q + 8
// in the low four bits.  |w / s| <= 7 (1 + 2^-8) here, so nothing is clamped;
// where s is so small that it has lost digits or 1 / s overflows, the
// division is done as such.
__device__ __forceinline__ uint32_t w4_codes(const uint32_t (&w)[4], float s) {
  uint32_t code = 0u;
  if (s >= 1e-30f && s <= 1e37f) {
    const float r = ptx::rcp_approx(s);
    constexpr float kGrid = 1.5f * 2048.0f, kInt = 1.5f * 8388608.0f + 8.0f;
    // Eight sums of 1.5 * 2^23 + 8 + q, shifted up and added: their constant
    // parts add up to kBase.
    constexpr uint32_t kOne = 0x4B400000u, kBase = kOne * 0x11111111u;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      code = (code << 4) + __float_as_uint(fmaf(bf16_hi(w[j]), r, kGrid) + (kInt - kGrid));
      code = (code << 4) + __float_as_uint(fmaf(bf16_lo(w[j]), r, kGrid) + (kInt - kGrid));
    }
    code -= kBase;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = (j & 1) ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
      int q = 0;
      if (s > 0.0f) q = max(-8, min(7, __float2int_rn(__fdiv_rn(x, s))));  // (NaN converts to 0)
      code |= static_cast<uint32_t>(q + 8) << (4 * j);
    }
  }
  return code;
}

__global__ void __launch_bounds__(256) w4_quantize_kernel(const W4Params p) {
  __shared__ uint16_t sc[8][32];
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31u);
  const int k = static_cast<int>(blockIdx.x) * 256 + lane * 8;
  const int n0 = static_cast<int>(blockIdx.y) * 32;
  const int lanes = 1 << (p.group_shift - 3);  // per group: 4 .. 32
  const int rows = k < p.K ? p.N - n0 - warp : 0;  // of this lane: row 8 i is one of them while 8 i < rows
  uint32_t w[4][4];
  const uint16_t* src = p.w + static_cast<long long>(n0 + warp) * p.ldw + k;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0u;
    if (8 * i < rows) ptx::ld_global_nc_v4(src, w[i][0], w[i][1], w[i][2], w[i][3]);
    src += 8 * p.ldw;
  }
  uint32_t m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m2 = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) m2 = __vmaxu2(m2, w[i][j] & 0x7FFF7FFFu);
    m[i] = max(m2 & 0xFFFFu, m2 >> 16);
  }
  for (int d = 1; d < lanes; d <<= 1) {  // (the four rows' shuffles in flight together)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], d));
  }
  uint8_t* dst = p.codes + static_cast<long long>(n0 + warp) * (p.K / 2) + k / 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // max / 7 by a product: like the quotients below, max / 7 is never within
    // 2^-12 of a bf16 rounding border without being a bf16 number itself.
    const __nv_bfloat16 sb = __float2bfloat16_rn(__uint_as_float(m[i] << 16) * (1.0f / 7.0f));
    const uint32_t code = w4_codes(w[i], __bfloat162float(sb));
    if (8 * i < rows) {
      *reinterpret_cast<uint32_t*>(dst) = code;
      if ((lane & (lanes - 1)) == 0) sc[lane >> (p.group_shift - 3)][warp + 8 * i] = __bfloat16_as_ushort(sb);
    }
    dst += 4ll * p.K;
  }
  __syncthreads();
  const int q = warp + (static_cast<int>(blockIdx.x) * 256 >> p.group_shift);
  if (warp < (256 >> p.group_shift) && q < (p.K >> p.group_shift) && n0 + lane < p.N)
    p.scales[static_cast<long long>(q) * p.N + n0 + lane] = sc[warp][lane];
}

// W[n,k] = bf16(s (q - 8)): 0x4300 is 128 in bf16 with a spacing of 1, so a
// code or-ed in gives 128 + q, and less 136 is exact; one bf16 multiplication
// per pair is the one rounding.  The same blocks; 4 bytes of codes and 16 of
// results per lane and row.
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const W4Params p) {
  __shared__ uint16_t sc[8][32];
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31u);
  const int k = static_cast<int>(blockIdx.x) * 256 + lane * 8;
  const int n0 = static_cast<int>(blockIdx.y) * 32;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + warp + 8 * i;
    w[i] = 0u;
    if (n < p.N && k < p.K)
      w[i] = __ldg(reinterpret_cast<const uint32_t*>(p.codes + static_cast<long long>(n) * (p.K / 2) + k / 2));
  }
  const int q = warp + (static_cast<int>(blockIdx.x) * 256 >> p.group_shift);
  if (warp < (256 >> p.group_shift) && q < (p.K >> p.group_shift) && n0 + lane < p.N)
    sc[warp][lane] = __ldg(p.scales + static_cast<long long>(q) * p.N + n0 + lane);
  __syncthreads();
  if (k >= p.K) return;
  const __nv_bfloat162 offset = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + warp + 8 * i;
    if (n >= p.N) continue;
    const __nv_bfloat16 s1 = __ushort_as_bfloat16(sc[lane >> (p.group_shift - 3)][warp + 8 * i]);
    const __nv_bfloat162 s2 = __halves2bfloat162(s1, s1);
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = ((w[i] >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 d = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v[j]), offset), s2);
      v[j] = *reinterpret_cast<const uint32_t*>(&d);
    }
    // pairs (k_j, k_j+4) back into order
    ptx::st_global_v4(p.w + static_cast<long long>(n) * p.ldw + k, __byte_perm(v[0], v[1], 0x5410),
                      __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                      __byte_perm(v[2], v[3], 0x7632));
  }
}

}  // namespace b200gemm
