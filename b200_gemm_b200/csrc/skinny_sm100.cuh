// Products of a few rows of activations with large weights for sm_100a, where
// reading the weights once from HBM is the whole cost:
//   Y = X W^T              W in 4 bits with group scales
//   H = act(X Wg^T) * (X Wu^T)   both weights bf16, or both in 4 bits
// X [M,K] bf16, at most 32 rows per CTA (blocks of 32 rows of X beyond that).
//
// 4-bit weights: W[n,k] = s[k / group, n] * (q[n,k] - 8), q in 0..15, two to a
// byte (even k in the low four bits), s bf16.  q - 8 is exact in bf16, so
// products of a group run on the tensor cores unscaled, summed in fp32, and
// each group's sum is multiplied by its scale in fp32: no weight is rounded.
//
// Rows of W are the M side of mma.sync m16n8k16, rows of X its N side.
// mma.sync, not tcgen05: 4-bit weights are expanded in registers, which
// mma.sync reads directly where tcgen05 would want them written back to
// shared memory first, and neither rate is near its limit here.  A CTA takes
// 64 rows of W (plain) or 32 of Wg and the same 32 of Wu (gated) and a K range;
// streams them through a ring of 128-byte-swizzled TMA boxes, of which its 4
// warps take whole stages in turn.  A stage has one reader, so the warp that
// has read it refills it itself: there is no producer warp and no second
// barrier to say that a stage is free.  The sum over k may run in any order as long as both operands use
// the same one, so a lane takes 8 consecutive k's of a row with a single load
// instead of the fragment's scattered ones.  The 4 warps' sums are added in
// shared memory and, where N is too narrow to occupy every SM, those of the
// K ranges of a cluster of up to 8 CTAs through distributed shared memory,
// always in the same order.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>

#include "ffn_sm100.cuh"
#include "gemm_sm100.cuh"

namespace b200gemm {

struct SkinnyParams {
  int M, N, K;             // gated: N = F
  int num_stages;          // ceil(K / stage K)
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

// G32: groups of 32, whose sums are scaled after every 32-k chunk (4-bit
// weights); without it a group holds 2, 4 or 8 chunks.
template <bool W4, bool GATED, int NT, bool G32 = false>
struct SkinnyCfg {
  static constexpr bool kW4 = W4;
  static constexpr bool kG32 = G32;
  static constexpr bool kGatedOut = GATED;
  static constexpr int kNT = NT;                       // tiles of 8 rows of X
  static constexpr int kTok = 8 * NT;
  static constexpr int kRows = 64;                     // weight rows per CTA
  static constexpr int kOutCols = GATED ? 32 : 64;     // output columns per CTA
  static constexpr int kWarps = 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStageK = W4 ? 256 : 64;        // 128 bytes of a weight row
  static constexpr int kChunks = kStageK / 32;         // 32 k's each
  static constexpr int kStageW = kRows * 128;
  static constexpr int kBoxX = kTok * 128;             // 64 k's of every row of X
  static constexpr int kStageX = kStageK / 64 * kBoxX;
  static constexpr int kStageBytes = kStageW + kStageX;
  // CTAs per SM and a ring that fits that often: small CTAs, so that all of
  // a launch's are resident at once and share HBM evenly.  (NT = 4 needs its
  // registers, and 24 KB stages for 4-bit weights.)
  static constexpr int kCtas = NT == 4 ? 2 : (W4 && NT == 2 ? 3 : 4);
  // A multiple of the warps, so that a stage has the same reader every time
  // around and that reader waits for its fillings in order: a wait by parity
  // for the filling after next would be satisfied before the next arrived.
  static constexpr int kStages = (NT == 4 ? 98304 : (W4 && NT == 2 ? 73728 : 53248)) / kStageBytes / kWarps * kWarps;
  static constexpr int kW = 0;
  static constexpr int kX = kW + kStages * kStageW;
  static constexpr int kFull = kX + kStages * kStageX;
  static constexpr int kAbort = kFull + 8 * kStages;
  static constexpr int kEnd = kAbort + 8;
  static constexpr int kSmemBytes = kEnd + 1024;
  // Sums, in the ring once it is drained: [4 warps][kTok][72], then the CTA's
  // own [kTok][72] (72: a lane group's 4 tokens x 8 rows fall into 32
  // different banks).
  static constexpr int kPitch = 72;
  static constexpr int kRed = 0;
  static constexpr int kPart = kRed + kWarps * kTok * kPitch * 4;
  static_assert(kPart + kTok * kPitch * 4 <= kFull, "sums alias the ring");
  static_assert(kStages >= kWarps && kStages % kWarps == 0, "one reader per stage");
  static_assert(kCtas * (kSmemBytes + 1024) <= 233472, "CTAs per SM");
};

__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with a zero accumulator going in.
__device__ __forceinline__ void mma_m16n8k16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// Eight codes of a word -> four bf16 pairs of q - 8: pair j holds codes j and
// j + 4.  0x4300 is 128 with a spacing of 1, so or-ing a code in gives
// 128 + q; 136 is subtracted, exactly.  And-or is one instruction on the
// logic pipe when mask and magic number come from registers (W4Const: opaque
// to the compiler, which otherwise keeps them as immediates and takes two).
struct W4Const {
  uint32_t mask, magic;
};
__device__ __forceinline__ W4Const w4_const() {
  W4Const c;
  asm volatile("mov.u32 %0, 0x000F000F;\n\tmov.u32 %1, 0x43004300;" : "=r"(c.mask), "=r"(c.magic));
  return c;
}
__device__ __forceinline__ void w4_expand(uint32_t w, const W4Const& k, uint32_t (&v)[4]) {
  const __nv_bfloat162 bias = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t x;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w >> (4 * j)), "r"(k.mask), "r"(k.magic));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), bias);
    v[j] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, Cfg::kCtas)
    skinny_sm100(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                 const __grid_constant__ CUtensorMap map_x, const SkinnyParams p) {
  constexpr int NT = Cfg::kNT;
  constexpr int STAGES = Cfg::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t full0 = base + Cfg::kFull;
  const int split = static_cast<int>(gridDim.x);   // CTAs of this cluster: K ranges
  const int rank = static_cast<int>(blockIdx.x);
  const int n0 = static_cast<int>(blockIdx.y) * Cfg::kOutCols;
  const int m0 = static_cast<int>(blockIdx.z) * 32;
  const int s_begin = rank * p.stages_per_cta;
  const int count = max(0, min(p.num_stages, s_begin + p.stages_per_cta) - s_begin);

  ptx::Watchdog wd;
  wd.abort_flag = base + Cfg::kAbort;
  wd.peer_abort_flag = ptx::mapa(wd.abort_flag, split > 1 ? static_cast<uint32_t>(rank ^ 1) : 0u);
  wd.status = p.status;
  wd.timeout_ns = p.timeout_ns;

  const uint64_t policy_w = ptx::policy_evict_first();  // read once (per 32 rows of X)
  const uint64_t policy_x = ptx::policy_evict_last();   // read by every CTA
  auto load_w = [&](int it, int s) {
    const uint32_t bar = full0 + 8 * s, dst = base + Cfg::kW + s * Cfg::kStageW;
    const int x = (s_begin + it) * (Cfg::kW4 ? 128 : 64);  // elements of the map: bytes (two codes) or bf16
    ptx::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
    ptx::tma_load_2d(dst, &map_w0, bar, x, n0, policy_w);
    if (Cfg::kGatedOut) ptx::tma_load_2d(dst + 32 * 128, &map_w1, bar, x, n0, policy_w);
  };
  auto load_x = [&](int it, int s) {
#pragma unroll
    for (int b = 0; b < Cfg::kStageK / 64; ++b)
      ptx::tma_load_2d(base + Cfg::kX + s * Cfg::kStageX + b * Cfg::kBoxX, &map_x, full0 + 8 * s,
                       (s_begin + it) * Cfg::kStageK + b * 64, m0, policy_x);
  };
  const int pre = min(STAGES, count);
  if (threadIdx.x == 0) {
    // The first ring is on its way before the other warps pass the barrier.
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(wd.abort_flag) : "memory");
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(full0 + 8 * s, 1);
    ptx::fence_mbar_init_cluster();
    ptx::fence_proxy_async_smem();
    if (p.pdl != kPdlWeightsEarly) ptx::griddep_wait();
    for (int it = 0; it < pre; ++it) load_w(it, it);
    if (p.pdl == kPdlWeightsEarly) ptx::griddep_wait();
    for (int it = 0; it < pre; ++it) load_x(it, it);
  }
  __syncthreads();

  // Fragment row (or column) g of 8 stands for row tok(g), so that the 8
  // lanes of a 16-byte access phase (two rows, 4 chunks each) hit all 8 chunk
  // places of the 128-byte swizzle.
  const uint32_t g = lane >> 2, t = lane & 3u;
  const uint32_t tokg = (g >> 1) | ((g & 1u) << 2);

  [[maybe_unused]] const W4Const w4c = w4_const();
  // acc[i][j]: weight rows 16 i .., tokens 8 j ..
  float acc[4][NT][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
  // Scales of a stage: lane l holds those of weight rows l and l + 32 for
  // the group that ends with chunk q, loaded one turn of this warp ahead.
  [[maybe_unused]] float lo_sc[Cfg::kChunks], hi_sc[Cfg::kChunks];
  [[maybe_unused]] uint32_t lo_next[Cfg::kChunks] = {}, hi_next[Cfg::kChunks] = {};
  const int chunk_mask = Cfg::kG32 || !Cfg::kW4 ? 0 : (1 << (p.group_shift - 5)) - 1;  // a group's chunks
  // (rows past N take the last row's scales: their sums are not written)
  const int na = min(n0 + static_cast<int>(lane), p.N - 1);
  const int nb = Cfg::kGatedOut ? na : min(n0 + static_cast<int>(lane) + 32, p.N - 1);
  const uint16_t* scales_a = p.scales0 + na;
  const uint16_t* scales_b = (Cfg::kGatedOut ? p.scales1 : p.scales0) + nb;
  auto load_scales = [&](int it) {
    if (it >= count) return;
    const int k0 = (s_begin + it) * Cfg::kStageK;
    const long long at = static_cast<long long>(k0 >> p.group_shift) * p.N;
    const uint16_t *pa = scales_a + at, *pb = scales_b + at;
    const int left = p.K - k0;  // k's past K: scale 0 (their weights and X are 0)
    if (left >= Cfg::kStageK) {
#pragma unroll
      for (int q = 0; q < Cfg::kChunks; ++q) {
        if ((q & chunk_mask) == chunk_mask) {
          lo_next[q] = __ldg(pa);
          hi_next[q] = __ldg(pb);
          pa += p.N;
          pb += p.N;
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < Cfg::kChunks; ++q) {
        if ((q & chunk_mask) == chunk_mask) {
          lo_next[q] = q * 32 < left ? __ldg(pa) : 0;
          hi_next[q] = q * 32 < left ? __ldg(pb) : 0;
          pa += p.N;
          pb += p.N;
        }
      }
    }
  };
  auto take_scales = [&]() {
#pragma unroll
    for (int q = 0; q < Cfg::kChunks; ++q) {
      lo_sc[q] = __uint_as_float(lo_next[q] << 16);
      hi_sc[q] = __uint_as_float(hi_next[q] << 16);
    }
  };
  if (p.pdl != kPdlWeightsEarly) ptx::griddep_wait();
  if constexpr (Cfg::kW4) load_scales(static_cast<int>(warp));
  for (int it = static_cast<int>(warp); it < count; it += Cfg::kWarps) {
    const int stage = it % STAGES;
    const uint32_t phase = static_cast<uint32_t>(it / STAGES) & 1u;
    if constexpr (Cfg::kW4) {
      take_scales();
      load_scales(it + Cfg::kWarps);
    }
    const bool got = ptx::mbar_wait_cta(full0 + 8 * stage, phase, wd, kSiteEpilogue, blockIdx.y);
    if (!__all_sync(0xFFFFFFFFu, got)) break;
    // Shared addresses: stages, boxes and groups of 8 rows are 1024-byte
    // aligned and a row is 128 bytes, so a chunk's place is one exclusive-or.
    const uint32_t aw = base + Cfg::kW + stage * Cfg::kStageW + tokg * 128u + (Cfg::kW4 ? (tokg << 4) + t * 4u : (t ^ tokg) << 4);
    const uint32_t ax = base + Cfg::kX + stage * Cfg::kStageX + tokg * 128u + ((t ^ tokg) << 4);
    [[maybe_unused]] float sum[4][NT][4];
#pragma unroll
    for (int q = 0; q < Cfg::kChunks; ++q) {
      // X's 8 k's of this lane for every tile of tokens
      uint32_t x[NT][4];
      const uint32_t axq = ax ^ (static_cast<uint32_t>(q & 1) << 6);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        ptx::ld_shared_v4(axq + (q >> 1) * Cfg::kBoxX + j * 1024u, x[j][0], x[j][1], x[j][2], x[j][3]);
      if constexpr (Cfg::kW4) {
        if (!Cfg::kG32 && (q == 0 || ((q - 1) & chunk_mask) == chunk_mask)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c) sum[i][j][c] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          // pairs (k_j, k_j+4), as w4_expand gives the weights
          const uint32_t x0 = x[j][0], x1 = x[j][1], x2 = x[j][2], x3 = x[j][3];
          x[j][0] = __byte_perm(x0, x2, 0x5410);
          x[j][1] = __byte_perm(x0, x2, 0x7632);
          x[j][2] = __byte_perm(x1, x3, 0x5410);
          x[j][3] = __byte_perm(x1, x3, 0x7632);
        }
        const uint32_t awq = aw ^ (static_cast<uint32_t>(q) << 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t lo[4], hi[4];
          w4_expand(ld_shared_u32(awq + i * 2048u), w4c, lo);
          w4_expand(ld_shared_u32(awq + i * 2048u + 1024u), w4c, hi);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (Cfg::kG32) mma_m16n8k16_zero(sum[i][j], lo[0], hi[0], lo[1], hi[1], x[j][0], x[j][1]);
            else mma_m16n8k16(sum[i][j], lo[0], hi[0], lo[1], hi[1], x[j][0], x[j][1]);
            mma_m16n8k16(sum[i][j], lo[2], hi[2], lo[3], hi[3], x[j][2], x[j][3]);
          }
        }
        if ((q & chunk_mask) == chunk_mask) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = i < 2 ? lo_sc[q] : hi_sc[q];
            const float s0 = __shfl_sync(0xFFFFFFFFu, v, (i & 1) * 16 + tokg);
            const float s1 = __shfl_sync(0xFFFFFFFFu, v, (i & 1) * 16 + 8 + tokg);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              acc[i][j][0] = fmaf(s0, sum[i][j][0], acc[i][j][0]);
              acc[i][j][1] = fmaf(s0, sum[i][j][1], acc[i][j][1]);
              acc[i][j][2] = fmaf(s1, sum[i][j][2], acc[i][j][2]);
              acc[i][j][3] = fmaf(s1, sum[i][j][3], acc[i][j][3]);
            }
          }
        }
      } else {
        const uint32_t awq = aw ^ (static_cast<uint32_t>(q) << 6);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t lo[4], hi[4];
          ptx::ld_shared_v4(awq + i * 2048u, lo[0], lo[1], lo[2], lo[3]);
          ptx::ld_shared_v4(awq + i * 2048u + 1024u, hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma_m16n8k16(acc[i][j], lo[0], hi[0], lo[1], hi[1], x[j][0], x[j][1]);
            mma_m16n8k16(acc[i][j], lo[2], hi[2], lo[3], hi[3], x[j][2], x[j][3]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && it + STAGES < count) {
      load_w(it + STAGES, stage);
      load_x(it + STAGES, stage);
    }
  }
  ptx::griddep_launch_dependents();
  // ------------------------------------------- the CTA's sum over its K range
  __syncthreads();  // the ring is drained
  auto* ring = reinterpret_cast<float*>(smem_raw + (base - ptx::smem_u32(smem_raw)));
  float* red = ring + Cfg::kRed / 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // column 2t + b of the fragment is token tok(2t + b) = t + 4b
        const uint32_t tok = j * 8u + t + 4u * (c & 1), row = i * 16u + 8u * (c >> 1) + tokg;
        red[(warp * Cfg::kTok + tok) * Cfg::kPitch + row] = acc[i][j][c];
      }
  __syncthreads();
  if (split > 1) {
    float* part = ring + Cfg::kPart / 4;
#pragma unroll
    for (int idx = static_cast<int>(threadIdx.x); idx < Cfg::kTok * 64; idx += 32 * Cfg::kWarps) {
      const int at = (idx >> 6) * Cfg::kPitch + (idx & 63);
      float v = red[at];
#pragma unroll
      for (int w = 1; w < Cfg::kWarps; ++w) v += red[w * Cfg::kTok * Cfg::kPitch + at];
      part[at] = v;
    }
  }
  if (split > 1) ptx::cluster_sync_all();

  // --------- the sum over the warps or over the cluster, whose CTAs share it out
  if (!ptx::aborted(wd)) {
    auto total = [&](int at) {
      if (split == 1) {
        const uint32_t a = base + Cfg::kRed + at * 4u;
        float v = __uint_as_float(ld_shared_u32(a));
#pragma unroll
        for (int w = 1; w < Cfg::kWarps; ++w)
          v += __uint_as_float(ld_shared_u32(a + w * Cfg::kTok * Cfg::kPitch * 4u));
        return v;
      }
      const uint32_t a = base + Cfg::kPart + at * 4u;
      float v = ld_cluster_f32(ptx::mapa(a, 0));
      for (int c = 1; c < split; ++c) v += ld_cluster_f32(ptx::mapa(a, static_cast<uint32_t>(c)));
      return v;
    };
    constexpr int kCols = Cfg::kOutCols;
    for (int idx = static_cast<int>(threadIdx.x) + 32 * Cfg::kWarps * rank; idx < Cfg::kTok * kCols;
         idx += 32 * Cfg::kWarps * split) {
      const int tok = idx / kCols, c = idx % kCols;
      if (m0 + tok >= p.M || n0 + c >= p.N) continue;
      float v = total(tok * Cfg::kPitch + c);
      if constexpr (Cfg::kGatedOut) {
        const float u = total(tok * Cfg::kPitch + 32 + c);
        switch (p.act) {
          case kActRelu: v = ffn_act<kActRelu>(v) * u; break;
          case kActGelu: v = ffn_act<kActGelu>(v) * u; break;
          case kActGeluTanh: v = ffn_act<kActGeluTanh>(v) * u; break;
          case kActSilu: v = ffn_act<kActSilu>(v) * u; break;
          default: v = v * u; break;
        }
      }
      const long long off = static_cast<long long>(m0 + tok) * p.ldo + n0 + c;
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
// scales are written row-contiguously through shared memory.
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

// W[n,k] = bf16(s (q - 8)): q - 8 is exact in bf16 (w4_expand), so one bf16
// multiplication per pair is the one rounding.  The same blocks; 4 bytes of
// codes and 16 of results per lane and row.
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
  const W4Const c = w4_const();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + warp + 8 * i;
    if (n >= p.N) continue;
    const __nv_bfloat16 s1 = __ushort_as_bfloat16(sc[lane >> (p.group_shift - 3)][warp + 8 * i]);
    const __nv_bfloat162 s2 = __halves2bfloat162(s1, s1);
    uint32_t v[4];
    w4_expand(w[i], c, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 d = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v[j]), s2);
      v[j] = *reinterpret_cast<const uint32_t*>(&d);
    }
    // pairs (k_j, k_j+4) back into order
    ptx::st_global_v4(p.w + static_cast<long long>(n) * p.ldw + k, __byte_perm(v[0], v[1], 0x5410),
                      __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                      __byte_perm(v[2], v[3], 0x7632));
  }
}

}  // namespace b200gemm
