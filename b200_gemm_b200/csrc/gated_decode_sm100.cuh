// Gated block for a few rows of activations (decode) on sm_100a, where reading
// the weights once from HBM is the whole cost:
//   H = act(X Wg^T) * (X Wu^T)     X [M,K], Wg, Wu [F,K] bf16
// at most 32 rows of X per CTA (blocks of 32 rows of X beyond that).
//
// Rows of the weights are the M side of mma.sync m16n8k16 (its rate is far
// from its limit here, and the sums stay in registers), rows of X its N side.
// A CTA takes 32 rows of Wg, the same 32 of Wu and a K range, and streams them
// through a ring of 128-byte-swizzled TMA boxes, of which its 4 warps take
// whole stages in turn.  A stage has one reader, so the warp that has read it
// refills it itself: there is no producer warp and no second barrier to say
// that a stage is free.  The sum over k may run in any order as long as both
// operands use the same one, so a lane takes 8 consecutive k's of a row with
// a single 16-byte load instead of the fragment's scattered ones.  The 4
// warps' sums are added in shared memory and, where F is too narrow to occupy
// every SM, those of the K ranges of a cluster of up to 8 CTAs through
// distributed shared memory, always in the same order.
//
// Measured: 1 x 14336 x 4096 38 us, 235 MB of weights at 6.2 TB/s (DRAM-bound;
// a copy reaches 6.5); 23 x 5003 x 2056 14 us for 41 MB, half of it what any
// launch takes: setting up, the first fetch, the sum over the cluster.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>

#include "ffn_sm100.cuh"
#include "gemm_sm100.cuh"

namespace b200gemm {

struct GatedDecodeParams {
  int M, F, K;
  int num_stages;          // ceil(K / 64)
  int stages_per_cta;      // of each CTA of a cluster
  int act;                 // kAct*
  uint16_t* out;           // H, bf16 bits
  long long ldo;           // elements
  uint16_t *gate, *up;     // G and U, or null
  long long ldgu;
  unsigned int* status;
  unsigned long long timeout_ns;
  int pdl;
};

// DEEP: twice the ring (or more) at half the CTAs per SM, for launches that
// do not fill the SMs otherwise: an SM needs some 64 KB of copies in flight
// to draw its share of HBM's bandwidth.
template <int NT, bool DEEP>
struct GatedDecodeCfg {
  static constexpr int kNT = NT;                       // tiles of 8 rows of X
  static constexpr int kTok = 8 * NT;
  static constexpr int kRows = 64;                     // weight rows per CTA: 32 of Wg, 32 of Wu
  static constexpr int kOutCols = 32;                  // output columns per CTA
  static constexpr int kWarps = 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStageK = 64;                   // 128 bytes of a weight row
  static constexpr int kStageW = kRows * 128;
  static constexpr int kStageX = kTok * 128;
  static constexpr int kStageBytes = kStageW + kStageX;
  // CTAs per SM and a ring that fits that often: small CTAs, so that all of
  // a launch's are resident at once and share HBM evenly.
  static constexpr int kCtas = (NT == 4 ? 2 : 4) / (DEEP ? 2 : 1);
  // A multiple of the warps, so that a stage has the same reader every time
  // around and that reader waits for its fillings in order: a wait by parity
  // for the filling after next would be satisfied before the next arrived.
  static constexpr int kStages = (233472 / kCtas - 1024 - 1024 - 256) / kStageBytes / kWarps * kWarps;
  static constexpr int kX = kStages * kStageW;
  static constexpr int kFull = kX + kStages * kStageX;
  static constexpr int kAbort = kFull + 8 * kStages;
  static constexpr int kEnd = kAbort + 8;
  static constexpr int kSmemBytes = kEnd + 1024;
  // Sums, in the ring once it is drained: [4 warps][kTok][72], then the CTA's
  // own [kTok][72] (72: a lane group's 4 tokens x 8 rows fall into 32
  // different banks).
  static constexpr int kPitch = 72;
  static constexpr int kPart = kWarps * kTok * kPitch * 4;
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

// act(gate) * up of one element.
__device__ __forceinline__ float gated_value(int act, float gate, float up) {
  switch (act) {
    case kActRelu: return ffn_act<kActRelu>(gate) * up;
    case kActGelu: return ffn_act<kActGelu>(gate) * up;
    case kActGeluTanh: return ffn_act<kActGeluTanh>(gate) * up;
    case kActSilu: return ffn_act<kActSilu>(gate) * up;
    default: return gate * up;
  }
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

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, Cfg::kCtas)
    gated_decode_sm100(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_u,
                       const __grid_constant__ CUtensorMap map_x, const GatedDecodeParams p) {
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
    const uint32_t bar = full0 + 8 * s, dst = base + s * Cfg::kStageW;
    ptx::mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
    ptx::tma_load_2d(dst, &map_g, bar, (s_begin + it) * Cfg::kStageK, n0, policy_w);
    ptx::tma_load_2d(dst + 32 * 128, &map_u, bar, (s_begin + it) * Cfg::kStageK, n0, policy_w);
  };
  auto load_x = [&](int it, int s) {
    ptx::tma_load_2d(base + Cfg::kX + s * Cfg::kStageX, &map_x, full0 + 8 * s, (s_begin + it) * Cfg::kStageK, m0,
                     policy_x);
  };
  if (threadIdx.x == 0) {
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(wd.abort_flag) : "memory");
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(full0 + 8 * s, 1);
    ptx::fence_mbar_init_cluster();
    ptx::fence_proxy_async_smem();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int pre = min(STAGES, count);
    if (p.pdl == kPdlWeightsEarly) {
      for (int it = 0; it < pre; ++it) load_w(it, it);
      ptx::griddep_wait();
      for (int it = 0; it < pre; ++it) load_x(it, it);
    } else {
      ptx::griddep_wait();
      for (int it = 0; it < pre; ++it) {  // stage by stage: a stage's X is not kept behind the next one's weights
        load_w(it, it);
        load_x(it, it);
      }
    }
  }
  __syncwarp();

  // Fragment row (or column) g of 8 stands for row tok(g), so that the 8
  // lanes of a 16-byte access phase (two rows, 4 chunks each) hit all 8 chunk
  // places of the 128-byte swizzle.
  const uint32_t g = lane >> 2, t = lane & 3u;
  const uint32_t tokg = (g >> 1) | ((g & 1u) << 2);
  // Shared addresses: stages and groups of 8 rows are 1024-byte aligned and a
  // row is 128 bytes, so the place of the second 32 k's is an exclusive-or.
  const uint32_t off = tokg * 128u + ((t ^ tokg) << 4);

  // acc[i][j]: weight rows 16 i .. (two tiles of Wg, two of Wu), tokens 8 j ..
  float acc[4][NT][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
  for (int it = static_cast<int>(warp); it < count; it += Cfg::kWarps) {
    const int stage = it % STAGES;
    const uint32_t phase = static_cast<uint32_t>(it / STAGES) & 1u;
    const bool got = ptx::mbar_wait_cta(full0 + 8 * stage, phase, wd, kSiteEpilogue, blockIdx.y);
    if (!__all_sync(0xFFFFFFFFu, got)) break;
    const uint32_t aw = base + stage * Cfg::kStageW + off;
    const uint32_t ax = base + Cfg::kX + stage * Cfg::kStageX + off;
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) {
      uint32_t x[NT][4];  // X's 8 k's of this lane for every tile of tokens
#pragma unroll
      for (int j = 0; j < NT; ++j)
        ptx::ld_shared_v4((ax ^ (q << 6)) + j * 1024u, x[j][0], x[j][1], x[j][2], x[j][3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t lo[4], hi[4];
        ptx::ld_shared_v4((aw ^ (q << 6)) + i * 2048u, lo[0], lo[1], lo[2], lo[3]);
        ptx::ld_shared_v4((aw ^ (q << 6)) + i * 2048u + 1024u, hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_m16n8k16(acc[i][j], lo[0], hi[0], lo[1], hi[1], x[j][0], x[j][1]);
          mma_m16n8k16(acc[i][j], lo[2], hi[2], lo[3], hi[3], x[j][2], x[j][3]);
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
  auto* sums = reinterpret_cast<float*>(smem_raw + (base - ptx::smem_u32(smem_raw)));
  constexpr int kSlab = Cfg::kTok * Cfg::kPitch;  // floats of one warp's sums
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // column 2t + b of the fragment is token tok(2t + b) = t + 4b
        const uint32_t tok = j * 8u + t + 4u * (c & 1), row = i * 16u + 8u * (c >> 1) + tokg;
        sums[warp * kSlab + tok * Cfg::kPitch + row] = acc[i][j][c];
      }
  __syncthreads();
  auto warp_sum = [&](int at) {
    float v = sums[at];
#pragma unroll
    for (int w = 1; w < Cfg::kWarps; ++w) v += sums[w * kSlab + at];
    return v;
  };
  if (split > 1) {
#pragma unroll
    for (int idx = static_cast<int>(threadIdx.x); idx < Cfg::kTok * 64; idx += Cfg::kThreads) {
      const int at = (idx >> 6) * Cfg::kPitch + (idx & 63);
      sums[Cfg::kPart / 4 + at] = warp_sum(at);
    }
    ptx::cluster_sync_all();
  }

  // --------- the sum over the warps or over the cluster, whose CTAs share it out
  if (!ptx::aborted(wd)) {
    auto total = [&](int at) {
      if (split == 1) return warp_sum(at);
      const uint32_t a = base + Cfg::kPart + at * 4u;
      float v = ld_cluster_f32(ptx::mapa(a, 0));
      for (int c = 1; c < split; ++c) v += ld_cluster_f32(ptx::mapa(a, static_cast<uint32_t>(c)));
      return v;
    };
    constexpr int kCols = Cfg::kOutCols;
    for (int idx = static_cast<int>(threadIdx.x) + Cfg::kThreads * rank; idx < Cfg::kTok * kCols;
         idx += Cfg::kThreads * split) {
      const int tok = idx / kCols, c = idx % kCols;
      if (m0 + tok >= p.M || n0 + c >= p.F) continue;
      const float gate = total(tok * Cfg::kPitch + c), up = total(tok * Cfg::kPitch + 32 + c);
      const long long r = m0 + tok;
      auto bits = [](float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); };
      p.out[r * p.ldo + n0 + c] = bits(gated_value(p.act, gate, up));
      if (p.gate != nullptr) {
        p.gate[r * p.ldgu + n0 + c] = bits(gate);
        p.up[r * p.ldgu + n0 + c] = bits(up);
      }
    }
  }
  if (threadIdx.x == 0 && ptx::aborted(wd)) ptx::sleep_ns_bounded(200000ull);
  __syncwarp();
  if (split > 1) ptx::cluster_sync_all();  // no CTA leaves while another reads its sums
}

}  // namespace b200gemm
