// Host side of the feed-forward entry points of include/b200gemm.h: argument
// checks, plans and launches of the kernels in ffn_sm100.cuh,
// gated_decode_sm100.cuh, w4_sm100.cuh and w4_mma_sm100.cuh.  Part of
// b200gemm.cu's translation unit (it uses the handle and the helpers there).
// Nothing here allocates, builds a table or waits, so every call can be captured
// into a CUDA graph from the first one.
#pragma once

namespace b200gemm {

// Stages fill shared memory next to the staging buffers: 3 x 48 KB + 64 KB,
// or 6 x 32 KB, 7 x 28 KB, 8 x 24 KB + 16 KB.
using FfnGated512 = FfnCfg<kGated, 2, 3>;
using FfnGated256 = FfnCfg<kGated, 1, 6>;
using FfnGated192 = FfnCfg<kGated, 1, 7, 192>;
using FfnGated128 = FfnCfg<kGated, 1, 8, 128>;
using FfnGrads512 = FfnCfg<kGrads, 2, 3>;
using FfnGrads256 = FfnCfg<kGrads, 1, 6>;
using FfnGrads128 = FfnCfg<kGrads, 1, 8, 128>;

template <class Cfg>
int prepare_ffn_kernel(int sm_count) {
  if (cudaFuncSetAttribute(ffn_gemm_sm100<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes) !=
      cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count & ~1), 1, 1);
  cfg.blockDim = dim3(Cfg::kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, ffn_gemm_sm100<Cfg>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return clusters;
}

// Smallest number of clusters that fit over all instances of the tiled
// feed-forward kernel (they differ only in registers), or 0 on failure.
int prepare_ffn_kernels(int sm_count) {
  const int c[] = {prepare_ffn_kernel<FfnGated512>(sm_count), prepare_ffn_kernel<FfnGated256>(sm_count),
                   prepare_ffn_kernel<FfnGated192>(sm_count), prepare_ffn_kernel<FfnGated128>(sm_count),
                   prepare_ffn_kernel<FfnGrads512>(sm_count), prepare_ffn_kernel<FfnGrads256>(sm_count),
                   prepare_ffn_kernel<FfnGrads128>(sm_count)};
  int least = c[0];
  for (int v : c) least = v < least ? v : least;
  return least;
}

template <class Kernel>
bool opt_in_smem(Kernel kernel, int bytes) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}

template <int NT>
bool prepare_gated_decode() {
  return opt_in_smem(gated_decode_sm100<GatedDecodeCfg<NT, false>>, GatedDecodeCfg<NT, false>::kSmemBytes) &&
         opt_in_smem(gated_decode_sm100<GatedDecodeCfg<NT, true>>, GatedDecodeCfg<NT, true>::kSmemBytes);
}
bool prepare_gated_decode_kernels() {
  return prepare_gated_decode<1>() && prepare_gated_decode<2>() && prepare_gated_decode<4>();
}

// Instances of the 4-bit product: 16-row tiles of W per warp (MT) that its
// registers and ring allow next to NT tiles of X's rows.
template <int NT>
constexpr int kW4MaxMT = NT == 1 ? 7 : 5;
// Rows of X up to which a 4-bit product runs on mma.sync, whose CTAs hold all
// of them (8 NT).
constexpr int kW4MaxSyncRows = 16;
static_assert(kW4MaxSyncRows <= W4NtCfg<false, false, 1, 2>::kTok, "rows of X of one CTA");

template <bool GATED, bool G32, int NT, int MT = kW4MaxMT<NT>>
bool prepare_w4_instances() {
  if constexpr (MT == 0) {
    return true;
  } else {
    using Cfg = W4NtCfg<GATED, G32, MT, NT>;
    return opt_in_smem(w4_nt_sm100<Cfg>, Cfg::kSmemBytes) && prepare_w4_instances<GATED, G32, NT, MT - 1>();
  }
}

template <bool GATED, bool G32>
bool prepare_w4_nt() {
  return prepare_w4_instances<GATED, G32, 1>() && prepare_w4_instances<GATED, G32, 2>();
}

template <bool GATED, int H, int TOK>
bool prepare_w4_mma() {
  using C1 = W4MmaCfg<GATED, H, 1, TOK>;
  using C2 = W4MmaCfg<GATED, H, 2, TOK>;
  using C4 = W4MmaCfg<GATED, H, 4, TOK>;
  return opt_in_smem(w4_mma_sm100<C1>, C1::kSmemBytes) && opt_in_smem(w4_mma_sm100<C2>, C2::kSmemBytes) &&
         opt_in_smem(w4_mma_sm100<C4>, C4::kSmemBytes);
}

bool prepare_w4_kernels() {
  return prepare_w4_mma<false, 1, 32>() && prepare_w4_mma<false, 2, 32>() && prepare_w4_mma<true, 2, 32>() &&
         prepare_w4_mma<false, 1, 64>() && prepare_w4_mma<false, 2, 64>() && prepare_w4_mma<true, 2, 64>() &&
         prepare_w4_nt<false, false>() && prepare_w4_nt<false, true>() && prepare_w4_nt<true, false>() &&
         prepare_w4_nt<true, true>();
}

// How many clusters of `split` CTAs of the 4-bit product, which fill an SM
// each, fit on the device at once.
int w4_clusters_fit(int sm_count, int split) {
  using Cfg = W4NtCfg<false, false, 7, 1>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(split), static_cast<unsigned>(sm_count / split), 1);
  cfg.blockDim = dim3(Cfg::kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, w4_nt_sm100<Cfg>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return clusters;
}

// The 79 kernel instances get their shared memory, and the clusters that fit
// are counted, at a handle's first call of their kind: who multiplies only
// neither waits nor fails for them (a process's first b200gemm_create 36 -> 32
// ms; the first gated call takes 1 ms instead, the first 4-bit product 3).  The
// handle's device is current and h->mu held; false on failure.  None of it is
// work on a stream, so a stream may be captured meanwhile.
bool gated_ready(b200gemm_handle* h) {
  if (h->ffn_clusters > 0) return true;
  if (!prepare_gated_decode_kernels()) return false;
  h->ffn_clusters = prepare_ffn_kernels(h->sm_count);
  return h->ffn_clusters > 0;
}
bool w4_ready(b200gemm_handle* h) {
  if (h->w4_clusters[0] > 0) return true;
  if (!prepare_w4_kernels()) return false;
  int fit[4];
  for (int i = 0; i < 4; ++i)
    if ((fit[i] = w4_clusters_fit(h->sm_count, 1 << i)) <= 0) return false;
  for (int i = 0; i < 4; ++i) h->w4_clusters[i] = fit[i];
  return true;
}

template <class Cfg>
cudaError_t launch_ffn(int clusters, cudaStream_t stream, const FfnMaps& m, const FfnParams& p, bool overlap) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * clusters), 1, 1);
  cfg.blockDim = dim3(Cfg::kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (overlap) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, ffn_gemm_sm100<Cfg>, m, p);
}

// Launch of a few-rows kernel: `split` CTAs a cluster, which share K.
template <class Kernel, class Params>
cudaError_t launch_rows(Kernel kernel, int threads, int smem, int split, int blocks, int token_blocks,
                        cudaStream_t stream, const CUtensorMap& w0, const CUtensorMap& w1, const CUtensorMap& x,
                        const Params& p) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(split), static_cast<unsigned>(blocks), static_cast<unsigned>(token_blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.pdl != kPdlOff) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, w0, w1, x, p);
}

// One matrix of a call, for the overlap check: rows of `width` bytes every
// `pitch` bytes.
struct Extent {
  const void* ptr;
  long long rows, width, pitch;
};

// Whether two matrices share a byte.  Column slices of one wide matrix
// (equal pitches) are told apart; other interleavings count as overlapping.
bool overlaps(const Extent& a, const Extent& b) {
  if (a.ptr == nullptr || b.ptr == nullptr || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  const auto pa = reinterpret_cast<uintptr_t>(a.ptr), pb = reinterpret_cast<uintptr_t>(b.ptr);
  const auto ea = pa + static_cast<uintptr_t>((a.rows - 1) * a.pitch + a.width);
  const auto eb = pb + static_cast<uintptr_t>((b.rows - 1) * b.pitch + b.width);
  if (ea <= pb || eb <= pa) return false;
  if (a.pitch != b.pitch || a.pitch <= 0) return true;
  const auto pitch = static_cast<uintptr_t>(a.pitch);
  const long long d = static_cast<long long>(pb >= pa ? (pb - pa) % pitch : (pitch - (pa - pb) % pitch) % pitch);
  return !(d >= a.width && d + b.width <= a.pitch);
}

// Outputs [0, outs) may share nothing with each other or with the inputs
// [outs, count).
bool outputs_distinct(const Extent* e, int outs, int count) {
  for (int i = 0; i < outs; ++i)
    for (int j = i + 1; j < count; ++j)
      if (overlaps(e[i], e[j])) return false;
  return true;
}

bool valid_activation(int act) { return act >= B200GEMM_ACT_NONE && act <= B200GEMM_ACT_SILU; }
bool group_shift_of(int group, int* shift) {
  for (int s = 5; s <= 8; ++s)
    if (group == (1 << s)) {
      *shift = s;
      return true;
    }
  return false;
}

constexpr int kMaxExtent = 0x7FFFFFFF - 4096;  // rows, columns: tile coordinates stay inside an int
constexpr long long kMaxPitch = 1ll << 38;     // elements: tensor maps take pitches below 2^40 bytes

// Time of one tile with `width` accumulator columns and num_kb K blocks, in
// the units and by the fit of tile_plan_cost; a 512-wide tile's epilogue is
// not hidden and costs `epi` more than the plain one.
double ffn_tile_time(int width, int num_kb, double epi) {
  if (width == 512) return (2.0 * num_kb + 13.0) * 0.8545 / 0.85 + epi;
  const double feed = (16384.0 + 64.0 * width) / 32768.0;
  return num_kb * (0.08 + 0.92 * feed) / 0.85 + 4.0;
}

// The same for a dW tile, which takes at least as long as its stores do: with
// one K block (dW of a few rows of X, 14336 x 4096) tiles of 512, 256 and 128
// columns took about 6.5, 4.5 and 3 us next to dX's.
double dw_tile_time(int width, int num_kb) {
  const double t = ffn_tile_time(width, num_kb, 0.0);
  const double stores = width == 512 ? 20.0 : (width == 256 ? 14.0 : 10.0);
  return t > stores ? t : stores;
}

// Accumulator columns of the gated block's tiles (twice H's): by waves of
// tiles.  A forced tile width asks for the nearest one there is.
int ffn_gated_width(const b200gemm_handle* h, int tiles_m, int F, int num_kb) {
  if (h->tile_width != 0) return h->tile_width >= 448 ? 512 : (h->tile_width >= 224 ? 256 : h->tile_width);
  int best = 0;
  double best_cost = 1e300;
  for (int width : {512, 256, 192, 128}) {
    const long long tiles = static_cast<long long>(tiles_m) * ((F + width / 2 - 1ll) / (width / 2));
    const double cost = static_cast<double>((tiles + h->ffn_clusters - 1) / h->ffn_clusters) *
                        ffn_tile_time(width, num_kb, 12.0);
    if (cost < best_cost) {
      best_cost = cost;
      best = width;
    }
  }
  return best;
}

// The same for the gradients, whose tiles fill the clusters' time together:
// the mean load and half a dW tile, or what the dX tiles take by themselves.
// Where dX has too few tiles for the clusters, its sum is split into up to 16
// ranges of at least 8 K blocks (another launch, and their partial sums, cost
// about 10 units).  The ranges are those of a call for all gradients also where
// dX alone is asked for, since the order of its sum goes by them.
struct GradsPlan {
  int width = 256, split = 1, slice_kb = 0, want = 1;
};
GradsPlan grads_plan(const b200gemm_handle* h, int m, int f, int k, bool dx, bool dw, bool may_split) {
  const int ranges = !dx || !may_split ? 1 : (dw ? 0 : grads_plan(h, m, f, k, true, true, true).want);  // 0: any
  GradsPlan best;
  double best_cost = 1e300;
  const double g = h->ffn_clusters;
  const int kb = 2 * ((f + 63) / 64);
  for (int width : {512, 256, 128}) {
    if (h->tile_width != 0 && width != (h->tile_width >= 448 ? 512 : (h->tile_width >= 192 ? 256 : 128))) continue;
    const double tn = static_cast<double>((k + width - 1ll) / width);
    const double n1 = dx ? tn * ((m + 255ll) / 256) : 0.0, n2 = dw ? 2.0 * tn * ((f + 255ll) / 256) : 0.0;
    const double t2 = dw_tile_time(width, (m + 63) / 64);
    for (int want = ranges > 0 ? ranges : 1; want <= (ranges > 0 ? ranges : 16); want *= 2) {
      const int slice = (kb + want - 1) / want, split = (kb + slice - 1) / slice;
      if (ranges == 0 && split > 1 && (slice < 8 || n1 * split > 2.0 * g)) break;
      const double t1 = ffn_tile_time(width, slice, 0.0);
      const double mean = (n1 * split * t1 + n2 * t2) / g + (n2 > 0.0 ? 0.5 * t2 : 0.0);
      double cost = static_cast<double>(static_cast<long long>((n1 * split + g - 1.0) / g)) * t1;
      if (mean > cost) cost = mean;
      const double dw_alone = n1 > 0.0 ? t2 : static_cast<double>(static_cast<long long>((n2 + g - 1.0) / g)) * t2;
      if (n2 > 0.0 && dw_alone > cost) cost = dw_alone;
      if (split > 1) cost += 10.0;
      if (cost < best_cost) {
        best_cost = cost;
        best.width = width;
        best.split = split;
        best.slice_kb = slice;
        best.want = want;
      }
    }
  }
  return best;
}

// Workspace of the gated block's gradients: dG, dU, and dX's partial sums.
unsigned long long grads_base_bytes(int M, int F) {
  return 4ull * static_cast<unsigned long long>(M) * ((static_cast<unsigned long long>(F) + 7) / 8 * 8);
}
unsigned long long grads_partial_bytes(int M, int K, int split) {
  return split > 1 ? 4ull * static_cast<unsigned long long>(split) * M * K : 0;
}

// bf16 operand maps of the tiled kernel: K-major boxes of 64 k x 128 rows (or
// as many as one CTA loads),
// MN-major boxes of 64 columns x 64 k, both one 128-byte swizzle row wide.
bool encode_kmajor(CUtensorMap* m, const void* ptr, int k, int rows, long long ld, int box_rows = 128) {
  return encode_2d(m, ptr, static_cast<uint64_t>(k), static_cast<uint64_t>(rows), static_cast<uint64_t>(ld) * 2,
                   kBlockK, static_cast<uint32_t>(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
}
bool encode_mnmajor(CUtensorMap* m, const void* ptr, int mn, int k, long long ld) {
  return encode_2d(m, ptr, static_cast<uint64_t>(mn), static_cast<uint64_t>(k), static_cast<uint64_t>(ld) * 2, 64, 64,
                   CU_TENSOR_MAP_SWIZZLE_128B);
}
bool encode_out(CUtensorMap* m, void* ptr, int cols, int rows, long long ld) {
  return encode_2d(m, ptr, static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), static_cast<uint64_t>(ld) * 2,
                   kCBoxCols, kCBoxRows, CU_TENSOR_MAP_SWIZZLE_64B);
}

// Whether the gated block runs on the decode kernel, which reads the weights
// once per 32 rows of X: always up to 32 rows, and as far as 128 where that is
// estimated to beat the tiled kernel, whose few tiles of a small block leave
// most SMs idle.  In microseconds, measured on B200: 0.315 per unit of
// ffn_tile_time; the weights at 5 TB/s with 32 rows of X; 4 of either launch.
// Never past the 65535 blocks of 32 columns that its grid takes.
bool gated_uses_decode(const b200gemm_handle* h, int M, int F, int K) {
  if (h->small_m == 0 || h->tile_width != 0 || M > 128 || F > 65535 * 32) return false;
  if (M <= 32) return true;
  const int num_kb = (K + kBlockK - 1) / kBlockK;
  const int width = ffn_gated_width(h, 1, F, num_kb);
  const long long tiles = (F + width / 2 - 1ll) / (width / 2);
  const double tiled = 0.315 * static_cast<double>((tiles + h->ffn_clusters - 1) / h->ffn_clusters) *
                       ffn_tile_time(width, num_kb, 12.0);
  return (M + 31) / 32 * (4e-6 / 5.0 * F * static_cast<double>(K)) < tiled;
}

// K ranges (CTAs of a cluster) of the decode kernel: the smallest power of two
// up to 8 that gives every SM a CTA, while each CTA's warps keep a few stages.
int gated_decode_split(const b200gemm_handle* h, long long ctas, int num_stages) {
  int split = 1;
  while (split < 8 && ctas * split < h->sm_count && num_stages >= 16 * split) split *= 2;
  return split;
}

template <int NT>
cudaError_t launch_gated_decode(const b200gemm_handle* h, int split, int blocks, int token_blocks, cudaStream_t stream,
                                const CUtensorMap& mg, const CUtensorMap& mu, const CUtensorMap& mx,
                                const GatedDecodeParams& p) {
  using Deep = GatedDecodeCfg<NT, true>;
  using Small = GatedDecodeCfg<NT, false>;
  if (static_cast<long long>(split) * blocks * token_blocks <= static_cast<long long>(Deep::kCtas) * h->sm_count)
    return launch_rows(gated_decode_sm100<Deep>, Deep::kThreads, Deep::kSmemBytes, split, blocks, token_blocks, stream,
                       mg, mu, mx, p);
  return launch_rows(gated_decode_sm100<Small>, Small::kThreads, Small::kSmemBytes, split, blocks, token_blocks, stream,
                     mg, mu, mx, p);
}

int run_gated_decode(b200gemm_t h, const void* Wg, const void* Wu, long long ldw, const void* X, long long ldx,
                     GatedDecodeParams p, cudaStream_t stream) {
  const int nt = p.M > 16 ? 4 : (p.M > 8 ? 2 : 1);
  const long long blocks = (static_cast<long long>(p.F) + 31) / 32;
  const int token_blocks = (p.M + 31) / 32;
  CUtensorMap mg, mu, mx;
  const auto encode = [&](CUtensorMap* m, const void* ptr, int rows, long long ld, int box_rows) {
    return encode_kmajor(m, ptr, p.K, rows, ld, box_rows);
  };
  if (!encode(&mg, Wg, p.F, ldw, 32) || !encode(&mu, Wu, p.F, ldw, 32) || !encode(&mx, X, p.M, ldx, 8 * nt))
    return B200GEMM_ERR_CUDA;
  p.num_stages = (p.K + 63) / 64;
  const int split = gated_decode_split(h, blocks * token_blocks, p.num_stages);
  p.stages_per_cta = (p.num_stages + split - 1) / split;
  {
    std::lock_guard<std::mutex> lock(h->mu);
    p.timeout_ns = h->timeout_ns;
    p.pdl = h->pdl;
  }
  p.status = h->status_dev;
  const int b = static_cast<int>(blocks);
  const cudaError_t e = nt == 1   ? launch_gated_decode<1>(h, split, b, token_blocks, stream, mg, mu, mx, p)
                        : nt == 2 ? launch_gated_decode<2>(h, split, b, token_blocks, stream, mg, mu, mx, p)
                                  : launch_gated_decode<4>(h, split, b, token_blocks, stream, mg, mu, mx, p);
  return e == cudaSuccess ? B200GEMM_OK : B200GEMM_ERR_CUDA;
}

// Rows of W per CTA, 16-row tiles per warp and K ranges of a 4-bit product: of
// the splits of K over clusters of 1, 2, 4 and 8 CTAs, the one with the least
// estimated time.  Rows are divided evenly over the clusters that fit at once
// (a second wave only where a CTA's registers and ring cannot hold its share).
// The estimate's unit, a warp's 16 x 64 weights times a tile of X, is some 0.2
// us; a CTA costs 6 of them besides, 10 in a cluster.  Measured with K in 1, 2,
// 4 and 8 ranges (us, * the choice; groups of 128 unless said otherwise):
//   1 x 4096 x 14336          18.6  13.5  11.6* 18.7
//   1 x 8192 x 8192           14.0  12.5* 16.8  21.6
//   1 x 28672 x 8192          27.8* 34.4  42.5  64.6
//   1 x 14336 x 4096          11.6  11.5* 16.1
//   8 x 2048 x 8192 (64)      11.4   7.7   6.7*  7.3
//   12 x 1024 x 8192 (32)     14.1   9.3   6.8*  7.0
//   16 x 4096 x 8192          12.9  11.2  11.1* 17.5
//   gated 5 x 14331 x 4096 (32) 18.7* 25.5  34.4
struct W4Plan {
  int rows = 0, mt = 0, split = 1;
  long long waves = 1;
};
W4Plan w4_plan(const b200gemm_handle* h, int N, int num_stages, int max_mt, bool gated) {
  const int tiles = gated ? 1 : 2;  // 16-row tiles of output per unit of mt
  W4Plan best;
  double best_cost = 1e300;
  for (int i = 0, split = 1; i < 4; ++i, split *= 2) {
    if (split > 1 && num_stages < 2 * split) break;
    const int fit = h->w4_clusters[i];
    const long long per_wave = 16ll * max_mt * tiles * fit;
    const long long waves = (N + per_wave - 1) / per_wave;
    const int rows = static_cast<int>((N + waves * fit - 1) / (waves * fit));
    const int mt = (rows + 16 * tiles - 1) / (16 * tiles);
    const int stages = (num_stages + split - 1) / split;
    const double cost = static_cast<double>(waves) * (stages * (mt + 1.0) + (split > 1 ? 10.0 : 6.0));
    if (cost < best_cost) {
      best_cost = cost;
      best.rows = rows;
      best.mt = mt;
      best.split = split;
      best.waves = waves;
    }
  }
  return best;
}

struct W4Launch {
  W4Plan plan;
  int blocks, token_blocks, tok;  // blocks of W, and of `tok` rows of X
  cudaStream_t stream;
  CUtensorMap w0, w1, x;
};

template <bool GATED, bool G32, int NT, int MT = kW4MaxMT<NT>>
cudaError_t launch_w4(const W4Launch& l, const W4NtParams& p) {
  if constexpr (MT == 0) {
    return cudaErrorInvalidValue;
  } else {
    using Cfg = W4NtCfg<GATED, G32, MT, NT>;
    if (l.plan.mt != MT) return launch_w4<GATED, G32, NT, MT - 1>(l, p);
    return launch_rows(w4_nt_sm100<Cfg>, Cfg::kThreads, Cfg::kSmemBytes, l.plan.split, l.blocks, 1,
                       l.stream, l.w0, l.w1, l.x, p);
  }
}

// The same for the tcgen05 kernel, whose CTA holds 128 rows of W or 256 (128
// of Wg and of Wu); plan.mt = 128-row blocks.  A stage of 256 k's takes some
// 1200 cycles with one block and 2100 with two, however few of their rows are
// there (a fit of whole calls; DRAM's share of 256 rows is 1400), and a CTA
// some 6000 besides, 700 more in a cluster.  Measured with K in 1, 2, 4 and 8
// ranges (us, * the choice; groups of 128 unless said otherwise):
//   32 x 8192 x 8192 (64)     26.4  17.9  18.7* 37.0
//   32 x 4096 x 14336         35.9  22.5  15.0* 29.3
//   32 x 1024 x 8192          22.2  14.9  10.2   7.9*
//   64 x 28416 x 8192         55.5* 66.9  78.8 107.3
W4Plan w4_mma_plan(const b200gemm_handle* h, int N, int token_blocks, int num_stages, bool gated) {
  W4Plan best;
  double best_cost = 1e300;
  for (int i = 0, split = 1; i < 4 && split <= num_stages; ++i, split *= 2) {
    const int fit = h->w4_clusters[i] / token_blocks > 0 ? h->w4_clusters[i] / token_blocks : 1;
    const long long max_rows = gated ? 128 : 256;
    const long long waves = (N + max_rows * fit - 1) / (max_rows * fit);
    const int rows = static_cast<int>((N + waves * fit - 1) / (waves * fit));
    const int blocks = gated || rows > 128 ? 2 : 1;
    const int stages = (num_stages + split - 1) / split;
    const double cost = static_cast<double>(waves) * (stages * (blocks == 2 ? 2100.0 : 1200.0) + (split > 1 ? 6700.0 : 6000.0));
    if (cost < best_cost) {
      best_cost = cost;
      best.rows = rows;
      best.mt = blocks;
      best.split = split;
      best.waves = waves;
    }
  }
  return best;
}

template <bool GATED, int H, int TOK>
cudaError_t launch_w4_mma_block(const W4Launch& l, const W4NtParams& p) {
  const auto go = [&](auto kernel, int threads, int smem) {
    return launch_rows(kernel, threads, smem, l.plan.split, l.blocks, l.token_blocks, l.stream, l.w0, l.w1, l.x, p);
  };
  using C1 = W4MmaCfg<GATED, H, 1, TOK>;
  using C2 = W4MmaCfg<GATED, H, 2, TOK>;
  using C4 = W4MmaCfg<GATED, H, 4, TOK>;
  if (p.group_shift == 5) return go(w4_mma_sm100<C4>, C4::kThreads, C4::kSmemBytes);
  if (p.group_shift == 6) return go(w4_mma_sm100<C2>, C2::kThreads, C2::kSmemBytes);
  return go(w4_mma_sm100<C1>, C1::kThreads, C1::kSmemBytes);
}

template <bool GATED>
cudaError_t launch_w4_mma(const W4Launch& l, const W4NtParams& p) {
  if (l.tok == 64) {
    if constexpr (!GATED)
      if (l.plan.mt == 1) return launch_w4_mma_block<false, 1, 64>(l, p);
    return launch_w4_mma_block<GATED, 2, 64>(l, p);
  }
  if constexpr (!GATED)
    if (l.plan.mt == 1) return launch_w4_mma_block<false, 1, 32>(l, p);
  return launch_w4_mma_block<GATED, 2, 32>(l, p);
}

template <bool GATED>
int run_w4(b200gemm_t h, const void* w0, const void* w1, const void* X, long long ldx, W4NtParams p,
           cudaStream_t stream) {
  // The grid takes 65535 blocks of rows of X: more of them in several launches.
  constexpr int kRowsPerLaunch = 65535 * 64;
  if (p.M > kRowsPerLaunch) {
    const long long row_bytes = p.ldo * (p.out_type == kOutF32 ? 4 : 2);
    for (long long m = 0; m < p.M; m += kRowsPerLaunch) {
      W4NtParams part = p;
      part.M = static_cast<int>(p.M - m < kRowsPerLaunch ? p.M - m : kRowsPerLaunch);
      part.out = static_cast<uint8_t*>(p.out) + m * row_bytes;
      const int rc = run_w4<GATED>(h, w0, w1, static_cast<const uint16_t*>(X) + m * ldx, ldx, part, stream);
      if (rc != B200GEMM_OK) return rc;
    }
    return B200GEMM_OK;
  }
  {
    std::lock_guard<std::mutex> lock(h->mu);
    if (!w4_ready(h)) return B200GEMM_ERR_CUDA;
    p.timeout_ns = h->timeout_ns;
    p.pdl = h->pdl;
  }
  p.status = h->status_dev;
  W4Launch l;
  l.tok = p.M > 32 ? 64 : 32;
  const long long token_blocks = (static_cast<long long>(p.M) + l.tok - 1) / l.tok;
  const auto stages = [&](int k) { return static_cast<int>((static_cast<long long>(p.K) + k - 1) / k); };
  l.token_blocks = static_cast<int>(token_blocks);
  l.stream = stream;
  // 16 rows of X and fewer: mma.sync, whose cost grows with them.  From 9 rows
  // on its registers hold 160 rows of W (gated: 80 of each) instead of 224:
  // where that means a second wave of CTAs and tcgen05 needs but one, that one,
  // except in groups of 32, whose sums it has to fetch four times per 128 k's.
  // (16 rows, mma.sync and tcgen05, us: gated 14336 x 4096 30.5 and 24.0, in
  // groups of 32 30.9 and 31.8; 28672 x 8192 46.5 and 43.5; two waves of both,
  // gated 20000 x 2048, 23.0 and 35.6.)
  const int nt = p.M > 8 ? 2 : 1;
  W4Plan sync_plan, mma_plan;
  if (p.M <= kW4MaxSyncRows)
    sync_plan = w4_plan(h, p.N, stages(512), nt == 1 ? kW4MaxMT<1> : kW4MaxMT<2>, GATED);
  bool mma = p.M > kW4MaxSyncRows || (nt == 2 && sync_plan.waves > 1 && p.group_shift > 5);
  if (mma) {
    mma_plan = w4_mma_plan(h, p.N, l.token_blocks, stages(256), GATED);
    mma = p.M > kW4MaxSyncRows || mma_plan.waves == 1;
  }
  l.plan = mma ? mma_plan : sync_plan;
  p.num_stages = stages(mma ? 256 : 512);
  l.blocks = (p.N + l.plan.rows - 1) / l.plan.rows;
  if (l.blocks > 65535) return B200GEMM_ERR_TOO_LARGE;
  p.rows = l.plan.rows;
  p.stages_per_cta = (p.num_stages + l.plan.split - 1) / l.plan.split;
  // Codes: boxes of 256 k's (128 swizzled bytes a row); X: 256 k's plain, or
  // 64 swizzled as the MMA reads them.
  const uint32_t box_rows = mma ? 128u : static_cast<uint32_t>((GATED ? 16 : 32) * l.plan.mt);
  const auto encode_w = [&](CUtensorMap* map, const void* w) {
    return encode_2d(map, w, static_cast<uint64_t>(p.K) / 2, static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.K) / 2,
                     128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_DATA_TYPE_UINT8);
  };
  if (!encode_w(&l.w0, w0) || (GATED && !encode_w(&l.w1, w1)) ||
      !encode_2d(&l.x, X, static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.M), static_cast<uint64_t>(ldx) * 2,
                 mma ? 64 : 256, mma ? static_cast<uint32_t>(l.tok) : static_cast<uint32_t>(8 * nt),
                 mma ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE)) {
    return B200GEMM_ERR_CUDA;
  }
  if (!GATED) l.w1 = l.w0;
  cudaError_t e;
  if (mma) {
    e = launch_w4_mma<GATED>(l, p);
  } else if (p.group_shift == 5) {
    e = nt == 1 ? launch_w4<GATED, true, 1>(l, p) : launch_w4<GATED, true, 2>(l, p);
  } else {
    e = nt == 1 ? launch_w4<GATED, false, 1>(l, p) : launch_w4<GATED, false, 2>(l, p);
  }
  return e == cudaSuccess ? B200GEMM_OK : B200GEMM_ERR_CUDA;
}

FfnSet ffn_set(int M, int N, int num_kb, int tile_n, int matrices) {
  FfnSet s;
  s.M = M;
  s.N = N;
  s.num_kb = num_kb;
  s.tiles_m = (M + kTileM - 1) / kTileM;
  s.tiles_n = (N + tile_n - 1) / tile_n;
  const long long tiles = static_cast<long long>(matrices) * s.tiles_m * s.tiles_n;
  s.tiles = tiles > (1ll << 29) ? -1 : static_cast<int>(tiles);  // -1: too many
  return s;
}

template <class Cfg>
int run_ffn(b200gemm_t h, const FfnMaps& maps, FfnParams p, cudaStream_t stream, bool overlap) {
  if (p.first.tiles < 0 || p.second.tiles < 0) return B200GEMM_ERR_TOO_LARGE;
  p.band = B200GEMM_DEFAULT_BAND;
  p.status = h->status_dev;
  {
    std::lock_guard<std::mutex> lock(h->mu);
    p.timeout_ns = h->timeout_ns;
  }
  const int tiles = p.first.tiles + p.second.tiles;
  const int clusters = tiles < h->ffn_clusters ? tiles : h->ffn_clusters;
  return launch_ffn<Cfg>(clusters, stream, maps, p, overlap) == cudaSuccess ? B200GEMM_OK : B200GEMM_ERR_CUDA;
}

// Blocks of 2048 columns, and enough rows of them for 32 blocks per SM.
template <int ACT>
void launch_gated_grad(const GatedGradParams& p, int sm_count, cudaStream_t stream) {
  const int bx = (p.F + 2047) / 2048;
  int by = (sm_count * 32 + bx - 1) / bx;
  if (by > p.M) by = p.M;
  gated_grad_kernel<ACT><<<dim3(static_cast<unsigned>(bx), static_cast<unsigned>(by)), 256, 0, stream>>>(p);
}

}  // namespace b200gemm

extern "C" int b200gemm_bf16_gated(b200gemm_t h, int M, int F, int K, const void* X, long long ldx, const void* Wg,
                                   const void* Wu, long long ldw, int activation, void* H, long long ldh, void* G,
                                   void* U, long long ldgu, void* stream_ptr) {
  if (h == nullptr || M < 0 || F < 0 || K < 0 || !valid_activation(activation)) return B200GEMM_ERR_INVALID_ARG;
  if ((G == nullptr) != (U == nullptr)) return B200GEMM_ERR_INVALID_ARG;
  if (M == 0 || F == 0) return B200GEMM_OK;
  if (K == 0) return B200GEMM_ERR_UNSUPPORTED;
  if (X == nullptr || Wg == nullptr || Wu == nullptr || H == nullptr) return B200GEMM_ERR_INVALID_ARG;
  if ((K % 8) != 0 || ldx < K || ldw < K || ldh < F || (ldx % 8) != 0 || (ldw % 8) != 0 || (ldh % 8) != 0)
    return B200GEMM_ERR_UNSUPPORTED;
  if (G != nullptr && (ldgu < F || (ldgu % 8) != 0)) return B200GEMM_ERR_UNSUPPORTED;
  for (const void* q : {X, Wg, Wu, static_cast<const void*>(H), static_cast<const void*>(G), static_cast<const void*>(U)})
    if (!aligned16(q)) return B200GEMM_ERR_UNSUPPORTED;
  if (M > kMaxExtent || F > kMaxExtent || K > kMaxExtent || ldx > kMaxPitch || ldw > kMaxPitch || ldh > kMaxPitch ||
      (G != nullptr && ldgu > kMaxPitch))
    return B200GEMM_ERR_TOO_LARGE;
  const Extent e[] = {{H, M, 2ll * F, 2 * ldh}, {G, M, 2ll * F, 2 * ldgu}, {U, M, 2ll * F, 2 * ldgu},
                      {X, M, 2ll * K, 2 * ldx}, {Wg, F, 2ll * K, 2 * ldw}, {Wu, F, 2ll * K, 2 * ldw}};
  if (!outputs_distinct(e, 3, 6)) return B200GEMM_ERR_INVALID_ARG;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  DeviceGuard guard(h->device);
  if (!guard.ok()) return B200GEMM_ERR_CUDA;

  bool small;
  int width;
  const int num_kb = (K + kBlockK - 1) / kBlockK;
  {
    std::lock_guard<std::mutex> lock(h->mu);
    if (!gated_ready(h)) return B200GEMM_ERR_CUDA;
    small = gated_uses_decode(h, M, F, K);
    width = ffn_gated_width(h, (M + kTileM - 1) / kTileM, F, num_kb);
  }
  if (small) {
    GatedDecodeParams p{};
    p.M = M;
    p.F = F;
    p.K = K;
    p.act = activation;
    p.out = static_cast<uint16_t*>(H);
    p.ldo = ldh;
    p.gate = static_cast<uint16_t*>(G);
    p.up = static_cast<uint16_t*>(U);
    p.ldgu = ldgu;
    return run_gated_decode(h, Wg, Wu, ldw, X, ldx, p, stream);
  }
  FfnMaps m;
  const int box_rows = width == 512 ? 128 : width / 2;
  if (!encode_kmajor(&m.a0, X, K, M, ldx) || !encode_kmajor(&m.b0, Wg, K, F, ldw, box_rows) ||
      !encode_kmajor(&m.b1, Wu, K, F, ldw, box_rows) || !encode_out(&m.c[0], H, F, M, ldh)) {
    return B200GEMM_ERR_CUDA;
  }
  m.a1 = m.w0 = m.w1 = m.x = m.a0;  // (not read)
  m.c[1] = m.c[2] = m.c[0];
  if (G != nullptr && (!encode_out(&m.c[1], G, F, M, ldgu) || !encode_out(&m.c[2], U, F, M, ldgu)))
    return B200GEMM_ERR_CUDA;
  FfnParams p{};
  p.first = ffn_set(M, F, num_kb, width / 2, 1);
  p.act = activation;
  p.save = G != nullptr ? 1 : 0;
  p.out[0] = {static_cast<uint16_t*>(H), ldh};
  p.out[1] = {static_cast<uint16_t*>(G), ldgu};
  p.out[2] = {static_cast<uint16_t*>(U), ldgu};
  switch (width) {
    case 512: return run_ffn<FfnGated512>(h, m, p, stream, false);
    case 192: return run_ffn<FfnGated192>(h, m, p, stream, false);
    case 128: return run_ffn<FfnGated128>(h, m, p, stream, false);
    default: return run_ffn<FfnGated256>(h, m, p, stream, false);
  }
}

extern "C" unsigned long long b200gemm_gated_backward_workspace(b200gemm_t h, int M, int F, int K) {
  if (h == nullptr || M <= 0 || F <= 0 || K <= 0 || M > kMaxExtent || F > kMaxExtent || K > kMaxExtent) return 0;
  DeviceGuard guard(h->device);
  std::lock_guard<std::mutex> lock(h->mu);
  if (!guard.ok() || !gated_ready(h)) return grads_base_bytes(M, F);
  return grads_base_bytes(M, F) + grads_partial_bytes(M, K, grads_plan(h, M, F, K, true, true, true).split);
}

extern "C" int b200gemm_bf16_gated_backward(b200gemm_t h, int M, int F, int K, const void* dH, long long lddh,
                                            const void* X, long long ldx, const void* Wg, const void* Wu,
                                            long long ldw, const void* G, const void* U, long long ldgu,
                                            int activation, void* dX, long long lddx, void* dWg, void* dWu,
                                            long long lddw, void* workspace, unsigned long long workspace_bytes,
                                            void* stream_ptr) {
  if (h == nullptr || M < 0 || F < 0 || K < 0 || !valid_activation(activation)) return B200GEMM_ERR_INVALID_ARG;
  if ((dWg == nullptr) != (dWu == nullptr)) return B200GEMM_ERR_INVALID_ARG;
  if (K == 0 || (dX == nullptr && dWg == nullptr)) return B200GEMM_OK;
  if (M == 0 && F == 0) return B200GEMM_OK;
  if ((K % 8) != 0) return B200GEMM_ERR_UNSUPPORTED;
  if (dX != nullptr && (lddx < K || (lddx % 8) != 0 || !aligned16(dX))) return B200GEMM_ERR_UNSUPPORTED;
  if (dWg != nullptr && (lddw < K || (lddw % 8) != 0 || !aligned16(dWg) || !aligned16(dWu)))
    return B200GEMM_ERR_UNSUPPORTED;
  if (M > kMaxExtent || F > kMaxExtent || K > kMaxExtent || (dX != nullptr && lddx > kMaxPitch) ||
      (dWg != nullptr && lddw > kMaxPitch))
    return B200GEMM_ERR_TOO_LARGE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (M == 0 || F == 0) {  // empty sums
    DeviceGuard guard(h->device);
    if (!guard.ok()) return B200GEMM_ERR_CUDA;
    const auto zero = [&](void* ptr, long long ld, int rows) {
      return ptr == nullptr || rows == 0 ||
             cudaMemset2DAsync(ptr, static_cast<size_t>(ld) * 2, 0, static_cast<size_t>(K) * 2,
                               static_cast<size_t>(rows), stream) == cudaSuccess;
    };
    return zero(dX, lddx, M) && zero(dWg, lddw, F) && zero(dWu, lddw, F) ? B200GEMM_OK : B200GEMM_ERR_CUDA;
  }
  if (dH == nullptr || X == nullptr || Wg == nullptr || Wu == nullptr || G == nullptr || U == nullptr ||
      workspace == nullptr)
    return B200GEMM_ERR_INVALID_ARG;
  if (lddh < F || ldx < K || ldw < K || ldgu < F || (lddh % 8) != 0 || (ldx % 8) != 0 || (ldw % 8) != 0 ||
      (ldgu % 8) != 0)
    return B200GEMM_ERR_UNSUPPORTED;
  for (const void* q : {dH, X, Wg, Wu, G, U, static_cast<const void*>(workspace)})
    if (!aligned16(q)) return B200GEMM_ERR_UNSUPPORTED;
  if (lddh > kMaxPitch || ldx > kMaxPitch || ldw > kMaxPitch || ldgu > kMaxPitch) return B200GEMM_ERR_TOO_LARGE;
  const long long f8 = (static_cast<long long>(F) + 7) / 8 * 8;
  const unsigned long long base_bytes = grads_base_bytes(M, F);
  if (workspace_bytes < base_bytes) return B200GEMM_ERR_UNSUPPORTED;
  const Extent e[] = {{workspace, 1, static_cast<long long>(workspace_bytes), 0},
                      {dX, M, 2ll * K, 2 * lddx},
                      {dWg, F, 2ll * K, 2 * lddw},
                      {dWu, F, 2ll * K, 2 * lddw},
                      {dH, M, 2ll * F, 2 * lddh},
                      {X, M, 2ll * K, 2 * ldx},
                      {Wg, F, 2ll * K, 2 * ldw},
                      {Wu, F, 2ll * K, 2 * ldw},
                      {G, M, 2ll * F, 2 * ldgu},
                      {U, M, 2ll * F, 2 * ldgu}};
  if (!outputs_distinct(e, 4, 10)) return B200GEMM_ERR_INVALID_ARG;
  DeviceGuard guard(h->device);
  if (!guard.ok()) return B200GEMM_ERR_CUDA;

  GradsPlan plan;
  {
    std::lock_guard<std::mutex> lock(h->mu);
    if (!gated_ready(h)) return B200GEMM_ERR_CUDA;
    plan = grads_plan(h, M, F, K, dX != nullptr, dWg != nullptr, true);
    if (plan.split > 1 && workspace_bytes < base_bytes + grads_partial_bytes(M, K, plan.split))
      plan = grads_plan(h, M, F, K, dX != nullptr, dWg != nullptr, false);
  }
  GatedGradParams gp{};
  gp.M = M;
  gp.F = F;
  gp.dh = static_cast<const uint16_t*>(dH);
  gp.g = static_cast<const uint16_t*>(G);
  gp.u = static_cast<const uint16_t*>(U);
  gp.lddh = lddh;
  gp.ldgu = ldgu;
  gp.dg = static_cast<uint16_t*>(workspace);
  gp.du = gp.dg + static_cast<long long>(M) * f8;
  gp.ldo = f8;
  switch (activation) {
    case B200GEMM_ACT_RELU: launch_gated_grad<kActRelu>(gp, h->sm_count, stream); break;
    case B200GEMM_ACT_GELU: launch_gated_grad<kActGelu>(gp, h->sm_count, stream); break;
    case B200GEMM_ACT_GELU_TANH: launch_gated_grad<kActGeluTanh>(gp, h->sm_count, stream); break;
    case B200GEMM_ACT_SILU: launch_gated_grad<kActSilu>(gp, h->sm_count, stream); break;
    default: launch_gated_grad<kActNone>(gp, h->sm_count, stream); break;
  }
  if (cudaGetLastError() != cudaSuccess) return B200GEMM_ERR_CUDA;

  const int f8i = static_cast<int>(f8);
  FfnMaps m;
  if (!encode_kmajor(&m.a0, gp.dg, f8i, M, f8) || !encode_kmajor(&m.a1, gp.du, f8i, M, f8) ||
      !encode_mnmajor(&m.b0, Wg, K, F, ldw) || !encode_mnmajor(&m.b1, Wu, K, F, ldw) ||
      !encode_mnmajor(&m.w0, gp.dg, f8i, M, f8) || !encode_mnmajor(&m.w1, gp.du, f8i, M, f8) ||
      !encode_mnmajor(&m.x, X, K, M, ldx) || (dX != nullptr && !encode_out(&m.c[0], dX, K, M, lddx)) ||
      (dWg != nullptr && (!encode_out(&m.c[1], dWg, K, F, lddw) || !encode_out(&m.c[2], dWu, K, F, lddw))))
    return B200GEMM_ERR_CUDA;
  if (dX == nullptr) m.c[0] = m.c[1];  // (not written)
  if (dWg == nullptr) m.c[1] = m.c[2] = m.c[0];
  const int width = plan.width;
  FfnParams p{};
  p.seg_kb = (F + kBlockK - 1) / kBlockK;
  p.split = plan.split;
  p.slice_kb = plan.slice_kb;
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + base_bytes);  // (a multiple of 32 bytes in)
  p.first = ffn_set(M, K, 2 * p.seg_kb, width, dX != nullptr ? plan.split : 0);
  p.second = ffn_set(F, K, (M + kBlockK - 1) / kBlockK, width, dWg != nullptr ? 2 : 0);
  p.ahead = static_cast<int>(ffn_tile_time(width, plan.split > 1 ? plan.slice_kb : p.first.num_kb, 0.0) /
                                 dw_tile_time(width, p.second.num_kb) + 0.5);
  p.out[0] = {static_cast<uint16_t*>(dX), lddx};
  p.out[1] = {static_cast<uint16_t*>(dWg), lddw};
  p.out[2] = {static_cast<uint16_t*>(dWu), lddw};
  const int rc = width == 512   ? run_ffn<FfnGrads512>(h, m, p, stream, true)
                 : width == 128 ? run_ffn<FfnGrads128>(h, m, p, stream, true)
                                : run_ffn<FfnGrads256>(h, m, p, stream, true);
  if (rc != B200GEMM_OK || dX == nullptr || plan.split == 1) return rc;
  const long long groups = static_cast<long long>(M) * (K / 8);
  dx_sum_kernel<<<static_cast<unsigned>((groups + 255) / 256), 256, 0, stream>>>(
      p.partials, plan.split, M, K, static_cast<uint16_t*>(dX), lddx);
  return cudaGetLastError() == cudaSuccess ? B200GEMM_OK : B200GEMM_ERR_CUDA;
}

namespace {

// Checks shared by the two 4-bit products; OK means "go on".
int w4_product_check(int K, int group, long long lda, const void* A, int* shift) {
  if (!group_shift_of(group, shift) || (K % group) != 0) return B200GEMM_ERR_UNSUPPORTED;
  if (lda < K || (lda % 8) != 0 || !aligned16(A)) return B200GEMM_ERR_UNSUPPORTED;
  return B200GEMM_OK;
}

bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

int w4_convert_check(b200gemm_t h, int N, int K, const void* W, long long ldw, int group, const void* codes,
                     const void* scales, int* shift) {
  if (h == nullptr || N < 0 || K < 0) return B200GEMM_ERR_INVALID_ARG;
  if (!group_shift_of(group, shift) || (K % group) != 0) return B200GEMM_ERR_UNSUPPORTED;
  if (N == 0 || K == 0) return B200GEMM_OK;
  if (W == nullptr || codes == nullptr || scales == nullptr) return B200GEMM_ERR_INVALID_ARG;
  if (ldw < K || (ldw % 8) != 0 || !aligned16(W) || !aligned16(codes) || !aligned2(scales))
    return B200GEMM_ERR_UNSUPPORTED;
  if ((static_cast<long long>(N) + 31) / 32 > 65535 || K > kMaxExtent || ldw > kMaxPitch) return B200GEMM_ERR_TOO_LARGE;
  return B200GEMM_OK;
}

}  // namespace

extern "C" int b200gemm_w4_quantize(b200gemm_t h, int N, int K, const void* W, long long ldw, int group, void* codes,
                                    void* scales, void* stream_ptr) {
  W4Params p{};
  const int rc = w4_convert_check(h, N, K, W, ldw, group, codes, scales, &p.group_shift);
  if (rc != B200GEMM_OK || N == 0 || K == 0) return rc;
  const Extent e[] = {{codes, 1, static_cast<long long>(N) * (K / 2), 0},
                      {scales, 1, 2ll * N * (K / group), 0},
                      {W, N, 2ll * K, 2 * ldw}};
  if (!outputs_distinct(e, 2, 3)) return B200GEMM_ERR_INVALID_ARG;
  DeviceGuard guard(h->device);
  if (!guard.ok()) return B200GEMM_ERR_CUDA;
  p.N = N;
  p.K = K;
  p.w = const_cast<uint16_t*>(static_cast<const uint16_t*>(W));
  p.ldw = ldw;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint16_t*>(scales);
  const dim3 grid(static_cast<unsigned>((K + 255) / 256), static_cast<unsigned>((N + 31) / 32));
  w4_quantize_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream_ptr)>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200GEMM_OK : B200GEMM_ERR_CUDA;
}

extern "C" int b200gemm_w4_dequantize(b200gemm_t h, int N, int K, const void* codes, const void* scales, int group,
                                      void* W, long long ldw, void* stream_ptr) {
  W4Params p{};
  const int rc = w4_convert_check(h, N, K, W, ldw, group, codes, scales, &p.group_shift);
  if (rc != B200GEMM_OK || N == 0 || K == 0) return rc;
  const Extent e[] = {{W, N, 2ll * K, 2 * ldw},
                      {codes, 1, static_cast<long long>(N) * (K / 2), 0},
                      {scales, 1, 2ll * N * (K / group), 0}};
  if (!outputs_distinct(e, 1, 3)) return B200GEMM_ERR_INVALID_ARG;
  DeviceGuard guard(h->device);
  if (!guard.ok()) return B200GEMM_ERR_CUDA;
  p.N = N;
  p.K = K;
  p.w = static_cast<uint16_t*>(W);
  p.ldw = ldw;
  p.codes = const_cast<uint8_t*>(static_cast<const uint8_t*>(codes));
  p.scales = const_cast<uint16_t*>(static_cast<const uint16_t*>(scales));
  const dim3 grid(static_cast<unsigned>((K + 255) / 256), static_cast<unsigned>((N + 31) / 32));
  w4_dequantize_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream_ptr)>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200GEMM_OK : B200GEMM_ERR_CUDA;
}

extern "C" int b200gemm_w4_nt(b200gemm_t h, int M, int N, int K, const void* A, long long lda, const void* codes,
                              const void* scales, int group, void* C, long long ldc, int out_type, void* stream_ptr) {
  if (h == nullptr || M < 0 || N < 0 || K < 0 || (out_type != B200GEMM_OUT_BF16 && out_type != B200GEMM_OUT_F32))
    return B200GEMM_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return B200GEMM_OK;
  if (K == 0) return B200GEMM_ERR_UNSUPPORTED;
  if (A == nullptr || codes == nullptr || scales == nullptr || C == nullptr) return B200GEMM_ERR_INVALID_ARG;
  W4NtParams p{};
  const int rc = w4_product_check(K, group, lda, A, &p.group_shift);
  if (rc != B200GEMM_OK) return rc;
  const int esize = out_type == B200GEMM_OUT_F32 ? 4 : 2;
  if (ldc < N || !aligned16(codes) || !aligned2(scales) ||
      (reinterpret_cast<uintptr_t>(C) & static_cast<uintptr_t>(esize - 1)) != 0)
    return B200GEMM_ERR_UNSUPPORTED;
  if (M > kMaxExtent || N > kMaxExtent || K > kMaxExtent || lda > kMaxPitch || ldc > kMaxPitch)
    return B200GEMM_ERR_TOO_LARGE;
  const Extent e[] = {{C, M, static_cast<long long>(esize) * N, esize * ldc},
                      {A, M, 2ll * K, 2 * lda},
                      {codes, 1, static_cast<long long>(N) * (K / 2), 0},
                      {scales, 1, 2ll * N * (K / group), 0}};
  if (!outputs_distinct(e, 1, 4)) return B200GEMM_ERR_INVALID_ARG;
  DeviceGuard guard(h->device);
  if (!guard.ok()) return B200GEMM_ERR_CUDA;
  p.M = M;
  p.N = N;
  p.K = K;
  p.out_type = out_type;
  p.scales0 = static_cast<const uint16_t*>(scales);
  p.out = C;
  p.ldo = ldc;
  return run_w4<false>(h, codes, nullptr, A, lda, p, static_cast<cudaStream_t>(stream_ptr));
}

extern "C" int b200gemm_w4_gated(b200gemm_t h, int M, int F, int K, const void* X, long long ldx,
                                 const void* gate_codes, const void* gate_scales, const void* up_codes,
                                 const void* up_scales, int group, int activation, void* H, long long ldh,
                                 void* stream_ptr) {
  if (h == nullptr || M < 0 || F < 0 || K < 0 || !valid_activation(activation)) return B200GEMM_ERR_INVALID_ARG;
  if (M == 0 || F == 0) return B200GEMM_OK;
  if (K == 0) return B200GEMM_ERR_UNSUPPORTED;
  if (X == nullptr || gate_codes == nullptr || gate_scales == nullptr || up_codes == nullptr || up_scales == nullptr ||
      H == nullptr)
    return B200GEMM_ERR_INVALID_ARG;
  W4NtParams p{};
  const int rc = w4_product_check(K, group, ldx, X, &p.group_shift);
  if (rc != B200GEMM_OK) return rc;
  if (ldh < F || !aligned16(gate_codes) || !aligned16(up_codes) || !aligned2(gate_scales) || !aligned2(up_scales) ||
      !aligned2(H))
    return B200GEMM_ERR_UNSUPPORTED;
  if (M > kMaxExtent || F > kMaxExtent || K > kMaxExtent || ldx > kMaxPitch || ldh > kMaxPitch)
    return B200GEMM_ERR_TOO_LARGE;
  const long long code_bytes = static_cast<long long>(F) * (K / 2), scale_bytes = 2ll * F * (K / group);
  const Extent e[] = {{H, M, 2ll * F, 2 * ldh},       {X, M, 2ll * K, 2 * ldx},
                      {gate_codes, 1, code_bytes, 0}, {gate_scales, 1, scale_bytes, 0},
                      {up_codes, 1, code_bytes, 0},   {up_scales, 1, scale_bytes, 0}};
  if (!outputs_distinct(e, 1, 6)) return B200GEMM_ERR_INVALID_ARG;
  DeviceGuard guard(h->device);
  if (!guard.ok()) return B200GEMM_ERR_CUDA;
  p.M = M;
  p.N = F;
  p.K = K;
  p.act = activation;
  p.out_type = kOutBf16;
  p.scales0 = static_cast<const uint16_t*>(gate_scales);
  p.scales1 = static_cast<const uint16_t*>(up_scales);
  p.out = H;
  p.ldo = ldh;
  return run_w4<true>(h, gate_codes, up_codes, X, ldx, p, static_cast<cudaStream_t>(stream_ptr));
}
