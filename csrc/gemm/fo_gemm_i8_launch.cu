// Instantiations of the 8-bit GEMM kernels and the choice between them.
#include "fo_gemm.h"
#include "fo_gemm_i8.h"
#include "fo_gemm_i8_sm100.cuh"

#include <algorithm>
#include <cmath>

namespace fo {

namespace {

template <typename Kernel>
cudaError_t prepare(Kernel kernel, int smem, bool* attr_set) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 16 && attr_set[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && dev >= 0 && dev < 16) attr_set[dev] = true;
  return e;
}

cudaLaunchConfig_t config(int64_t grid, int threads, int smem, int cluster, cudaStream_t stream, cudaLaunchAttribute (&attr)[2]) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cfg;
}

// CTA pairs of the wide kernel that run at once on the current device.
template <bool BF16, bool GROUPED, int MT>
int resident_pairs() {
  static int cache[16] = {};  // 0: not asked yet
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16) return 1;
  if (cache[dev] == 0) {
    int sm_count = 0, clusters = 0;
    cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = config(sm_count & ~1, kI8WideThreads, I8WideSmem<GROUPED, MT>::kTotalBytes, 2, nullptr, attr);
    cfg.attrs = attr + 1;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters, fo_gemm_i8_wide_kernel<BF16, GROUPED, MT>, &cfg) != cudaSuccess || clusters < 1) {
      cudaGetLastError();
      clusters = 1;
    }
    cache[dev] = clusters;
  }
  return cache[dev];
}

template <bool BF16, bool GROUPED, int MT>
cudaError_t launch_wide(const GemmI8Maps& maps, const GemmI8Params& p, cudaStream_t stream) {
  constexpr int smem = I8WideSmem<GROUPED, MT>::kTotalBytes;
  static_assert(smem <= 227 * 1024, "shared memory of this configuration exceeds 227 KB");
  static bool attr_set[16] = {};
  auto kernel = fo_gemm_i8_wide_kernel<BF16, GROUPED, MT>;
  const cudaError_t e = prepare(kernel, smem, attr_set);
  if (e != cudaSuccess) return e;
  // with offsets, every expert may end in a tile of its own
  const int64_t units = ((p.M + MT * kI8Rows - 1) / (MT * kI8Rows) + (GROUPED ? std::min(p.experts, p.M) : 0)) * static_cast<int64_t>(p.tiles_n);
  const int64_t resident = resident_pairs<BF16, GROUPED, MT>();
  const int64_t pairs = MT == 1 && (GROUPED || 2 * units <= resident) ? std::min(2 * units, resident) : std::min(units, resident);
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(2 * pairs, kI8WideThreads, smem, 2, stream, attr);
  return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

template <bool BF16, int TN, int S>
cudaError_t launch_narrow(const GemmI8Maps& maps, const GemmI8Params& p, cudaStream_t stream) {
  constexpr int smem = I8NarrowSmem<TN, S>::kTotalBytes;
  static_assert(smem <= 227 * 1024, "shared memory of this configuration exceeds 227 KB");
  static bool attr_set[16] = {};
  auto kernel = fo_gemm_i8_narrow_kernel<BF16, TN, S>;
  const cudaError_t e = prepare(kernel, smem, attr_set);
  if (e != cudaSuccess) return e;
  const int64_t grid = static_cast<int64_t>(p.token_tiles) * ((p.N + 127) / 128) * S;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(grid, kI8NarrowThreads, smem, S, stream, attr);
  return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

template <bool BF16, int TN>
cudaError_t dispatch_split(int split, const GemmI8Maps& maps, const GemmI8Params& p, cudaStream_t stream) {
  switch (split) {
    case 1: return launch_narrow<BF16, TN, 1>(maps, p, stream);
    case 2: return launch_narrow<BF16, TN, 2>(maps, p, stream);
    case 4: return launch_narrow<BF16, TN, 4>(maps, p, stream);
    default: break;
  }
  if constexpr (TN >= 32) {
    if (split == 8) return launch_narrow<BF16, TN, 8>(maps, p, stream);
  }
  return cudaErrorInvalidValue;
}

template <bool BF16>
cudaError_t dispatch(const GemmI8Plan& plan, const GemmI8Maps& maps, const GemmI8Params& p, cudaStream_t stream) {
  switch (plan.tokens) {
    case 0:
      if (p.offsets != nullptr) return launch_wide<BF16, true, 1>(maps, p, stream);
      return plan.split == 2 ? launch_wide<BF16, false, 2>(maps, p, stream) : launch_wide<BF16, false, 1>(maps, p, stream);
    case 16: return dispatch_split<BF16, 16>(plan.split, maps, p, stream);
    case 32: return dispatch_split<BF16, 32>(plan.split, maps, p, stream);
    case 64: return dispatch_split<BF16, 64>(plan.split, maps, p, stream);
    case 128: return dispatch_split<BF16, 128>(plan.split, maps, p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

// ---------------------------------------------------------------------------- choice of a kernel
//
// A model of the time of one call, in us, with what was measured on a B200 (cold, less 8 us that an empty call reads):
//  * the wide kernel's pairs take 0.34 us a k-block of 128 for a 256 x 256 tile (3.7 PFLOP/s), 0.23 us for a half, and 2.5 us at
//    the end of a wave; 256 x 8192 x 28672: 51 us in halves, 1024 x 28672 x 8192: 133 us.  Its loads reach 5.9 TB/s;
//  * a narrow kernel's SM takes in 140 KB/us, a CTA with half an SM's memory 92 at most, all together 6.3 TB/s of weights; the epilogue
//    takes 0.045 us a token (64 tokens x 1024 deep: 2.8 us of products, 2.9 us of stores), the exchange of a split 0.7 us and 26 KB/us.
// The two sides for one token x 8192 x 28672: 94 us wide, 34 us as 16 tokens split in four; 128 x 8192 x 28672: 51 and 41;
// 256 x 28672 x 8192: 47 and 80; 192 x 1024 x 8192: 14 and 6; 4096 rows of 64 experts x 3584 x 4096: 162 and 188, 512 rows: 137 and 125.
namespace {

constexpr int kPairs = 74;  // of a whole B200; where fewer SMs are seen the choice is for more of them, the launch asks the device

// Weight matrices that are used, and the tiles of `rows` tokens that each has: about half of a tile is empty at an expert's end.
// The counts are on the device, so every expert is taken to have its share.  Shares that fall with the expert's rank to the power of 1.5
// cost little (64 experts x 3584 x 4096, chosen and best: 256 rows 92 and 91 us, 512 rows 117 and 115, 4096 rows 249 and 227), all rows
// for one expert more (256 rows 29 and 10 us, 512 rows 41 and 11, 4096 rows 46 and 45).
struct I8Load {
  double matrices, tiles_each;
};
I8Load i8_load(int M, int experts, bool grouped, int rows) {
  if (!grouped) return I8Load{1.0, static_cast<double>((M + rows - 1) / rows)};
  const double used = std::min(experts, M);
  return I8Load{used, std::max(1.0, M / used / rows + 0.5)};
}

// mt: 1, or 2 for tiles of 512 x 256.  Those save power, which is what binds sustained calls, but nothing hides their epilogue, so they want
// a long K, and whole waves of their larger tiles.  Sustained, tiles of 256 and of 512 rows, us: 8192 x 8192 x 8192 377, 384; x 12288 568, 566;
// x 16384 763, 747; x 20480 959, 928; x 28672 1342, 1288; 1024 x 8192 x 28672 187, 176; but 8192 x 28672 x 8192 1340, 1378; 4096 x
// 8192 x 28672 (3.5 waves of large tiles) 675, 690; 8192 x 5120 x 17920 535, 547.  0.66 us a k-block is their rate under load and 0.34 the
// other tiles' by themselves (0.42 under load), so that the model takes tall tiles only where their waves are well filled: it does in the cases
// above from 20480 on that they win, leaves 2 % at 16384 and 4 % of 2048 x 8192 x 28672 (357, 344), and takes them in none that they lose.
constexpr int kTallTilesK = 16384;

double wide_time(int M, int N, int K, int experts, bool grouped, int mt = 1) {
  const double num_kb = (K + kI8BK - 1) / kI8BK;
  const I8Load l = i8_load(M, experts, grouped, mt * kI8Rows);
  const int64_t units = static_cast<int64_t>(l.matrices * l.tiles_each + 0.5) * ((N + kI8Cols - 1) / kI8Cols);
  const int64_t left = units % kPairs;
  if (mt == 2) return static_cast<double>((units + kPairs - 1) / kPairs) * (0.66 * num_kb + 3.5);
  const double last = left == 0 ? 0.0 : (2 * left <= kPairs ? 0.23 : 0.34) * num_kb;
  const double weights = 1e-6 * l.matrices * N * K / 5.9;
  return std::max(units / kPairs * 0.34 * num_kb + last, weights) + 2.5;
}

double narrow_time(int M, int N, int K, int experts, bool grouped, int tokens, int split) {
  const int num_kb = ((K + kI8BK - 1) / kI8BK + split - 1) / split;
  const I8Load l = i8_load(M, experts, grouped, tokens);
  const double ctas = l.matrices * l.tiles_each * ((N + 127) / 128) * split;
  const int slots = tokens == 128 ? 2 * kPairs : 4 * kPairs;
  auto wave = [&](double n) {
    const double rate = n > 2 * kPairs ? 140e3 * 2 * kPairs / slots : (tokens == 128 ? 140e3 : 92e3);
    const double loads = num_kb * (16384.0 + 128.0 * tokens) / rate;
    const double weights = n / l.tiles_each * num_kb * 16384.0 / 6.3e6;
    return std::max(loads, weights) + 0.045 * tokens / split;
  };
  const double full = std::floor(ctas / slots), rest = ctas - full * slots;
  const double exchange = split > 1 ? 0.7 + tokens * 512.0 * (split - 1) / split / 26e3 : 0.0;
  if (split > 1 && ctas > slots) return 1e30;  // clusters in a second wave wait for room for all of their CTAs
  return full * wave(slots) + (rest > 0 ? wave(rest) : 0.0) + exchange;
}

}  // namespace

GemmI8Plan choose_i8(int M, int N, int K, int experts, bool grouped) {
  GemmI8Plan plan{0, 1};
  double best = wide_time(M, N, K, experts, grouped);
  if (!grouped && K >= kTallTilesK) {
    const double t = wide_time(M, N, K, experts, grouped, 2);
    if (t < best) {
      best = t;
      plan = GemmI8Plan{0, 2};
    }
  }
  for (int tokens : {16, 32, 64, 128}) {
    for (int split : {1, 2, 4, 8}) {
      if (4 * split > tokens || (split > 1 && split * kI8BK > K)) continue;  // sums are exchanged four tokens at a time
      const double t = narrow_time(M, N, K, experts, grouped, tokens, split);
      if (t < best) {
        best = t;
        plan = GemmI8Plan{tokens, split};
      }
    }
  }
  return plan;
}

std::string gemm_i8_launch(const GemmI8Plan& plan, GemmI8Params p, const void* A, const void* B, bool bf16,
                           cudaStream_t stream) {
  GemmI8Maps maps;
  const bool wide = plan.tokens == 0;
  std::string e = encode_tmap_8bit(&maps.a, A, 1, p.M, p.K, wide ? 128 : plan.tokens, false);
  if (!e.empty()) return "A: " + e;
  e = encode_tmap_8bit(&maps.b, B, p.experts, p.N, p.K, 128, true);
  if (!e.empty()) return "B: " + e;
  if (wide) {
    e = encode_tmap_8bit(&maps.b_half, B, p.experts, p.N, p.K, 64, true);
    if (!e.empty()) return "B: " + e;
    e = encode_tmap_16bit(&maps.c, p.C, p.M, p.N, 32);
    if (!e.empty()) return "C: " + e;
  }
  p.tiles_n = (p.N + kI8Cols - 1) / kI8Cols;
  p.raster_sw = std::min(8, p.tiles_n);
  if (!wide) {
    // with offsets: the tiles that the rows can have at most, one more than they fill for each expert
    p.token_tiles = p.offsets == nullptr ? (p.M + plan.tokens - 1) / plan.tokens
                                         : p.M / plan.tokens + std::min(p.experts, p.M);
  }
  const cudaError_t r = bf16 ? dispatch<true>(plan, maps, p, stream) : dispatch<false>(plan, maps, p, stream);
  if (r == cudaSuccess) return "";
  cudaGetLastError();  // reported to the caller, not left for the next one
  return std::string("launch: ") + cudaGetErrorString(r);
}

}  // namespace fo
