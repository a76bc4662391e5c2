// Host side of the block-scaled fp8 products: shared-memory attributes once per device, cluster launches.
#include "fp8_launch.h"

#include <atomic>

#include "fp8_gemm.cuh"
#include "fp8_pair_gemm.cuh"

namespace b200dq {

namespace {

constexpr int kMaxDevices = 32;

template <bool TOK_LANE, int TN>
cudaError_t prepare_tile(int* dev) {
  static bool attr_set[kMaxDevices] = {};
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return e;
  if (*dev < 0 || *dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!attr_set[*dev]) {
    e = cudaFuncSetAttribute(fp8_tile_gemm_kernel<TOK_LANE, TN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Fp8TileConfig<TN>::kSmemBytes);
    if (e != cudaSuccess) return e;
    attr_set[*dev] = true;
  }
  return cudaSuccess;
}

template <bool TOK_LANE, int TN>
cudaError_t launch_tile(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const Fp8GemmParams& p, long long tiles,
                        cudaStream_t stream) {
  int dev = 0;
  const cudaError_t e = prepare_tile<TOK_LANE, TN>(&dev);
  if (e != cudaSuccess) return e;
  if (tiles * p.split > 0x7fffffffll) return cudaErrorInvalidValue;
  return chain_launch(fp8_tile_gemm_kernel<TOK_LANE, TN>, static_cast<unsigned>(tiles * p.split), Fp8TileConfig<TN>::kThreads,
                      Fp8TileConfig<TN>::kSmemBytes, stream, static_cast<unsigned>(p.split), tmap_a, tmap_w, p);
}

// Clusters of every size that the device holds at once; a cluster lies within one group of SMs, so this is
// less than the SMs divided by the size (148 SMs hold 144 single CTAs in clusters of 3 at best).
template <bool TOK_LANE, int TN>
cudaError_t resident_clusters(int split, int* clusters) {
  static std::atomic<int> known[kMaxDevices][9] = {};
  int dev = 0;
  cudaError_t e = prepare_tile<TOK_LANE, TN>(&dev);
  if (e != cudaSuccess) return e;
  int n = known[dev][split].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(split));
    cfg.blockDim = dim3(Fp8TileConfig<TN>::kThreads);
    cfg.dynamicSmemBytes = Fp8TileConfig<TN>::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&n, fp8_tile_gemm_kernel<TOK_LANE, TN>, &cfg);
    if (e != cudaSuccess) return e;
    known[dev][split].store(n, std::memory_order_relaxed);
  }
  *clusters = n;
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_fp8_tile_gemm(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const Fp8GemmParams& p,
                                 bool tokens_on_lanes, int tile_tokens, long long tiles, cudaStream_t stream) {
  if (tokens_on_lanes) return launch_tile<true, 128>(tmap_a, tmap_w, p, tiles, stream);
  switch (tile_tokens) {
    case 16: return launch_tile<false, 16>(tmap_a, tmap_w, p, tiles, stream);
    case 32: return launch_tile<false, 32>(tmap_a, tmap_w, p, tiles, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t fp8_resident_clusters(int tile_tokens, int split, int* clusters) {
  if (split < 1 || split > 8) return cudaErrorInvalidValue;
  switch (tile_tokens) {
    case 16: return resident_clusters<false, 16>(split, clusters);
    case 32: return resident_clusters<false, 32>(split, clusters);
    case 128: return resident_clusters<true, 128>(split, clusters);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_fp8_pair_gemm(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const CUtensorMap& tmap_c,
                                 const Fp8GemmParams& p, int pairs, cudaStream_t stream) {
  static_assert(kFp8PairMaxGroups == kPairMaxGroups, "tile table");
  static bool attr_set[kMaxDevices][2] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  const bool gated = p.gate_codes != nullptr;
  auto kernel = gated ? fp8_pair_gemm_kernel<true> : fp8_pair_gemm_kernel<false>;
  if (!attr_set[dev][gated]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmemBytes);
    if (e != cudaSuccess) return e;
    attr_set[dev][gated] = true;
  }
  return chain_launch(kernel, 2 * pairs, kPairThreads, kPairSmemBytes, stream, 2, tmap_a, tmap_w, tmap_c, p);
}

}  // namespace b200dq
