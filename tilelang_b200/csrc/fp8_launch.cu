// Host side of the block-scaled fp8 products: shared-memory attributes once per device, cluster launches.
#include "fp8_launch.h"

#include "fp8_gemm.cuh"
#include "fp8_pair_gemm.cuh"

namespace b200dq {

namespace {

constexpr int kMaxDevices = 32;

template <bool TOK_LANE, int TN>
cudaError_t launch_tile(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const Fp8GemmParams& p, long long tiles,
                        cudaStream_t stream) {
  using C = Fp8TileConfig<TN>;
  static bool attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  auto kernel = fp8_tile_gemm_kernel<TOK_LANE, TN>;
  if (!attr_set[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  if (tiles * p.split > 0x7fffffffll) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.split));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, tmap_a, tmap_w, p);
}

}  // namespace

cudaError_t launch_fp8_tile_gemm(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const Fp8GemmParams& p,
                                 bool tokens_on_lanes, int tile_tokens, long long tiles, cudaStream_t stream) {
  if (tokens_on_lanes) return launch_tile<true, 128>(tmap_a, tmap_w, p, tiles, stream);
  switch (tile_tokens) {
    case 16: return launch_tile<false, 16>(tmap_a, tmap_w, p, tiles, stream);
    case 32: return launch_tile<false, 32>(tmap_a, tmap_w, p, tiles, stream);
    case 64: return launch_tile<false, 64>(tmap_a, tmap_w, p, tiles, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_fp8_pair_gemm(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const Fp8GemmParams& p, int pairs,
                                 cudaStream_t stream) {
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
  kernel<<<2 * pairs, kPairThreads, kPairSmemBytes, stream>>>(tmap_a, tmap_w, p);
  return cudaGetLastError();
}

}  // namespace b200dq
