// Host side of the token exchange: chunk sizes, launches.
#include "exchange_launch.h"

#include <algorithm>

#include "exchange.cuh"

namespace b200dq {

namespace {

template <typename MOVE>
cudaError_t dispatch(const ExchangeSortParams& s, const ExchangeRowsParams& r, cudaStream_t stream) {
  const long long pairs = s.tokens * s.top_k;
  const int bins = s.num_experts + 1;
  if (pairs <= kExchangeOneLaunchPairs) {
    const int per = static_cast<int>((s.tokens + 295) / 296);              // two CTAs an SM
    const int grid = static_cast<int>((s.tokens + per - 1) / per);
    return chain_launch(exchange_dispatch_small_kernel<MOVE>, grid, 256, 2 * bins * sizeof(int), stream, 0, s, r, per);
  }
  const long long per = std::max<long long>(512, (pairs + kExchangeMaxChunks - 1) / kExchangeMaxChunks);
  const int chunks = static_cast<int>((pairs + per - 1) / per);
  cudaError_t e = chain_launch(exchange_count_kernel, chunks, 256, bins * sizeof(int), stream, 0, s, per);
  if (e != cudaSuccess) return e;
  e = chain_launch(exchange_place_kernel, chunks, kPlaceWarps * 32, (kPlaceWarps + 2) * bins * sizeof(int), stream, 0, s, per);
  if (e != cudaSuccess) return e;
  const int grid = static_cast<int>(std::min<long long>(s.tokens, 148 * 32));
  return chain_launch(exchange_move_kernel<MOVE>, grid, 256, 0, stream, 0, s, r);
}

template <typename T>
cudaError_t dispatch_quant(const ExchangeSortParams& s, const ExchangeRowsParams& r, cudaStream_t stream) {
  return r.fp8_type == FP8_E4M3 ? dispatch<QuantMove<T, FP8_E4M3>>(s, r, stream) : dispatch<QuantMove<T, FP8_E5M2>>(s, r, stream);
}

}  // namespace

cudaError_t launch_exchange_dispatch(const ExchangeSortParams& s, const ExchangeRowsParams& r, cudaStream_t stream) {
  if (r.scales == nullptr) return dispatch<CopyMove>(s, r, stream);
  if (r.type == EXCHANGE_F16) return dispatch_quant<__half>(s, r, stream);
  if (r.type == EXCHANGE_BF16) return dispatch_quant<__nv_bfloat16>(s, r, stream);
  return dispatch_quant<float>(s, r, stream);
}

cudaError_t launch_exchange_sum(const ExchangeSumParams& p, cudaStream_t stream) {
  const int items = p.vec ? p.width / (p.type == EXCHANGE_F32 ? 4 : 8) : p.width;
  const int threads = std::min(256, (items + 31) / 32 * 32);
  const int grid = static_cast<int>(std::min<long long>(p.tokens, 148 * 64));
  return chain_launch(p.type == EXCHANGE_F16 ? exchange_sum_kernel<__half> : p.type == EXCHANGE_BF16 ? exchange_sum_kernel<__nv_bfloat16> : exchange_sum_kernel<float>,
                      grid, threads, 0, stream, 0, p);
}

cudaError_t launch_exchange_sum_grad(const ExchangeSumGradParams& p, cudaStream_t stream) {
  const int grid = static_cast<int>(std::min<long long>((p.tokens * p.top_k + 7) / 8, 148 * 64));
  return chain_launch(p.type == EXCHANGE_F16 ? exchange_sum_grad_kernel<__half> : p.type == EXCHANGE_BF16 ? exchange_sum_grad_kernel<__nv_bfloat16> : exchange_sum_grad_kernel<float>,
                      grid, 256, 0, stream, 0, p);
}

}  // namespace b200dq
